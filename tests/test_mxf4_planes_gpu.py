"""Batches of rows times MX-FP4 weights on the block-scaled tensor-core kernel: activations as three (bf16) or four (fp16)
E5M2 planes.  Tolerance: that of test_mxf4_product_gpu (products exact, fp32 sums, one rounding of C) and what the planes leave
of an element, less than 2^-36 of its block's largest, times the weights it meets."""
import numpy as np
import pytest

import helpers as H
import mxf4_plain as MX
import skl_b200 as S
from test_mxf4_product_gpu import bits, call, f64, tolerance

pytestmark = pytest.mark.gpu

SHAPES = [(5, 1, 128), (9, 17, 128), (16, 256, 256), (17, 257, 384), (33, 300, 512), (61, 520, 1024), (64, 1000, 2048), (100, 129, 768),
          (128, 512, 4096), (129, 260, 640), (200, 96, 1280), (256, 513, 256), (255, 200, 128), (31, 2000, 14336), (42, 70, 96), (43, 70, 100), (64, 33, 4099), (65, 300, 1000)]


def run(skl, ta, tc, m, n, k, alpha, beta, pad, g, a, codes, scales):
    kb = -(-k // 32)
    rsa, rsb, rss, rsc = k + pad, 16 * kb + 8 * pad, kb + pad, n + pad
    A = np.full(m * rsa, bits(ta, np.array([99.0]))[0])
    A.reshape(m, rsa)[:, :k] = a
    B, SC = np.full(n * rsb, 0x77, np.uint8), np.full(n * rss, 200, np.uint8)
    B.reshape(n, rsb)[:, : 16 * kb] = codes
    SC.reshape(n, rss)[:, :kb] = scales
    C = bits(tc, g.standard_normal(m * rsc))
    got = call(skl, ta, tc, False, m, n, k, alpha, A, rsa, B, rsb, SC, rss, beta, C, rsc).reshape(m, rsc)
    assert skl.skl_b200_last_path() == S.PATH_TCGEN05 and skl.skl_b200_last_launch_count() == 2
    assert np.array_equal(got[:, n:], C.reshape(m, rsc)[:, n:]), "the gap behind a row of C was written"
    return got[:, :n], f64(tc, C.reshape(m, rsc)[:, :n])


@pytest.mark.parametrize("ta,tc", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
def test_batches(skl, ta, tc):
    for i, (m, n, k) in enumerate(SHAPES):
        g = H.rng(100 * i + m)
        codes, scales = MX.random_packed(g, (n, k), 112, 122)
        # rows of different size, elements down to 2^-20 of their neighbours
        a = bits(ta, g.standard_normal((m, k)) * np.exp2(g.integers(-4, 4, (m, 1))) * np.exp2(-g.integers(0, 21, (m, k)) * (g.random((m, k)) < 0.2)))
        alpha, beta, pad = (1.0, -0.5)[i % 2], (0.0, 1.5)[i % 2], (0, 8, 3)[i % 3]
        got, old = run(skl, ta, tc, m, n, k, alpha, beta, pad, g, a, codes, scales)
        x, W = f64(ta, a), MX.values(codes, scales, k)
        want = alpha * (x @ W.T) + beta * old
        block = np.abs(np.pad(x, ((0, 0), (0, -k % 32)))).reshape(m, -1, 32).max(-1).repeat(32, 1)[:, :k]
        absum = abs(alpha) * (np.abs(x) @ np.abs(W).T) + abs(beta) * np.abs(old)
        left = abs(alpha) * 2.0 ** -36 * (block @ np.abs(W).T)
        tol = tolerance(tc, want, absum + left / (2 * ((1 + 2.0 ** -24) ** (k + 2) - 1)), k)
        err = np.abs(f64(tc, got) - want)
        assert np.all(err <= tol), (m, n, k, float(np.max(err / tol)), np.argwhere(err > tol)[:4])


@pytest.mark.parametrize("ta", ["bf16", "f16"])
def test_whole_numbers_are_exact(skl, ta):
    """Whole activations (8 and 11 significant bits) and one scale: every product and sum is a multiple of 1/2 below 2^24."""
    g = H.rng(1)
    m, n, k = 70, 300, 512
    codes, _ = MX.random_packed(g, (n, k))
    scales = np.full((n, k // 32), 127, np.uint8)
    a = g.integers(-255, 256, (m, k)) if ta == "bf16" else g.integers(-2047, 2048, (m, k))
    got, _ = run(skl, ta, "f32", m, n, k, 1.0, 0.0, 0, g, bits(ta, a.astype(np.float64)), codes, scales)
    assert np.array_equal(got, (a.astype(np.float64) @ MX.values(codes, scales, k).T).astype(np.float32))


@pytest.mark.parametrize("m", [40, 200])
def test_each_block_meets_its_scale(skl, m):
    n, k = 600, 1024
    g = H.rng(2)
    for row, blk, col in ((0, 0, 0), (7, 1, 31), (31, 2, 32), (33, 3, 127), (5, 13, 128), (39, 31, 255), (20, 17, 256), (38, 22, 511), (11, 30, 599)):
        codes, scales = np.full((n, k // 2), 0x22, np.uint8), np.full((n, k // 32), 127, np.uint8)
        scales[col, blk] = 130
        a = np.ones((m, k))
        a[row, blk * 32:blk * 32 + 32] = 2.0 ** -9  # a scale of its own for this block of A
        got, _ = run(skl, "bf16", "f32", m, n, k, 1.0, 0.0, 0, g, bits("bf16", a), codes, scales)
        want = np.full((m, n), float(k))
        want[row] += 32 * (2.0 ** -9 - 1)
        want[:, col] += 32 * 7
        want[row, col] += 32 * 7 * (2.0 ** -9 - 1)
        assert np.array_equal(got, want.astype(np.float32)), (row, blk, col, np.argwhere(got != want)[:4])


def test_extreme_scales_and_values_that_are_not_finite(skl):
    g = H.rng(3)
    m, n, k = 48, 300, 256
    codes, scales = MX.random_packed(g, (n, k), 100, 140)
    scales[5, 3], scales[290, 0] = 255, 255
    a = g.standard_normal((m, k)) * np.exp2(g.integers(-60, 60, (m, 1)))
    a[3, 40], a[7, 255], a[9, 0] = np.nan, np.inf, -np.inf
    a[11], a[12] = 0.0, 2.0 ** -126
    b = bits("bf16", a)
    got, _ = run(skl, "bf16", "f32", m, n, k, 1.0, 0.0, 0, g, b, codes, scales)
    ok = np.ones((m, n), bool)
    ok[:, [5, 290]] = ok[[3, 7, 9]] = False
    assert np.all(np.isnan(got[:, [5, 290]])) and not np.any(np.isfinite(got[[3, 7, 9]]))
    x, W = np.where(np.isfinite(f64("bf16", b)), f64("bf16", b), 0.0), np.where(np.isnan(MX.values(codes, scales, k)), 0.0, MX.values(codes, scales, k))
    want, absum = x @ W.T, np.abs(x) @ np.abs(W).T
    block = np.abs(np.pad(x, ((0, 0), (0, -k % 32)))).reshape(m, -1, 32).max(-1).repeat(32, 1)[:, :k]
    tol = tolerance("f32", want, absum, k) + 2.0 ** -36 * (block @ np.abs(W).T)
    assert np.all(np.abs(got.astype(np.float64) - want)[ok] <= tol[ok])


def test_same_bits_every_time(skl):
    g = H.rng(4)
    m, n, k = 77, 700, 3200
    codes, scales = MX.random_packed(g, (n, k), 112, 122)
    a = bits("bf16", g.standard_normal((m, k)))
    first, _ = run(skl, "bf16", "f32", m, n, k, 1.0, 0.0, 0, g, a, codes, scales)
    for _ in range(3):
        again, _ = run(skl, "bf16", "f32", m, n, k, 1.0, 0.0, 0, g, a, codes, scales)
        assert np.array_equal(first.view(np.uint32), again.view(np.uint32))


@pytest.mark.parametrize("ta,m", [("bf16", 8), ("bf16", 60), ("bf16", 130), ("f16", 100)])
def test_expired_wait_is_reported_and_the_context_survives(skl, ta, m):
    """One, two, three and four tiles to a stage: the loads are announced and not issued, the waits run out after 5 ms, the call says
    so in time, and the next call is right."""
    import time

    n, k = 700, 4096
    g = H.rng(m)
    codes, _ = MX.random_packed(g, (n, k))
    scales = np.full((n, k // 32), 127, np.uint8)
    a = g.integers(-8, 9, (m, k)).astype(np.float64)
    args = (skl, ta, "f32", False, m, n, k, 1.0, bits(ta, a), k, codes.reshape(-1), k // 2, scales.reshape(-1), k // 32, 0.0,
            np.zeros(m * n, np.float32), n)
    want = (a @ MX.values(codes, scales, k).T).astype(np.float32)
    assert np.array_equal(call(*args).reshape(m, n), want)
    skl.skl_b200_set_wait_limit(5)
    skl.skl_b200_debug_skip_loads(1)
    try:
        t0 = time.perf_counter()
        with pytest.raises(S.SklB200Error, match="stage code 0x40[123]"):
            call(*args)
        assert time.perf_counter() - t0 < 1.0, "the give-up path must not take longer than a few wait limits"
        assert skl.skl_b200_last_status() == 4 and skl.skl_b200_last_path() == S.PATH_TCGEN05
    finally:
        skl.skl_b200_debug_skip_loads(0)
        skl.skl_b200_set_wait_limit(0)
    assert np.array_equal(call(*args).reshape(m, n), want)
