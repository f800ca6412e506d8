"""16-bit activations times MX-FP4 weights in both directions, through the C ABI, against 64-bit arithmetic on the same values.

Tolerance: every product is exact (8 or 11 by 2 significant bits), so what is left is the fp32 summation, for which the
reference suite's own forward bound of a k-deep sum is used, 2 ((1 + 2^-24)^(k + 2) - 1) (|alpha| |A||W| + |beta| |C|); a
narrowed C adds half a step of its type (2^-8 of the value for bf16, 2^-11 or half the smallest subnormal for fp16)."""
import numpy as np
import pytest

import helpers as H
import mxf4_plain as MX
import skl_b200 as S

pytestmark = pytest.mark.gpu

NP = {"f32": np.float32, "bf16": np.uint16, "f16": np.uint16}
PAIRS = [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")]


def bits(t, x):
    with np.errstate(over="ignore"):
        return {"f32": lambda v: v.astype(np.float32), "bf16": lambda v: H.f32_to_bf16_bits(v.astype(np.float32)),
                "f16": lambda v: v.astype(np.float16).view(np.uint16)}[t](np.asarray(x))


def f64(t, b):
    return {"f32": lambda v: v, "bf16": H.bf16_bits_to_f32, "f16": lambda v: v.view(np.float16)}[t](b).astype(np.float64)


def tolerance(tc, want, absum, k):
    tol = 2 * ((1 + 2.0 ** -24) ** (k + 2) - 1) * absum + 2.0 ** -140
    if tc == "bf16":
        tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
    elif tc == "f16":
        tol = tol + np.maximum(2.0 ** -11 * (np.abs(want) + tol), 2.0 ** -25)
    return tol


def call(skl, ta, tc, grad, m, n, k, alpha, A, rsa, codes, rsb, scales, rss, beta, C, rsc, where="device", off=0, off_b=0):
    """A: flat bits; codes / scales: flat bytes; C: flat bits (updated copy is returned)."""
    import torch

    fn = getattr(skl, f"skl_gemm_{ta}_mxf4e2m1{'r' if grad else ''}_{tc}_sm100a")
    if where == "host":
        C = C.copy()
        fn(m, n, k, alpha, S.ptr(A) + 2 * off, rsa, S.ptr(codes) + off_b, rsb, S.ptr(scales) + off_b, rss, beta, S.ptr(C), rsc)
        S.check()
        return C
    dA, dB, dS, dC = (torch.from_numpy(v.view(np.uint8)).cuda() for v in (A, codes, scales, C))
    fn(m, n, k, alpha, dA.data_ptr() + 2 * off, rsa, dB.data_ptr() + off_b, rsb, dS.data_ptr() + off_b, rss, beta, dC.data_ptr(), rsc)
    S.check()
    return dC.cpu().numpy().view(C.dtype)


def case(skl, ta, tc, grad, m, n, k, alpha=1.0, beta=0.0, pad=0, off=0, off_b=0, where="device", seed=0, lo=118, hi=134):
    g = H.rng(seed * 1000003 + m * 7919 + n * 31 + k)
    rows, length = (k, n) if grad else (n, k)
    kb = -(-length // 32)
    codes, scales = MX.random_packed(g, (rows, length), lo, hi)
    rsa, rsb, rss, rsc = k + pad, 16 * kb + pad, kb + pad, n + pad
    a = bits(ta, g.standard_normal((m, k)) * np.exp2(g.integers(-8, 8, (m, 1))))
    A = np.full(off + m * rsa + 16, bits(ta, np.array([99.0]))[0])
    A[off:off + m * rsa].reshape(m, rsa)[:, :k] = a
    B, SC = np.full(off_b + rows * rsb, 0x77, np.uint8), np.full(off_b + rows * rss, 200, np.uint8)
    B[off_b:].reshape(rows, rsb)[:, : 16 * kb] = codes
    SC[off_b:].reshape(rows, rss)[:, :kb] = scales
    C = bits(tc, g.standard_normal(m * rsc))
    got = call(skl, ta, tc, grad, m, n, k, alpha, A, rsa, B, rsb, SC, rss, beta, C, rsc, where, off, off_b).reshape(m, rsc)
    assert np.array_equal(got[:, n:], C.reshape(m, rsc)[:, n:]), "the gap behind a row of C was written"
    W = MX.values(codes, scales, length)
    W = W if grad else W.T
    old = f64(tc, C.reshape(m, rsc)[:, :n])
    want = alpha * (f64(ta, a) @ W) + (beta * old if beta else 0.0)
    absum = abs(alpha) * (np.abs(f64(ta, a)) @ np.abs(W)) + abs(beta) * np.abs(old)
    tol = tolerance(tc, want, absum, k)
    value = f64(tc, got[:, :n])
    if tc == "f16":
        # a sum s with |s| >= 65520 (half a step above the largest finite fp16, 65504) rounds to the infinity of its sign, any
        # smaller one to a finite value; s is within tol of want, so only a want within tol of 65520 may go either way
        over = np.isinf(value)
        assert np.all(np.sign(value[over]) == np.sign(want[over])) and np.all((np.abs(want) + tol)[over] >= 65520)
        assert np.all((np.abs(want) - tol)[~over] < 65520)
        value, want = np.where(over, 0.0, value), np.where(over, 0.0, want)
    err = np.abs(value - want)
    assert np.all(err <= tol), (m, n, k, float(np.max(err / tol)), np.argwhere(err > tol)[:4])
    return got[:, :n], want


FORWARD = [(1, 1, 1), (1, 16, 32), (1, 17, 31), (2, 15, 33), (1, 300, 4096), (2, 64, 14336), (3, 33, 257), (4, 130, 1000),
           (5, 100, 544), (7, 48, 2080), (8, 257, 4099), (9, 50, 96), (17, 140, 300), (61, 520, 1024), (100, 129, 777), (130, 256, 512)]


@pytest.mark.parametrize("ta,tc", PAIRS)
def test_forward(skl, ta, tc):
    for i, (m, n, k) in enumerate(FORWARD):
        case(skl, ta, tc, False, m, n, k, alpha=(1.0, -0.5)[i % 2], beta=(0.0, 0.0, 1.5)[i % 3], seed=i)


@pytest.mark.parametrize("ta,tc", PAIRS)
def test_forward_strides_and_alignment(skl, ta, tc):
    """Leading strides beyond the row, activations and packed rows that no 16-byte load can take."""
    for i, (m, n, k) in enumerate([(1, 40, 512), (2, 33, 290), (6, 64, 300), (20, 70, 200)]):
        for pad, off, off_b in ((16, 0, 0), (8, 1, 0), (3, 0, 1), (1, 3, 5)):
            case(skl, ta, tc, False, m, n, k, beta=0.5, pad=pad, off=off, off_b=off_b, seed=i)


@pytest.mark.parametrize("ta,tc", PAIRS)
def test_gradient(skl, ta, tc):
    for i, (m, n, k) in enumerate([(1, 1, 1), (1, 70, 33), (3, 32, 100), (40, 257, 96), (128, 300, 513), (77, 64, 1030)]):
        case(skl, ta, tc, True, m, n, k, alpha=(1.0, 0.25)[i % 2], beta=(0.0, 2.0)[i % 2], pad=(0, 5, 8)[i % 3], seed=i)


@pytest.mark.parametrize("ta,tc", PAIRS)
@pytest.mark.parametrize("grad", [False, True])
def test_activations_on_any_boundary_run_on_the_tensor_cores(skl, ta, tc, grad):
    """Rows of odd length, rows at odd pitches and bases off 16 bytes, above the batches of the block-scaled kernel (and for the
    gradient from one row on): the path is the one that the header names."""
    for i, (m, n, k) in enumerate([(600, 136, 515), (520, 257, 72), (1 if grad else 513, 300, 4099)]):
        for pad, off in ((0, 0), (5, 0), (8, 1), (2, 7)):
            case(skl, ta, tc, grad, m, n, k, alpha=(1.0, -0.5)[i % 2], beta=(0.0, 0.5)[i % 2], pad=pad, off=off, seed=i)
            assert skl.skl_b200_last_path() == S.PATH_TCGEN05, (m, n, k, pad, off)
    case(skl, ta, tc, grad, 530, 40, 333, where="host")
    assert skl.skl_b200_last_path() == S.PATH_TCGEN05


def test_captured_with_activations_off_16_bytes(skl):
    """The copy's scratch belongs to the graph, as the widened weights' does; the activations are read at each replay."""
    import torch

    m, n, k = 300, 64, 259
    a, b, s, want, tol = tensors(m, n, k, 31)
    kb, c = -(-k // 32), torch.zeros(m, n, device="cuda")
    run = lambda: skl.skl_gemm_bf16_mxf4e2m1_f32_sm100a(m, n, k, 1.0, a.data_ptr(), k, b.data_ptr(), 16 * kb, s.data_ptr(), kb,  # noqa: E731
                                                        0.0, c.data_ptr(), n)
    run()
    S.check()
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    skl.skl_b200_set_async(1)
    try:
        skl.skl_b200_set_stream(st.cuda_stream)
        with torch.cuda.graph(graph, stream=st):
            run()
            assert skl.skl_b200_last_status() == 0 and skl.skl_b200_last_path() == S.PATH_TCGEN05
    finally:
        skl.skl_b200_set_stream(None)
        skl.skl_b200_set_async(0)
    old = a.clone()
    for flip in (0, 1):
        a.copy_(old)
        a.view(-1)[1::2] ^= 0x80 * flip  # the sign of every element
        torch.cuda.synchronize()
        c.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.all(np.abs(c.cpu().numpy() - (1 - 2 * flip) * want) <= tol)


@pytest.mark.parametrize("grad", [False, True])
def test_host_operands(skl, grad):
    for m, n, k in ((1, 40, 100), (12, 33, 64)):
        case(skl, "bf16", "f32", grad, m, n, k, beta=1.0, pad=3, where="host")
        case(skl, "f16", "f16", grad, m, n, k, pad=1, where="host")


@pytest.mark.parametrize("m", [1, 2, 4, 8, 16, 40])
def test_exact_sums_are_exact(skl, m):
    """Small whole activations and one scale: every partial sum is a multiple of 1/2 below 2^24, any order gives it exactly."""
    g = H.rng(m)
    n, k = 96, 700
    codes, _ = MX.random_packed(g, (n, k))
    scales = np.full((n, 22), 127, np.uint8)
    a = g.integers(-8, 9, (m, k)).astype(np.float64)
    got = call(skl, "bf16", "f32", False, m, n, k, 1.0, bits("bf16", a), k, codes.reshape(-1), 352, scales.reshape(-1), 22, 0.0,
               np.zeros(m * n, np.float32), n)
    assert np.array_equal(got.reshape(m, n), (a @ MX.values(codes, scales, k).T).astype(np.float32))


@pytest.mark.parametrize("m", [1, 2, 3, 8, 24])
def test_each_block_meets_its_scale(skl, m):
    """All weights 1, one block scaled up: the result names the row and the block that the scale reached."""
    n, k = 40, 1056
    for row, blk in ((0, 0), (7, 1), (8, 5), (15, 32), (16, 31), (39, 18)):
        codes, scales = np.full((n, 16 * 33), 0x22, np.uint8), np.full((n, 33), 127, np.uint8)
        scales[row, blk] = 130
        a = np.ones((m, k))
        a[:, blk * 32] = np.arange(m) + 2
        got = call(skl, "bf16", "f32", False, m, n, k, 1.0, bits("bf16", a), k, codes.reshape(-1), 528, scales.reshape(-1), 33,
                   0.0, np.zeros(m * n, np.float32), n).reshape(m, n)
        want = np.repeat((k + 1.0 + np.arange(m))[:, None], n, 1)
        want[:, row] += 7 * (32 + 1 + np.arange(m))
        assert np.array_equal(got, want), (row, blk)


@pytest.mark.parametrize("m", [1, 3, 8, 20])
def test_far_scales(skl, m):
    """The smallest and the largest scales, and activations 2^-20 of their block's largest next to it."""
    case(skl, "bf16", "f32", False, m, 33, 96, seed=5, lo=0, hi=3)
    case(skl, "bf16", "f32", False, m, 33, 96, seed=6, lo=236, hi=240)
    g = H.rng(9)
    n, k = 20, 64
    codes, scales = MX.random_packed(g, (n, k), 120, 130)
    codes[:, :16] &= 0xF0  # the large activations meet zeros
    a = g.standard_normal((m, k))
    a[:, 0:32:2] *= 2.0 ** 20
    b = bits("bf16", a)
    got = call(skl, "bf16", "f32", False, m, n, k, 1.0, b, k, codes.reshape(-1), 32, scales.reshape(-1), 2, 0.0,
               np.zeros(m * n, np.float32), n).reshape(m, n)
    W = MX.values(codes, scales, k).T
    want = f64("bf16", b) @ W
    assert np.all(np.abs(got - want) <= tolerance("f32", want, np.abs(f64("bf16", b)) @ np.abs(W), k))


@pytest.mark.parametrize("m", [1, 2, 3, 4, 8, 60, 300])
@pytest.mark.parametrize("top", [-118, -100, 104, 118, 119, 123, 127])
def test_large_activations_meet_small_scales(skl, m, top):
    """Activations up to the largest bf16 numbers whose products with small weights are ordinary numbers, and the reverse; in
    every other row the activations are ordinary, and some blocks of weights have the smallest scale or none but zero codes."""
    g = H.rng(abs(top + m))
    n, k = 37, 520
    codes, scales = MX.random_packed(g, (n, k), 128 - top, 134 - top) if top < 127 else MX.random_packed(g, (n, k), 1, 6)
    scales[g.random(scales.shape) < 0.1] = 0
    codes[3, 32:48] = 0
    a = g.uniform(0.5, 0.99, (m, k)) * np.where(g.random((m, k)) < 0.5, -1, 1) * 2.0 ** (top + 1)
    a[:, ::5] *= 2.0 ** -12
    a[1::2] *= 2.0 ** -top
    b = bits("bf16", a)
    assert np.all(np.isfinite(f64("bf16", b)))
    got = call(skl, "bf16", "f32", False, m, n, k, 1.0, b, k, codes.reshape(-1), 16 * 17, scales.reshape(-1), 17, 0.0,
               np.zeros(m * n, np.float32), n).reshape(m, n)
    W = MX.values(codes, scales, k).T
    want = f64("bf16", b) @ W
    absum = np.abs(f64("bf16", b)) @ np.abs(W)
    # every partial sum is at most the sum of the magnitudes: where that is below 2^127 nothing may overflow (the ordinary rows
    # under scales of 2^118 and more pass the range of 32 bits by their definition and are not compared)
    inside = absum < 2.0 ** 127
    assert np.all(inside) or top == -118
    with np.errstate(invalid="ignore"):
        err = np.abs(got - want)
    assert np.all(err[inside] <= tolerance("f32", want, absum, k)[inside])


def test_a_block_of_large_and_equal_activations(skl):
    """One row, 32 activations of 2^123, codes of 6, scale 2^-20: 32 * 6 * 2^103."""
    got = call(skl, "bf16", "f32", False, 1, 1, 32, 1.0, bits("bf16", np.full(32, 2.0 ** 123)), 32, np.full(16, 0x77, np.uint8), 16,
               np.full(1, 107, np.uint8), 1, 0.0, np.zeros(1, np.float32), 1)
    assert got[0] == np.float32(192 * 2.0 ** 103)


@pytest.mark.parametrize("m", [1, 3, 8])
def test_a_sum_past_the_range_is_infinite_and_a_scale_of_255_stays(skl, m):
    """Large activations again: zero codes under the largest scale stay zero, sums past fp32's range become infinities of
    their sign, a block of scale 255 makes its column NaN, all in the same blocks of activations."""
    n, k = 4, 64
    codes, scales = np.full((n, 32), 0x22, np.uint8), np.full((n, 2), 127 - 110, np.uint8)  # ones times 2^-110
    codes[1, :16], scales[1, 0] = 0, 252
    codes[2, :] = 0xAA  # minus ones
    scales[2] = 200
    scales[3, 1] = 255
    b = bits("bf16", np.full((m, k), 2.0 ** 125))
    got = call(skl, "bf16", "f32", False, m, n, k, 1.0, b, k, codes.reshape(-1), 32, scales.reshape(-1), 2, 0.0,
               np.zeros(m * n, np.float32), n).reshape(m, n)
    assert np.all(got[:, 0] == 64 * 2.0 ** 15) and np.all(got[:, 1] == 32 * 2.0 ** 15)
    assert np.all(got[:, 2] == -np.inf) and np.all(np.isnan(got[:, 3]))


@pytest.mark.parametrize("ta", ["bf16", "f16"])
@pytest.mark.parametrize("m", [2, 8, 24])
def test_not_finite_values_stay_where_they_are(skl, ta, m):
    g = H.rng(4)
    n, k = 35, 320
    codes, scales = MX.random_packed(g, (n, k), 120, 130)
    scales[5, 3] = 255
    a = g.standard_normal((m, k))
    a[1, 40], a[m - 1, 300] = np.nan, np.inf
    got = f64("f32", call(skl, ta, "f32", False, m, n, k, 1.0, bits(ta, a), k, codes.reshape(-1), 160, scales.reshape(-1), 10, 0.0,
                          np.zeros(m * n, np.float32), n).reshape(m, n))
    ok = np.ones((m, n), bool)
    ok[:, 5] = ok[1] = ok[m - 1] = False
    assert np.all(np.isfinite(got[ok])) and np.all(np.isnan(got[:, 5])) and np.all(np.isnan(got[1]))
    assert not np.any(np.isfinite(got[m - 1]))


def test_no_k_and_no_rows(skl):
    import torch

    c = torch.arange(12, dtype=torch.float32, device="cuda")
    skl.skl_gemm_bf16_mxf4e2m1_f32_sm100a(3, 4, 0, 1.0, None, 0, None, 0, None, 0, 2.0, c.data_ptr(), 4)
    S.check()
    assert torch.equal(c.cpu(), 2 * torch.arange(12, dtype=torch.float32))
    skl.skl_gemm_bf16_mxf4e2m1_f32_sm100a(3, 4, 0, 1.0, None, 0, None, 0, None, 0, 0.0, c.data_ptr(), 4)
    S.check()
    assert not c.any()
    for m, n in ((0, 4), (4, 0)):
        skl.skl_gemm_f16_mxf4e2m1r_f16_sm100a(m, n, 8, 1.0, None, 8, None, 16, None, 1, 0.0, None, 4)
        S.check()


def tensors(m, n, k, seed, grad=False):
    import torch

    g = H.rng(seed)
    rows, length = (k, n) if grad else (n, k)
    codes, scales = MX.random_packed(g, (rows, length))
    a = bits("bf16", g.standard_normal((m, k)))
    W = MX.values(codes, scales, length)
    want = f64("bf16", a) @ (W if grad else W.T)
    absum = np.abs(f64("bf16", a)) @ np.abs(W if grad else W.T)
    return [torch.from_numpy(v.view(np.uint8).copy()).cuda() for v in (a, codes, scales)] + [want, tolerance("f32", want, absum, k)]


@pytest.mark.parametrize("ta", ["bf16", "f16"])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("m,n,k", [(2048, 4096, 992), (1100, 5000, 1515)])
def test_several_rounds_of_tiles(skl, ta, grad, m, n, k):
    """Widened products with more tiles than the chip takes at once, on pairs of SMs where the shape allows; compared on the GPU."""
    import torch

    g = H.rng(m + n)
    rows, length = (k, n) if grad else (n, k)
    kb = -(-length // 32)
    codes, scales = MX.random_packed(g, (rows, length), 112, 122)
    a = bits(ta, g.standard_normal((m, k)) * np.exp2(g.integers(-4, 4, (m, 1))))
    A, B, SC = (torch.from_numpy(np.ascontiguousarray(v).view(np.uint8)).cuda() for v in (a, codes, scales))
    c = torch.zeros(m, n, device="cuda")
    fn = getattr(skl, f"skl_gemm_{ta}_mxf4e2m1{'r' if grad else ''}_f32_sm100a")
    fn(m, n, k, 1.0, A.data_ptr(), k, B.data_ptr(), 16 * kb, SC.data_ptr(), kb, 0.0, c.data_ptr(), n)
    S.check()
    assert skl.skl_b200_last_path() == S.PATH_TCGEN05
    x, W = torch.from_numpy(f64(ta, a)).cuda(), torch.from_numpy(MX.values(codes, scales, length)).cuda()
    W = W if grad else W.T
    absum = x.abs() @ W.abs()
    assert torch.all((c.double() - x @ W).abs() <= tolerance("f32", 0.0, absum, k))


@pytest.mark.parametrize("m", [1, 40])
def test_two_graphs_side_by_side(skl, m):
    """Two captured products, replayed together on two streams, then after a larger call has come and gone."""
    import torch

    n, k = 200, 1024
    sets = [tensors(m, n, k, s) for s in (1, 2)]
    outs = [torch.zeros(m, n, device="cuda") for _ in sets]
    fn = skl.skl_gemm_bf16_mxf4e2m1_f32_sm100a

    def go(i):
        a, b, s = sets[i][:3]
        fn(m, n, k, 1.0, a.data_ptr(), k, b.data_ptr(), k // 2, s.data_ptr(), k // 32, 0.0, outs[i].data_ptr(), n)

    go(0)  # first call of the thread: status words and kernel attributes
    streams, graphs = [torch.cuda.Stream() for _ in sets], []
    skl.skl_b200_set_async(1)
    try:
        for i, st in enumerate(streams):
            skl.skl_b200_set_stream(st.cuda_stream)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                go(i)
                assert skl.skl_b200_last_status() == 0
            graphs.append(graph)
        skl.skl_b200_set_stream(None)
        for after in range(2):
            torch.cuda.synchronize()
            for o in outs:
                o.zero_()
            torch.cuda.synchronize()
            for _ in range(5):
                for graph, st in zip(graphs, streams):
                    with torch.cuda.stream(st):
                        graph.replay()
            torch.cuda.synchronize()
            for s, o in zip(sets, outs):
                assert np.all(np.abs(o.cpu().numpy() - s[3]) <= s[4])
            skl.skl_b200_set_async(0)
            big = tensors(64, 1000, 2048, 3)
            c = torch.zeros(64, 1000, device="cuda")
            fn(64, 1000, 2048, 1.0, big[0].data_ptr(), 2048, big[1].data_ptr(), 1024, big[2].data_ptr(), 64, 0.0, c.data_ptr(), 1000)
            S.check()
            assert np.all(np.abs(c.cpu().numpy() - big[3]) <= big[4])
            skl.skl_b200_release_workspace()
    finally:
        skl.skl_b200_set_stream(None)
        skl.skl_b200_set_async(0)


@pytest.mark.parametrize("m", [1, 8, 33])
def test_same_bits_every_time(skl, m):
    import torch

    n, k = 500, 3000
    a, b, s, want, tol = tensors(m, n, k, 8)
    kb = -(-k // 32)
    first = None
    for _ in range(4):
        c = torch.zeros(m, n, device="cuda")
        skl.skl_gemm_bf16_mxf4e2m1_f32_sm100a(m, n, k, 1.0, a.data_ptr(), k, b.data_ptr(), 16 * kb, s.data_ptr(), kb, 0.0, c.data_ptr(), n)
        S.check()
        first = c if first is None else first
        assert torch.equal(c, first)
    assert np.all(np.abs(first.cpu().numpy() - want) <= tol)


def test_declared_static_weights_give_the_same_bits(skl):
    import torch

    m, n, k = 2, 320, 2048
    a, b, s, want, tol = tensors(m, n, k, 11)
    out = [torch.zeros(m, n, device="cuda") for _ in range(2)]
    for i in (0, 1):
        skl.skl_b200_set_static_weights(i)
        try:
            for _ in range(3):
                skl.skl_gemm_bf16_mxf4e2m1_f32_sm100a(m, n, k, 1.0, a.data_ptr(), k, b.data_ptr(), k // 2, s.data_ptr(), k // 32,
                                                      0.0, out[i].data_ptr(), n)
                S.check()
        finally:
            skl.skl_b200_set_static_weights(0)
    assert torch.equal(out[0], out[1]) and np.all(np.abs(out[0].cpu().numpy() - want) <= tol)


def test_quantise_multiply_and_gradient_as_a_layer_uses_them(skl):
    """fp32 weights K x N quantised along k by columns; y = x W; dx = dy W^T with the same packed matrix; and the gradient
    against differences of the forward product (y is linear in x: a difference of two products, exact up to their sums)."""
    import torch

    m, n, k = 24, 160, 288
    g = H.rng(21)
    w = g.standard_normal((k, n)).astype(np.float32) * 0.1
    dw = torch.from_numpy(w).cuda()
    codes, scales = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda"), torch.zeros(n, k // 32, dtype=torch.uint8, device="cuda")
    skl.skl_cvt_f32rc_mxf4e2m1_sm100a(codes.data_ptr(), k // 2, scales.data_ptr(), k // 32, dw.data_ptr(), 1, n, n, k)
    S.check()
    W = MX.values(*MX.quantise(w.T), k)  # [n][k]
    x, dy = bits("bf16", g.standard_normal((m, k))), bits("bf16", g.standard_normal((m, n)))

    def forward(xb):
        return call(skl, "bf16", "f32", False, m, n, k, 1.0, xb, k, codes.cpu().numpy().reshape(-1), k // 2,
                    scales.cpu().numpy().reshape(-1), k // 32, 0.0, np.zeros(m * n, np.float32), n).reshape(m, n).astype(np.float64)

    y = forward(x)
    want = f64("bf16", x) @ W.T
    assert np.all(np.abs(y - want) <= tolerance("f32", want, np.abs(f64("bf16", x)) @ np.abs(W).T, k))
    # dx = dy W: contraction over n, the packed rows of W are its rows
    dx = call(skl, "bf16", "f32", True, m, k, n, 1.0, dy, n, codes.cpu().numpy().reshape(-1), k // 2, scales.cpu().numpy().reshape(-1),
              k // 32, 0.0, np.zeros(m * k, np.float32), k).reshape(m, k).astype(np.float64)
    wantdx = f64("bf16", dy) @ W
    assert np.all(np.abs(dx - wantdx) <= tolerance("f32", wantdx, np.abs(f64("bf16", dy)) @ np.abs(W), n))
    for col in (0, 31, 32, 287):
        up = f64("bf16", x).copy()
        up[:, col] += 4.0  # exact in bf16 or not, the difference below uses what was stored
        ub = bits("bf16", up)
        step = f64("bf16", ub)[:, col] - f64("bf16", x)[:, col]
        diff = ((forward(ub) - y) * f64("bf16", dy)).sum(1)
        slack = 2 * tolerance("f32", want, (np.abs(f64("bf16", x)) + 8) @ np.abs(W).T, k)
        assert np.all(np.abs(diff - step * dx[:, col]) <= (slack * np.abs(f64("bf16", dy))).sum(1) + 8 * 2.0 ** -16 * np.abs(wantdx).max())


@pytest.mark.parametrize("m,ta,grad", [(2, "bf16", False), (9, "bf16", False), (9, "f16", False), (300, "bf16", False), (9, "f16", True)])
def test_offsets_past_32_bits(skl, m, ta, grad):
    """The last rows of every operand lie more than 4 GiB behind the first.  Whole numbers: the sums are exact."""
    import torch

    n, k = 40, 96
    rows, length = (k, n) if grad else (n, k)
    kb = -(-length // 32)
    step = lambda r: (((1 << 32) // (r - 1) + 4096) // 256) * 256  # noqa: E731  bytes from row to row
    g = H.rng(m)
    codes, _ = MX.random_packed(g, (rows, length))
    scales = np.full((rows, kb), 127, np.uint8)
    a = g.integers(-8, 9, (m, k)).astype(np.float64)

    def far(v):
        v = np.ascontiguousarray(v).view(np.uint8).reshape(v.shape[0], -1)
        by = step(v.shape[0])
        buf = torch.empty((v.shape[0] - 1) * by + v.shape[1], dtype=torch.uint8, device="cuda")
        torch.as_strided(buf, v.shape, (by, 1)).copy_(torch.from_numpy(v).cuda())
        return buf, by

    (da, sa), (db, sb), (ds, ss), (dc, sc) = (far(v) for v in (bits(ta, a), codes, scales, np.zeros((m, n), np.float32)))
    fn = getattr(skl, f"skl_gemm_{ta}_mxf4e2m1{'r' if grad else ''}_f32_sm100a")
    fn(m, n, k, 1.0, da.data_ptr(), sa // 2, db.data_ptr(), sb, ds.data_ptr(), ss, 0.0, dc.data_ptr(), sc // 4)
    S.check()
    got = torch.as_strided(dc, (m, 4 * n), (sc, 1)).contiguous().cpu().numpy().view(np.float32)
    W = MX.values(codes, scales, length)
    assert np.array_equal(got, (a @ (W if grad else W.T)).astype(np.float32))


@pytest.mark.parametrize("m,grad", [(1, False), (4, False), (30, False), (300, False), (2, True)])
def test_profiled_calls_are_counted_and_timed(skl, m, grad):
    """skl_b200_profile_begin / _end around the products of every path: as many records as calls, no more than were asked for."""
    import ctypes

    import torch

    n, k = 2048, 1024
    a, b, s, want, tol = tensors(m, n, k, m, grad)
    kb, c = -(-(n if grad else k) // 32), torch.zeros(m, n, device="cuda")
    fn = skl.skl_gemm_bf16_mxf4e2m1r_f32_sm100a if grad else skl.skl_gemm_bf16_mxf4e2m1_f32_sm100a
    for asked, calls in ((3, 3), (2, 4)):
        skl.skl_b200_profile_begin(asked)
        for _ in range(calls):
            fn(m, n, k, 1.0, a.data_ptr(), k, b.data_ptr(), 16 * kb, s.data_ptr(), kb, 0.0, c.data_ptr(), n)
            S.check()
        ms = ctypes.c_double(0.0)
        assert skl.skl_b200_profile_end(ctypes.byref(ms)) == min(asked, calls)
        assert 0.0 < ms.value < 100.0
    assert np.all(np.abs(c.cpu().numpy() - want) <= tol)


def test_two_threads_at_once(skl):
    """Every path from two threads, each on a stream of its own; the calls share the library's pool of scratch memory."""
    import threading

    import torch

    lib, n, k = S.lib(), 520, 1024
    shapes = [(2, False), (30, False), (400, False), (50, True)]
    jobs = []
    for t in range(2):
        g = H.rng(t)
        for m, grad in shapes:
            rows, length = (k, n) if grad else (n, k)
            codes, _ = MX.random_packed(g, (rows, length))
            scales = np.full((rows, -(-length // 32)), 127, np.uint8)
            a = g.integers(-8, 9, (m, k)).astype(np.float64)
            W = MX.values(codes, scales, length)
            jobs.append((t, m, grad, *(torch.from_numpy(v.view(np.uint8)).cuda() for v in (bits("bf16", a), codes, scales)), length,
                         torch.zeros(m, n, device="cuda"), (a @ (W if grad else W.T)).astype(np.float32)))
    torch.cuda.synchronize()
    failed = []

    def work(t):
        torch.cuda.set_device(0)
        stream = torch.cuda.Stream()
        lib.skl_b200_set_stream(stream.cuda_stream)
        lib.skl_b200_set_async(1)
        for _ in range(20):
            for owner, m, grad, a, b, s, length, c, _want in jobs:
                if owner == t:
                    fn = lib.skl_gemm_bf16_mxf4e2m1r_f32_sm100a if grad else lib.skl_gemm_bf16_mxf4e2m1_f32_sm100a
                    kb = -(-length // 32)
                    fn(m, n, k, 1.0, a.data_ptr(), k, b.data_ptr(), 16 * kb, s.data_ptr(), kb, 0.0, c.data_ptr(), n)
                    if lib.skl_b200_last_status() != 0:
                        failed.append((t, m, grad))
        lib.skl_b200_synchronize()
        if lib.skl_b200_last_status() != 0:
            failed.append((t, "synchronize"))

    threads = [threading.Thread(target=work, args=(t,)) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    torch.cuda.synchronize()
    for _t, m, grad, _a, _b, _s, _l, c, want in jobs:
        assert np.array_equal(c.cpu().numpy(), want), (m, grad)
