"""Quantisation to MX-FP4 and the way back, through the C ABI.  Both are defined down to the bit (the header gives scale and
rounding), so every comparison is of bits; the oracle is tests/mxf4_plain.py in 64 bits."""
import numpy as np
import pytest

import helpers as H
import mxf4_plain as MX
import skl_b200 as S

pytestmark = pytest.mark.gpu

TYPES = ["f32", "bf16", "f16"]


def to_bits(t, x):
    with np.errstate(over="ignore"):
        return {"f32": lambda v: v.astype(np.float32), "bf16": lambda v: H.f32_to_bf16_bits(v.astype(np.float32)),
                "f16": lambda v: v.astype(np.float16).view(np.uint16)}[t](x)


def to_f64(t, b):
    return {"f32": lambda v: v, "bf16": H.bf16_bits_to_f32, "f16": lambda v: v.view(np.float16)}[t](b).astype(np.float64)


def hard_values(g, m, k, t):
    """Values of very different sizes: subnormals, exact powers of two, ties between neighbours, zeros of both signs, a
    block of zeros, and (from row 3 on) infinities and NaN in some blocks."""
    x = g.standard_normal((m, k)) * np.exp2(g.integers(-14 if t == "f16" else -126, 10 if t == "f16" else 100, (m, 1)))
    x[0] = np.round(x[0] * 8) / 8 if m == 1 else 0.0
    if m > 1:
        x[1] = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.0, 4.0, -0.0, -0.25, -2.5, -5.0])[g.integers(0, 14, k)]
    if m > 2:
        x[2] = np.exp2(g.integers(-10, 10, k)) * np.where(g.random(k) < 0.5, -1, 1)
    for i in range(3, m, 3):
        x[i, g.integers(0, k)] = [np.inf, -np.inf, np.nan][i // 3 % 3]
    if m > 5:
        x[5] = g.standard_normal(k) * (1e-40 if t != "f16" else 1e-6)
    return to_bits(t, x)


def run_quant(skl, t, buf, off, rs, cs, m, k, where, pad=0, dst_off=0):
    """buf: flat source array.  Returns (codes [m, rsd], scales [m, rss]) with canaries in the padding."""
    import torch

    kb = -(-k // 32)
    rsd, rss = 16 * kb + pad, kb + pad
    codes, scales = np.full(dst_off + m * rsd, 0xA5, np.uint8), np.full(dst_off + m * rss, 0x5A, np.uint8)
    fn = getattr(skl, f"skl_cvt_{t}rc_mxf4e2m1_sm100a")
    if where == "host":
        fn(S.ptr(codes) + dst_off, rsd, S.ptr(scales) + dst_off, rss, S.ptr(buf) + off * buf.itemsize, rs, cs, m, k)
        S.check()
    else:
        dc, ds, db = (torch.from_numpy(v.view(np.uint8)).cuda() for v in (codes, scales, buf))
        fn(dc.data_ptr() + dst_off, rsd, ds.data_ptr() + dst_off, rss, db.data_ptr() + off * buf.itemsize, rs, cs, m, k)
        S.check()
        codes, scales = dc.cpu().numpy(), ds.cpu().numpy()
    assert np.all(codes[:dst_off] == 0xA5) and np.all(scales[:dst_off] == 0x5A)
    codes, scales = codes[dst_off:].reshape(m, rsd), scales[dst_off:].reshape(m, rss)
    assert np.all(codes[:, 16 * kb:] == 0xA5) and np.all(scales[:, kb:] == 0x5A), "padding was written"
    return codes[:, : 16 * kb], scales[:, :kb]


SHAPES = [(1, 1), (1, 31), (1, 32), (1, 4096), (2, 33), (7, 64), (9, 250), (64, 256), (65, 257), (130, 1000), (300, 96)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layout", ["rows", "padded", "odd", "columns", "columns_odd", "both"])
def test_quantised_bits(skl, t, layout):
    """Every layout of the source: 16-byte aligned rows, a longer leading stride, rows no vector divides, columns of a
    row-major matrix, and two strides of which neither is 1."""
    for n, (m, k) in enumerate(SHAPES):
        g = H.rng(1000 * TYPES.index(t) + n)
        vals = hard_values(g, m, k, t)
        rs, cs = {"rows": (k, 1), "padded": (-(-k // 16) * 16 + 16, 1), "odd": (k + 3, 1), "columns": (1, -(-m // 8) * 8),
                  "columns_odd": (1, m + 1), "both": (2 * k + 5, 2)}[layout]
        off = 1 if layout in ("odd", "columns_odd") else 0
        buf = np.full(off + (m - 1) * rs + (k - 1) * cs + 1, to_bits(t, np.array([77.0]))[0])
        buf[off + np.arange(m)[:, None] * rs + np.arange(k)[None, :] * cs] = vals
        want = MX.quantise(to_f64(t, vals))
        got = run_quant(skl, t, buf, off, rs, cs, m, k, "device", pad=(0, 4, 3)[n % 3], dst_off=(0, 16, 5)[n % 3])
        assert np.array_equal(got[1], want[1]), (m, k, np.argwhere(got[1] != want[1])[:4])
        assert np.array_equal(got[0], want[0]), (m, k, np.argwhere(got[0] != want[0])[:4])


@pytest.mark.parametrize("t", TYPES)
def test_host_operands(skl, t):
    g = H.rng(7)
    vals = hard_values(g, 13, 100, t)
    want = MX.quantise(to_f64(t, vals))
    got = run_quant(skl, t, vals.reshape(-1), 0, 100, 1, 13, 100, "host", pad=5)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_every_tie_and_every_exponent(skl):
    """fp32: for each exponent a block can have, the magnitudes around every rounding border of a block of that size."""
    border = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    rows = []
    for e in range(-149, 128):
        around = np.concatenate([border, np.nextafter(border, 0, dtype=np.float32), np.nextafter(border, 9, dtype=np.float32), -border])
        around[0] = 4.0  # fixes the block's exponent
        with np.errstate(over="ignore", under="ignore"):
            rows.append((around[:32] * 2.0 ** (e - 2)).astype(np.float32))
    x = np.array(rows)
    want = MX.quantise(x)
    got = run_quant(skl, "f32", x.reshape(-1), 0, 32, 1, len(x), 32, "device")
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def rounded(t, v):
    """64-bit values as the type's bits; values of MX-FP4 have two significant bits, so going through fp32 rounds once."""
    with np.errstate(over="ignore", invalid="ignore"):
        return to_bits(t, v.astype(np.float32))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("where", ["device", "host"])
def test_read_back(skl, t, where):
    import torch

    for n, (m, k) in enumerate(SHAPES):
        g = H.rng(50 + n)
        pad, off = (0, 4, 3)[n % 3], (0, 16, 1)[n % 3]
        codes, scales = MX.random_packed(g, (m, k), 0, 256)
        kb = scales.shape[1]
        rsa, rss, rsd = 16 * kb + pad, kb + pad, k + (0, 8, 5)[n % 3]
        c, s = np.zeros(off + m * rsa, np.uint8), np.zeros(m * rss, np.uint8)
        c[off:].reshape(m, rsa)[:, : 16 * kb] = codes
        s.reshape(m, rss)[:, :kb] = scales
        out = np.full(m * rsd, 3, np.float32 if t == "f32" else np.uint16)
        fn = getattr(skl, f"skl_cvt_mxf4e2m1_{t}_sm100a")
        if where == "host":
            fn(S.ptr(out), rsd, S.ptr(c) + off, rsa, S.ptr(s), rss, m, k)
            S.check()
        else:
            dc, ds, do = (torch.from_numpy(v.view(np.uint8)).cuda() for v in (c, s, out))
            fn(do.data_ptr(), rsd, dc.data_ptr() + off, rsa, ds.data_ptr(), rss, m, k)
            S.check()
            out = do.cpu().numpy().view(out.dtype)
        out = out.reshape(m, rsd)
        assert np.all(out[:, k:] == 3), "the gap behind a row was written"
        want = MX.values(codes, scales, k)
        got = out[:, :k]
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(to_f64(t, got)), nan)
        assert np.array_equal(got[~nan].view(np.uint32 if t == "f32" else np.uint16),
                              rounded(t, want)[~nan].view(np.uint32 if t == "f32" else np.uint16)), (m, k)


def test_quantised_operands_go_through_the_block_scaled_product(skl):
    """Activations and weights quantised by the library, multiplied by its MX-FP4 GEMM: k = 100 is filled up to 128 with
    zeros.  Sums of 128 products of 2-bit values; the bound is the reference's forward bound on the quantised values."""
    import torch

    m, n, k = 37, 130, 100
    g = H.rng(3)
    a, w = g.standard_normal((m, k)).astype(np.float32), g.standard_normal((k, n)).astype(np.float32)
    da, dw = torch.from_numpy(a).cuda(), torch.from_numpy(w).cuda()
    pa, sa = torch.empty(m, 64, dtype=torch.uint8, device="cuda"), torch.empty(m, 4, dtype=torch.uint8, device="cuda")
    pw, sw = torch.empty(n, 64, dtype=torch.uint8, device="cuda"), torch.empty(n, 4, dtype=torch.uint8, device="cuda")
    c = torch.zeros(m, n, device="cuda")
    skl.skl_cvt_f32rc_mxf4e2m1_sm100a(pa.data_ptr(), 64, sa.data_ptr(), 4, da.data_ptr(), k, 1, m, k)
    skl.skl_cvt_f32rc_mxf4e2m1_sm100a(pw.data_ptr(), 64, sw.data_ptr(), 4, dw.data_ptr(), 1, n, n, k)
    skl.skl_gemm_mxf4e2m1_mxf4e2m1_f32_sm100a(m, n, 128, 1.0, pa.data_ptr(), 64, sa.data_ptr(), 4, pw.data_ptr(), 64,
                                              sw.data_ptr(), 4, 0.0, c.data_ptr(), n)
    S.check()
    A, W = MX.values(*MX.quantise(a), 128), MX.values(*MX.quantise(w.T), 128)
    bound = 2 * ((1 + 2.0 ** -24) ** 130 - 1) * (np.abs(A) @ np.abs(W).T)
    assert np.all(np.abs(c.cpu().numpy() - A @ W.T) <= bound)


def test_empty_and_long_strides(skl):
    for fn, args in ((skl.skl_cvt_f32rc_mxf4e2m1_sm100a, (None, 0, None, 0, None, 0, 1, 0, 5)),
                     (skl.skl_cvt_mxf4e2m1_f32_sm100a, (None, 0, None, 0, None, 0, 5, 0))):
        fn(*args)
        S.check()
        assert skl.skl_b200_last_launch_count() == 0


def test_offsets_past_32_bits(skl):
    """Two packed rows and two source rows more than 4 GiB apart."""
    import torch

    k, far = 64, (1 << 32) + 256
    buf = torch.zeros(far + 4096, dtype=torch.uint8, device="cuda")
    out = torch.zeros(far + 4096, dtype=torch.uint8, device="cuda")
    x = np.arange(2 * k, dtype=np.float32).reshape(2, k) - 40
    for i in range(2):
        buf[i * far:i * far + 4 * k] = torch.from_numpy(x[i].view(np.uint8)).cuda()
    skl.skl_cvt_f32rc_mxf4e2m1_sm100a(out.data_ptr(), far, out.data_ptr() + 1024, far, buf.data_ptr(), far // 4, 1, 2, k)
    S.check()
    codes, scales = MX.quantise(x)
    for i in range(2):
        assert np.array_equal(out[i * far:i * far + 32].cpu().numpy(), codes[i])
        assert np.array_equal(out[i * far + 1024:i * far + 1026].cpu().numpy(), scales[i])
    skl.skl_cvt_mxf4e2m1_f32_sm100a(buf.data_ptr(), far // 4, out.data_ptr(), far, out.data_ptr() + 1024, far, 2, k)
    S.check()
    for i in range(2):
        assert np.array_equal(buf[i * far:i * far + 4 * k].cpu().numpy().view(np.float32), MX.values(codes, scales, k)[i].astype(np.float32))


def test_captured_and_replayed(skl):
    import torch

    x = torch.randn(33, 1000, device="cuda")
    codes = torch.zeros(33, 512, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(33, 32, dtype=torch.uint8, device="cuda")
    y = torch.zeros(33, 1000, device="cuda")
    stream = torch.cuda.Stream()
    skl.skl_b200_set_stream(stream.cuda_stream)
    skl.skl_b200_set_async(1)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            skl.skl_cvt_f32rc_mxf4e2m1_sm100a(codes.data_ptr(), 512, scales.data_ptr(), 32, x.data_ptr(), 1000, 1, 33, 1000)
            skl.skl_cvt_mxf4e2m1_f32_sm100a(y.data_ptr(), 1000, codes.data_ptr(), 512, scales.data_ptr(), 32, 33, 1000)
            assert skl.skl_b200_last_status() == 0
        for _ in range(3):
            x.normal_()
            graph.replay()
            torch.cuda.synchronize()
            a = x.cpu().numpy()
            assert np.array_equal(y.cpu().numpy(), MX.values(*MX.quantise(a), 1000).astype(np.float32))
    finally:
        skl.skl_b200_set_stream(None)
        skl.skl_b200_set_async(0)
