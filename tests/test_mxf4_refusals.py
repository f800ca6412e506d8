"""What the MX-FP4 entry points refuse, before any device is touched (runs without a GPU)."""
import numpy as np
import pytest

import skl_b200 as S

INVALID, UNSUPPORTED = 1, 5
B = S.ptr(np.zeros(4096, np.uint8))


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_cvt_refusals(skl, t):
    to, back = getattr(skl, f"skl_cvt_{t}rc_mxf4e2m1_sm100a"), getattr(skl, f"skl_cvt_mxf4e2m1_{t}_sm100a")
    good_to, good_back = [B, 32, B, 2, B, 33, 1, 2, 33], [B, 33, B, 32, B, 2, 2, 33]
    for at, bad in [(0, 0), (2, 0), (4, 0), (1, 31), (3, 1), (7, 1 << 31), (8, 1 << 31)]:
        args = list(good_to)
        args[at] = bad
        to(*args)
        assert skl.skl_b200_last_status() == INVALID, (at, bad)
    for at, bad in [(0, 0), (2, 0), (4, 0), (1, 32), (3, 31), (5, 1), (6, 1 << 31), (7, 1 << 31)]:
        args = list(good_back)
        args[at] = bad
        back(*args)
        assert skl.skl_b200_last_status() == INVALID, (at, bad)


@pytest.mark.parametrize("name", ["bf16_mxf4e2m1_f32", "bf16_mxf4e2m1_bf16", "f16_mxf4e2m1_f32", "f16_mxf4e2m1_f16",
                                  "bf16_mxf4e2m1r_f32", "bf16_mxf4e2m1r_bf16", "f16_mxf4e2m1r_f32", "f16_mxf4e2m1r_f16"])
def test_product_refusals(skl, name):
    """m, n, k, alpha, a, rsa, b, rsb, sb, rssb, beta, c, rsc with n = k = 33: two blocks to a packed row either way."""
    fn = getattr(skl, f"skl_gemm_{name}_sm100a")
    good = [2, 33, 33, 1.0, B, 33, B, 32, B, 2, 0.0, B, 33]
    for at, bad in [(4, 0), (6, 0), (8, 0), (11, 0), (5, 32), (7, 31), (9, 1), (12, 32), (0, 1 << 31), (1, 1 << 31), (2, 1 << 31)]:
        args = list(good)
        args[at] = bad
        fn(*args)
        assert skl.skl_b200_last_status() == INVALID, (at, bad)


@pytest.mark.parametrize("mx", [False, True])
def test_moe_refusals(skl, mx):
    fn = skl.skl_moe_swiglu_bf16_mxf4e2m1_bf16_sm100a if mx else skl.skl_moe_swiglu_bf16_bf16_bf16_sm100a
    size = skl.skl_b200_moe_workspace_size(2, 16, 4, 2)
    assert size >= 2 * 2 * 16 * 4 and skl.skl_b200_moe_workspace_size(65, 16, 4, 2) == 0
    weights = [B] * (4 if mx else 2)
    good = [2, 32, 16, 4, 2, 1, B, 4, B, 32, *weights, B, 32, B, B, B, size]
    y = 10 + len(weights)
    for at, bad, status in [(1, 0, INVALID), (2, 0, INVALID), (4, 0, INVALID), (4, 5, INVALID), (6, 0, INVALID), (7, 3, INVALID),
                            (8, 0, INVALID), (9, 31, INVALID), (10, 0, INVALID), (y - 1, 0, INVALID), (y, 0, INVALID),
                            (y + 1, 31, INVALID), (y + 2, 0, INVALID), (y + 3, 0, INVALID), (y + 4, 0, INVALID),
                            (y + 4, B + 2, INVALID), (y + 5, size - 1, INVALID), (0, 65, UNSUPPORTED)]:
        args = list(good)
        args[at] = bad
        fn(*args)
        assert skl.skl_b200_last_status() == status, (at, bad)
    for at, bad in [(1, 32769), (2, 32769), (3, 1025), (4, 33)]:
        args = list(good)
        args[3], args[7], args[9], args[y + 1] = 1024, 4096, 40000, 40000
        args[at] = bad
        fn(*args)
        assert skl.skl_b200_last_status() == UNSUPPORTED, (at, bad)
