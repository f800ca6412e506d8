"""The block-scaled 4-bit operators and the experts' layer: what is timed, on which inputs, and the plain arithmetic they stand for.

Four operators around OCP MX-FP4 data (E2M1 elements, two per byte, low nibble first; one E8M0 scale byte per block of
32 consecutive elements of a row; a row whose length is no multiple of 32 ends in a block padded with zeros):

* ``quant``: a matrix is quantised to MX-FP4 and read back.  The scale exponent of a block is floor(log2(largest
  magnitude)) - 2, the elements are rounded to nearest even and saturate at 6 times the scale.
* ``read``: packed rows are widened to bf16, fp16 or fp32.
* ``gemm``: 16-bit activations times MX-FP4 weights.  ``grad`` false: C[m, n] = A[m, k] W[n, k]^T; true: the product of
  the backward pass, C[m, n] = A[m, k] W[k, n], where A is the gradient of the layer's output.
* ``moe``: a mixture-of-experts layer for few tokens.  From the router's fp32 logits: the topk largest (ties to the lowest
  index), their softmax as gates; y = sum_j gate_j * W2[e_j] (silu(G x) * (U x)), G and U the two halves of W1[e_j].

A case is a dict of plain values; `run` makes one pass, in elementary torch operations in 32 bits, or, where `own` is
true, through skl_b200's entry points.  `exact` computes the same from the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_ES = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token's activations before a 4-bit product: latency of the smallest call
        {"name": "quant_one_token", "op": "quant", "m": 1, "k": 4096, "src": "bf16", "out": "bf16", "columns": False},
        # the activations of a long batch
        {"name": "quant_batch", "op": "quant", "m": 16384, "k": 4096, "src": "bf16", "out": "bf16", "columns": False},
        # fp32 master weights stored K x N, quantised along K (a column of the source becomes a packed row)
        {"name": "quant_weights_by_column", "op": "quant", "m": 14336, "k": 4096, "src": "f32", "out": "bf16", "columns": True},
        # packed weights widened for a layer that wants them in 16 bits
        {"name": "read_weights", "op": "read", "m": 14336, "k": 4096, "out": "bf16"},
        # an odd slice for inspection: ragged last block, rows that no vector width divides
        {"name": "read_odd", "op": "read", "m": 333, "k": 4099, "out": "f32"},
        # a decode step: one token through the up projection, and two through the down projection
        {"name": "gemm_one_token", "op": "gemm", "m": 1, "n": 14336, "k": 4096, "a": "bf16", "out": "bf16", "grad": False},
        {"name": "gemm_two_tokens_down", "op": "gemm", "m": 2, "n": 4096, "k": 14336, "a": "f16", "out": "f32", "grad": False},
        # a batch of decode steps, odd in m
        {"name": "gemm_decode_batch", "op": "gemm", "m": 61, "n": 14336, "k": 4096, "a": "bf16", "out": "bf16", "grad": False},
        # a prompt, or a training step over frozen weights
        {"name": "gemm_prompt", "op": "gemm", "m": 4096, "n": 14336, "k": 4096, "a": "bf16", "out": "bf16", "grad": False},
        # the gradient of that step's input, for half as many tokens
        {"name": "gemm_gradient", "op": "gemm", "m": 2048, "n": 4096, "k": 14336, "a": "bf16", "out": "bf16", "grad": True},
        # one token through 8 of 64 experts, 16-bit weights
        {"name": "moe_one_token", "op": "moe", "m": 1, "d": 2048, "f": 1024, "experts": 64, "topk": 8, "w": "bf16"},
        # a small batch of tokens that meets nearly every expert, 4-bit weights
        {"name": "moe_batch_4bit", "op": "moe", "m": 16, "d": 2048, "f": 1024, "experts": 64, "topk": 8, "w": "mxf4"},
    ]


def draw(rng):
    def size(lo, hi, step=1):
        """log-uniform in [lo, hi]; two in three are a multiple of 32 (or of `step`), where that is no smaller than lo"""
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        unit = 32 if rng.random() < 0.67 else step
        return min(hi, max(lo, v // unit * unit if v >= unit else v))

    op = rng.choice(["quant", "quant", "read", "gemm", "gemm", "gemm", "moe", "moe"])
    if op in ("quant", "read"):
        while True:
            m, k = size(1, 16384), size(16, 16384)
            if m * k <= 16384 * 4096:
                break
        if op == "read":
            return {"op": op, "m": m, "k": k, "out": rng.choice(["bf16", "f16", "f32"])}
        src = rng.choice(["bf16", "f16", "f32"])
        return {"op": op, "m": m, "k": k, "src": src, "out": rng.choice([src, "f32"]), "columns": rng.random() < 0.4}
    if op == "gemm":
        a = rng.choice(["bf16", "bf16", "f16"])
        while True:
            m, n, k = rng.choice([size(1, 16), size(1, 512), size(16, 4096)]), size(64, 14336), size(64, 14336)
            if m * n * k <= 4096 * 14336 * 4096 and n * k >= 1 << 18 and n * k <= 14336 * 4096:
                break
        return {"op": op, "m": m, "n": n, "k": k, "a": a, "out": rng.choice([a, "f32"]), "grad": rng.random() < 0.25}
    while True:
        m, d, f = rng.choice([1, 2, 3, 4, size(1, 32), size(1, 32)]), size(256, 4096, 8), size(128, 2048, 8)
        e = rng.choice([8, 16, 32, 60, 64, 128])
        topk = rng.choice([1, 2, 4, 6, 8])
        if e * d * f <= 64 * 2048 * 1024 and m * topk * d * f <= 16 * 8 * 2048 * 1024:
            break
    return {"op": op, "m": m, "d": d, "f": f, "experts": e, "topk": topk, "w": rng.choice(["bf16", "mxf4"])}


# ------------------------------------------------------------------------------------------ MX-FP4 in plain operations
def _blocks(k):
    return (k + 31) // 32


def _power(byte):
    """2^(byte - 127) in fp32 from its bit pattern (0: the subnormal 2^-127, 255: NaN): a pow() on the GPU need not be exact."""
    byte = byte.to(torch.int32)
    bits = torch.where(byte == 0, 0x00400000, torch.where(byte == 255, 0x7FC00000, byte << 23))
    return bits.to(torch.int32).view(torch.float32)


def _quantised(x):
    """(elements in units of the scale, scale exponents) of the rows of x: [m, blocks, 32] and [m, blocks] in fp32 / int32."""
    m, k = x.shape
    x = x.to(torch.float32)
    if k % 32:
        x = torch.cat([x, x.new_zeros(m, 32 - k % 32)], 1)
    x = x.reshape(m, -1, 32)
    top = x.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, torch.full_like(top, -127, dtype=torch.int32)).clamp_min(-127)
    y = x * _power(127 - e).unsqueeze(-1)
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp_max(6.0), y), e


def _packed(x):
    """(codes uint8 [m, 16 blocks], scales uint8 [m, blocks]) of the rows of x."""
    q, e = _quantised(x)
    a = q.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) + 8 * (torch.signbit(q)).to(torch.uint8)
    code = code.reshape(x.shape[0], -1, 2)
    return (code[..., 0] | (code[..., 1] << 4)).contiguous(), (e + 127).to(torch.uint8)


def _values(codes, scales, k):
    """fp32 values of packed rows (any leading dimensions), cut to k columns."""
    nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int32)
    mag = nib & 7
    v = torch.where(mag < 4, mag * 0.5, torch.where(mag < 6, mag - 2.0, mag * 2.0 - 8.0))
    v = torch.where(nib >= 8, -v, v).reshape(*scales.shape, 32)
    return (v * _power(scales).unsqueeze(-1)).flatten(-2)[..., :k]


# ------------------------------------------------------------------------------------------------------------ inputs
def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _activations(gen, m, k):
    """Normal values, one channel in a hundred twenty times as large, rows of different size."""
    x = _normal(gen, m, k) * torch.exp2(torch.randint(-3, 4, (m, 1), device="cuda", generator=gen).float())
    return x * torch.where(torch.rand(k, device="cuda", generator=gen) < 0.01, 20.0, 1.0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, s = case["op"], dict(case)
    if op == "quant":
        m, k = case["m"], case["k"]
        x = _activations(gen, m, k) if not case["columns"] else _normal(gen, k, m) * 0.02
        s["x"] = x.to(_DT[case["src"]])
        s["codes"] = torch.zeros(m, 16 * _blocks(k), dtype=torch.uint8, device="cuda")
        s["scales"] = torch.zeros(m, _blocks(k), dtype=torch.uint8, device="cuda")
        s["y"] = torch.zeros(m, k, dtype=_DT[case["out"]], device="cuda")
    elif op == "read":
        s["codes"], s["scales"] = _packed(_normal(gen, case["m"], case["k"]) * 0.02)
        s["y"] = torch.zeros(case["m"], case["k"], dtype=_DT[case["out"]], device="cuda")
    elif op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        x = _activations(gen, m, k) if not case["grad"] else _normal(gen, m, k) * 0.01
        s["x"] = x.to(_DT[case["a"]])
        # a packed row runs along k for the forward product, along n for the gradient's
        s["codes"], s["scales"] = _packed(_normal(gen, *((k, n) if case["grad"] else (n, k))) / math.sqrt(k))
        s["y"] = torch.zeros(m, n, dtype=_DT[case["out"]], device="cuda")
    else:
        m, d, f, e = case["m"], case["d"], case["f"], case["experts"]
        s["x"] = _normal(gen, m, d).to(torch.bfloat16)
        s["logits"] = _normal(gen, m, e) * 2.0
        for name, rows, cols in (("w1", 2 * f, d), ("w2", d, f)):
            if case["w"] == "bf16":
                s[name] = torch.empty(e, rows, cols, dtype=torch.bfloat16, device="cuda")
                for i in range(e):
                    s[name][i] = _normal(gen, rows, cols) / math.sqrt(cols)
            else:
                s[name] = torch.empty(e, rows, 16 * _blocks(cols), dtype=torch.uint8, device="cuda")
                s["s" + name[1]] = torch.empty(e, rows, _blocks(cols), dtype=torch.uint8, device="cuda")
                for i in range(e):
                    s[name][i], s["s" + name[1]][i] = _packed(_normal(gen, rows, cols) / math.sqrt(cols))
        s["y"] = torch.zeros(m, d, dtype=torch.bfloat16, device="cuda")
        s["ids"] = torch.zeros(m, case["topk"], dtype=torch.int32, device="cuda")
        s["gates"] = torch.zeros(m, case["topk"], dtype=torch.float32, device="cuda")
        # the layer keeps its intermediate values in a buffer of the caller's, one for each call in flight
        s["work"] = torch.zeros(1 << 16 | (m * case["topk"] * (f + 64) * 8), dtype=torch.uint8, device="cuda")
    return s


# --------------------------------------------------------------------------------------------------------------- run
def _library():
    """skl_b200's functions, on torch's current stream, without waiting for the device after each call."""
    import skl_b200

    lib = skl_b200.lib()
    lib.skl_b200_set_stream(torch.cuda.current_stream().cuda_stream)
    lib.skl_b200_set_async(1)
    return lib


def _run_own(s):
    lib, op = _library(), s["op"]
    if op == "quant":
        m, k = s["m"], s["k"]
        c, e, x, y = s["codes"], s["scales"], s["x"], s["y"]
        rs, cs = (1, m) if s["columns"] else (k, 1)
        getattr(lib, "skl_cvt_%src_mxf4e2m1_sm100a" % s["src"])(c.data_ptr(), c.shape[1], e.data_ptr(), e.shape[1], x.data_ptr(), rs, cs, m, k)
        getattr(lib, "skl_cvt_mxf4e2m1_%s_sm100a" % s["out"])(y.data_ptr(), k, c.data_ptr(), c.shape[1], e.data_ptr(), e.shape[1], m, k)
        return y
    if op == "read":
        c, e, y = s["codes"], s["scales"], s["y"]
        getattr(lib, "skl_cvt_mxf4e2m1_%s_sm100a" % s["out"])(y.data_ptr(), s["k"], c.data_ptr(), c.shape[1], e.data_ptr(), e.shape[1], s["m"], s["k"])
        return y
    if op == "gemm":
        m, n, k = s["m"], s["n"], s["k"]
        c, e, x, y = s["codes"], s["scales"], s["x"], s["y"]
        fn = getattr(lib, "skl_gemm_%s_mxf4e2m1%s_%s_sm100a" % (s["a"], "r" if s["grad"] else "", s["out"]))
        fn(m, n, k, 1.0, x.data_ptr(), k, c.data_ptr(), c.shape[1], e.data_ptr(), e.shape[1], 0.0, y.data_ptr(), n)
        return y
    m, d, f = s["m"], s["d"], s["f"]
    head = (m, d, f, s["experts"], s["topk"], 1, s["logits"].data_ptr(), s["experts"], s["x"].data_ptr(), d)
    tail = (s["y"].data_ptr(), d, s["ids"].data_ptr(), s["gates"].data_ptr(), s["work"].data_ptr(), s["work"].numel())
    if s["w"] == "bf16":
        lib.skl_moe_swiglu_bf16_bf16_bf16_sm100a(*head, s["w1"].data_ptr(), s["w2"].data_ptr(), *tail)
    else:
        lib.skl_moe_swiglu_bf16_mxf4e2m1_bf16_sm100a(*head, s["w1"].data_ptr(), s["s1"].data_ptr(), s["w2"].data_ptr(), s["s2"].data_ptr(), *tail)
    return s["y"], s["ids"], s["gates"]


def run(s):
    if own:
        return _run_own(s)
    op = s["op"]
    if op == "quant":
        q, e = _quantised(s["x"].t() if s["columns"] else s["x"])
        return (q * _power(e + 127).unsqueeze(-1)).flatten(-2)[:, : s["k"]].to(s["y"].dtype)
    if op == "read":
        return _values(s["codes"], s["scales"], s["k"]).to(s["y"].dtype)
    if op == "gemm":
        w = _values(s["codes"], s["scales"], s["n"] if s["grad"] else s["k"])
        return (s["x"].float() @ (w if s["grad"] else w.t())).to(s["y"].dtype)
    x, f = s["x"].float(), s["f"]
    top, ids = torch.sort(s["logits"], dim=-1, descending=True, stable=True)
    top, ids = top[:, : s["topk"]], ids[:, : s["topk"]]
    g = torch.exp(top - top[:, :1])
    g = g / g.sum(-1, keepdim=True)
    if s["w"] == "bf16":
        w1, w2 = s["w1"][ids].float(), s["w2"][ids].float()
    else:
        w1, w2 = _values(s["w1"][ids], s["s1"][ids], s["d"]), _values(s["w2"][ids], s["s2"][ids], f)
    h = (w1 @ x[:, None, :, None]).squeeze(-1)
    h = h[..., :f] / (1 + torch.exp(-h[..., :f])) * h[..., f:]
    y = ((w2 @ h.unsqueeze(-1)).squeeze(-1) * g.unsqueeze(-1)).sum(1)
    return y.to(torch.bfloat16), ids.to(torch.int32), g


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op in ("quant", "read"):
        m, k = case["m"], case["k"]
        packed = m * _blocks(k) * 17
        return {"bytes": packed + m * k * (_ES[case["out"]] + (_ES[case["src"]] if op == "quant" else 0)), "flops": 0}
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        packed = k * _blocks(n) * 17 if case["grad"] else n * _blocks(k) * 17
        return {"bytes": packed + m * k * 2 + m * n * _ES[case["out"]], "flops": 2 * m * n * k}
    m, d, f, e, t = case["m"], case["d"], case["f"], case["experts"], case["topk"]
    met = e * (1 - (1 - min(t, e) / e) ** m)  # experts that some token meets, for even routing
    per = 6 * d * f if case["w"] == "bf16" else (2 * f * _blocks(d) + d * _blocks(f)) * 17
    return {"bytes": met * per + m * (4 * d + 4 * e + 8 * t), "flops": 6 * m * t * d * f}


# ------------------------------------------------------------------------------------------------------------- exact
_GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _unit64(e):
    """2^e for whole e in [-127, 128), from a table."""
    return torch.from_numpy(np.ldexp(1.0, np.arange(-127, 128))).cuda()[e.long() + 127]


def _decode64(codes, scales, k):
    """Values of packed rows by table, in 64 bits."""
    table = torch.from_numpy(np.concatenate([_GRID, -_GRID])).cuda()
    pairs = torch.stack([table[(codes % 16).long()], table[torch.div(codes, 16, rounding_mode="floor").long()]], -1)
    return (pairs.reshape(codes.shape[0], -1) * _unit64(scales.long() - 127).repeat_interleave(32, 1))[:, :k]


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "quant":
        out = []
        for rows in (s["x"].t() if case["columns"] else s["x"]).split(2048):
            x = torch.nn.functional.pad(rows.double(), (0, -case["k"] % 32)).unflatten(1, (-1, 32))
            top = x.abs().max(-1, keepdim=True).values
            # the power of two that is no larger than the largest magnitude, looked up: a log2() need not be exact at powers
            powers = torch.from_numpy(np.ldexp(1.0, np.arange(-160, 128))).cuda()
            unit = _unit64(torch.clamp(torch.searchsorted(powers, top.contiguous(), right=True) - 161 - 2, min=-127))
            a, n = x.abs() / unit, 0
            # midpoints of neighbours; one that ties goes to the neighbour of even index
            for i in range(7):
                mid = (_GRID[i] + _GRID[i + 1]) / 2
                n = n + ((a >= mid) if i % 2 else (a > mid)).long()
            out.append((torch.from_numpy(_GRID).cuda()[n] * torch.sign(x) * unit).flatten(1)[:, : case["k"]])
        return torch.cat(out)
    if op == "read":
        return _decode64(s["codes"], s["scales"], case["k"])
    if op == "gemm":
        w = _decode64(s["codes"], s["scales"], case["n"] if case["grad"] else case["k"])
        return torch.matmul(s["x"].double(), w if case["grad"] else w.T)
    m, d, f, t = case["m"], case["d"], case["f"], case["topk"]
    logits = s["logits"].double().cpu().numpy()
    ids = np.stack([np.lexsort((np.arange(logits.shape[1]), -row))[:t] for row in logits])
    gates = np.exp(np.take_along_axis(logits, ids, 1) - logits.max(1, keepdims=True))
    gates /= gates.sum(1, keepdims=True)
    y = torch.zeros(m, d, dtype=torch.float64, device="cuda")
    for e in sorted(set(ids.reshape(-1).tolist())):
        tok, slot = np.nonzero(ids == e)
        w1 = s["w1"][e].double() if case["w"] == "bf16" else _decode64(s["w1"][e], s["s1"][e], d)
        w2 = s["w2"][e].double() if case["w"] == "bf16" else _decode64(s["w2"][e], s["s2"][e], f)
        rows = torch.from_numpy(tok).cuda()
        gate, up = (s["x"][rows].double() @ w1.T).split(f, 1)
        h = gate * torch.sigmoid(gate) * up
        y.index_add_(0, rows, (h @ w2.T) * torch.from_numpy(gates[tok, slot]).cuda()[:, None])
    return y, torch.from_numpy(ids.astype(np.int64)), torch.from_numpy(gates).cuda()
