"""The experts' layer through the C ABI against 64-bit arithmetic.

Tolerances, carried forward step by step (u = 2^-24, gamma(k) = 2 ((1 + u)^(k + 2) - 1), the reference suite's bound of a
k-deep fp32 sum): the first products are off by gamma(d) |W1||x| (and 2^-38 of a block's largest |x| per product in the
4-bit form); silu has a slope below 1.1, so h is off by 1.1 e_gate |up| + |silu| e_up + e_gate e_up + 2^-20 |h|; h enters the
second product with 11 significant bits of its own or, below 2^-17 of its block's largest, 2^-39 of that (4-bit weights), or
with 16 bits (two bf16 values); the second sums add gamma(f + topk); gates are off by 2^-20 of themselves; the result is
rounded to bf16, 2^-8 of the value."""
import os

import numpy as np
import pytest

import helpers as H
import mxf4_plain as MX
import skl_b200 as S

pytestmark = pytest.mark.gpu


def gamma(k):
    return 2 * ((1 + 2.0 ** -24) ** (k + 2) - 1)


def bf(x):
    return H.f32_to_bf16_bits(np.asarray(x, np.float32))


def f64(b):
    return H.bf16_bits_to_f32(b).astype(np.float64)


def choose(logits, topk, renormalise):
    """ids and gates of the definition: NaN first, then by value, ties to the lowest index; masked slots get gate 0."""
    l = logits.astype(np.float64)
    ids = np.stack([np.lexsort((np.arange(l.shape[1]), -np.where(np.isnan(r), np.inf, r), ~np.isnan(r)))[:topk] for r in l])
    val = np.take_along_axis(l, ids, 1)
    with np.errstate(invalid="ignore", over="ignore"):
        e = np.where(val == -np.inf, 0.0, np.exp(val - val[:, :1]))
        total = e.sum(1, keepdims=True) if renormalise else np.where(l == -np.inf, 0.0, np.exp(l - val[:, :1])).sum(1, keepdims=True)
        gates = np.where(val == -np.inf, 0.0, e / np.where(total == 0, 1.0, total))
    return ids, gates, val != -np.inf


def layer(x, w1, w2, ids, gates, routed, mx):
    """y and its tolerance before the last rounding; w1 [E][2f][d], w2 [E][d][f] in 64 bits."""
    m, d = x.shape
    f = w1.shape[1] // 2
    y, tol = np.zeros((m, d)), np.zeros((m, d))
    for i in range(m):
        for j, e in enumerate(ids[i]):
            if not routed[i, j]:
                continue
            full, absf = w1[e] @ x[i], np.abs(w1[e]) @ np.abs(x[i])
            err = gamma(d) * absf
            if mx:
                blocks = np.abs(np.pad(x[i], (0, -d % 32)).reshape(-1, 32)).max(1).repeat(32)[:d]
                err = err + 2.0 ** -38 * (np.abs(w1[e]) @ blocks)
            g, u, eg, eu = full[:f], full[f:], err[:f], err[f:]
            silu = g / (1 + np.exp(-g))
            h = silu * u
            eh = 1.1 * eg * np.abs(u) + np.abs(silu) * eu + 1.1 * eg * eu + 2.0 ** -20 * np.abs(h)
            if mx:
                top = np.abs(np.pad(h, (0, -f % 32)).reshape(-1, 32)).max(1).repeat(32)[:f]
                eh = eh + np.maximum(2.0 ** -11 * np.abs(h), 2.0 ** -39 * top)
            else:
                eh = eh + 2.0 ** -16 * np.abs(h)
            part, absp = w2[e] @ h, np.abs(w2[e]) @ (np.abs(h) + eh)
            ep = np.abs(w2[e]) @ eh + gamma(f + ids.shape[1]) * absp
            y[i] += gates[i, j] * part
            tol[i] += gates[i, j] * (ep + (2.0 ** -20 + gamma(ids.shape[1])) * (np.abs(part) + ep))
    return y, tol


class Case:
    def __init__(self, m, d, f, experts, topk, mx, renormalise=1, seed=0, pad=0, logits=None, off=0):
        import torch

        g = H.rng(seed * 7919 + m * 131 + d * 7 + f + experts * 3 + topk)
        self.shape, self.mx, self.renormalise = (m, d, f, experts, topk), mx, renormalise
        self.logits = g.standard_normal((m, experts)).astype(np.float32) * 2 if logits is None else np.asarray(logits, np.float32)
        self.rsl, self.rsx, self.rsy = experts + pad, d + pad, d + pad
        x = bf(g.standard_normal((m, d)))
        self.x = f64(x)
        L, X = np.full((m, self.rsl), 9e9, np.float32), bf(np.full((m, self.rsx), 5.0))
        L[:, :experts], X[:, :d] = self.logits, x
        put = lambda v, o=0: self._put(torch, v, o)  # noqa: E731
        self.tl, self.tx = put(L), put(X, 2 * off)
        if mx:
            # weights of about 1 / sqrt(columns): scale bytes around 127 - log2(3 sqrt(columns))
            c1, s1 = MX.random_packed(g, (experts, 2 * f, d), 121 - int(np.log2(d) / 2), 125 - int(np.log2(d) / 2))
            c2, s2 = MX.random_packed(g, (experts, d, f), 121 - int(np.log2(f) / 2), 125 - int(np.log2(f) / 2))
            self.w = [put(v, off) for v in (c1, s1, c2, s2)]
            self.w1, self.w2 = MX.values(c1, s1, d), MX.values(c2, s2, f)
        else:
            b1, b2 = bf(g.standard_normal((experts, 2 * f, d)) / np.sqrt(d)), bf(g.standard_normal((experts, d, f)) / np.sqrt(f))
            self.w = [put(v, 2 * off) for v in (b1, b2)]
            self.w1, self.w2 = f64(b1), f64(b2)
        self.out()

    @staticmethod
    def _put(torch, v, off):
        raw = np.concatenate([np.zeros(off, np.uint8), np.ascontiguousarray(v).view(np.uint8).reshape(-1)])
        return torch.from_numpy(raw).cuda()[off:]

    def out(self):
        import torch

        m, d, f, experts, topk = self.shape
        self.y = torch.full((m, self.rsy), 7.0, dtype=torch.bfloat16, device="cuda")
        self.ids = torch.full((m, topk), -7, dtype=torch.int32, device="cuda")
        self.gates = torch.full((m, topk), -7.0, device="cuda")
        size = S.lib().skl_b200_moe_workspace_size(m, f, experts, topk)
        self.work = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")
        self.size = size

    def call(self):
        lib = S.lib()
        m, d, f, experts, topk = self.shape
        fn = lib.skl_moe_swiglu_bf16_mxf4e2m1_bf16_sm100a if self.mx else lib.skl_moe_swiglu_bf16_bf16_bf16_sm100a
        fn(m, d, f, experts, topk, self.renormalise, self.tl.data_ptr(), self.rsl, self.tx.data_ptr(), self.rsx,
           *[w.data_ptr() for w in self.w], self.y.data_ptr(), self.rsy, self.ids.data_ptr(), self.gates.data_ptr(),
           self.work.data_ptr(), self.size)
        assert lib.skl_b200_last_status() == 0

    def check(self):
        import torch

        torch.cuda.synchronize()
        m, d, f, experts, topk = self.shape
        ids, gates, routed = choose(self.logits, topk, self.renormalise)
        assert np.array_equal(self.ids.cpu().numpy(), ids)
        got = self.gates.cpu().numpy().astype(np.float64)
        nan = np.isnan(gates)
        assert np.array_equal(np.isnan(got), nan)
        assert np.all(np.abs(got - gates)[~nan] <= 2.0 ** -20 * gates[~nan] + 2.0 ** -126)
        y = f64(self.y.view(torch.int16).cpu().numpy().view(np.uint16))
        assert np.all(y[:, d:] == 7.0), "the gap behind a row of y was written"
        assert torch.all(self.work[self.size:] == 255), "written behind the workspace"
        bad = nan.any(1)
        want, tol = layer(self.x, self.w1, self.w2, ids, np.where(nan, 0.0, gates), routed, self.mx)
        tol = tol + 2.0 ** -8 * (np.abs(want) + tol) + 2.0 ** -130
        assert np.all(np.isnan(y[bad, :d]))
        err = np.abs(y[:, :d] - want)[~bad]
        assert np.all(err <= tol[~bad]), (self.shape, float(np.max(err / tol[~bad])))


SHAPES = [(1, 64, 32, 4, 2), (1, 256, 256, 8, 8), (2, 512, 128, 16, 4), (3, 300, 100, 6, 3), (4, 1024, 512, 8, 1), (5, 40, 17, 3, 2),
          (8, 33, 65, 60, 6), (16, 384, 272, 32, 8), (17, 128, 96, 2, 2), (40, 160, 64, 5, 4), (64, 96, 32, 1, 1), (64, 64, 64, 128, 8)]


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_layer(skl, shape, mx):
    for renormalise in (0, 1):
        c = Case(*shape, mx, renormalise, seed=renormalise)
        c.call()
        c.check()


@pytest.mark.parametrize("mx", [False, True])
def test_larger_layer(skl, mx):
    c = Case(16, 2048, 1024, 16, 4, mx)
    c.call()
    c.check()
    c = Case(1, 4096, 1000, 8, 2, mx, seed=3)
    c.call()
    c.check()


@pytest.mark.parametrize("mx", [False, True])
def test_strides_and_alignment(skl, mx):
    for pad, off in ((8, 0), (3, 0), (0, 1), (5, 3)):
        c = Case(3, 256, 256, 4, 2, mx, pad=pad, off=off, seed=pad)
        c.call()
        c.check()


@pytest.mark.parametrize("mx", [False, True])
def test_workspace_at_any_word(skl, mx):
    """The workspace needs no more than its words' alignment, and no byte outside the asked-for size is touched."""
    c = Case(5, 96, 80, 6, 3, mx)
    for off in (4, 8, 12):
        c.out()
        whole = c.work
        c.work = whole[off:]
        c.call()
        c.check()
        import torch

        assert torch.all(whole[:off] == 255)


@pytest.mark.parametrize("mx", [False, True])
def test_largest_routing_and_rows(skl, mx):
    """64 tokens, 1024 experts, 32 of them to a token, rows of 32768 elements."""
    c = Case(64, 32768, 1, 1024, 32, mx)
    c.call()
    c.check()


@pytest.mark.parametrize("mx", [False, True])
def test_long_hidden_rows(skl, mx):
    c = Case(6, 3, 32768, 4, 2, mx)
    c.call()
    c.check()


@pytest.mark.parametrize("mx", [False, True])
def test_every_token_to_one_expert(skl, mx):
    """More tokens of one expert than a pass takes."""
    logits = np.zeros((37, 5), np.float32)
    logits[:, 3] = 5.0
    c = Case(37, 128, 96, 5, 1, mx, logits=logits)
    c.call()
    c.check()


def test_ties_masks_and_nan(skl):
    inf = np.inf
    rows = [[0, 0, 0, 0, 0, 0], [1, 3, 3, 3, 0, 1], [-0.0, 0.0, -0.0, -1, -1, 0.0], [-inf, 2, -inf, -inf, -inf, -inf], [-inf] * 6,
            [5, -inf, 5, -inf, 4, -inf], [1e38, -1e38, 0, 0, 0, 0], [-200, -201, -300, -299, -inf, -200.5], [0, np.nan, 1, 2, 3, 4]]
    for mx in (False, True):
        for renormalise in (0, 1):
            c = Case(len(rows), 64, 48, 6, 3, mx, renormalise, logits=rows)
            c.call()
            c.check()
            assert np.all(f64(c.y.view(__import__("torch").int16).cpu().numpy().view(np.uint16))[4, :64] == 0.0)


@pytest.mark.parametrize("mx", [False, True])
def test_a_masked_expert_may_hold_anything(skl, mx):
    """NaN and infinities in the weights of an expert that no unmasked logit chooses do not reach the output."""
    import torch

    logits = np.array([[1.0, -np.inf, -np.inf]] * 2)
    c = Case(2, 64, 32, 3, 2, mx, logits=logits)
    if mx:
        c.w[1].view(3, -1)[1:] = 255
        c.w[3].view(3, -1)[1:] = 255
    else:
        for w in c.w:
            w.view(torch.int16).view(3, -1)[1:] = 0x7FC0
    c.w1[1:], c.w2[1:] = 0.0, 0.0
    c.call()
    c.check()


@pytest.mark.parametrize("m", [1, 2, 5, 9])
def test_large_values_and_small_scales(skl, m):
    """4-bit weights: tokens near the largest bf16 numbers under small scales of w1, then h that large under small scales of w2."""
    import torch

    d, f, experts = 192, 96, 2
    put = lambda v: torch.from_numpy(np.ascontiguousarray(v).view(np.uint8).reshape(-1)).cuda()  # noqa: E731
    c = Case(m, d, f, experts, 2, True, seed=m)
    c.x = c.x * 2.0 ** 122
    c.tx = put(bf(c.x))
    c.w[1] -= 116
    c.w1 = c.w1 * 2.0 ** -116
    assert np.all(np.isfinite(f64(bf(c.x))))
    c.call()
    c.check()
    c = Case(m, d, f, experts, 2, True, seed=m + 20)
    c.w[1].view(experts, 2 * f, -1)[:, f:] += 120
    c.w1[:, f:] *= 2.0 ** 120
    c.w[3] -= 116
    c.w2 = c.w2 * 2.0 ** -116
    c.call()
    c.check()


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("d,f", [(64, 64), (64, 192), (128, 320), (64, 128), (72, 40)])
def test_nothing_behind_a_row_of_the_second_weights_is_used(skl, d, f, mx):
    """NaN in masked experts on both sides of the one that is used, and in memory behind the last row of w2: rows that are whole
    128-byte steps but no whole items of the kernel (f = 64, 192, 320 in 16 bits) end where they end."""
    import torch

    for used in range(3):  # the used expert's last row is followed by another expert's first, or by the end of w2
        logits = np.full((3, 3), -np.inf)
        logits[:, used] = 1.0
        c = Case(3, d, f, 3, 2, mx, logits=logits, seed=used)
        for i, w in enumerate(c.w):
            room = torch.empty(w.numel() + 4096, dtype=torch.uint8, device="cuda")
            if mx:
                room.fill_(255)
            else:
                room.view(torch.int16).fill_(0x7FFF)
            per = w.numel() // 3
            room[used * per:(used + 1) * per] = w[used * per:(used + 1) * per]
            c.w[i] = room
        for e in range(3):
            if e != used:
                c.w1[e], c.w2[e] = 0.0, 0.0
        c.call()
        c.check()


def test_a_row_of_the_second_weights_may_hold_nan(skl):
    """... and its NaN reaches that row's output only, not the row's before it."""
    import torch

    m, d, f = 2, 64, 192
    c = Case(m, d, f, 2, 1, False, logits=np.array([[1.0, 0.0]] * m))
    c.call()
    torch.cuda.synchronize()
    plain = c.y.clone()
    c.w[1].view(torch.int16).view(2, d, f)[:, 1::2] = 0x7FFF
    c.out()
    c.call()
    torch.cuda.synchronize()
    assert torch.equal(c.y[:, 0:d:2], plain[:, 0:d:2]) and torch.all(torch.isnan(c.y[:, 1:d:2]))


@pytest.mark.parametrize("mx", [False, True])
def test_same_bits_every_time(skl, mx):
    import torch

    c = Case(9, 512, 320, 12, 4, mx)
    first = None
    for _ in range(4):
        c.out()
        c.call()
        torch.cuda.synchronize()
        first = c.y if first is None else first
        assert torch.equal(first, c.y)
    c.check()


@pytest.mark.parametrize("mx", [False, True])
def test_captured_side_by_side_and_on_other_streams(skl, mx):
    """Two captured layers with a workspace each, replayed together; new inputs between replays change the routing."""
    import torch

    cases = [Case(4, 256, 192, 8, 3, mx, seed=s) for s in (1, 2)]
    cases[0].call()
    streams, graphs = [torch.cuda.Stream() for _ in cases], []
    skl.skl_b200_set_async(1)
    try:
        for c, st in zip(cases, streams):
            skl.skl_b200_set_stream(st.cuda_stream)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                c.call()
            graphs.append(graph)
        for turn in range(3):
            for c in cases:
                c.logits = H.rng(50 + turn).standard_normal((4, 8)).astype(np.float32)
                c.tl.copy_(torch.from_numpy(c.logits.view(np.uint8).reshape(-1)))
            torch.cuda.synchronize()
            for _ in range(3):
                for graph, st in zip(graphs, streams):
                    with torch.cuda.stream(st):
                        graph.replay()
            for c in cases:
                c.check()
    finally:
        skl.skl_b200_set_stream(None)
        skl.skl_b200_set_async(0)


@pytest.mark.parametrize("mx", [False, True])
def test_values_that_are_not_finite_stay_with_their_tokens(skl, mx):
    """An infinity and a NaN in two tokens' activations, a NaN in a weight of an expert that some tokens have: every other token's
    result is what it is without them."""
    import torch

    m, d, f, experts, topk = 9, 192, 160, 6, 2
    logits = H.rng(77).standard_normal((m, experts)).astype(np.float32)
    logits[:, 5] = -9.0
    logits[3, 5] = 9.0  # only this token has expert 5
    c = Case(m, d, f, experts, topk, mx, logits=logits, seed=77)
    c.call()
    torch.cuda.synchronize()
    plain = c.y.clone()
    x = bf(c.x)
    x[1, 40], x[6, 191] = 0x7F80, 0x7FC0
    c.tx = torch.from_numpy(x.view(np.uint8).reshape(-1)).cuda()
    if mx:
        c.w[1].view(experts, 2 * f, -1)[5, f + 7, 3] = 255  # an element of h
        c.w[3].view(experts, d, -1)[5, 11, 0] = 255  # and a row of the result
    else:
        c.w[0].view(torch.int16).view(experts, 2 * f, d)[5, f + 7, 100] = 0x7FC0
        c.w[1].view(torch.int16).view(experts, d, f)[5, 11, 3] = 0x7FC0
    c.out()
    c.call()
    torch.cuda.synchronize()
    fine = [i for i in range(m) if i not in (1, 3, 6)]
    assert torch.equal(c.y[fine], plain[fine])
    assert not torch.any(torch.isfinite(c.y[1])) and torch.all(torch.isnan(c.y[[3, 6]]))


@pytest.mark.parametrize("byte", [0, 1, 245, 252])
def test_scales_at_the_ends_of_their_range(skl, byte):
    """4-bit weights whose gate rows and down rows have the smallest or the largest scales; the activations make up for them."""
    import torch

    m, d, f, experts = 3, 96, 64, 2
    c = Case(m, d, f, experts, 2, True, seed=byte)
    c.x = c.x * 2.0 ** (100 if byte < 118 else -100)
    c.tx = torch.from_numpy(bf(c.x).view(np.uint8).reshape(-1)).cuda()
    c.w[1].fill_(byte)
    c.w[1].view(experts, 2 * f, -1)[:, f:] = 120
    c.w[3].fill_(byte)
    rows = lambda v, n: v.cpu().numpy().reshape(experts, n, -1)  # noqa: E731
    c.w1, c.w2 = MX.values(rows(c.w[0], 2 * f), rows(c.w[1], 2 * f), d), MX.values(rows(c.w[2], d), rows(c.w[3], d), f)
    with np.errstate(over="ignore"):
        c.call()
        c.check()


@pytest.mark.parametrize("mx", [False, True])
def test_weights_past_32_bits(skl, mx):
    """1024 experts whose last one lies more than 4 GiB behind the first in both matrices; nothing else of them is used."""
    import torch

    d, f, experts = (4096, 4096, 1024) if mx else (2048, 2048, 1024)
    logits = np.full((2, experts), -np.inf, np.float32)
    logits[:, -1] = 0.5
    small = Case(2, d, f, 1, 1, mx, logits=logits[:, -1:], seed=5)
    c = object.__new__(Case)
    c.__dict__.update(small.__dict__)
    c.shape, c.logits, c.rsl = (2, d, f, experts, 1), logits, experts
    c.tl = torch.from_numpy(logits.view(np.uint8).reshape(-1)).cuda()
    c.w = []
    for w in small.w:
        big = torch.empty(w.numel() * experts, dtype=torch.uint8, device="cuda")
        big[-w.numel():] = w
        c.w.append(big)
    assert min(w.numel() - w.numel() // experts for w in c.w[::2 if mx else 1]) > 1 << 32
    c.out()
    c.call()
    torch.cuda.synchronize()
    want, tol = layer(small.x, small.w1, small.w2, np.zeros((2, 1), int), np.ones((2, 1)), np.ones((2, 1), bool), mx)
    tol = tol + 2.0 ** -8 * (np.abs(want) + tol) + 2.0 ** -130
    assert torch.all(c.ids == experts - 1) and torch.all(c.gates == 1.0)
    got = f64(c.y.view(torch.int16).cpu().numpy().view(np.uint16))
    assert np.all(np.abs(got - want) <= tol)


def test_two_threads_at_once(skl):
    """Both kinds of weights from two threads that start together in a new process, each on a stream and a workspace of its own."""
    import subprocess
    import sys

    code = """
import threading, torch
import test_moe_gpu as T
torch.zeros(1, device="cuda")
jobs = [[T.Case(3 + t, 128 * (t + 1), 192, 6, 2, mx, seed=t) for mx in (False, True)] for t in range(2)]
torch.cuda.synchronize()
gate, failed = threading.Barrier(2), []
def work(t):
    try:
        torch.cuda.set_device(0)
        lib, stream = T.S.lib(), torch.cuda.Stream()
        lib.skl_b200_set_stream(stream.cuda_stream)
        lib.skl_b200_set_async(1)
        gate.wait()
        for _ in range(20):
            for c in jobs[t]:
                c.call()
        lib.skl_b200_synchronize()
        assert lib.skl_b200_last_status() == 0
    except BaseException as e:
        failed.append(repr(e))
threads = [threading.Thread(target=work, args=(t,)) for t in range(2)]
[t.start() for t in threads]
[t.join() for t in threads]
assert not failed, failed
for cases in jobs:
    for c in cases:
        c.check()
print("fine")
"""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(here), os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and r.stdout.strip().endswith("fine"), r.stdout + r.stderr


def test_from_the_router_on(skl):
    """The run of a layer: logits from the library's GEMM, weights quantised by the library, the experts on the result."""
    import torch

    m, d, f, experts, topk = 6, 128, 64, 8, 2
    g = H.rng(12)
    c = Case(m, d, f, experts, topk, True, seed=4)
    router = bf(g.standard_normal((d, experts)) / np.sqrt(d))
    tr = torch.from_numpy(router.view(np.int16)).cuda()
    skl.skl_gemm_bf16_bf16_f32_sm100a(m, experts, d, 1.0, c.tx.data_ptr(), d, tr.data_ptr(), experts, 0.0, c.tl.data_ptr(), experts)
    S.check()
    c.logits = c.tl.cpu().numpy().view(np.float32).reshape(m, experts).copy()
    assert np.allclose(c.logits, c.x @ f64(router), atol=1e-3)
    for i, (rows, cols) in enumerate(((2 * f, d), (d, f))):
        w = (g.standard_normal((experts * rows, cols)) / np.sqrt(cols)).astype(np.float32)
        tw = torch.from_numpy(w).cuda()
        skl.skl_cvt_f32rc_mxf4e2m1_sm100a(c.w[2 * i].data_ptr(), cols // 2, c.w[2 * i + 1].data_ptr(), cols // 32, tw.data_ptr(), cols,
                                          1, experts * rows, cols)
        S.check()
        setattr(c, f"w{i + 1}", MX.values(*MX.quantise(w), cols).reshape(experts, rows, cols))
    c.call()
    c.check()


def test_host_pointers_are_refused(skl):
    c = Case(2, 64, 32, 4, 2, False)
    host = np.zeros(2 * 64, np.uint16)
    skl.skl_moe_swiglu_bf16_bf16_bf16_sm100a(2, 64, 32, 4, 2, 1, c.tl.data_ptr(), 4, S.ptr(host), 64, c.w[0].data_ptr(),
                                             c.w[1].data_ptr(), c.y.data_ptr(), 64, c.ids.data_ptr(), c.gates.data_ptr(),
                                             c.work.data_ptr(), c.size)
    assert skl.skl_b200_last_status() == 1 and skl.skl_b200_last_launch_count() == 0
