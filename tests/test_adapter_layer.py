"""The operators of a decoder layer for requests with their own adapters over a 4-bit paged cache,
run together: projection with adapters, q/k norm and rotary positions with several axes into the
cache, attention (chunked prefill, then decode steps) and the output projection.

Two comparisons. The chain of kernels equals the same kernels called one at a time on inputs
copied in between (streams, dependent launches, graphs and shared workspaces change nothing), bit
for bit. And each step's result lies within that step's own tolerance of a 64-bit form of it, fed
with what the kernels before it left: the projections as in their own test; the attention 2^-8 of
the output for its rounding, and of sum(p u) for each of P's rounding and V's, u being |v| or, as
decode multiplies (code - 8) by P times the scale, 8 scales where that is more; 2^-11 of sum(p u)
holds the 32-bit sums, the exponentials and the roundings of q and K to fp16."""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

BF16, I32 = torch.bfloat16, torch.int32
H, HKV, D, K, RANK, ADAPTERS, BS = 8, 2, 128, 1024, 16, 3, 32
WIDTH = (H + 2 * HKV) * D


@pytest.fixture(scope="module")
def kx():
    from voiceagent_b200 import kernels

    return kernels


class Layer:
    """Weights, adapters and the cache of one layer, and a batch of requests over it."""

    def __init__(self, kx, lengths, seed=0, device="cuda"):
        self.kx, self.device = kx, device
        gen = torch.Generator().manual_seed(seed)
        bf = lambda *s, scale: (torch.randn(*s, generator=gen) * scale).bfloat16().to(device)  # noqa: E731
        self.w_qkv, self.w_o = bf(WIDTH, K, scale=K ** -0.5), bf(K, H * D, scale=(H * D) ** -0.5)
        self.a_qkv, self.b_qkv = bf(ADAPTERS, RANK, K, scale=K ** -0.5), bf(ADAPTERS, WIDTH, RANK, scale=RANK ** -0.5)
        self.a_o, self.b_o = bf(ADAPTERS, RANK, H * D, scale=(H * D) ** -0.5), bf(ADAPTERS, K, RANK, scale=RANK ** -0.5)
        self.scales = (0.5 + torch.rand(ADAPTERS, generator=gen)).to(device)
        self.qw, self.kw = bf(D, scale=1.0), bf(D, scale=1.0)
        inv = 10000.0 ** (-torch.arange(0, D, 2).double() / D)
        angle = torch.arange(4096).double()[:, None] * inv
        self.table = torch.cat([angle.cos(), angle.sin()], 1).float().to(device)
        self.axis = kx.mrope_freq_axis([24, 20, 20], interleaved=True, device=device)
        self.lengths = list(lengths)
        pages = [(n + BS - 1) // BS + 1 for n in lengths]
        order = torch.randperm(sum(pages), generator=gen)
        self.tables = torch.full((len(lengths), max(pages)), -1, dtype=I32)
        at = 0
        for b, n in enumerate(pages):
            self.tables[b, :n] = order[at:at + n].int()
            at += n
        self.slots_of = [[int(self.tables[b, i // BS]) * BS + i % BS for i in range(pages[b] * BS)]
                         for b in range(len(lengths))]
        self.tables = self.tables.to(device)
        self.cache = kx.kv4_cache(sum(pages), BS, HKV, D, device)
        self.err = torch.zeros(1, dtype=I32, device=device)
        self.gen = gen

    def tokens(self, counts, starts):
        """hidden rows, adapters, positions, slots and offsets of `counts` tokens from `starts` on."""
        total = sum(counts)
        x = torch.randn(total, K, generator=self.gen).bfloat16().to(self.device)
        on = lambda v: torch.tensor(v, dtype=I32, device=self.device)  # noqa: E731
        ids = on([b % (ADAPTERS + 1) - 1 for b, n in enumerate(counts) for _ in range(n)])
        where = [(b, s + i) for b, (n, s) in enumerate(zip(counts, starts)) for i in range(n)]
        pos = torch.tensor([[f(b, p) for b, p in where] for f in (lambda b, p: p, lambda b, p: p // 2 + b, lambda b, p: p // 3)],
                           dtype=torch.int64, device=self.device)
        slots = on([self.slots_of[b][p] for b, p in where])
        cu = lambda v: on(np.concatenate([[0], np.cumsum(v)]).tolist())  # noqa: E731
        return x, ids, pos, slots, cu(counts), cu([n + s for n, s in zip(counts, starts)])

    def run(self, batch, *, decode, between=lambda *t: t):
        """The layer on a batch; `between` sees (and may copy) what one call hands the next."""
        kx, (x, ids, pos, slots, cu_q, cu_k) = self.kx, batch
        qkv = kx.lora_linear(x, self.w_qkv, self.a_qkv, self.b_qkv, self.scales, ids, error_flag=self.err)
        qkv, = between(qkv)
        q = torch.empty(x.shape[0], H, D, dtype=BF16, device=self.device)
        codes, vcodes, params = self.cache
        kx.qk_norm_mrope_store(qkv, pos, self.axis, num_heads=H, num_kv_heads=HKV, head_dim=D, q_weight=self.qw,
                               k_weight=self.kw, eps=1e-6, cos_sin_cache=self.table, q_out=q, k_codes=codes,
                               v_codes=vcodes, kv_params=params, slot_mapping=slots, error_flag=self.err)
        q, = between(q)
        out = torch.empty_like(q)
        most = int(self.tables.shape[1]) * BS
        if decode:
            kx.paged_decode4(q, *self.cache, cu_k, self.tables, max_seqlen_k=most, scale=D ** -0.5, out=out,
                             error_flag=self.err)
        else:
            kx.paged_prefill4(q, *self.cache, cu_q, cu_k, self.tables, max_seqlen_q=most, max_seqlen_k=most,
                              scale=D ** -0.5, out=out, error_flag=self.err)
        out, = between(out)
        y = kx.lora_linear(out.view(-1, H * D), self.w_o, self.a_o, self.b_o, self.scales, ids, error_flag=self.err)
        return qkv, q, out, y

    def schedule(self):
        """Chunked prefill of all but the last three tokens of each request, then three decode steps."""
        first = [max(0, (n - 3) * 2 // 3) for n in self.lengths]
        rest = [n - 3 - f for n, f in zip(self.lengths, first)]
        yield self.tokens(first, [0] * len(first)), False
        yield self.tokens(rest, first), False
        for i in range(3):
            yield self.tokens([1] * len(first), [n - 3 + i for n in self.lengths]), True


def apart(*tensors):
    torch.cuda.synchronize()
    out = tuple(t.clone() for t in tensors)
    torch.cuda.synchronize()
    return out


SHORT, LONG = [3, 40, 129, 500, 31, 64], [4, 1500, 700, 2600]


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [SHORT, LONG])
@pytest.mark.parametrize("pdl", [False, True])
def test_the_chain_equals_its_calls_one_at_a_time(kx, lengths, pdl):
    one, two = Layer(kx, lengths, 3), Layer(kx, lengths, 3)
    was = kx.pdl_enabled()
    kx.set_pdl(pdl)
    try:
        for (batch, decode), (same, _) in zip(one.schedule(), two.schedule()):
            kx.set_pdl(pdl)
            got = one.run(batch, decode=decode)
            torch.cuda.synchronize()
            kx.set_pdl(False)
            want = two.run(same, decode=decode, between=apart)
            for g, w in zip(got, want):
                assert torch.equal(g, w)
    finally:
        kx.set_pdl(was)
    for a, b in zip(one.cache, two.cache):
        assert torch.equal(a, b)
    assert one.err.item() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [SHORT, LONG])
def test_each_step_against_64_bits(kx, lengths):
    layer = Layer(kx, lengths, 5)
    d = lambda t: t.double().cpu().numpy()  # noqa: E731

    def projection(x, w, a, b, ids):
        x, w, a, b, s = d(x), d(w), d(a), d(b), d(layer.scales)
        base, size, extra = x @ w.T, np.abs(x) @ np.abs(w).T, np.zeros((len(x), len(w)))
        for t, i in enumerate(ids.tolist()):
            if i >= 0:
                down = s[i] * (x[t] @ a[i].T)
                base[t] += down @ b[i].T
                extra[t] = np.abs(down) @ np.abs(b[i]).T
                size[t] += s[i] * (np.abs(x[t]) @ np.abs(a[i]).T) @ np.abs(b[i]).T
        return base, 2.0 ** -8 * (np.abs(base) + extra) + 2.0 ** -15 * size

    def within(got, out, tol):
        over = np.abs(d(got).reshape(out.shape) - out) - tol
        assert (over <= 0).all(), over.max()

    for batch, decode in layer.schedule():
        x, ids, pos, slots, cu_q, cu_k = batch
        qkv, q, out, y = layer.run(batch, decode=decode)
        within(qkv, *projection(x, layer.w_qkv, layer.a_qkv, layer.b_qkv, ids))
        within(y, *projection(out.view(-1, H * D), layer.w_o, layer.a_o, layer.b_o, ids))
        q = d(q)
        for b in range(len(lengths)):
            lo, hi = int(cu_q[b]), int(cu_q[b + 1])
            n = int(cu_k[b + 1] - cu_k[b])
            if lo == hi:
                continue
            at = torch.tensor(layer.slots_of[b][:n], dtype=I32, device="cuda")
            codes = [d(c.view(-1, HKV, D // 2)[at.long()]).astype(np.int64) for c in layer.cache[:2]]
            par = d(layer.cache[2].view(-1, HKV, 4)[at.long()])
            kv = [par[:, :, 2 * i + 1, None] + par[:, :, 2 * i, None] *
                  np.stack([c & 15, c >> 4], -1).reshape(n, HKV, D) for i, c in enumerate(codes)]
            for h in range(H):
                k, v = kv[0][:, h // (H // HKV)], kv[1][:, h // (H // HKV)]
                s = q[lo:hi, h] @ k.T * D ** -0.5
                s[np.arange(n)[None] > (n - (hi - lo) + np.arange(hi - lo))[:, None]] = -np.inf
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                u = np.maximum(np.abs(v), 8 * par[:, h // (H // HKV), 2, None])
                within(out[lo:hi, h], p @ v, 2.0 ** -8 * np.abs(p @ v) + (2 * 2.0 ** -8 + 2.0 ** -11) * (p @ u))
    assert layer.err.item() == 0


@pytest.mark.gpu
def test_a_captured_step_replayed_on_new_contents(kx):
    one, two = Layer(kx, LONG, 7), Layer(kx, LONG, 7)
    steps = list(zip(one.schedule(), two.schedule()))
    for (batch, decode), (same, _) in steps[:2]:
        one.run(batch, decode=decode)
        two.run(same, decode=decode)
    held = [t.clone() for t in steps[2][0][0]]
    one.run(held, decode=True)  # warm-up; the first replay does the same step again
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = one.run(held, decode=True)
    for (batch, _), (same, _) in steps[2:]:
        for h, t in zip(held, batch):
            h.copy_(t)
        graph.replay()
        for g, w in zip(got, two.run(same, decode=True)):
            assert torch.equal(g, w)
    for a, b in zip(one.cache, two.cache):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_layers_on_two_streams_and_threads_at_once(kx):
    seeds = (11, 12)
    want = []
    for seed in seeds:
        layer = Layer(kx, LONG, seed)
        want.append([t for batch, decode in layer.schedule() for t in layer.run(batch, decode=decode)])
    layers = [Layer(kx, LONG, seed) for seed in seeds]
    steps = [list(layer.schedule()) for layer in layers]
    torch.cuda.synchronize()
    got, failed = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for batch, decode in steps[i]:
                    got[i] += layers[i].run(batch, decode=decode)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for w, g in zip(want, got):
        assert len(w) == len(g) and all(torch.equal(a, b) for a, b in zip(w, g))


@pytest.mark.gpu
def test_an_empty_batch(kx):
    layer = Layer(kx, [5], 1)
    before = [t.clone() for t in layer.cache]
    x, ids, pos, slots, cu_q, cu_k = layer.tokens([0], [0])
    for decode in (False, True):
        one = torch.zeros(1, dtype=I32, device="cuda") if decode else cu_q
        for t in layer.run((x, ids, pos, slots, one, one), decode=decode):
            assert t.shape[0] == 0
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, layer.cache)) and layer.err.item() == 0
