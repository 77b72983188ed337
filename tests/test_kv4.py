"""The 4-bit paged KV cache: rows in and out, and attention over it, against plain 64-bit forms.

Tolerances of the attention outputs are element by element, from the roundings the kernels make:

* the output to bf16: 2^-8 of its value;
* a probability times its V scale to bf16 before the product with the centred code (code - 8):
  2^-8 of sum_t p_t vs_t |code_t - 8|;
* the score's 32-bit accumulation, whose terms are up to (1024 + 15) |q_i| for at most
  D / 16 + 1 additions of 2^-23 each: an absolute error e of the score (base e) changes each
  probability by the factor exp(+-e), so the output by at most 2 e sum_t p_t |v_t - out|
  <= 2 e (sum_t p_t |v_t| + |out|);
* prefill takes q, K, V and P as fp16 (2^-11 of the value each; below fp16's smallest normal
  number, 2^-27 of the largest of a q row or of 32 K rows, 2^-24 for V, which no test reaches
  unless it says so): a score (base e) moves by at most e = |scale| (2 * 2^-11 + 2^-20)
  sum_i |q_i k_i|, 2^-20 for the 32-bit sums, and the output by 2 * 2^-11 of sum_t p_t |v_t|;
* 2^-16 of sum_t p_t (|v_t| + |zero_t|) for the other 32-bit sums, exp2 and the division (up to a
  few hundred additions of 2^-24 each and exp2 within 2^-22).
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

BF16 = torch.bfloat16


# --------------------------------------------------------------------------- plain forms


def f32(x: torch.Tensor) -> np.ndarray:
    return x.detach().float().cpu().numpy()


def bf16_of(bits: np.ndarray) -> np.ndarray:
    return (bits.astype(np.uint32) << 16).view(np.float32)


def plain_quantise(x: np.ndarray):
    """codes [..., D], scale [...], zero [...] of bf16-valued float32 rows, scale by search."""
    lo, hi = x.min(-1), x.max(-1)
    wide = (hi - lo).astype(np.float32)
    guess = (wide / np.float32(15)).astype(np.float32).view(np.uint32) >> 16
    scale = np.full(wide.shape, np.inf, np.float32)
    for step in (2, 1, 0, -1, -2):  # from above: the last that still reaches is the smallest
        s = bf16_of(np.maximum(guess.astype(np.int64) + step, 0))
        scale = np.where(15 * s.astype(np.float64) >= wide, s, scale)
    scale = np.where(wide < 2.0 ** -100, 0, scale).astype(np.float32)
    d = (x - lo[..., None]).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.rint(d / scale[..., None])
    code = np.where(scale[..., None] > 0, np.clip(code, 0, 15), 0).astype(np.int64)
    return code, scale, lo


def unpack_codes(c: torch.Tensor) -> np.ndarray:
    c = c.cpu().numpy().astype(np.int64)
    return np.stack((c & 15, c >> 4), -1).reshape(*c.shape[:-1], -1)


def sequence_rows(cache, table, n):
    """(k values, v codes, v scale, v zero) of a sequence's first n tokens in 64 bits."""
    kc, vc, par = cache
    bs = kc.shape[1]
    pos = torch.arange(n)
    blk = table.cpu().long()[pos // bs]
    at = pos % bs
    kc, vc, par = kc.cpu()[blk, at], vc.cpu()[blk, at], par.cpu()[blk, at].double().numpy()
    k = unpack_codes(kc) * par[..., 0:1] + par[..., 1:2]
    return k, unpack_codes(vc).astype(np.float64), par[..., 2:3], par[..., 3:4], par[..., 0:1]


def plain_attention(q, cache, table, n, scale, prefill=False, bf16_v=False):
    """out [q_len, H, D] and its tolerance, causal with the mask aligned bottom-right."""
    q = q.double().cpu().numpy()
    m, heads, d = q.shape
    out, tol = np.zeros_like(q), np.zeros_like(q)
    if n == 0:
        return out, tol
    k, vcode, vs, vz, ks = sequence_rows(cache, table, n)
    v = vcode * vs + vz
    group = heads // k.shape[1]
    for i in range(m):
        seen = n - (m - 1 - i)
        if seen <= 0:
            continue
        for h in range(heads):
            g = h // group
            s = k[:seen, g] @ q[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            o = p @ v[:seen, g]
            mass = p @ np.abs(v[:seen, g])
            if prefill:  # a key's e weighs with its probability
                e = (2 * 2.0 ** -11 + 2.0 ** -20) * abs(scale) * (np.abs(k[:seen, g]) @ np.abs(q[i, h]))
                rounded = (2 * 2.0 ** -8 if bf16_v else 2 * 2.0 ** -11) * mass
                moved = (p * e) @ np.abs(v[:seen, g]) + (p @ e) * np.abs(o)  # exp(x) - 1 <= x exp(x)
                moved = moved * np.exp(e.max())
            else:
                e = abs(scale) * ks[:seen, g].max() * 1040 * np.abs(q[i, h]).sum() * (d / 16 + 1) * 2.0 ** -23
                rounded = 2.0 ** -8 * (p @ (vs[:seen, g] * np.abs(vcode[:seen, g] - 8)))
                moved = 2 * e * (mass + np.abs(o))
            out[i, h] = o
            tol[i, h] = (2.0 ** -8 * np.abs(o) + rounded + moved
                         + 2.0 ** -16 * (mass + p @ np.abs(vz[:seen, g] * np.ones(d))))
    return out, tol


def check_close(got, want, tol, what):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all(), f"{what}: not finite"
    over = np.abs(got - want) - tol * 1.0001
    assert (over <= 0).all(), f"{what}: {over.max():.3e} past the tolerance at {np.unravel_index(over.argmax(), over.shape)}"


# -------------------------------------------------------------------------------- inputs


def filled(seed, blocks, bs, hkv, d, layout="slots", spread=1.0):
    """A random cache; ``layout`` "heads" keeps a block's rows of one head together."""
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(2, blocks, bs, hkv, d, generator=gen) * spread).bfloat16().float().numpy()
    out = []
    params = np.zeros((blocks, bs, hkv, 4), np.float32)
    for i in range(2):
        code, params[..., 2 * i], params[..., 2 * i + 1] = plain_quantise(x[i])
        out.append(torch.from_numpy((code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8)).cuda())
    out.append(torch.from_numpy(params).bfloat16().cuda())
    if layout == "heads":
        out = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in out]
    return out


def paged(seed, lens, bs, extra=1):
    rng = np.random.default_rng(seed)
    used = [(n + bs - 1) // bs for n in lens]
    blocks = sum(used) + extra
    order = rng.permutation(blocks)
    table = np.full((len(lens), max(used + [1])), -1, np.int32)
    c = 0
    for i, u in enumerate(used):
        table[i, :u] = order[c:c + u]
        c += u
    return torch.from_numpy(table).cuda(), blocks


def poison_unused(cache, table, lens):
    """NaN parameters and 0xff codes in every row no sequence holds."""
    kc, vc, par = cache
    bs = kc.shape[1]
    keep = torch.zeros(kc.shape[0], bs, dtype=torch.bool)
    for row, n in zip(table.cpu().long(), lens):
        pos = torch.arange(n)
        keep[row[pos // bs], pos % bs] = True
    drop = ~keep.cuda()
    kc[drop] = 255
    vc[drop] = 255
    par[drop] = float("nan")


def starts(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).cuda()


@pytest.fixture(scope="module")
def kx():
    from voiceagent_b200 import kernels

    return kernels


# ---------------------------------------------------------------------- refusals (CPU)


def _kv4_struct(**over):
    from voiceagent_b200._lib import Kv4

    d = dict(k_codes=256, v_codes=256, params=256, code_stride=(256 * 512, 512, 64),
             param_stride=(256 * 32, 32, 4), num_blocks=4, block_size=256, num_kv_heads=8, head_dim=128)
    d.update(over)
    return Kv4(d["k_codes"], d["v_codes"], d["params"], d["code_stride"], d["param_stride"],
               d["num_blocks"], d["block_size"], d["num_kv_heads"], d["head_dim"])


@pytest.mark.parametrize("over,says", [
    (dict(head_dim=96), "head_dim"), (dict(code_stride=(8, 512, 64)), "aligned"),
    (dict(param_stride=(256 * 32, 30, 4)), "aligned"), (dict(k_codes=258), "aligned"),
    (dict(params=260), "aligned"), (dict(block_size=0), "cache sizes"), (dict(params=None), "null"),
])
def test_c_entries_refuse_bad_caches(over, says):
    from voiceagent_b200._lib import lib

    p = ctypes.c_void_p(256)
    c = ctypes.byref(_kv4_struct(**over))
    for rc in (lib.b200asr_store_kvcache4(p, 1024, 128, p, 1024, 128, c, p, 3, None, None),
               lib.b200asr_load_kvcache4(c, p, 3, p, 1024, 128, p, 1024, 128, None, None),
               lib.b200asr_paged_decode4(p, 2048, 128, c, 16, p, p, 4, 4, 2, 100, 1.0, p, 2048, 128,
                                         None, 0, None, None)):
        assert rc == 1 and says in lib.b200asr_last_error().decode()


def test_c_entries_refuse_bad_calls():
    from voiceagent_b200._lib import lib

    p, c = ctypes.c_void_p(256), ctypes.byref(_kv4_struct())
    err = lambda: lib.b200asr_last_error().decode()  # noqa: E731
    assert lib.b200asr_store_kvcache4(p, 1020, 128, p, 1024, 128, c, p, 3, None, None) == 1 and "aligned" in err()
    assert lib.b200asr_store_kvcache4(p, 1024, 128, p, 1024, 128, None, p, 3, None, None) == 1 and "null" in err()
    assert lib.b200asr_store_kvcache4(None, 8, 8, None, 8, 8, c, None, 0, None, None) == 0
    dec = lambda **k: lib.b200asr_paged_decode4(  # noqa: E731
        p, k.get("qs", 2048), 128, c, k.get("heads", 16), p, p, 4, 4, k.get("batch", 2),
        k.get("longest", 100), 1.0, p, 2048, 128, None, 0, None, None)
    assert dec(heads=12) == 1 and "multiple" in err()
    assert dec(qs=2044) == 1 and "aligned" in err()
    assert dec(longest=-1) == 1 and "sizes" in err()
    assert dec(batch=0) == 0
    pre = lambda **k: lib.b200asr_paged_prefill4(  # noqa: E731
        p, 2048, 128, c, k.get("heads", 16), p, p, p, 4, 4, k.get("batch", 2), k.get("rows", 9), 1.0, p,
        k.get("os", 2048), 128, k.get("ws"), 1 << 20, None, None)
    assert pre(ws=ctypes.c_void_p(264)) == 1 and "workspace" in err()
    size = lib.b200asr_paged_prefill4_workspace_size
    assert size(200, 1, 1024, 16, 8, 128) == size(0, 1, 5000, 16, 8, 128) == size(10**6, 1, 5000, 16, 8, 128) == 0
    assert pre(heads=12) == 1 and "multiple" in err()
    assert pre(os=2044) == 1 and "aligned" in err()
    assert pre(rows=-1) == 1 and "sizes" in err()
    assert pre(batch=0) == 0 and pre(rows=0) == 0


def test_wrappers_refuse_cpu_tensors_and_wrong_types(kx):
    kc, vc, par = kx.kv4_cache(2, 16, 2, 64, device="cpu")
    x = torch.zeros(3, 2, 64, dtype=BF16)
    slots = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kx.store_kvcache4(x, x, kc, vc, par, slots)
    with pytest.raises(ValueError, match="uint8"):
        kx.store_kvcache4(x, x, kc.int(), vc, par, slots)
    with pytest.raises(ValueError, match="parameters"):
        kx.load_kvcache4(kc, vc, par[:, :, :1], slots)
    with pytest.raises(ValueError, match="alike"):
        kx.load_kvcache4(kc, vc[:, :8], par, slots)
    with pytest.raises(ValueError, match="64 or 128"):
        kx.kv4_cache(2, 16, 2, 96, device="cpu")
    table, starts = torch.zeros(3, 1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    wide = torch.empty(1, dtype=torch.uint8).expand(1 << 26)
    with pytest.raises(ValueError, match="contiguous workspace"):
        kx.paged_decode4(x, kc, vc, par, starts, table, max_seqlen_k=2000, scale=1.0, out=x, workspace=wide)
    with pytest.raises(ValueError, match="contiguous workspace"):
        kx.paged_prefill4(x, kc, vc, par, starts, starts, table, max_seqlen_q=1, max_seqlen_k=2000, scale=1.0, out=x,
                          workspace=wide)


# ---------------------------------------------------------------------- rows in and out


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,hkv,d,bs,layout", [
    (1, 8, 128, 256, "slots"), (37, 8, 128, 256, "slots"), (300, 2, 64, 16, "slots"),
    (65, 3, 64, 48, "heads"), (513, 1, 128, 16, "heads")])
def test_store_and_load(kx, tokens, hkv, d, bs, layout):
    gen = torch.Generator().manual_seed(tokens)
    wide = torch.randn(tokens, 2 * hkv + 1, d, generator=gen) * torch.exp(3 * torch.randn(tokens, 1, 1, generator=gen))
    wide = wide.bfloat16()
    wide[0, 0] = 1.5  # a flat row
    if tokens > 3:
        wide[1, 0] = torch.arange(d).bfloat16() * 0.25  # codes on exact ties
        wide[2, hkv, 3] = float("nan")
        wide[3, hkv, 5] = float("inf")
        wide[3, 0] = -0.0
    rows = wide.cuda()  # key and value as strided views of one projection
    key, value = rows[:, :hkv], rows[:, hkv:2 * hkv]
    blocks = (tokens + bs - 1) // bs + 2
    cache = filled(3, blocks, bs, hkv, d, layout)
    before = [t.clone() for t in cache]
    slots = torch.from_numpy(np.random.default_rng(1).permutation(blocks * bs)[:tokens].astype(np.int32)).cuda()
    if tokens > 10:
        slots[7] = -1
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    kx.store_kvcache4(key, value, *cache, slots, error_flag=err)
    k, v = kx.load_kvcache4(*cache, slots, error_flag=err)
    assert err.item() == 0
    kept = (slots >= 0).cpu().numpy()
    for got, x, codes, col in ((k, f32(key), cache[0], 0), (v, f32(value), cache[1], 2)):
        code, scale, zero = plain_quantise(np.where(np.isfinite(x), x, 0))
        want = (code * scale[..., None].astype(np.float64) + zero[..., None]).astype(np.float32)
        want = torch.from_numpy(want).bfloat16().float().numpy()
        bad = ~np.isfinite(x).all(-1)
        want[bad] = np.nan
        want[~kept] = 0
        np.testing.assert_array_equal(f32(got), want)
        blk, at = slots.long() // bs, slots.long() % bs
        held = unpack_codes(codes[blk.clamp(min=0), at.clamp(min=0)])
        np.testing.assert_array_equal(held[kept & ~bad.any(-1)], code[kept & ~bad.any(-1)])
        good = kept[:, None] & ~bad  # half a step and one rounding of the read-back row
        off = np.abs(want - x).max(-1)
        assert (off <= 0.5 * scale * (1 + 2.0 ** -20) + 2.0 ** -8 * np.abs(x).max(-1))[good].all()
    untouched = torch.ones(blocks * bs, dtype=torch.bool, device="cuda")
    untouched[slots[slots >= 0].long()] = False
    for was, now in zip(before, cache):
        was, now = (t.reshape(blocks * bs, *t.shape[2:])[untouched] for t in (was, now))
        assert torch.equal(was, now)


@pytest.mark.gpu
def test_slots_outside_the_cache_are_flagged_and_skipped(kx):
    cache = filled(5, 2, 16, 2, 64)
    before = [t.clone() for t in cache]
    x = torch.randn(4, 2, 64, device="cuda").bfloat16()
    slots = torch.tensor([32, -2, -1, 1 << 30], dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    kx.store_kvcache4(x, x, *cache, slots, error_flag=err)
    assert err.item() == 1 and all(torch.equal(a, b) for a, b in zip(before, cache))
    k, v = kx.load_kvcache4(*cache, slots, error_flag=err)
    assert not k.any() and not v.any()


# ------------------------------------------------------------------------------- decode

LENS = [0, 1, 2, 31, 32, 33, 127, 128, 129, 300, 511, 512]


def run_decode(kx, q, cache, table, lens, scale, longest=None, **kw):
    out = torch.full_like(q, float("nan"))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    kx.paged_decode4(q, *cache, starts(lens), table, max_seqlen_k=max(lens) if longest is None else longest,
                     scale=scale, out=out, error_flag=err, **kw)
    torch.cuda.synchronize()
    assert err.item() == 0
    return out


def check_decode(kx, lens, heads, hkv, d, bs, layout="slots", longest=None, q_scale=1.5, seed=0):
    table, blocks = paged(seed, lens, bs)
    cache = filled(seed + 1, blocks, bs, hkv, d, layout)
    poison_unused(cache, table, lens)
    gen = torch.Generator().manual_seed(seed + 2)
    q = (torch.randn(len(lens) + 2, heads, d, generator=gen) * q_scale).bfloat16().cuda()
    scale = d ** -0.5
    out = run_decode(kx, q, cache, table, lens, scale, longest)
    assert out[len(lens):].isnan().all()  # rows past the batch are left alone
    for b, n in enumerate(lens):
        want, tol = plain_attention(q[b:b + 1], cache, table[b], n, scale)
        check_close(out[b:b + 1], want, tol, f"row {b} of {n} keys")


@pytest.mark.gpu
@pytest.mark.parametrize("heads,hkv,d,bs,layout", [
    (16, 8, 128, 256, "slots"), (16, 8, 128, 16, "heads"), (7, 1, 128, 48, "slots"),
    (14, 2, 64, 32, "heads"), (4, 4, 64, 1, "slots"), (9, 1, 64, 16, "slots"), (34, 2, 128, 256, "slots")])
@pytest.mark.parametrize("longest", [512, 1300])
def test_decode_against_64_bits(kx, heads, hkv, d, bs, layout, longest):
    lens = LENS if longest == 512 else LENS + [513, 640, 1025, 1300]
    check_decode(kx, lens, heads, hkv, d, bs, layout, longest)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[137], [0], [0, 0, 5], [5000], [20000, 1, 3]])
def test_decode_few_long_and_empty(kx, lens):
    check_decode(kx, lens, 16, 8, 128, 256, seed=11)


@pytest.mark.gpu
def test_decode_peaked_scores(kx):
    check_decode(kx, [40, 700, 1500], 16, 8, 128, 256, q_scale=12.0, seed=21)


@pytest.mark.gpu
def test_decode_many_rows(kx):
    rng = np.random.default_rng(3)
    check_decode(kx, [int(n) for n in rng.integers(0, 40, size=300)] + [1600], 2, 1, 64, 16, seed=31)


@pytest.mark.gpu
def test_decode_is_the_same_every_time_and_under_capture(kx):
    lens = [3000, 1, 0, 777]
    table, blocks = paged(1, lens, 256)
    cache = filled(2, blocks, 256, 8, 128)
    q = torch.randn(4, 16, 128, device="cuda").bfloat16()
    cu = starts(lens)
    first = run_decode(kx, q, cache, table, lens, 0.1)
    outs, graphs = [torch.empty_like(q) for _ in range(2)], []
    side = torch.cuda.Stream()
    for out in outs:  # two graphs, replayed at once on two streams
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kx.paged_decode4(q, *cache, cu, table, max_seqlen_k=4096, scale=0.1, out=out)
        graphs.append(graph)
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    again = run_decode(kx, q, cache, table, lens, 0.1, longest=4096)
    for out in outs:
        assert torch.equal(out, again)
    assert torch.equal(run_decode(kx, q, cache, table, lens, 0.1), first)


@pytest.mark.gpu
def test_decode_reads_strided_queries_and_a_given_workspace(kx):
    lens = [1900, 33]
    table, blocks = paged(5, lens, 16)
    cache = filled(6, blocks, 16, 2, 64)
    wide = torch.randn(2, 3, 8, 64, device="cuda").bfloat16()
    q = wide[:, 1, ::2]  # 4 heads, every second one of a wider row
    out = torch.empty(2, 8, 64, dtype=BF16, device="cuda")[:, ::2]
    ws = torch.full((kx.paged_decode4_workspace_size(1900, 4, 2, 64),), 255, dtype=torch.uint8, device="cuda")
    kx.paged_decode4(q, *cache, starts(lens), table, max_seqlen_k=1900, scale=0.125, out=out, workspace=ws)
    for b, n in enumerate(lens):
        want, tol = plain_attention(q[b:b + 1], cache, table[b], n, 0.125)
        check_close(out[b:b + 1], want, tol, f"row {b}")
    with pytest.raises(RuntimeError, match="workspace"):
        kx.paged_decode4(q, *cache, starts(lens), table, max_seqlen_k=1900, scale=0.125, out=out, workspace=ws[:-16])


@pytest.mark.gpu
def test_decode_flags_bad_pages_and_lengths(kx):
    lens = [40, 700]
    table, blocks = paged(7, lens, 16)
    cache = filled(8, blocks, 16, 2, 64)
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    out, err = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device="cuda")
    bad = table.clone()
    bad[0, 1], bad[1, 3] = blocks, -7
    kx.paged_decode4(q, *cache, starts(lens), bad, max_seqlen_k=700, scale=0.1, out=out, error_flag=err)
    assert err.item() == 2
    err.zero_()
    kx.paged_decode4(q, *cache, starts(lens), table[:, :2], max_seqlen_k=700, scale=0.1, out=out, error_flag=err)
    assert err.item() == 8  # both cut at 32 tokens
    for b in range(2):
        want, tol = plain_attention(q[b:b + 1], cache, table[b], 32, 0.1)
        check_close(out[b:b + 1], want, tol, f"row {b}, cut")


@pytest.mark.gpu
def test_decode_not_finite_rows_reach_only_their_sequence(kx):
    lens = [100, 100, 100]
    table, blocks = paged(9, lens, 16)
    cache = filled(10, blocks, 16, 2, 64)
    q = torch.randn(3, 4, 64, device="cuda").bfloat16()
    clean = run_decode(kx, q, cache, table, lens, 0.1)
    cache[2][table[1, 2].long(), 5] = float("nan")
    out = torch.empty_like(q)
    kx.paged_decode4(q, *cache, starts(lens), table, max_seqlen_k=100, scale=0.1, out=out)
    assert out[1].isnan().all() and torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])


# ------------------------------------------------------------------------------ prefill


def check_prefill(kx, q_lens, k_lens, heads, hkv, d, bs, layout="slots", q_scale=1.5, seed=0, scale=None, spread=1.0):
    table, blocks = paged(seed, k_lens, bs)
    cache = filled(seed + 1, blocks, bs, hkv, d, layout, spread)
    poison_unused(cache, table, k_lens)
    gen = torch.Generator().manual_seed(seed + 2)
    total = sum(q_lens)
    q = (torch.randn(total + 3, heads, d, generator=gen) * q_scale).bfloat16().cuda()
    scale = d ** -0.5 if scale is None else scale
    out = torch.full_like(q, float("nan"))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    kx.paged_prefill4(q, *cache, starts(q_lens), starts(k_lens), table, max_seqlen_q=max(q_lens),
                      max_seqlen_k=max(k_lens), scale=scale, out=out, error_flag=err)
    torch.cuda.synchronize()
    assert err.item() == 0 and out[total:].isnan().all()
    at = 0
    for b, (m, n) in enumerate(zip(q_lens, k_lens)):
        want, tol = plain_attention(q[at:at + m], cache, table[b], n, scale, prefill=True, bf16_v=spread != 1.0)
        check_close(out[at:at + m], want, tol, f"sequence {b}: {m} rows, {n} keys")
        at += m


@pytest.mark.gpu
@pytest.mark.parametrize("heads,hkv,d,bs,layout", [
    (16, 8, 128, 256, "slots"), (4, 2, 128, 16, "heads"), (7, 1, 128, 48, "slots"), (14, 2, 64, 32, "heads"),
    (3, 3, 64, 1, "slots"), (9, 1, 64, 16, "slots"), (34, 2, 128, 256, "slots")])
def test_prefill_against_64_bits(kx, heads, hkv, d, bs, layout):
    check_prefill(kx, [1, 5, 0, 64, 33, 1, 2], [1, 5, 17, 64, 300, 129, 140], heads, hkv, d, bs, layout)


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,k_lens", [
    ([200], [200]), ([128], [128]), ([129], [1000]), ([1], [0]), ([3, 4], [0, 2]), ([300, 7], [290, 3]), ([1], [2500])])
def test_prefill_lengths(kx, q_lens, k_lens):
    check_prefill(kx, q_lens, k_lens, 4, 2, 128, 16, seed=4)


SPLIT = [([200], [5000]), ([1, 300, 0, 17, 4], [4000, 1300, 2000, 0, 3]), ([40, 40, 40, 1], [3000, 1500, 1025, 9]),
         ([500, 3], [1400, 5]), ([600], [100])]


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,k_lens", SPLIT)
@pytest.mark.parametrize("heads,hkv,d,bs", [(4, 2, 128, 256), (7, 1, 64, 16)])
def test_prefill_contexts_split_over_ctas(kx, q_lens, k_lens, heads, hkv, d, bs):
    assert kx.paged_prefill4_workspace_size(sum(q_lens) + 3, len(q_lens), max(max(k_lens), 1025), heads, hkv, d) > 0
    check_prefill(kx, q_lens, k_lens, heads, hkv, d, bs)


@pytest.mark.gpu
def test_prefill_split_any_workspace_the_same_every_time_and_under_capture(kx):
    q_lens, k_lens = SPLIT[1]
    table, blocks = paged(3, k_lens, 32)
    cache = filled(4, blocks, 32, 2, 128)
    poison_unused(cache, table, k_lens)
    q = torch.randn(sum(q_lens), 8, 128, device="cuda").bfloat16()
    slot = 256 * 132 * 4

    def call(ws, out=None):
        return kx.paged_prefill4(q, *cache, starts(q_lens), starts(k_lens), table, max_seqlen_q=300, max_seqlen_k=4000,
                                 scale=0.09, out=torch.empty_like(q) if out is None else out, workspace=ws)

    want = call(None)
    for slots in (0, 1, 2, 9, 50, 400):  # split less, or not at all
        ws = torch.full((slots * slot + 16,), 255, dtype=torch.uint8, device="cuda")  # (NaN)
        got = call(ws)
        assert torch.equal(got, call(ws))
        at = 0
        for b, (m, n) in enumerate(zip(q_lens, k_lens)):
            check_close(got[at:at + m], *plain_attention(q[at:at + m], cache, table[b], n, 0.09, prefill=True),
                        f"{slots} slots, sequence {b}")
            at += m
    cq, ck, out = starts(q_lens), starts(k_lens), torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kx.paged_prefill4(q, *cache, cq, ck, table, max_seqlen_q=300, max_seqlen_k=4000, scale=0.09, out=out)
    for _ in range(2):
        out.fill_(float("nan"))
        graph.replay()
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_prefill_scales(kx, scale):
    check_prefill(kx, [70, 1], [200, 140], 4, 2, 128, 256, seed=5, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("spread,q_scale", [(1e-5, 1e5), (1e6, 1e-6), (1e30, 1e-30), (1e-30, 1e30)])
def test_prefill_values_outside_fp16(kx, spread, q_scale):
    """K and V of any size of bf16 (V then goes through as bf16, 2^-8 for it and for P)."""
    check_prefill(kx, [70, 1], [200, 140], 4, 2, 128, 256, seed=5, spread=spread, q_scale=q_scale)


@pytest.mark.gpu
def test_decode_values_of_any_size(kx):
    for spread in (1e-30, 1e-5, 1e6, 1e30):
        table, blocks = paged(3, [700, 33], 256)
        cache = filled(4, blocks, 256, 2, 128, spread=spread)
        q = (torch.randn(2, 4, 128, device="cuda") / spread).bfloat16()
        out = run_decode(kx, q, cache, table, [700, 33], 0.08)
        for b, n in enumerate((700, 33)):
            want, tol = plain_attention(q[b:b + 1], cache, table[b], n, 0.08)
            check_close(out[b:b + 1], want, tol, f"spread {spread}, row {b}")


@pytest.mark.gpu
def test_prefill_more_items_than_ctas(kx):
    rng = np.random.default_rng(1)
    q = [int(n) for n in rng.integers(0, 6, size=200)]
    check_prefill(kx, q, [n + int(rng.integers(0, 20)) for n in q], 4, 2, 64, 16, seed=6)


@pytest.mark.gpu
def test_prefill_equals_decode_on_single_rows(kx):
    """One query token per sequence is what paged_decode4 computes (which rounds less)."""
    lens = [1, 50, 700, 1290]
    table, blocks = paged(3, lens, 256)
    cache = filled(4, blocks, 256, 8, 128)
    q = torch.randn(4, 16, 128, device="cuda").bfloat16()
    one = run_decode(kx, q, cache, table, lens, 0.08)
    out = torch.empty_like(q)
    kx.paged_prefill4(q, *cache, starts([1] * 4), starts(lens), table, max_seqlen_q=1, max_seqlen_k=1290, scale=0.08,
                      out=out)
    for b, n in enumerate(lens):
        _, tol = plain_attention(q[b:b + 1], cache, table[b], n, 0.08, prefill=True)
        _, tol1 = plain_attention(q[b:b + 1], cache, table[b], n, 0.08)
        check_close(out[b:b + 1], one[b:b + 1].double().cpu().numpy(), tol + tol1, f"row {b}")


@pytest.mark.gpu
def test_prefill_not_finite_keys_reach_only_the_rows_that_see_them(kx):
    table, blocks = paged(2, [100, 100], 16)
    cache = filled(3, blocks, 16, 2, 128)
    q = torch.randn(200, 4, 128, device="cuda").bfloat16()
    call = lambda: kx.paged_prefill4(  # noqa: E731
        q, *cache, starts([100, 100]), starts([100, 100]), table, max_seqlen_q=100, max_seqlen_k=100, scale=0.1,
        out=torch.empty_like(q))
    clean = call()
    for half in (slice(0, 2), slice(2, 4)):  # K, then V, of key 60 of the second sequence
        kept = cache[2].clone()
        cache[2][table[1, 3].long(), 12, 1, half] = float("nan")
        got = call()
        cache[2].copy_(kept)
        hit = torch.zeros(200, 4, dtype=torch.bool, device="cuda")
        hit[160:, 2:] = True
        assert got[hit].isnan().all() and torch.equal(got[~hit], clean[~hit])


@pytest.mark.gpu
def test_prefill_largest_values_reach_only_the_rows_that_see_them(kx):
    """A V row whose top code lies past the largest bf16 is no infinity to rows behind the mask."""
    table, blocks = paged(2, [100, 100], 16)
    cache = filled(3, blocks, 16, 2, 128)
    q = torch.randn(200, 4, 128, device="cuda").bfloat16()
    call = lambda: kx.paged_prefill4(  # noqa: E731
        q, *cache, starts([100, 100]), starts([100, 100]), table, max_seqlen_q=100, max_seqlen_k=100, scale=0.1,
        out=torch.empty_like(q))
    clean = call()
    most = torch.finfo(BF16).max
    row = cache[2][table[1, 4].long(), 6, 1]  # key 70 of the second sequence
    row[2:] = torch.tensor([most / 15 * (1 + 2 ** -7), 0.0], device="cuda").bfloat16()
    assert 15 * row[2].double().item() > most * (1 + 2 ** -9)
    got = call()
    hit = torch.zeros(200, 4, dtype=torch.bool, device="cuda")
    hit[170:, 2:] = True
    # rows that do not see the key, in the 32 keys whose P is now rounded to bf16 (2^-8 of values
    # up to 15 steps past the zero): those of keys 64 to 69
    near = torch.zeros_like(hit)
    near[164:170, 2:] = True
    assert torch.equal(got[~hit & ~near], clean[~hit & ~near])
    top = (cache[2][..., 2].abs() * 15 + cache[2][..., 3].abs()).view(-1, 2)
    top = top[top < 1e30].max().item()
    assert (got[near].float() - clean[near].float()).abs().max().item() <= 4 * 2 ** -8 * top


@pytest.mark.gpu
def test_prefill_flags_and_capture(kx):
    q_lens, k_lens = [30, 40], [60, 300]
    table, blocks = paged(7, k_lens, 16)
    cache = filled(8, blocks, 16, 2, 64)
    q = torch.randn(70, 4, 64, device="cuda").bfloat16()
    out, err = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device="cuda")
    cq, ck = starts(q_lens), starts(k_lens)
    call = lambda t: kx.paged_prefill4(  # noqa: E731
        q, *cache, cq, ck, t, max_seqlen_q=40, max_seqlen_k=300, scale=0.1, out=out, error_flag=err)
    bad = table.clone()
    bad[1, 3] = -5
    call(bad)
    assert err.item() == 2
    err.zero_()
    call(table[:, :8])
    assert err.item() == 8
    err.zero_()
    call(table)
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(table)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want) and err.item() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_maximum_that_jumps(kx, d):
    """Scores that rise by 2^8, 2^15 and far beyond within a tile and from tile to tile."""
    n, m = 400, 130
    table, blocks = paged(1, [n], 256)
    gen = torch.Generator().manual_seed(d)
    rows = torch.randn(n, 1, d, generator=gen) * 0.3
    rows[:, 0, 0] = torch.arange(n) % 97 * 0.07  # within a tile
    for key, size in ((40, 30.0), (70, 55.0), (129, 80.0), (300, 140.0), (301, 90.0)):
        rows[key, 0, 0] = size
    cache = kx.kv4_cache(blocks, 256, 1, d)
    slots = (table[0].long()[torch.arange(n) // 256] * 256 + torch.arange(n).cuda() % 256).int()
    value = torch.randn(n, 1, d, generator=gen).bfloat16().cuda()
    kx.store_kvcache4(rows.bfloat16().cuda(), value, *cache, slots)
    q = torch.randn(m, 2, d, generator=gen) * 0.2
    q[:, 0, 0], q[:, 1, 0] = 1.0, -1.0
    q = q.bfloat16().cuda()
    out = torch.empty_like(q)
    kx.paged_prefill4(q, *cache, starts([m]), starts([n]), table, max_seqlen_q=m, max_seqlen_k=n, scale=0.6, out=out)
    want, tol = plain_attention(q, cache, table[0], n, 0.6, prefill=True)
    check_close(out, want, tol, "jumps")
