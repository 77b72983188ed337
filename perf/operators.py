"""Operators of a multi-tenant decoder layer over a 4-bit paged KV cache, and what they cost.

Five operators, used in this order by one decoder layer that serves many requests at once:

* ``lora``    a projection shared by all requests plus each request's own low-rank adapter,
* ``rope``    q/k RMS norm and rotary positions with several axes (time, height, width),
              fused with the store into the paged cache (16-bit or 4-bit),
* ``store``   K/V rows quantised to 4 bits into paged slots, and rows read back as bf16,
* ``decode``  attention of one new token per request over the 4-bit cache,
* ``prefill`` causal attention of many new tokens per request over the 4-bit cache.

The 4-bit format: a cached head row of D values is D / 2 bytes (value 2j in the low half of
byte j) plus a bf16 scale and a bf16 zero; value = zero + code * scale. ``zero`` is the row's
minimum and ``scale`` the smallest bf16 with 15 * scale >= maximum - minimum.

``run`` computes the operators in plain torch operations, or calls the framework's own kernels
where ``own`` is true.
"""

import math
import random

import torch

own = False

BLOCK = 256  # tokens of a cache block, as the engine allocates them
EPS = 1e-6


# ------------------------------------------------------------------------------- cases


def listed():
    return [
        # the rows one decode step of a full batch adds to the cache
        dict(name="store, 32 new rows", op="store", tokens=32, kv_heads=8, dim=128, key=1),
        # a prefill batch's rows (the token budget of one engine step)
        dict(name="store, 8192 rows", op="store", tokens=8192, kv_heads=8, dim=128, key=2),
        # q/k norm + 3-axis rotation of one decode step, 4-bit cache
        dict(name="rope, 32 rows, 4-bit", op="rope", tokens=32, heads=16, kv_heads=8, dim=128,
             axes=3, interleaved=1, bits=4, key=3),
        # the same for a prefill batch with image grids in its prompts, 16-bit cache
        dict(name="rope, 7829 rows", op="rope", tokens=7829, heads=16, kv_heads=8, dim=128,
             axes=3, interleaved=0, bits=16, key=4),
        # one interactive request
        dict(name="decode, 1 x 137", op="decode", batch=1, low=137, high=137, heads=16,
             kv_heads=8, dim=128, empty=0, key=5),
        # a full decode bucket of short requests, two of its rows without any key
        dict(name="decode, 32 x 64..1024", op="decode", batch=32, low=64, high=1024, heads=16,
             kv_heads=8, dim=128, empty=2, key=6),
        # long contexts, which is what a 4-bit cache is for
        dict(name="decode, 32 x 8k..32k", op="decode", batch=32, low=8192, high=32768, heads=16,
             kv_heads=8, dim=128, empty=0, key=7),
        # a mixed batch: new prompts, chunks behind a cached prefix, single decode rows
        dict(name="prefill, mixed", op="prefill", batch=7, q_low=1, q_high=600, k_extra=2000,
             heads=16, kv_heads=8, dim=128, key=8),
        # long chunks behind long cached prefixes
        dict(name="prefill, 4 x 2k of 8k", op="prefill", batch=4, q_low=1800, q_high=2048,
             k_extra=6144, heads=16, kv_heads=8, dim=128, key=9),
        # the qkv projection of a decode step, 8 tenants, some rows without an adapter
        dict(name="lora, 13 rows", op="lora", rows=13, k=1024, n=4096, rank=16, adapters=8, key=10),
        # a full decode bucket where almost every row has its own adapter
        dict(name="lora, 64 rows", op="lora", rows=64, k=2048, n=4096, rank=64, adapters=48, key=11),
        # a prefill batch of several requests
        dict(name="lora, 7829 rows", op="lora", rows=7829, k=2048, n=4096, rank=32, adapters=16,
             key=12),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["store", "rope", "decode", "decode", "prefill", "prefill", "lora", "lora"])
    key = rng.randrange(1 << 20)
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (16, 16), (16, 2), (14, 2), (32, 8), (20, 4), (7, 1)])
    dim = rng.choice([128, 128, 64])
    if op == "store":
        return dict(op=op, tokens=_spread(rng, 1, 8192), kv_heads=kv_heads, dim=dim, key=key)
    if op == "rope":
        return dict(op=op, tokens=_spread(rng, 1, 8192 * 16 // max(16, heads)), heads=heads,
                    kv_heads=kv_heads, dim=dim, axes=rng.choice([2, 3, 3, 4]),
                    interleaved=rng.randrange(2), bits=rng.choice([4, 16]), key=key)
    if op == "decode":
        batch = _spread(rng, 1, 64)
        top = min(32768, 600_000 // (batch * kv_heads) * 8)
        high = _spread(rng, 1, top)
        return dict(op=op, batch=batch, low=max(1, high // rng.choice([1, 2, 16])), high=high, heads=heads,
                    kv_heads=kv_heads, dim=dim, empty=rng.choice([0, 0, 1]) if batch > 1 else 0, key=key)
    if op == "prefill":
        batch = _spread(rng, 1, 12)
        q_high = _spread(rng, 1, max(16, 7000 // batch))
        return dict(op=op, batch=batch, q_low=max(1, q_high // rng.choice([1, 2, 50])), q_high=q_high,
                    k_extra=rng.choice([0, _spread(rng, 1, 6144)]), heads=min(heads, 16),
                    kv_heads=min(kv_heads, 8) if heads != 16 else kv_heads, dim=dim, key=key)
    rows = _spread(rng, 1, 7829)
    return dict(op=op, rows=rows, k=64 * _spread(rng, 4, 32), n=64 * _spread(rng, 4, 64),
                rank=rng.choice([8, 16, 16, 24, 32, 64]), adapters=_spread(rng, 1, 48 if rows <= 64 else 16),
                key=key)


def _lens(case):
    """Key lengths (and query lengths for prefill) of a case's requests."""
    rng = random.Random(case["key"])
    if case["op"] == "decode":
        k = [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]
        k[0] = case["high"]
        for i in range(case["empty"]):
            k[-1 - i] = 0
        return k, [1] * len(k)
    q = [_spread(rng, case["q_low"], case["q_high"]) for _ in range(case["batch"])]
    q[0] = case["q_high"]
    return [n + (rng.randint(0, case["k_extra"]) if i % 3 else case["k_extra"]) for i, n in enumerate(q)], q


def work(case):
    op = case["op"]
    if op == "store":
        values = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        rows = 2 * case["tokens"] * case["kv_heads"]
        return {"bytes": values * 2 + 2 * (values // 2 + rows * 4) + values * 2 + case["tokens"] * 8,
                "flops": 4 * values}
    if op == "rope":
        t, d = case["tokens"], case["dim"]
        read = t * (case["heads"] + 2 * case["kv_heads"]) * d * 2 + t * case["axes"] * 8 + t * d * 4 + t * 4
        kv = 2 * t * case["kv_heads"] * d * 2
        wrote = t * case["heads"] * d * 2 + (kv if case["bits"] == 16 else kv + 2 * (kv // 4 + 8 * t * case["kv_heads"]))
        return {"bytes": read + wrote, "flops": 10 * t * (case["heads"] + case["kv_heads"]) * d}
    if op in ("decode", "prefill"):
        k, q = _lens(case)
        cache = sum(k) * case["kv_heads"] * (case["dim"] + 8)
        rows = sum(q) * case["heads"] * case["dim"] * 2 * 2
        tables = 4 * sum((n + BLOCK - 1) // BLOCK for n in k)
        pairs = sum(m * n - m * (m - 1) // 2 for n, m in zip(k, q) if n)
        return {"bytes": cache + rows + tables, "flops": 4 * case["heads"] * case["dim"] * pairs}
    t, k, n, r = case["rows"], case["k"], case["n"], case["rank"]
    used = min(case["adapters"], t)
    return {"bytes": 2 * (t * k + n * k + t * n + used * r * (k + n)) + 4 * t + 4 * used,
            "flops": 2 * t * n * k + 2 * t * r * (k + n)}


# ------------------------------------------------------------------------------ inputs


def _generator(seed, case):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1_000_003 + case["key"])


def _randn(gen, *shape, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen) * scale).bfloat16()


def _quantise(x):
    """bf16 rows [..., D] as 4-bit codes [..., D / 2], a bf16 scale and a bf16 zero [...]."""
    x = x.float()
    low, high = x.amin(-1), x.amax(-1)
    wide = high - low
    # the smallest bf16 whose 15 steps reach the row's maximum (15 * scale is exact in 32 bits);
    # a row narrower than 2^-100 is held as its minimum
    scale = (wide / 15).bfloat16()
    scale = _step(scale, 15 * scale.float() < wide, 1)
    below = _step(scale, scale > 0, -1)
    scale = torch.where(15 * below.float() >= wide, below, scale)
    scale = torch.where(wide < 2.0 ** -100, torch.zeros_like(scale), scale)
    step = scale.float().unsqueeze(-1)
    code = torch.where(step > 0, (x - low.unsqueeze(-1)) / step, torch.zeros_like(x))
    code = code.round().clamp(0, 15).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale, low.bfloat16()


def _step(x, where, by):
    """The next bf16 up or down of positive values, where asked."""
    return torch.where(where, (x.view(torch.int16) + by).view(torch.bfloat16), x)


def _values(codes, scale, zero):
    """What 4-bit rows stand for, in 32 bits."""
    x = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    return x * scale.float().unsqueeze(-1) + zero.float().unsqueeze(-1)


def _filled_cache(gen, blocks, kv_heads, dim):
    """A cache whose rows hold normalised keys (some channels larger, as rotary keys have) and values."""
    kc = torch.empty(blocks, BLOCK, kv_heads, dim // 2, dtype=torch.uint8, device="cuda")
    vc = torch.empty_like(kc)
    params = torch.empty(blocks, BLOCK, kv_heads, 4, dtype=torch.bfloat16, device="cuda")
    channel = 1 + 2 * (torch.rand(kv_heads, dim, device="cuda", generator=gen) > 0.95).float()
    for i in range(0, blocks, 256):
        n = min(256, blocks - i)
        k = (torch.randn(n, BLOCK, kv_heads, dim, device="cuda", generator=gen) * channel).bfloat16()
        kc[i:i + n], params[i:i + n, ..., 0], params[i:i + n, ..., 1] = _quantise(k)
        v = torch.randn(n, BLOCK, kv_heads, dim, device="cuda", generator=gen).bfloat16()
        vc[i:i + n], params[i:i + n, ..., 2], params[i:i + n, ..., 3] = _quantise(v)
    return kc, vc, params


def _paged(gen, lens):
    """Block tables [B, W] int32 over shuffled blocks (rows padded with -1), and the block count."""
    used = [(n + BLOCK - 1) // BLOCK for n in lens]
    blocks = sum(used) + 1
    order = torch.randperm(blocks, device="cuda", generator=gen).int()
    column = torch.arange(max(1, max(used)), device="cuda")
    counts = torch.tensor(used, device="cuda")
    first = torch.cumsum(counts, 0) - counts
    at = (first[:, None] + column).clamp_(max=blocks - 1)
    return torch.where(column < counts[:, None], order[at], -1).int().contiguous(), blocks


def _starts(lens):
    return torch.tensor([0] + lens, device="cuda").cumsum(0).int()


def _grid_positions(tokens, axes):
    """Positions [axes, T]: text runs (all axes equal) between grids of 15 x 22 patches."""
    i = torch.arange(tokens, device="cuda")
    grid = 15 * 22
    run, inside = i // (grid + 70), i % (grid + 70)
    base = run * (70 + 22)
    text = inside < 70
    patch = (inside - 70).clamp(min=0)
    step = [patch // grid, patch // 22, patch % 22, patch % 7]
    rows = [torch.where(text, base + inside, base + 70 + step[a % 4]) for a in range(axes)]
    return torch.stack(rows).contiguous()


def _axis_of(dim, axes, interleaved):
    """Which axis each of the D / 2 frequencies turns by: the axes in turn (the first takes what
    is left over), or one run of frequencies per axis."""
    half = dim // 2
    if interleaved:
        share = half // (axes + 1)
        return [j % axes if j < axes * share else 0 for j in range(half)]
    share = half // axes
    return [min(j // share, axes - 1) for j in range(half)]


def _rope_table(dim, positions):
    inverse = 1.0 / 1_000_000.0 ** (torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inverse
    return torch.cat((angle.cos(), angle.sin()), -1).float()


def prepare(case, seed):
    gen = _generator(seed, case)
    op = case["op"]
    s = dict(op=op, case=case)
    if op in ("store", "rope"):
        t, h, d = case["tokens"], case["kv_heads"], case["dim"]
        blocks = (t + BLOCK - 1) // BLOCK + 1
        slots = torch.randperm(blocks * BLOCK, device="cuda", generator=gen)[:t].int()
        slots[t // 2::97] = -1  # rows that are not cached (prompt padding)
        s["slots"] = slots
        s["read"] = slots[torch.randperm(t, device="cuda", generator=gen)]
        s["k_codes"], s["v_codes"], s["params"] = _filled_cache(gen, blocks, h, d)
    if op == "store":
        channel = 1 + 2 * (torch.rand(h, d, device="cuda", generator=gen) > 0.95).float()
        s["key"] = (torch.randn(t, h, d, device="cuda", generator=gen) * channel).bfloat16()
        s["value"] = _randn(gen, t, h, d)
    elif op == "rope":
        s["qkv"] = _randn(gen, t, (case["heads"] + 2 * h) * d, scale=2.0)
        s["q_weight"] = (1 + 0.3 * torch.randn(d, device="cuda", generator=gen)).bfloat16()
        s["k_weight"] = (1 + 0.3 * torch.randn(d, device="cuda", generator=gen)).bfloat16()
        s["positions"] = _grid_positions(t, case["axes"])
        s["axis"] = torch.tensor(_axis_of(d, case["axes"], case["interleaved"]), device="cuda").int()
        s["table"] = _rope_table(d, 65536)
        if case["bits"] == 16:
            s["k_cache"] = _randn(gen, blocks, BLOCK, h, d)
            s["v_cache"] = _randn(gen, blocks, BLOCK, h, d)
    elif op in ("decode", "prefill"):
        k, q = _lens(case)
        s["tables"], blocks = _paged(gen, k)
        s["k_codes"], s["v_codes"], s["params"] = _filled_cache(gen, blocks, case["kv_heads"], case["dim"])
        s["cu_k"], s["cu_q"], s["max_k"], s["max_q"] = _starts(k), _starts(q), max(k), max(q)
        s["q"] = _randn(gen, sum(q), case["heads"], case["dim"], scale=1.5)
        s["scale"] = case["dim"] ** -0.5
    elif op == "lora":
        t, k, n, r, a = case["rows"], case["k"], case["n"], case["rank"], case["adapters"]
        s["x"] = _randn(gen, t, k)
        s["weight"] = _randn(gen, n, k, scale=k ** -0.5)
        s["a"] = _randn(gen, a, r, k, scale=k ** -0.5)
        s["b"] = _randn(gen, a, n, r, scale=0.5 * r ** -0.5)
        s["scales"] = 0.5 + 1.5 * torch.rand(a, device="cuda", generator=gen)
        if t <= 64:  # a decode step: one row per request
            s["rows"] = torch.randint(-1, a, (t,), device="cuda", generator=gen).int()
        else:  # a prefill batch: each request's rows follow one another
            cuts = torch.rand(2 * a, device="cuda", generator=gen).mul(t).long()
            request = (torch.arange(t, device="cuda")[:, None] >= cuts).sum(1)
            s["rows"] = torch.randint(-1, a, (2 * a + 1,), device="cuda", generator=gen).int()[request]
    return s


# ------------------------------------------------------------------------------ passes


def run(s):
    return {"store": _store, "rope": _rope, "decode": _decode, "prefill": _prefill, "lora": _lora}[s["op"]](s)


def _put(s, key, value):
    """Rows into their slots; a slot of -1 is left out."""
    at = torch.nonzero(s["slots"] >= 0).squeeze(1)
    to = s["slots"][at].long()
    params = s["params"].flatten(0, 1)
    s["k_codes"].flatten(0, 1)[to], params[to, :, 0], params[to, :, 1] = (x[at] for x in _quantise(key))
    s["v_codes"].flatten(0, 1)[to], params[to, :, 2], params[to, :, 3] = (x[at] for x in _quantise(value))


def _get(s):
    """The rows of slots as bf16; a slot of -1 reads as zeros."""
    at = s["read"].long().clamp(min=0)
    p = s["params"].flatten(0, 1)[at]
    keep = (s["read"] >= 0)[:, None, None]
    k = _values(s["k_codes"].flatten(0, 1)[at], p[..., 0], p[..., 1])
    v = _values(s["v_codes"].flatten(0, 1)[at], p[..., 2], p[..., 3])
    return torch.where(keep, k, 0.0).bfloat16(), torch.where(keep, v, 0.0).bfloat16()


def _store(s):
    if own:
        from voiceagent_b200 import kernels as kx

        kx.store_kvcache4(s["key"], s["value"], s["k_codes"], s["v_codes"], s["params"], s["slots"])
        k, v = kx.load_kvcache4(s["k_codes"], s["v_codes"], s["params"], s["read"])
    else:
        _put(s, s["key"], s["value"])
        k, v = _get(s)
    return {"key": k, "value": v}


def _rope(s):
    c = s["case"]
    heads, h, d = c["heads"], c["kv_heads"], c["dim"]
    t = s["qkv"].shape[0]
    if own:
        from voiceagent_b200 import kernels as kx

        q = torch.empty(t, heads, d, dtype=torch.bfloat16, device=s["qkv"].device)
        to = (dict(k_cache=s["k_cache"], v_cache=s["v_cache"]) if c["bits"] == 16 else
              dict(k_codes=s["k_codes"], v_codes=s["v_codes"], kv_params=s["params"]))
        kx.qk_norm_mrope_store(s["qkv"], s["positions"], s["axis"], num_heads=heads, num_kv_heads=h, head_dim=d,
                               q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS, cos_sin_cache=s["table"],
                               q_out=q, slot_mapping=s["slots"], **to)
        if c["bits"] == 16:
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        k, v = kx.load_kvcache4(s["k_codes"], s["v_codes"], s["params"], s["read"])
        return {"q": q, "key": k, "value": v}
    x = s["qkv"].view(t, heads + 2 * h, d)
    y = x[:, :heads + h].float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
    weight = torch.cat((s["q_weight"].expand(heads, d), s["k_weight"].expand(h, d))).float()
    y = y * weight
    half = d // 2
    column = torch.arange(half, device=y.device)
    at = s["positions"][s["axis"].long()].t()  # [T, D / 2]: each frequency's own position
    cos, sin = s["table"][at, column][:, None], s["table"][at, half + column][:, None]
    first, second = y[..., :half], y[..., half:]
    y = torch.cat((first * cos - second * sin, second * cos + first * sin), -1).bfloat16()
    q, key, value = y[:, :heads].contiguous(), y[:, heads:], x[:, heads + h:]
    if c["bits"] == 4:
        _put(s, key, value)
        k, v = _get(s)
        return {"q": q, "key": k, "value": v}
    at = torch.nonzero(s["slots"] >= 0).squeeze(1)
    to = s["slots"][at].long()
    s["k_cache"].flatten(0, 1)[to] = key[at]
    s["v_cache"].flatten(0, 1)[to] = value[at]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _rows_of(s):
    """Every request's cached rows, padded to the longest: values [B, Hkv, L, D] and the lengths."""
    lens = (s["cu_k"][1:] - s["cu_k"][:-1]).long()
    place = torch.arange(max(1, s["max_k"]), device=lens.device)
    slot = s["tables"].long()[:, place // BLOCK].clamp(min=0) * BLOCK + place % BLOCK
    p = s["params"].flatten(0, 1)[slot]
    k = _values(s["k_codes"].flatten(0, 1)[slot], p[..., 0], p[..., 1]).transpose(1, 2)
    v = _values(s["v_codes"].flatten(0, 1)[slot], p[..., 2], p[..., 3]).transpose(1, 2)
    return k, v, lens, place


def _softmax_rows(score, seen):
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)  # a row that sees nothing gives zeros


def _decode(s):
    q = s["q"]
    if own:
        from voiceagent_b200 import kernels as kx

        return kx.paged_decode4(q, s["k_codes"], s["v_codes"], s["params"], s["cu_k"], s["tables"],
                                max_seqlen_k=s["max_k"], scale=s["scale"], out=torch.empty_like(q))
    b, heads, d = q.shape
    k, v, lens, place = _rows_of(s)
    score = torch.matmul(q.float().view(b, k.shape[1], -1, d), k.transpose(2, 3)) * s["scale"]
    p = _softmax_rows(score, (place < lens[:, None])[:, None, None])
    return torch.matmul(p, v).view(b, heads, d).bfloat16()


def _prefill(s):
    q = s["q"]
    if own:
        from voiceagent_b200 import kernels as kx

        return kx.paged_prefill4(q, s["k_codes"], s["v_codes"], s["params"], s["cu_q"], s["cu_k"], s["tables"],
                                 max_seqlen_q=s["max_q"], max_seqlen_k=s["max_k"], scale=s["scale"],
                                 out=torch.empty_like(q))
    t, heads, d = q.shape
    k, v, k_len, place = _rows_of(s)
    b, h = k.shape[:2]
    q_len = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    row = torch.arange(t, device=q.device)
    request = torch.searchsorted(s["cu_q"][1:].contiguous(), row.int(), right=True)
    inside = row - s["cu_q"].long()[request]
    padded = torch.zeros(b, s["max_q"], heads, d, device=q.device)
    padded[request, inside] = q.float()
    padded = padded.view(b, s["max_q"], h, -1, d).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, Hkv, G * Lq, D]
    score = torch.matmul(padded, k.transpose(2, 3)) * s["scale"]
    last = torch.arange(s["max_q"], device=q.device) + (k_len - q_len)[:, None]  # the last key a row sees
    seen = (place <= last[:, :, None]).repeat(1, heads // h, 1)[:, None]
    out = torch.matmul(_softmax_rows(score, seen), v)
    out = out.view(b, h, heads // h, s["max_q"], d).permute(0, 3, 1, 2, 4).reshape(b, s["max_q"], heads, d)
    return out[request, inside].bfloat16()


def _lora(s):
    if own:
        from voiceagent_b200 import kernels as kx

        return kx.lora_linear(s["x"], s["weight"], s["a"], s["b"], s["scales"], s["rows"])
    x, rows = s["x"].float(), s["rows"].long()
    adapters, rank = s["a"].shape[:2]
    y = x @ s["weight"].float().t()
    mine = torch.arange(adapters, device=x.device) == rows[:, None]  # [T, adapters]
    down = (x @ s["a"].float().flatten(0, 1).t()).view(-1, adapters, rank)
    down = (down * (mine * s["scales"])[..., None]).flatten(1)
    y = y + down @ s["b"].float().transpose(1, 2).reshape(adapters * rank, -1)
    return y.bfloat16()


# ------------------------------------------------------------------- the same in 64 bits


def _exact_rows(x):
    """The 4-bit values that rows of 64-bit numbers are held as, rounded to bf16 before."""
    x = x.to(torch.bfloat16).double()
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    wide = high - low
    fifteenth = wide / torch.full_like(wide, 15)
    mantissa, _ = torch.frexp(fifteenth)
    unit = fifteenth / mantissa / 256  # the step of bf16 at this size
    scale = torch.where(wide >= 2.0 ** -100, torch.ceil(wide / (15 * unit)) * unit, 0.0)
    code = torch.where(scale > 0, torch.round((x - low) / scale.clamp(min=1e-300)), 0.0)
    return low + code.clamp(0, 15) * scale


def _exact_cached(s, which):
    """A filled cache's values in 64 bits, one row per slot."""
    codes = s["k_codes" if which == 0 else "v_codes"].flatten(0, 1).long()
    p = s["params"].flatten(0, 1).double()
    x = torch.empty(*codes.shape[:2], 2 * codes.shape[2], dtype=torch.float64, device=codes.device)
    x[..., 0::2] = p[..., 2 * which + 1:2 * which + 2] + (codes % 16) * p[..., 2 * which:2 * which + 1]
    x[..., 1::2] = p[..., 2 * which + 1:2 * which + 2] + (codes // 16) * p[..., 2 * which:2 * which + 1]
    return x


def _exact_read(s, key, value):
    """What read slots give after key and value rows were stored."""
    out = {}
    inverse = torch.full((int(s["slots"].max()) + 1,), -1, dtype=torch.long, device="cuda")
    for i, slot in enumerate(s["slots"].tolist()):
        if slot >= 0:
            inverse[slot] = i
    for name, x in (("key", key), ("value", value)):
        rows = torch.zeros(len(s["read"]), *x.shape[1:], dtype=torch.float64, device="cuda")
        held = _exact_rows(x)
        wanted = s["read"] >= 0
        rows[wanted] = held[inverse[s["read"][wanted].long()]]
        out[name] = rows
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "store":
        return _exact_read(s, s["key"].double(), s["value"].double())
    if op == "rope":
        heads, h, d = case["heads"], case["kv_heads"], case["dim"]
        x = s["qkv"].double().reshape(-1, heads + 2 * h, d)
        norm = torch.sqrt((x * x).sum(-1, keepdim=True) / d + EPS)
        y = x / norm
        y[:, :heads] *= s["q_weight"].double()
        y[:, heads:heads + h] *= s["k_weight"].double()
        turned = y.clone()
        for j, axis in enumerate(s["axis"].tolist()):
            entry = s["table"][s["positions"][axis]].double()
            cos, sin = entry[:, None, j], entry[:, None, j + d // 2]
            turned[..., j] = y[..., j] * cos - y[..., j + d // 2] * sin
            turned[..., j + d // 2] = y[..., j + d // 2] * cos + y[..., j] * sin
        q, key, value = turned[:, :heads], turned[:, heads:heads + h], x[:, heads + h:]
        if case["bits"] == 4:
            return {"q": q, **_exact_read(s, key, value)}
        out = {"q": q, "k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double()}
        stored = s["slots"] >= 0
        out["k_cache"].view(-1, h, d)[s["slots"][stored].long()] = key[stored]
        out["v_cache"].view(-1, h, d)[s["slots"][stored].long()] = value[stored]
        return out
    if op in ("decode", "prefill"):
        k_lens, q_lens = _lens(case)
        d, group = case["dim"], case["heads"] // case["kv_heads"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        begin = 0
        for b, (n, m) in enumerate(zip(k_lens, q_lens)):
            if n:
                blocks = s["tables"][b, :(n + BLOCK - 1) // BLOCK].long()
                part = {name: s[name][blocks] for name in ("k_codes", "v_codes", "params")}
                k, v = _exact_cached(part, 0)[:n], _exact_cached(part, 1)[:n]
                hidden = torch.ones(m, n, dtype=torch.bool, device="cuda").triu(n - m + 1)
                for head in range(case["heads"]):
                    logit = s["q"][begin:begin + m, head].double() @ k[:, head // group].T / math.sqrt(d)
                    weight = torch.softmax(logit.masked_fill(hidden, -math.inf), -1)
                    out[begin:begin + m, head] = weight @ v[:, head // group]
            begin += m
        return out
    x, rows = s["x"].double(), s["rows"]
    y = x @ s["weight"].double().T
    for i in range(case["adapters"]):
        mine = rows == i
        y[mine] += s["scales"][i].double() * ((x[mine] @ s["a"][i].double().T) @ s["b"][i].double().T)
    return y
