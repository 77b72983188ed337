"""q/k norm + rotary positions with several axes + the paged store, against 64 bits.

The kernel computes in 32 bits and rounds to bf16 once, so an output is within 2^-8 of its
value, plus 2^-19 of the terms it is a difference of (a few 2^-24 roundings and rsqrt's 2^-22)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from tests.test_kv4 import filled, f32, plain_quantise

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def kx():
    from voiceagent_b200 import kernels

    return kernels


def table(d, n=4096):
    inv = 1e6 ** (-np.arange(0, d, 2) / d)
    ang = np.arange(n)[:, None] * inv
    return torch.from_numpy(np.concatenate([np.cos(ang), np.sin(ang)], -1).astype(np.float32)).cuda()


def plain(qkv, positions, axis, heads, hkv, d, qw, kw, eps, tab):
    """Rotated q and k heads [T, H + Hkv, D], their tolerance, and v."""
    x = qkv.double().cpu().numpy().reshape(len(qkv), heads + 2 * hkv, d)
    w = np.concatenate([np.tile(qw.double().cpu().numpy(), (heads, 1)), np.tile(kw.double().cpu().numpy(), (hkv, 1))])
    y = x[:, :heads + hkv]
    y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * w
    pos, ax = positions.cpu().numpy(), axis.cpu().numpy()
    tab = tab.double().cpu().numpy()
    j = np.arange(d // 2)
    at = pos[ax].T  # [T, D / 2]
    c, s = tab[at, j][:, None], tab[at, d // 2 + j][:, None]
    a, b = y[..., :d // 2], y[..., d // 2:]
    out = np.concatenate([a * c - b * s, b * c + a * s], -1)
    terms = np.concatenate([np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)], -1)
    return out, 2.0 ** -8 * np.abs(out) + 2.0 ** -19 * terms, x[:, heads + hkv:]


def inputs(tokens, heads, hkv, d, axes, seed=0, pad=0):
    gen = torch.Generator().manual_seed(seed)
    qkv = (2 * torch.randn(tokens, (heads + 2 * hkv) * d + pad, generator=gen)).bfloat16().cuda()
    qkv = qkv[:, :(heads + 2 * hkv) * d]
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=gen)).bfloat16().cuda() for _ in range(2))
    positions = torch.randint(0, 4096, (axes, tokens), generator=gen).cuda()
    return qkv, qw, kw, positions


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 33, 700])
@pytest.mark.parametrize("heads,hkv,d,axes,interleaved", [
    (16, 8, 128, 3, True), (16, 8, 128, 3, False), (7, 1, 128, 2, False), (14, 2, 64, 4, True), (5, 3, 64, 1, False)])
@pytest.mark.parametrize("bits", [16, 4])
def test_against_64_bits(kx, tokens, heads, hkv, d, axes, interleaved, bits):
    qkv, qw, kw, positions = inputs(tokens, heads, hkv, d, axes, tokens, pad=8)
    share = [d // 2 - (axes - 1) * (d // 2 // (axes + 1))] + [d // 2 // (axes + 1)] * (axes - 1)
    axis = kx.mrope_freq_axis(share, interleaved=interleaved)
    tab = table(d)
    bs, blocks = 16, tokens // 16 + 2
    slots = torch.from_numpy(np.random.default_rng(2).permutation(bs * blocks)[:tokens].astype(np.int32)).cuda()
    slots[tokens // 2::5] = -1
    kept = (slots >= 0).cpu().numpy()
    q = torch.empty(tokens, heads, d, dtype=BF16, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    call = dict(num_heads=heads, num_kv_heads=hkv, head_dim=d, q_weight=qw, k_weight=kw, eps=1e-6,
                cos_sin_cache=tab, slot_mapping=slots, error_flag=err)
    kc, vc = (torch.full((blocks, bs, hkv, d), 7.0, dtype=BF16, device="cuda") for _ in range(2))
    kx.qk_norm_mrope_store(qkv, positions, axis, q_out=q, k_cache=kc, v_cache=vc, **call)
    want, tol, v = plain(qkv, positions, axis, heads, hkv, d, qw, kw, 1e-6, tab)
    assert (np.abs(f32(q) - want[:, :heads]) <= tol[:, :heads]).all()
    at = slots[slots >= 0].long()
    k_rows, v_rows = kc.view(-1, hkv, d)[at], vc.view(-1, hkv, d)[at]
    assert (np.abs(f32(k_rows) - want[kept, heads:]) <= tol[kept, heads:]).all()
    np.testing.assert_array_equal(f32(v_rows), v[kept])
    others = torch.ones(blocks * bs, dtype=torch.bool, device="cuda")
    others[at] = False
    assert (kc.view(-1, hkv, d)[others] == 7).all() and (vc.view(-1, hkv, d)[others] == 7).all()
    if bits == 4:  # the same rows, quantised from the bf16 K and V, bit for bit
        cache = filled(1, blocks, bs, hkv, d)
        before = [t.clone() for t in cache]
        q4 = torch.empty_like(q)
        kx.qk_norm_mrope_store(qkv, positions, axis, q_out=q4, k_codes=cache[0], v_codes=cache[1],
                               kv_params=cache[2], **call)
        assert torch.equal(q, q4)
        kx.store_kvcache4(k_rows, v_rows, *before, slots[slots >= 0].contiguous())
        assert all(torch.equal(a, b) for a, b in zip(cache, before))
        code, scale, zero = plain_quantise(f32(k_rows))
        held = before[2].view(-1, hkv, 4)[at]
        np.testing.assert_array_equal(f32(held[..., 0]), scale)
        np.testing.assert_array_equal(f32(held[..., 1]), zero)
    assert err.item() == 0


@pytest.mark.gpu
def test_one_axis_is_the_plain_rotation(kx):
    """Equal position rows give qk_norm_rope_store's rotation (which rounds three times)."""
    qkv, qw, kw, positions = inputs(70, 16, 8, 128, 1)
    positions = positions.expand(3, -1).contiguous()
    axis = kx.mrope_freq_axis([24, 20, 20], interleaved=True)
    tab = table(128)
    q, q1 = (torch.empty(70, 16, 128, dtype=BF16, device="cuda") for _ in range(2))
    call = dict(num_heads=16, num_kv_heads=8, head_dim=128, q_weight=qw, k_weight=kw, eps=1e-6, cos_sin_cache=tab)
    kx.qk_norm_mrope_store(qkv, positions, axis, q_out=q, **call)
    kx.qk_norm_rope_store(qkv, positions[0].contiguous(), q_out=q1, **call)
    size = f32(qkv).reshape(70, 32, 128)[:, :16]
    norm = np.abs(size / np.sqrt((size ** 2).mean(-1, keepdims=True)) * f32(qw))
    pair = norm + np.roll(norm, 64, -1)  # two roundings of each partner, one of each result
    assert (np.abs(f32(q) - f32(q1)) <= 2.0 ** -7 * pair * 1.02 + 2 * 2.0 ** -8 * np.abs(f32(q1))).all()


@pytest.mark.gpu
def test_bad_positions_axes_and_slots_are_flagged(kx):
    qkv, qw, kw, positions = inputs(4, 2, 1, 64, 2)
    tab = table(64, 100)
    positions %= 100
    axis = kx.mrope_freq_axis([16, 16], interleaved=False)
    kc, vc = (torch.zeros(2, 16, 1, 64, dtype=BF16, device="cuda") for _ in range(2))
    call = dict(num_heads=2, num_kv_heads=1, head_dim=64, q_weight=qw, k_weight=kw, eps=1e-6,
                cos_sin_cache=tab, q_out=torch.empty(4, 2, 64, dtype=BF16, device="cuda"), k_cache=kc, v_cache=vc)
    ok = torch.arange(4, dtype=torch.int32, device="cuda")

    def flag(p, ax, slots):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        kx.qk_norm_mrope_store(qkv, p, ax, slot_mapping=slots, error_flag=err, **call)
        return err.item()

    assert flag(positions, axis, ok) == 0
    far = positions.clone()
    far[1, 2] = 100
    assert flag(far, axis, ok) == 4
    far[1, 2] = -1
    assert flag(far, axis, ok) == 4
    assert flag(positions, axis + 1, ok) == 4
    kc.zero_()
    assert flag(positions, axis, torch.tensor([32, -5, -1, -1], dtype=torch.int32, device="cuda")) == 1
    assert not kc.any()


def test_c_entry_refuses(kx):
    from voiceagent_b200._lib import lib
    from tests.test_kv4 import _kv4_struct

    p = ctypes.c_void_p(256)
    err = lambda: lib.b200asr_last_error().decode()  # noqa: E731

    def call(d=128, stride=4096, axes=3, slots=p, kc=p, vc=p, n=1000, c4=None, tokens=5):
        return lib.b200asr_qk_norm_mrope_store(p, stride, p, 5, axes, p, tokens, 16, 8, d, p, p, 1e-6, p, 100, p,
                                               2048, slots, kc, vc, n, c4, None, None)

    assert call(d=96) == 1 and "head_dim" in err()
    assert call(stride=4100) == 1 and "aligned" in err()
    assert call(axes=0) == 1 and "sizes" in err()
    assert call(kc=None) == 1 and "cache" in err()
    assert call(c4=ctypes.byref(_kv4_struct())) == 1 and "cache" in err()
    assert call(kc=None, vc=None, c4=ctypes.byref(_kv4_struct(num_kv_heads=4))) == 1 and "cache" in err()
    assert call(tokens=0) == 0


def test_freq_axis(kx):
    assert kx.mrope_freq_axis([3, 2], interleaved=False, device="cpu").tolist() == [0, 0, 0, 1, 1]
    got = kx.mrope_freq_axis([24, 20, 20], interleaved=True, device="cpu").tolist()
    assert got[:6] == [0, 1, 2, 0, 1, 2] and [got.count(a) for a in range(3)] == [24, 20, 20] and got[60:] == [0] * 4
    with pytest.raises(ValueError, match="reach past"):
        kx.mrope_freq_axis([0, 20, 2], interleaved=True, device="cpu")
    with pytest.raises(ValueError, match="positions"):
        x = torch.zeros(2, 256, dtype=BF16)
        kx.qk_norm_mrope_store(x, torch.zeros(2, dtype=torch.int64), torch.zeros(32, dtype=torch.int32), num_heads=2,
                               num_kv_heads=1, head_dim=64, q_weight=x[0, :64], k_weight=x[0, :64], eps=1e-6,
                               cos_sin_cache=torch.zeros(4, 64), q_out=torch.zeros(2, 2, 64, dtype=BF16))
