"""A shared projection with the rows' own low-rank adapters, against 64 bits.

Tolerances, element by element: the output's rounding (2^-8 of its value); for batches beyond
a decode step, whose t = s x A^T is rounded to bf16, 2^-8 of |t| |B|^T; and 2^-15 of the
absolute terms for the 32-bit sums (at most 2048 + 128 additions in tiles of 16 at 2^-23 each)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def kx():
    from voiceagent_b200 import kernels

    return kernels


def inputs(rows, k, n, rank, adapters, seed=0, device="cuda"):
    gen = torch.Generator().manual_seed(seed)
    bf = lambda *s, scale: (torch.randn(*s, generator=gen) * scale).bfloat16().to(device)  # noqa: E731
    return (bf(rows, k, scale=1), bf(n, k, scale=k ** -0.5), bf(adapters, rank, k, scale=k ** -0.5),
            bf(adapters, n, rank, scale=rank ** -0.5), (0.5 + torch.rand(adapters, generator=gen)).to(device))


def plain(x, w, a, b, s, rows):
    """(out, tolerance)."""
    d = lambda t: t.double().cpu().numpy()  # noqa: E731
    x, w, a, b, s = map(d, (x, w, a, b, s))
    base, size = x @ w.T, np.abs(x) @ np.abs(w).T
    part, part_size, t_size = (np.zeros_like(base) for _ in range(3))
    for t, i in enumerate(rows.tolist()):
        if 0 <= i < len(a):
            part[t] = s[i] * (x[t] @ a[i].T) @ b[i].T
            t_size[t] = np.abs(s[i] * (x[t] @ a[i].T)) @ np.abs(b[i]).T
            part_size[t] = s[i] * (np.abs(x[t]) @ np.abs(a[i]).T) @ np.abs(b[i]).T
    out = base + part
    tol = 2.0 ** -8 * np.abs(out) + 2.0 ** -15 * (size + part_size)
    return out, tol + (2.0 ** -8 * t_size if len(x) > 64 or w.shape[0] % 128 or w.shape[1] % 64 else 0)


def check(got, want, what=""):
    out, tol = want
    over = np.abs(got.double().cpu().numpy() - out) - tol
    assert np.isfinite(over).all() and (over <= 0).all(), f"{what}: {over.max():.3e} past the tolerance"


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 13, 33, 64, 65, 200])
@pytest.mark.parametrize("k,n,rank,adapters", [
    (1024, 4096, 16, 8), (2048, 256, 64, 40), (192, 128, 8, 3), (72, 40, 24, 5), (1024, 328, 128, 2), (8, 8, 8, 1)])
def test_against_64_bits(kx, rows, k, n, rank, adapters):
    args = inputs(rows, k, n, rank, adapters, rows)
    ids = torch.from_numpy(np.random.default_rng(rows).integers(-1, adapters, rows).astype(np.int32)).cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = kx.lora_linear(*args, ids, error_flag=err)
    check(got, plain(*args, ids))
    assert err.item() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [40, 333])
def test_no_adapter_one_adapter_and_runs(kx, rows):
    args = inputs(rows, 512, 384, 32, 6, 3)
    for ids in (np.full(rows, -1), np.full(rows, 5), np.sort(np.random.default_rng(0).integers(-1, 6, rows))):
        ids = torch.from_numpy(ids.astype(np.int32)).cuda()
        check(kx.lora_linear(*args, ids), plain(*args, ids))
    none = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    got = kx.lora_linear(*args, none)
    check(got, plain(*args, none))
    if rows <= 64:  # the same kernel with nothing to add
        assert torch.equal(got, kx.linear_small(args[0], args[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [512, 513, 700])
@pytest.mark.parametrize("k,n,rank,adapters", [(1024, 256, 16, 8), (320, 136, 64, 40), (72, 40, 24, 5), (264, 128, 128, 2)])
def test_many_rows_against_64_bits(kx, rows, k, n, rank, adapters):
    """The down product that streams 32 rows of x: runs of rows, and every row another adapter."""
    args = inputs(rows, k, n, rank, adapters, rows + 1)
    rng = np.random.default_rng(rows)
    for ids in (np.sort(rng.integers(-1, adapters, rows)), rng.integers(-1, adapters, rows), np.full(rows, -1)):
        ids = torch.from_numpy(ids.astype(np.int32)).cuda()
        wide = torch.full((rows, args[0].shape[1] + 8), float("nan"), dtype=BF16, device="cuda")
        wide[:, :args[0].shape[1]] = args[0]
        check(kx.lora_linear(wide[:, :args[0].shape[1]], *args[1:], ids), plain(*args, ids))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [9, 90])
def test_strided_rows_given_out_and_nan_of_other_adapters(kx, rows):
    x, w, a, b, s = inputs(rows, 256, 128, 16, 4, 7)
    wide = torch.randn(rows, 3 * 256, device="cuda").bfloat16()
    x = wide[:, 256:512]
    ids = torch.arange(rows, device="cuda").remainder(3).int()  # adapter 3 is not used
    a[3], b[3], s[3] = float("nan"), float("nan"), float("nan")
    keep = torch.full((rows, 3 * 128), 5.0, dtype=BF16, device="cuda")
    out = keep[:, 128:256]
    assert kx.lora_linear(x, w, a, b, s, ids, out=out).data_ptr() == out.data_ptr()
    check(out, plain(x, w, a, b, s, ids))
    assert (keep[:, :128] == 5).all() and (keep[:, 256:] == 5).all()
    a[0, 0, 0] = float("inf")  # reaches the rows of adapter 0 alone
    got = kx.lora_linear(x, w, a, b, s, ids)
    assert not got[ids == 0].isfinite().any() and torch.equal(got[ids != 0], out[ids != 0])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [40, 300, 600])
def test_values_that_are_not_finite_in_b_reach_their_adapter_alone(kx, rows):
    """Rows of several adapters share a tile of the product: 0 * inf must not join them."""
    x, w, a, b, s = inputs(rows, 128, 256, 16, 4, 9)
    ids = torch.arange(rows, device="cuda").remainder(5).sub(1).int()
    want = plain(x, w, a, b, s, ids)
    b[2, 7, 3], b[2, 200, 0] = float("inf"), float("nan")
    b[3, 40:80] = float("nan")
    got = kx.lora_linear(x, w, a, b, s, ids)
    wild = torch.zeros(rows, 256, dtype=torch.bool, device="cuda")
    wild[ids == 2, 7] = wild[ids == 2, 200] = True
    wild[(ids == 3)[:, None] & (torch.arange(256, device="cuda") // 40 == 1)] = True
    assert not got[wild].isfinite().any()
    got[wild] = torch.from_numpy(want[0]).cuda()[wild].to(BF16)
    check(got, want)
    w[5, 9] = float("nan")  # the shared weights reach every row
    x[1] = float("inf")     # and a row of x its own
    got = kx.lora_linear(x, w, a, b, s, ids)
    wild[:, 5] = wild[1] = True
    assert not got[wild].isfinite().any()
    got[wild] = torch.from_numpy(want[0]).cuda()[wild].to(BF16)
    check(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 70])
def test_bad_indices_are_flagged_and_count_as_none(kx, rows):
    args = inputs(rows, 128, 128, 8, 2)
    ids = torch.zeros(rows, dtype=torch.int32, device="cuda")
    ids[1], ids[3] = 2, -7
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = kx.lora_linear(*args, ids, error_flag=err)
    assert err.item() == 32
    ids[ids != 0] = -1
    assert torch.equal(got, kx.lora_linear(*args, ids))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [16, 130])
def test_under_capture(kx, rows):
    args = inputs(rows, 512, 256, 16, 4)
    ids = torch.arange(rows, device="cuda").remainder(5).sub(1).int()
    out = torch.empty(rows, 256, dtype=BF16, device="cuda")
    want = kx.lora_linear(*args, ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kx.lora_linear(*args, ids, out=out)
    graph.replay()
    assert torch.equal(out, want)
    ids.copy_(ids.flip(0))  # the adapters are read at replay
    graph.replay()
    assert torch.equal(out, kx.lora_linear(*args, ids))


def test_refusals(kx):
    x, w, a, b, s = inputs(3, 64, 32, 8, 2, device="cpu")
    ids = torch.zeros(3, dtype=torch.int32)
    for args, says in (((x, w, a, b, s, ids), "CUDA"), ((x, w, a, b, s, ids.long()), "row_adapter"),
                       ((x, w, a, b[:, :16].contiguous(), s, ids), "lora_b"), ((x, w, a, b, s[:1], ids), "scales"),
                       ((x, w[:, :32], a, b, s, ids), "weight"), ((x, w, a[..., :32], b, s, ids), "lora_a"),
                       ((x, w, a[:, :4].contiguous(), b[..., :4].contiguous(), s, ids), "rank"),
                       ((x.float(), w, a, b, s, ids), "x bf16")):
        with pytest.raises(ValueError, match=says):
            kx.lora_linear(*args)


def test_c_entries_refuse():
    from voiceagent_b200._lib import lib

    p = ctypes.c_void_p(256)
    err = lambda: lib.b200asr_last_error().decode()  # noqa: E731
    down = lambda k=64, r=8, st=64, rows=3: lib.b200asr_lora_down(p, st, rows, k, p, 2, r, p, p, p, None, None)  # noqa: E731
    assert down(k=60) == 1 and "multiple of 8" in err()
    assert down(r=12) == 1 and "rank" in err()
    assert down(r=136) == 1 and "rank" in err()
    assert down(st=60) == 1 and "aligned" in err()
    assert down(rows=0) == 0
    big = lambda n=64, y=p, st=64, ws=1 << 20: lib.b200asr_lora_rows(  # noqa: E731
        p, 64, 3, 64, p, n, p, p, 2, 8, p, p, y, st, p, ws, None, None)
    assert big(n=60) == 1 and "multiple" in err()
    assert big(y=None) == 1 and "null" in err()
    assert big(st=63) == 1 and "aligned" in err()
    assert big(ws=lib.b200asr_lora_rows_workspace_size(3, 8) - 1) == 4 and "workspace" in err()
    up = lambda m=3, n=128, r=8: lib.b200asr_linear_small_lora(p, 64, m, 64, p, n, p, p, 2, r, p, p, 128, None, None)  # noqa: E731
    assert up(m=65) == 1 and "64" in err()
    assert up(n=120) == 1 and "multiple" in err()
    assert up(r=4) == 1 and "rank" in err()
