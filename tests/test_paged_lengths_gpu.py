"""Paged attention over every way in which pieces are cut, all rows against the definition in 64 bits, so that a lost tile of keys shows."""
import math

import pytest
import torch

from paged_cases import bound, make

BF16, FP16 = torch.bfloat16, torch.float16


def definition(d, leave_out=None):
    """``paged_oracle.attention`` with all rows of a sequence at once: → output, and the same average of the values' magnitudes.  ``leave_out (row, key)``:
    a tile of 64 keys from there on is not seen by that row."""
    q, kc, vc = d["q"], d["k_cache"], d["v_cache"]
    B, W, H, D = q.shape
    ps, Hkv = kc.shape[1:3]
    out = torch.zeros(B, W, H, D, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    for b in range(B):
        first, m = int(d["positions"][b]), W if d["lens"] is None else int(d["lens"][b])
        if first < 0 or m <= 0:
            continue
        n = first + m
        pages = d["table"][b].long().clone()
        if d["shared_pages"] is not None:
            pages[:len(d["shared_pages"])] = d["shared_pages"].long()
        j = torch.arange(n, device=q.device)
        k, v = (c[pages[j // ps], j % ps].double().repeat_interleave(H // Hkv, 1) for c in (kc, vc))          # [n, H, D]
        s = torch.einsum("whd,nhd->hwn", q[b, :m].double(), k) / math.sqrt(D)
        unseen = j > first + torch.arange(m, device=q.device)[:, None]
        if leave_out is not None and leave_out[0] == b:
            unseen |= (j >= leave_out[1]) & (j < leave_out[1] + 64)
        p = torch.softmax(s.masked_fill(unseen, -math.inf), -1)
        out[b, :m] = torch.einsum("hwn,nhd->whd", p, v)
        size[b, :m] = torch.einsum("hwn,nhd->whd", p, v.abs())
    return out, size


def case(device, dtype, W, H, Hkv, shared, most, B=60, D=64):
    g = torch.Generator().manual_seed(1000 * W + most)
    positions = (96 + torch.randint(0, most, (B,), generator=g)).tolist()
    lens = torch.randint(1, W + 1, (B,), generator=g).tolist()
    return make(50 + W, device, dtype, B, W, H, Hkv, D, 32, positions, lens, shared)


def wrong(d, got, want, size):
    return (got.double() - want).abs() > bound(d["q"].dtype, want, size)


CASES = [(5, 8, 1), (3, 16, 2), (20, 8, 1), (40, 8, 1), (1, 16, 2), (1, 2, 2)]


@pytest.mark.parametrize("W, H, Hkv", [(5, 8, 1), (3, 16, 2)])
def test_a_lost_tile_would_show(W, H, Hkv):
    """On the CPU, without a kernel: the definition without one tile of 64 keys is outside the bound, for the shortest and for the longest sequences."""
    for most in (130, 4000):
        d = case("cpu", FP16, W, H, Hkv, 0, most, B=4)
        want, size = definition(d)
        assert not bool(wrong(d, want.to(FP16), want, size).any())
        for b in range(4):
            for key in (0, 64 * (int(d["positions"][b]) // 128)):
                less, _ = definition(d, (b, key))
                assert bool(wrong(d, less.to(FP16), want, size)[b].any()), (most, b, key)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, D", [(FP16, 64), (BF16, 128)])
@pytest.mark.parametrize("W, H, Hkv", CASES)
@pytest.mark.parametrize("shared", [0, 3])
def test_windows_of_many_lengths(dtype, D, W, H, Hkv, shared):
    from test_paged_gpu import attend

    for most in (130, 700, 4000):
        d = case("cuda", dtype, W, H, Hkv, shared, most, D=D)
        want, size = definition(d)
        off = wrong(d, attend(d), want, size)
        assert not bool(off.any()), (most, off.nonzero()[:4].tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, D", [(FP16, 64), (BF16, 128), (BF16, 64)])
@pytest.mark.parametrize("B, W, H, Hkv, shared, most", [(5, 1, 8, 8, 0, 700), (5, 1, 8, 1, 0, 3000), (3, 4, 8, 2, 0, 500), (7, 2, 16, 2, 0, 1500),
                                                        (2, 2, 8, 2, 3, 300), (1, 1, 8, 1, 33, 200)])
def test_weights_of_few_rows_are_not_rounded(dtype, D, B, W, H, Hkv, shared, most):
    """Up to 16 query rows of a sequence and key/value head (and of the batch, over shared pages): the bound of `bound` without the rounding of the weights
    to the type; what is left of it, a half step of a half step (2^-17 in bf16; 2^-25 of a weight of 1 in fp16, of up to 4000 of them), lies within the
    2^-13 of products and exponentials with which it is added."""
    from test_paged_gpu import attend

    d = case("cuda", dtype, W, H, Hkv, shared, most, B=B, D=D)
    want, size = definition(d)
    u = torch.finfo(dtype).eps / 2
    off = (attend(d).double() - want).abs() - (u * want.abs() + (2.0 ** -13 + 4000 * 2.0 ** -25) * size + 1e-7)
    assert bool((off <= 0).all()), (float(off.max()), off.argmax())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_dealt_out_many(dtype):
    """More sequences than threads that look for places, in tables that few-row launches are dealt out for."""
    from test_paged_gpu import attend, widen

    B = 1100
    d = make(60, "cuda", dtype, B, 1, 2, 1, 64, 16, [(37 * b) % 190 - 1 for b in range(B)])
    want, size = definition(d)
    for _ in range(2):
        off = wrong(d, attend(d), want, size)
        assert not bool(off.any()), off.nonzero()[:4].tolist()
        d = widen(d, 20000)


@pytest.mark.gpu
@pytest.mark.parametrize("W", [1, 3, 24, 300])
def test_tables_without_a_column(W):
    """Nobody sees a key: zeros, and nothing is written."""
    from neuronx_distributed_b200 import ops

    d = make(61, "cuda", BF16, 3, W, 8, 2, 128, 16, [5, 0, -1])
    got = ops.paged.attention(d["q"], d["k_cache"], d["v_cache"], d["table"][:, :0], d["positions"])
    assert got.shape == d["q"].shape and not bool(got.any())
    cos, sin = ops.rope.rope_tables(400, 128, device="cuda")
    before, lost = d["k_cache"].clone(), torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.paged.rope_append(d["q"], d["k"], d["v"], d["positions"], cos, sin, d["k_cache"], d["v_cache"], d["table"][:, :0], lost=lost)
    assert torch.equal(before.nan_to_num(), d["k_cache"].nan_to_num()) and int(lost) == 1
