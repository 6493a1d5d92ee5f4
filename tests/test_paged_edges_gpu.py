"""Calls of the paged operators that their documentation allows and ordinary programs seldom make."""
import pytest
import torch

from paged_cases import make
from test_paged_gpu import attend, check
from test_verify_edges_cpu import odd_rows

from neuronx_distributed_b200 import ops

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype, D", [(BF16, 128), (FP16, 64)])
@pytest.mark.parametrize("B, W, H, Hkv", [(1, 1, 8, 8), (4, 2, 4, 2), (3, 5, 2, 2), (5, 1, 16, 2), (6, 6, 8, 2), (40, 2, 8, 1), (9, 14, 8, 1)])
@pytest.mark.parametrize("last", [-1, 0, 37, 94, 95])
def test_shared_pages_that_nobody_sees_to_the_end(dtype, D, B, W, H, Hkv, last):
    """Every row stands inside the shared pages (or is idle): what lies there behind the last key that any of them sees may be anything."""
    positions = [max(-1, last - W + 1 - 3 * b) for b in range(B)]
    lens = [W if b % 3 else max(1, W - 1) for b in range(B)]
    lens[0] = min(W, last + 1)
    d = make(40, "cuda", dtype, B, W, H, Hkv, D, 16, positions, lens, 6)
    end = max([p + n for p, n in zip(positions, lens) if p >= 0] + [0])
    results = []
    for x in (float("nan"), float("inf"), 0.0):
        for i in range(end, 96):
            for t in ("k_cache", "v_cache"):
                d[t][d["shared_pages"][i // 16].long(), i % 16] = x
        results.append(attend(d))
    check(d, results[0])
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])


@pytest.mark.parametrize("dtype", [torch.float32, BF16, FP16])
@pytest.mark.parametrize("V", [9, 1000, 32016])
def test_verify_counts_negative_numbers_and_nan_as_zero(dtype, V):
    args, want = odd_rows(V, dtype)
    got = ops.select.verify_drafts(*[t.cuda() for t in args])
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_shared_pages_under_very_many_heads():
    """The join of parts has a warp for every row and key/value head: 128 rows of 2048 heads are more than a launch takes; the shared pages are then the
    first of every sequence's own."""
    d = make(41, "cuda", BF16, 1, 128, 2048, 2048, 64, 16, [20], [128], 1, spare=1)
    got = attend(d)
    # the same heads 512 at a time (8 of them against the definition)
    for h in range(0, 2048, 512):
        part = {**d, "q": d["q"][:, :, h:h + 512], "k_cache": d["k_cache"][:, :, h:h + 512], "v_cache": d["v_cache"][:, :, h:h + 512]}
        few = {**d, "q": d["q"][:, :, h:h + 2], "k_cache": d["k_cache"][:, :, h:h + 2], "v_cache": d["v_cache"][:, :, h:h + 2]}
        check(few, got[:, :, h:h + 2])
        check(few, attend(part)[:, :, :2])


@pytest.fixture
def waits():
    """→ a function that sets after how many ns the tile kernel's waits give up; negative: with keys that never come."""
    call = ops._ext.ext().paged_wait_ns
    before = call(2_000_000_000)
    yield call
    call(before)


def live_rows(d):
    w = torch.arange(d["q"].shape[1], device="cuda")
    n = torch.full_like(d["positions"], len(w)) if d["lens"] is None else d["lens"]
    return (w < n[:, None]) & (d["positions"] >= 0)[:, None]


@pytest.mark.parametrize("dtype, D", [(BF16, 128), (FP16, 64)])
@pytest.mark.parametrize("B, W, H, Hkv, shared, most", [
    (3, 300, 8, 2, 0, 500), (2, 100, 8, 2, 0, 5000), (30, 10, 8, 1, 0, 3000), (3, 40, 2, 2, 0, 40), (40, 5, 8, 1, 0, 30), (1, 700, 4, 1, 0, 1),
    (20, 1, 16, 2, 5, 600), (9, 9, 8, 2, 33, 300), (24, 20, 16, 2, 5, 2000), (2, 9, 8, 2, 5, 50),
])
def test_waits_that_run_out(waits, dtype, D, B, W, H, Hkv, shared, most):
    """Keys that never come: every row that counts is NaN, whatever was left of the output and the workspace before; the next call is as ever."""
    g = torch.Generator().manual_seed(W)
    positions = (shared * 16 + torch.randint(0, most, (B,), generator=g)).tolist()
    lens = torch.randint(1, W + 1, (B,), generator=g).tolist()
    if B > 2:
        positions[1] = -1
    lens[0] = W
    d = make(42, "cuda", dtype, B, W, H, Hkv, D, 16, positions, lens, shared)
    want = attend(d)
    torch.cuda.synchronize()
    live = live_rows(d)
    for left in (0.0, 1.0):
        spare = torch.full((want.numel() * 8 + 300 * 256 * (D + 2) * 4,), left, device="cuda")         # what the allocator hands out next
        del spare
        waits(-1_000_000)
        bad = attend(d)
        torch.cuda.synchronize()
        waits(2_000_000_000)
        assert bool(bad[live].isnan().all()) and not bool(bad[~live].any())
        assert torch.equal(attend(d), want)
    check(d, want)
