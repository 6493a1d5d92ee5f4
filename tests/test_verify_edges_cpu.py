"""Drafted tokens whose rows hold negative numbers and NaN, which count as 0 on both sides."""
import pytest
import torch

from neuronx_distributed_b200 import ops


def odd_rows(V, dtype):
    """→ arguments, and what the definition says of each row."""
    nan = float("nan")
    p, q = torch.zeros(6, 2, V), torch.zeros(6, 1, V)
    tokens, accept, sample = torch.zeros(6, 1, dtype=torch.long), torch.full((6, 1), 0.5), torch.full((6,), 0.5)
    last = V - 1
    # a token that the target never gives, drafted with a negative number: 0.5 * 0 < 0 does not hold; the next from p, at its only number
    p[0, 0, 3], q[0, 0, 0] = 0.5, -1.0
    # a NaN of the draft at the drafted token: 0 < 0.25, taken; behind it p's only number
    p[1, 0, 0], q[1, 0, 0], p[1, 1, last] = 0.25, nan, 1.0
    # refused at 0 (0.5 * 1 < 0.25 does not hold); of what is left of p - q, numbers with a NaN or a negative one of q weigh p itself: 0.125 at 2, 0.5 at
    # the end, whose running sum passes half of 0.625
    p[2, 0, 0], q[2, 0, 0], p[2, 0, 2], q[2, 0, 2], p[2, 0, last], q[2, 0, last] = 0.25, 1.0, 0.125, nan, 0.5, -8.0
    # negative on both sides: nothing, not their difference
    p[3, 0, 0], q[3, 0, 0], p[3, 0, 1], q[3, 0, 1], p[3, 0, 4] = 0.25, 1.0, -0.5, -2.0, 0.125
    # a negative number of the target at the drafted token: 0 < 0 does not hold
    p[4, 0, 0], q[4, 0, 0], p[4, 0, 5] = -0.5, -2.0, 0.125
    # a NaN of the target there, and nothing left of p - q: from p
    p[5, 0, 0], q[5, 0, 0], p[5, 0, 6], q[5, 0, 6] = nan, nan, 0.125, 0.25
    want = torch.tensor([[3, -1], [0, last], [last, -1], [4, -1], [5, -1], [6, -1]]), torch.tensor([0, 1, 0, 0, 0, 0])
    return [tokens, q.to(dtype), p.to(dtype), accept, sample], want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [9, 1000])
def test_negative_numbers_and_nan_count_as_zero(dtype, V):
    args, want = odd_rows(V, dtype)
    got = ops.select.verify_drafts(*args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), got
