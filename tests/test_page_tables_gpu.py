"""The kernel of page tables (``csrc/page_tables.cu``) against the definition."""
import pytest
import torch

from page_tables_cases import CASES, seeded, state, step
from paged_int4_cases import assign
from test_page_tables_cpu import one_row_for_all, refusals

from neuronx_distributed_b200 import ops

pytestmark = pytest.mark.gpu


def cuda(*t):
    return [None if x is None else x.cuda() for x in t]


@pytest.mark.parametrize("case", CASES + [(2500, 9, 9000, 16, 1, 2), (1, 5000, 8000, 16, 0, 3), (3, 1301, 1500, 16, 5, 40), (37, 257, 4000, 16, 3, 9), (130, 64, 3000, 16, 0, 20)])
@pytest.mark.parametrize("mode", ["tokens", "turnover"])
@pytest.mark.parametrize("in_place", [False, True])
def test_assign(case, mode, in_place):
    B, n, P, ps, shared, new = case
    rng = seeded(B + n + in_place)
    for trim in (False, True):
        table, held, free, span = state(rng, B, n, P, ps, shared)
        dev = cuda(table, held, free, span)
        for _ in range(3):
            positions, lens, lengths = step(rng, B, n, ps, held, shared, new, mode)
            want = assign(table, held, free, span, positions, new, ps, lens, lengths, shared, trim)
            before = [t.clone() for t in dev]
            short = torch.zeros(1, dtype=torch.int32, device="cuda")
            p, l, g = cuda(positions, lens, lengths)
            got = ops.page_tables.assign(*dev, p, new, ps, lens=l, lengths=g, shared=shared, trim=trim, short=short, in_place=in_place)
            for name, t, w in zip(got._fields, got, want):
                assert t.tolist() == w, name
            assert bool(short) == want[5]
            if in_place:
                assert all(a is b for a, b in zip(got, dev))
            else:
                assert all(torch.equal(a, b) for a, b in zip(before, dev))
            dev = list(got[:4])
            table, held, free, span = (t.cpu() for t in dev)


def test_tables_in_wider_rows_and_other_integers():
    rng = seeded(2)
    B, n, P, ps = 5, 6, 40, 16
    table, held, free, span = state(rng, B, n, P, ps)
    positions, lens, _ = step(rng, B, n, ps, held, 0, 3, "tokens")
    want = assign(table, held, free, span, positions, 3, ps, lens)
    for in_place in (False, True):
        wide = torch.full((B, n + 3), 99, dtype=torch.int32, device="cuda")
        wide[:, :n] = table.cuda()
        got = ops.page_tables.assign(wide[:, :n], *cuda(held, free, span), positions.int().cuda(), 3, ps, lens=lens.int().cuda(), in_place=in_place)
        assert [t.tolist() for t in got] == list(want[:5]) and bool((wide[:, n:] == 99).all())


def test_captured_on_another_stream():
    """A captured call takes pages whenever it is replayed, for the positions that stand there then."""
    B, n, P, ps = 4, 5, 20, 16
    table, held, free, span = cuda(torch.full((B, n), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32), torch.randperm(P).int(), torch.tensor([0, P]))
    positions = torch.zeros(B, dtype=torch.long, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.page_tables.assign(table, held, free, span, positions, 1, ps, lens=torch.zeros_like(positions), in_place=True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            slots = ops.page_tables.assign(table, held, free, span, positions, 1, ps, in_place=True).slots
        state = [t.cpu() for t in (table, held, free, span)]
        for at in ([0, 15, -1, 3], [16, 16, 0, 4], [32, 17, 16, 5], [70, 18, 17, 40]):
            positions.copy_(torch.tensor(at))
            graph.replay()
            *state, want, _ = assign(*state, torch.tensor(at), 1, ps)
            state = [torch.tensor(state[0], dtype=torch.int32), torch.tensor(state[1], dtype=torch.int32), torch.tensor(state[2], dtype=torch.int32), torch.tensor(state[3])]
            assert slots.tolist() == want
            assert all(torch.equal(a.cpu(), b) for a, b in zip((table, held, free, span), state))
    torch.cuda.current_stream().wait_stream(side)


def test_refusals():
    refusals("cuda")
    with pytest.raises(ValueError):
        one_row_for_all("cuda")
    with pytest.raises(ValueError):
        ops.page_tables.assign(torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32, device="cuda"),
                               torch.zeros(2, dtype=torch.long, device="cuda"), torch.zeros(2, dtype=torch.long, device="cuda"), 1, 16)


@pytest.mark.parametrize("in_place", [False, True])
def test_no_rows(in_place):
    got = ops.page_tables.assign(*cuda(torch.zeros(0, 3, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), torch.arange(4, dtype=torch.int32), torch.tensor([1, 3]),
                                       torch.zeros(0, dtype=torch.long)), 2, 16, in_place=in_place)
    assert got.free.tolist() == [0, 1, 2, 3] and got.span.tolist() == [1, 3] and got.slots.shape == (0, 2)
