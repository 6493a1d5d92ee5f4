"""Page tables and slots from the lengths of requests (``ops.page_tables``) against their definition, and what they refuse."""
import pytest
import torch

from page_tables_cases import CASES, seeded, state, step
from paged_int4_cases import assign

from neuronx_distributed_b200 import ops


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("mode", ["tokens", "turnover"])
@pytest.mark.parametrize("trim", [False, True])
def test_assign(case, mode, trim):
    B, n, P, ps, shared, new = case
    rng = seeded(B + n)
    for in_place in (False, True):
        table, held, free, span = state(rng, B, n, P, ps, shared)
        for _ in range(3):
            positions, lens, lengths = step(rng, B, n, ps, held, shared, new, mode)
            want = assign(table, held, free, span, positions, new, ps, lens, lengths, shared, trim)
            before = [t.clone() for t in (table, held, free, span)]
            short = torch.zeros(1, dtype=torch.int32)
            got = ops.page_tables.assign(table, held, free, span, positions, new, ps, lens=lens, lengths=lengths, shared=shared, trim=trim, short=short,
                                         in_place=in_place)
            assert [t.tolist() for t in got] == list(want[:5]) and bool(short) == want[5]
            assert in_place == all(a is b for a, b in zip(got, (table, held, free, span)))
            if not in_place:
                assert all(torch.equal(a, b) for a, b in zip(before, (table, held, free, span)))
            table, held, free, span = got[:4]


def test_pages_stay_whole():
    """Over many steps no page gets lost or belongs to two."""
    rng = seeded(5)
    B, n, P, ps, shared = 9, 8, 50, 16, 1
    table, held, free, span = state(rng, B, n, P, ps, shared)
    common = int(table[0, 0])
    for i in range(40):
        positions, lens, lengths = step(rng, B, n, ps, held, shared, 4, "turnover" if i % 3 == 0 else "tokens")
        table, held, free, span, _ = ops.page_tables.assign(table, held, free, span, positions, 4, ps, lens=lens, lengths=lengths, shared=shared, trim=i % 2 == 0)
        mine = [int(p) for b in range(B) for p in table[b, shared:held[b]]]
        left = [int(free[int(x) % P]) for x in range(int(span[0]), int(span[1]))]
        assert sorted(mine + left) == [p for p in range(P) if p != common]


def test_all_rows_behind_one_that_finds_too_few_take_none():
    table = torch.full((3, 4), -1, dtype=torch.int32)
    held, free, span = torch.zeros(3, dtype=torch.int32), torch.arange(4, dtype=torch.int32), torch.tensor([0, 4])
    short = torch.zeros(1, dtype=torch.int32)
    got = ops.page_tables.assign(table, held, free, span, torch.tensor([0, 0, 0]), 0, 16, lengths=torch.tensor([32, 64, 16]), short=short)
    assert got.held.tolist() == [2, 0, 0] and got.span.tolist() == [2, 4] and got.slots.shape == (3, 0) and int(short) == 1


def refusals(device):
    z = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
    good = dict(page_table=z(2, 3), held=z(2), free=z(4), span=z(2, dtype=torch.long), positions=z(2, dtype=torch.long), new=1, page_size=16)
    for name, value in [("page_table", z(2, 3, dtype=torch.long)), ("page_table", z(6)), ("page_table", z(3, 2).t()), ("held", z(3)),
                        ("held", z(2, dtype=torch.long)), ("free", z(0)), ("free", z(4, dtype=torch.long)), ("free", z(8)[::2]), ("span", z(2)),
                        ("span", z(3, dtype=torch.long)), ("positions", z(3, dtype=torch.long)), ("lens", z(1, dtype=torch.long)),
                        ("lengths", z(2, 2, dtype=torch.long)), ("new", -1), ("new", 1 << 31), ("page_size", 0), ("page_size", 1 << 30), ("shared", 4), ("shared", -1),
                        ("short", z(1, dtype=torch.long)), ("short", z(2))]:
        with pytest.raises(ValueError):
            ops.page_tables.assign(**{**good, name: value})
    ops.page_tables.assign(**good)


def test_refusals():
    refusals("cpu")
    with pytest.raises(ValueError):
        one_row_for_all("cpu")


def one_row_for_all(device):
    """Rows that are one another's memory are not changed in place."""
    z = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
    state = z(1, 3).expand(2, 3), z(2), z(4), z(2, dtype=torch.long), z(2, dtype=torch.long)
    ops.page_tables.assign(*state, 1, 16)
    ops.page_tables.assign(*state, 1, 16, in_place=True)


def test_no_rows():
    got = ops.page_tables.assign(torch.zeros(0, 3, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), torch.arange(4, dtype=torch.int32), torch.tensor([1, 3]),
                                 torch.zeros(0, dtype=torch.long), 2, 16)
    assert got.free.tolist() == [0, 1, 2, 3] and got.span.tolist() == [1, 3] and got.slots.shape == (0, 2)
