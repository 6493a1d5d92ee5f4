"""States of page tables as a server's steps leave them."""
import random

import torch


def state(rng, B, n, P, ps, shared=0):
    """Random rows over a pool of ``P`` pages, some of them free; → table, held, free, span."""
    pages = list(range(P))
    rng.shuffle(pages)
    common, pages = pages[:shared], pages[shared:]
    table, held = [], []
    for _ in range(B):
        h = rng.randint(0, min(n - shared, len(pages)))
        own, pages = pages[:h], pages[h:]
        table.append(common + own + [-1] * (n - shared - h))
        held.append(shared + h)
    head = rng.randint(0, 3 * P)
    free = [-1] * P
    for i, page in enumerate(pages):
        free[(head + i) % P] = page
    return (torch.tensor(table, dtype=torch.int32).view(B, n), torch.tensor(held, dtype=torch.int32), torch.tensor(free, dtype=torch.int32),
            torch.tensor([head, head + len(pages)]))


def step(rng, B, n, ps, held, shared, new, mode):
    """Positions, lens and lengths of a step: all rows go on (``tokens``), or some end, begin or shrink (``turnover``)."""
    positions, lens, lengths = [], [], []
    for b in range(B):
        end = rng.randint(max(0, (int(held[b]) - 1) * ps), n * ps + (1 if rng.random() < 0.05 else 0))
        m = rng.randint(0, new)
        first = max(end - m, shared * ps) if rng.random() < 0.9 else -1
        positions.append(first)
        lens.append(m)
        lengths.append(rng.choice([0, -1, first + m if first >= 0 else -1, rng.randint(1, n * ps)]))
    as_long = lambda v: torch.tensor(v, dtype=torch.long)  # noqa: E731
    return as_long(positions), as_long(lens), as_long(lengths) if mode == "turnover" else None


CASES = [(1, 1, 1, 16, 0, 1), (1, 3, 5, 16, 1, 2), (4, 6, 20, 16, 0, 1), (7, 9, 40, 48, 2, 30), (33, 5, 100, 32, 0, 5), (70, 12, 500, 16, 3, 1),
         (600, 4, 2000, 16, 1, 3), (3, 700, 1500, 16, 5, 40), (2, 40, 64, 128, 0, 1000)]     # rows, columns, pages, page size, shared, new


def seeded(seed):
    return random.Random(seed)
