"""The kernels of a cache in pages (``csrc/paged.cu``, ``csrc/verify.cu``) against their definitions in 64 bits."""
import pytest
import torch

import paged_oracle as oracle
from paged_cases import bound, make

from neuronx_distributed_b200 import ops

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def attend(d, **kw):
    return ops.paged.attention(d["q"], d["k_cache"], d["v_cache"], d["table"], d["positions"], lens=d["lens"], shared_pages=d["shared_pages"], **kw)


def check(d, got, scale=None):
    want, size = oracle.attention(d["q"], d["k_cache"], d["v_cache"], d["table"], d["positions"], scale=scale, lens=d["lens"], shared_pages=d["shared_pages"])
    off = (got.double() - want).abs() - bound(d["q"].dtype, want, size)
    assert bool((off <= 0).all()), (float(off.max()), (off > 0).nonzero()[:4].tolist())


# ------------------------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype, D", [(BF16, 128), (BF16, 64), (FP16, 96), (torch.float32, 16), (torch.float32, 40)])
@pytest.mark.parametrize("B, W, H, Hkv, ps, positions, lens", [
    (1, 1, 4, 4, 16, [0], None),
    (3, 1, 8, 1, 16, [15, 16, 200], None),
    (4, 7, 6, 2, 48, [-1, 41, 48, 0], [7, 7, 0, 3]),
    (2, 130, 4, 2, 128, [0, 100], [130, 64]),
])
@pytest.mark.parametrize("layout", ["rows", "heads", "slice"])
def test_append(dtype, D, B, W, H, Hkv, ps, positions, lens, layout):
    if D * dtype.itemsize % 32:
        pytest.skip("halves of no whole packets")
    d = make(1, "cuda", dtype, B, W, H, Hkv, D, ps, positions, lens, layout=layout)
    cos, sin = ops.rope.rope_tables(300, D, device="cuda")
    want_q, want_k, want_v, written = oracle.append(d["q"], d["k"], d["v"], d["positions"], cos, sin, d["k_cache"], d["v_cache"], d["table"], d["lens"])
    old = d["k_cache"].clone(), d["v_cache"].clone()
    q = ops.paged.rope_append(d["q"], d["k"], d["v"], d["positions"], cos, sin, d["k_cache"], d["v_cache"], d["table"], lens=d["lens"])
    assert q.dtype == dtype and q.transpose(0, 1).is_contiguous()
    # one rounding to the type, and three in 32 bits of numbers below 6
    near = lambda got, want: bool(((got.double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 6 * 3 * 2.0 ** -24).all())
    assert near(q, want_q)
    written = written.cuda()
    for got, want, before in ((d["k_cache"], want_k, old[0]), (d["v_cache"], want_v, old[1])):
        assert near(got[written], want[written])
        assert torch.equal(got[~written].nan_to_num(), before[~written].nan_to_num())


def test_append_takes_sections_and_odd_views():
    """Sections of a projection's output, and views that begin at no packet."""
    B, W, H, Hkv, D = 2, 3, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    cos, sin = ops.rope.rope_tables(64, D, device="cuda")
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    positions = torch.tensor([5, 14], device="cuda")
    flat = torch.randn(W, B, (H + 2 * Hkv) * D + 3, generator=g, device="cuda").to(BF16)
    for qkv in (flat[..., :-3], flat[..., 3:]):
        q, k, v = (s.unflatten(-1, (-1, D)).transpose(0, 1) for s in qkv.split([H * D, Hkv * D, Hkv * D], -1))
        caches = [torch.zeros(4, 16, Hkv, D, dtype=BF16, device="cuda") for _ in range(4)]
        a = ops.paged.rope_append(q, k, v, positions, cos, sin, caches[0], caches[1], table)
        b = ops.paged.rope_append(q.contiguous(), k.contiguous(), v.contiguous(), positions, cos, sin, caches[2], caches[3], table)
        assert torch.equal(a, b) and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])
        odd = torch.zeros(cos.numel() + 1, device="cuda")
        odd[1:] = cos.flatten()
        assert torch.equal(a, ops.paged.rope_append(q, k, v, positions, odd[1:].view_as(cos), sin, caches[2], caches[3], table))


# --------------------------------------------------------------------------------------------------------------- attention
HEADS = [(8, 8), (8, 4), (6, 2), (8, 2), (5, 1), (16, 2), (12, 1), (24, 1)]


@pytest.mark.parametrize("dtype, D", [(BF16, 128), (FP16, 64), (BF16, 64), (FP16, 128)])
@pytest.mark.parametrize("H, Hkv", HEADS)
def test_one_token(dtype, D, H, Hkv):
    d = make(3, "cuda", dtype, 5, 1, H, Hkv, D, 16, [0, 15, 16, 257, 700])
    check(d, attend(d))


@pytest.mark.parametrize("ps", [16, 32, 48, 64, 80, 128, 256])
@pytest.mark.parametrize("positions", [[63], [64], [0, -1, 1, 1000], [-1, -1]])
def test_pages(ps, positions):
    d = make(4, "cuda", BF16, len(positions), 1, 8, 2, 128, ps, positions)
    check(d, attend(d))


@pytest.mark.parametrize("W", [2, 3, 4, 5, 8, 17, 33, 64, 129, 300])
@pytest.mark.parametrize("H, Hkv", [(8, 8), (8, 2), (16, 2)])
def test_windows(W, H, Hkv):
    d = make(5, "cuda", BF16, 3, W, H, Hkv, 128, 32, [0, 31, 333], [W, max(1, W - 1), W // 2])
    check(d, attend(d))


@pytest.mark.parametrize("W, H, Hkv", [(5, 8, 1), (3, 16, 2), (20, 8, 1), (40, 8, 1)])
@pytest.mark.parametrize("shared", [0, 3])
def test_windows_of_many_lengths(W, H, Hkv, shared):
    """Every number of key tiles in a block's pieces, odd ones before even ones and ones of a single tile among them."""
    g = torch.Generator().manual_seed(W)
    for most in (130, 700, 4000):
        positions = (96 + torch.randint(0, most, (60,), generator=g)).tolist()
        lens = torch.randint(1, W + 1, (60,), generator=g).tolist()
        d = make(6, "cuda", BF16, 60, W, H, Hkv, 64, 32, positions, lens, shared)
        got = attend(d)
        one = [ops.paged.attention(d["q"][b:b + 1], d["k_cache"], d["v_cache"], d["table"][b:b + 1], d["positions"][b:b + 1], lens=d["lens"][b:b + 1])
               for b in range(60)]
        # other cuts of the same sums: weights rounded relative to other maxima, results rounded once each
        size = oracle_size(d)
        assert bool(((got - torch.cat(one)).double().abs() <= 2 * bound(BF16, got.double(), size)).all())
        assert torch.equal(got, attend(d))


@pytest.mark.parametrize("B, W, H, Hkv, shared", [(30, 5, 8, 1, 0), (30, 10, 8, 1, 0), (30, 10, 8, 1, 3), (24, 20, 16, 2, 0), (24, 40, 16, 2, 0), (2, 300, 8, 2, 0)])
@pytest.mark.parametrize("D", [64, 128])
def test_short_pairs_and_long_ones(B, W, H, Hkv, shared, D):
    """Pairs that one block takes whole beside pairs that are cut, over all sizes of row tiles; rows that do not count and sequences without tokens."""
    g = torch.Generator().manual_seed(W)
    for most in (40, 500, 3000):
        positions = (48 + torch.randint(0, most, (B,), generator=g)).tolist()
        lens = torch.randint(0, W + 1, (B,), generator=g).tolist()
        lens[0], positions[-1], lens[-1] = W, 2200, W
        d = make(7, "cuda", BF16, B, W, H, Hkv, D, 16, positions, lens, shared)
        check(d, attend(d))


def oracle_size(d):
    """A bound of the weighted average of the values' magnitudes, without its softmax: the largest that a row sees."""
    v = d["v_cache"].double().nan_to_num(0.0)
    return v.abs().amax()


@pytest.mark.parametrize("dtype, D", [(FP16, 128), (BF16, 64), (FP16, 64)])
@pytest.mark.parametrize("W", [4, 40, 200])
def test_windows_of_other_types(dtype, D, W):
    d = make(6, "cuda", dtype, 2, W, 12, 4, D, 48, [100, 7], [W, 0])
    check(d, attend(d))


@pytest.mark.parametrize("layout", ["heads", "slice"])
@pytest.mark.parametrize("W", [1, 40])
@pytest.mark.parametrize("shared", [0, 3])
def test_layouts(layout, W, shared):
    d = make(7, "cuda", BF16, 3, W, 8, 2, 128, 48, [200, 150, 333], None, shared, layout=layout)
    check(d, attend(d))


def test_long_and_short_sequences_together():
    positions = [9000, 3, -1, 40, 4000, 0, 700, 701, 702, 703]
    d = make(8, "cuda", BF16, len(positions), 1, 8, 1, 128, 16, positions)
    check(d, attend(d))


def widen(d, keys):
    """The same sequences in tables for ones of `keys` tokens: few-row launches are dealt out then, not given to clusters."""
    ps = d["k_cache"].shape[1]
    more = keys // ps - d["table"].shape[1]
    d["table"] = torch.cat([d["table"], torch.full((d["table"].shape[0], more), -1, dtype=torch.int32, device="cuda")], 1)
    return d


@pytest.mark.parametrize("dtype, D", [(BF16, 128), (FP16, 64)])
@pytest.mark.parametrize("H, Hkv", HEADS)
@pytest.mark.parametrize("positions", [[0, 15, 16, 257, 700], [9000, 3, -1, 40, 4000, 0, 700, 701, 702, 703], [-1, -1], [5]])
def test_dealt_out(dtype, D, H, Hkv, positions):
    d = make(8, "cuda", dtype, len(positions), 1, H, Hkv, D, 16, positions)
    near = attend(d)
    d = widen(d, 20000)
    check(d, attend(d))
    assert torch.equal(near == 0, attend(d) == 0)


@pytest.mark.parametrize("W", [2, 8])
def test_dealt_out_windows(W):
    d = widen(make(8, "cuda", BF16, 5, W, 4, 2, 128, 48, [3000, -1, 47, 0, 900], [W, W, 0, 1, W]), 48 * 500)
    check(d, attend(d))


def test_dealt_out_many():
    """More sequences than threads that look for places."""
    B = 1100
    positions = [(37 * b) % 190 - 1 for b in range(B)]
    d = make(9, "cuda", BF16, B, 1, 2, 1, 64, 16, positions)
    want = attend(d)
    got = attend(widen(d, 20000))
    assert bool(((got - want).double().abs() <= 2 * bound(BF16, got.double(), oracle_size(d))).all())
    check({**d, **{k: d[k][-40:] for k in ("q", "table", "positions")}}, got[-40:])


@pytest.mark.parametrize("B", [129, 300])
def test_many_sequences(B):
    positions = [(37 * b) % 90 - 1 for b in range(B)]
    d = make(9, "cuda", BF16, B, 1, 4, 2, 64, 16, positions)
    check(d, attend(d))


@pytest.mark.parametrize("W", [1, 24])
def test_holes(W):
    """Entries outside the pool: nobody sees their keys; a sequence of nothing else sees none."""
    d = make(10, "cuda", BF16, 4, W, 8, 2, 128, 32, [200, 100, 150, 90], None)
    d["table"][0, 2], d["table"][0, 0], d["table"][1, 3] = -1, 2 ** 31 - 1, -5
    d["table"][2] = d["k_cache"].shape[0]
    got = attend(d)
    check(d, got)
    assert not bool(got[2].any())


@pytest.mark.parametrize("W", [1, 3, 24])
def test_positions_beyond_everything(W):
    """Positions and lengths that no table has: nothing is read or written outside; the row sees the whole table."""
    far = make(11, "cuda", BF16, 3, W, 8, 2, 128, 16, [40, 17, 70])
    far["positions"][0], far["positions"][1] = 2 ** 63 - 1, -2 ** 63
    d = {**far, "lens": torch.tensor([2 ** 62, W, -5], device="cuda")}
    d["k_cache"].nan_to_num_(0.0)
    d["v_cache"].nan_to_num_(0.0)
    cos, sin = ops.rope.rope_tables(64, 128, device="cuda")
    before = d["k_cache"].clone()
    q = ops.paged.rope_append(d["q"], d["k"], d["v"], d["positions"], cos, sin, d["k_cache"], d["v_cache"], d["table"], lens=d["lens"])
    assert not bool(q.any()) and torch.equal(before, d["k_cache"])
    got = attend(d)
    end = {**d, "positions": torch.tensor([d["table"].shape[1] * 16 - 1, -1, 70], device="cuda"), "lens": torch.tensor([W, 0, 0], device="cuda")}
    want, size = oracle.attention(end["q"], end["k_cache"], end["v_cache"], end["table"], end["positions"], lens=end["lens"])
    assert bool(((got[0].double() - want[0]).abs() <= bound(BF16, want[0], size[0])).all())
    assert not bool(got[1:].any())


def test_positions_behind_the_table():
    d = make(11, "cuda", BF16, 2, 4, 8, 2, 128, 16, [30, 62], cols=6)
    d["table"] = d["table"][:, :3].contiguous()
    check(d, attend(d))


def test_garbage_where_nobody_looks():
    """Infinities and NaN in rows that no token sees, and zeros in their place, give the same bits."""
    for W, shared in ((1, 0), (5, 0), (50, 0), (3, 2)):
        a, b = (make(12, "cuda", BF16, 3, W, 8, 2, 128, 32, [100, 80, 200], None, shared, garbage=x) for x in (float("nan"), 0.0))
        c = make(12, "cuda", BF16, 3, W, 8, 2, 128, 32, [100, 80, 200], None, shared, garbage=float("-inf"))
        x = attend(a)
        assert torch.equal(x, attend(b)) and torch.equal(x, attend(c))


def test_nan_and_large_scores():
    d = make(13, "cuda", BF16, 3, 1, 8, 2, 128, 16, [100, 100, 100])
    d["q"][1] *= 200
    d["q"][2, 0, 3, 5] = float("nan")
    got = attend(d)
    assert bool(got[2, 0, 3].isnan().all()) and not bool(got[2, 0, 4].isnan().any())
    d["q"][2, 0, 3, 5] = 1.0
    got[2, 0, 3] = attend(d)[2, 0, 3]
    # scores to 2000: products in 32 bits leave 128 * 2^-24 * 2000 = 2^-6 of a weight
    want, size = oracle.attention(d["q"], d["k_cache"], d["v_cache"], d["table"], d["positions"])
    assert bool(((got.double() - want).abs() <= bound(BF16, want, size) + 2.0 ** -6 * size).all())


@pytest.mark.parametrize("scale", [0.01, 1.0])
def test_scale(scale):
    d = make(14, "cuda", BF16, 2, 2, 8, 2, 64, 16, [100, 37])
    d["q"] *= 0.25
    check(d, attend(d, scale=scale), scale)


# ----------------------------------------------------------------------------------------------------------- shared prefix
@pytest.mark.parametrize("dtype, D", [(BF16, 128), (FP16, 64)])
@pytest.mark.parametrize("B, W, H, Hkv", [(1, 1, 8, 8), (2, 1, 8, 2), (20, 1, 16, 2), (9, 3, 6, 2), (3, 1, 4, 4), (40, 2, 8, 1)])
@pytest.mark.parametrize("shared", [1, 5, 33])
def test_shared(dtype, D, B, W, H, Hkv, shared):
    positions = [shared * 16 + (53 * b) % 170 for b in range(B)]
    d = make(15, "cuda", dtype, B, W, H, Hkv, D, 16, positions, [1 + (b % W) for b in range(B)], shared)
    check(d, attend(d))


def test_shared_with_idle_rows_and_rows_inside():
    """Rows whose tokens stand inside the shared pages see their part of them."""
    d = make(16, "cuda", BF16, 6, 3, 8, 2, 128, 32, [-1, 0, 50, 94, 95, 500], [3, 3, 3, 3, 3, 0], 3)
    check(d, attend(d))


def test_shared_holes():
    d = make(17, "cuda", BF16, 3, 1, 8, 2, 128, 16, [200, 100, 79], None, 4)
    d["shared_pages"][1] = -1
    d["shared_pages"][2] = 10 ** 8
    check(d, attend(d))


def test_shared_is_what_the_tables_say():
    """The first columns of the tables are not looked at."""
    d = make(18, "cuda", BF16, 4, 1, 8, 2, 128, 64, [200, 150, 400, 129], None, 2)
    a = attend(d)
    d["table"][:, :2] = -1
    assert torch.equal(a, attend(d))


@pytest.mark.parametrize("W", [1, 16, 17, 40, 100])
def test_shared_windows_and_portions(W):
    """Few rows, tiles of them, and portions of prompts, which read the shared pages as their own."""
    d = make(19, "cuda", BF16, 3, W, 8, 1, 128, 32, [96, 150, 260], [W, 1, W], 3)
    a = attend(d)
    check(d, a)
    d["table"][:, :3] = -1
    assert torch.equal(a, attend(d))
    none = {**d, "shared_pages": d["shared_pages"][:0], "table": torch.cat([d["shared_pages"].expand(3, 3), d["table"][:, 3:]], 1)}
    check(none, attend(none))


def test_long_shared_prefix():
    d = make(19, "cuda", BF16, 7, 1, 8, 1, 128, 128, [8000, 8064, 8063, 8200, 8100, 9000, 8065], None, 63)
    check(d, attend(d))


# ------------------------------------------------------------------------------------------------------------- as programs
def test_offsets_pass_32_bits():
    """A pool of more than 2^32 bytes (and 2^31 numbers): pages at its end."""
    pages, ps, Hkv, D = 70000, 16, 16, 128
    kc, vc = (torch.empty(pages, ps, Hkv, D, dtype=BF16, device="cuda") for _ in range(2))
    d = make(20, "cuda", BF16, 2, 3, 16, 16, D, ps, [100, 37])
    n = d["k_cache"].shape[0]
    kc[-n:], vc[-n:] = d["k_cache"], d["v_cache"]
    table = d["table"] + (pages - n)
    got = ops.paged.attention(d["q"], kc, vc, table, d["positions"])
    assert torch.equal(got, attend(d))
    cos, sin = ops.rope.rope_tables(128, D, device="cuda")
    ops.paged.rope_append(d["q"], d["k"], d["v"], d["positions"], cos, sin, kc, vc, table)
    ops.paged.rope_append(d["q"], d["k"], d["v"], d["positions"], cos, sin, d["k_cache"], d["v_cache"], d["table"])
    assert torch.equal(kc[-n:].nan_to_num(), d["k_cache"].nan_to_num()) and torch.equal(vc[-n:].nan_to_num(), d["v_cache"].nan_to_num())


def test_results_repeat():
    for W, shared in ((1, 0), (40, 0), (2, 20)):
        d = make(21, "cuda", BF16, 4, W, 16, 2, 128, 16, [2000, 321, 900, 1500], None, shared)
        a = attend(d)
        assert all(torch.equal(a, attend(d)) for _ in range(3))


@pytest.mark.parametrize("W, shared", [(1, 0), (5, 0), (30, 0), (1, 8)])
def test_captured_and_replayed(W, shared):
    """One graph over append and attention; positions, tables and tokens change between replays, and two graphs take turns."""
    cos, sin = ops.rope.rope_tables(2000, 128, device="cuda")

    def program(d):
        q = ops.paged.rope_append(d["q"], d["k"], d["v"], d["positions"], cos, sin, d["k_cache"], d["v_cache"], d["table"], lens=d["lens"])
        return q, attend({**d, "q": q})

    sets = [make(22 + i, "cuda", BF16, 3, W, 16, 4, 128, 16, p, n, shared, cols=100)
            for i, (p, n) in enumerate((([150, 700, 300], [W, W, W]), ([1000, -1, 129], [1, W, W])))]
    want = [program({k: (v.clone() if torch.is_tensor(v) else v) for k, v in d.items()}) for d in sets]
    live = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in sets[0].items()}
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        program(live)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = program(live)
        graphs.append((g, out))
    for i in (1, 0, 1):
        for g, out in graphs:
            for k, v in live.items():
                if torch.is_tensor(v):
                    v.copy_(sets[i][k])
            g.replay()
            assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])


def test_two_streams_at_once():
    ds = [make(24 + i, "cuda", BF16, 4, 1 + 3 * i, 16, 4, 128, 16, [900, 300, 1200, 50]) for i in range(2)]
    want = [attend(d) for d in ds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ds]
    got = [[], []]
    for _ in range(20):
        for i, (s, d) in enumerate(zip(streams, ds)):
            with torch.cuda.stream(s):
                got[i].append(attend(d))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_general_way_for_other_types():
    """32-bit numbers and other head sizes go the general way, with the same results as far as their types allow."""
    for dtype, D in ((torch.float32, 64), (BF16, 32), (BF16, 80)):
        d = make(26, "cuda", dtype, 3, 2, 8, 2, D, 16, [100, 5, -1], [2, 1, 2])
        check(d, attend(d))


def test_refused_on_the_device():
    d = make(27, "cuda", BF16, 2, 1, 8, 2, 128, 16, [40, 20])
    good = [d["q"], d["k_cache"], d["v_cache"], d["table"], d["positions"]]
    ops.paged.attention(*good)
    for which, change in ((0, lambda t: t[0]), (0, lambda t: t[:, :, :3]), (0, lambda t: t.half()), (1, lambda t: t[:, :, :1]), (1, lambda t: t.half()),
                          (2, lambda t: t[:1]), (3, lambda t: t[:1]), (3, lambda t: t.cpu()), (4, lambda t: t[:1]), (4, lambda t: t.cpu())):
        args = list(good)
        args[which] = change(args[which])
        with pytest.raises(ValueError):
            ops.paged.attention(*args)
    pages = torch.zeros(40, 16, 2, 128, dtype=BF16, device="cuda")
    with pytest.raises(ValueError):
        ops.paged.attention(d["q"], pages[:, :8], pages[:, :8], d["table"], d["positions"])
    with pytest.raises(ValueError):
        ops.paged.attention(*good, shared_pages=torch.zeros(9, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        ops.paged.attention(*good, lens=torch.ones(3, dtype=torch.long, device="cuda"))
    cos, sin = ops.rope.rope_tables(64, 128, device="cuda")
    with pytest.raises(ValueError):
        ops.paged.rope_append(d["q"], d["k"], d["v"], d["positions"], cos[:, :8], sin[:, :8], d["k_cache"], d["v_cache"], d["table"])
    with pytest.raises(ValueError):
        ops.paged.rope_append(d["q"], d["k"][:, :, :1], d["v"][:, :, :1], d["positions"], cos, sin, d["k_cache"], d["v_cache"], d["table"])


# ------------------------------------------------------------------------------------------------------- drafted tokens
def drafts(seed, B, K, V, dtype=torch.float32, close=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn(B, K + 1, V, generator=g, device="cuda") * 2
    target = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits[:, :K] + close * torch.randn(B, K, V, generator=g, device="cuda"), -1).to(dtype)
    tokens = torch.multinomial(draft.float().reshape(B * K, V), 1, generator=g).view(B, K) if K else torch.zeros(B, 0, dtype=torch.long, device="cuda")
    return [tokens, draft, target, torch.rand(B, K, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")]


def same(args):
    """The plain path on the CPU: the same comparisons and sums, in another order."""
    got, n = ops.select.verify_drafts(*args)
    want, m = ops.select.verify_drafts(*[t.cpu() for t in args])
    assert torch.equal(n.cpu(), m) and torch.equal(got.cpu(), want)
    return got, n


@pytest.mark.parametrize("V", [1, 5, 128, 1000, 32000, 32016, 50257, 100352])
@pytest.mark.parametrize("B, K", [(1, 1), (3, 4), (5, 0), (2, 40), (70, 7)])
def test_verify(V, B, K):
    if B * (K + 1) * V > 2e7:
        B = 9
    same(drafts(30, B, K, V))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("V", [37, 32000])
def test_verify_half_types(dtype, V):
    same(drafts(31, 6, 3, V, dtype))


def test_verify_all_and_none():
    args = drafts(32, 8, 4, 1000, close=0.0)
    args[3] *= 0.9                                       # p = q: every u below 1 accepts
    _, n = same(args)
    assert bool((n == 4).all())
    args[3].fill_(1.0)                                   # and u = 1 refuses; nothing of p - q is left
    got, n = same(args)
    assert bool((n == 0).all()) and bool((got[:, 1:] == -1).all())


def test_verify_odd_rows():
    args = drafts(33, 10, 3, 517)
    args[0][0, 1], args[0][1, 0], args[0][2] = -1, 517, 2 ** 40
    args[2][3] = 0.0
    args[2][4, :, 5] = float("nan")
    args[2][5, 0] = -1.0
    args[1][6] = 0.0
    args[4][7], args[4][8] = 0.0, 1.0 - 2.0 ** -24
    args[4][9] = 1.0
    got, _ = same(args)
    assert int(got[3, 0]) == -1


def test_verify_one_weight():
    """Only the last, or the first, of a row's numbers is not zero, in every block's and warp's stretch."""
    V = 32016
    for at in (0, 1, 511, 512, 4095, 4096, V // 2, V - 1):
        args = drafts(34, 2, 1, V)
        args[0].fill_(-1)
        args[2].zero_()
        args[2][:, 0, at] = 2.0 ** -100
        got, _ = same(args)
        assert got[:, 0].tolist() == [at, at]


def test_verify_views_and_capture():
    args = drafts(35, 4, 3, 1001)
    want, n = ops.select.verify_drafts(*args)
    wide = torch.zeros(4, 4, 2 * 1001 + 1, device="cuda")
    wide[:, :, 1:1002] = args[2]
    turned = args[1].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    got, m = ops.select.verify_drafts(args[0], turned, wide[:, :, 1:1002], args[3], args[4])
    assert torch.equal(got, want) and torch.equal(n, m)
    live = [t.clone() for t in args]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, k = ops.select.verify_drafts(*live)
    for seed in (36, 35):
        other = drafts(seed, 4, 3, 1001)
        for a, b in zip(live, other):
            a.copy_(b)
        g.replay()
        want, n = ops.select.verify_drafts(*other)
        assert torch.equal(out, want) and torch.equal(k, n)
