"""The kernels of the cache in 4 bits (``csrc/paged_int4.cu``) against their definitions in 64 bits."""
import pytest
import torch

from paged_int4_cases import append, assign, attention, bound, lay, make, packed, values
from test_paged_int4_cpu import refusals

from neuronx_distributed_b200 import ops
from neuronx_distributed_b200.ops.paged_int4 import Pages

pytestmark = pytest.mark.gpu
BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32


def attend(d, **kw):
    return ops.paged_int4.attention(d["q"], d["k_pages"], d["v_pages"], d["table"], d["positions"], lens=d["lens"], shared_pages=d["shared_pages"], **kw)


def check(d, got, scale=None):
    want, size = attention(d, scale)
    off = (got.double() - want).abs() - bound(d["q"].dtype, want, size)
    assert bool((off <= 0).all()), (float(off.max()), (~(off <= 0)).nonzero()[:4].tolist())


# ------------------------------------------------------------------------------------------------------------------ append
def check_append(q, k, v, positions, cos, sin, slots, pages, got, before, interleaved):
    """Queries within a half step of their type and three roundings in 32 bits of numbers below 6; steps and codes those of exact numbers, everything else
    as it was."""
    dtype, ps = q.dtype, pages[0].codes.shape[1]
    tokens = pages[0].codes.shape[0] * ps
    want_q, written = append(q.cpu(), k.cpu(), v.cpu(), positions.cpu(), cos.cpu(), sin.cpu(), slots.cpu(), tokens, interleaved)
    assert got.dtype == dtype and got.transpose(0, 1).is_contiguous()
    assert bool(((got.double().cpu() - want_q).abs() <= torch.finfo(dtype).eps / 2 * want_q.abs() + 6 * 3 * 2.0 ** -24).all())
    for i, p in enumerate(pages):
        codes, steps = p.codes.cpu(), p.steps.cpu()
        for slot in range(tokens):
            at = slot // ps, slot % ps
            want = packed(written[slot][i]) if slot in written else Pages(before[i].codes[at].cpu(), before[i].steps[at].cpu())
            assert torch.equal(codes[at], want.codes) and torch.equal(steps[at].view(torch.int16), want.steps.view(torch.int16)), (i, slot)


@pytest.mark.parametrize("dtype, D", [(BF16, 128), (BF16, 64), (FP16, 96), (F32, 128), (F32, 32)])
@pytest.mark.parametrize("B, W, H, Hkv, ps, positions", [(1, 1, 4, 4, 16, [0]), (3, 2, 8, 1, 16, [15, 16, 200]), (4, 7, 6, 2, 48, [0, 41, 48, 296]), (2, 65, 4, 2, 128, [0, 100])])
@pytest.mark.parametrize("rotation", ["halves", "pairs", "part", "part_pairs", "none"])
@pytest.mark.parametrize("layout", ["heads", "rows", "slice"])
def test_append(dtype, D, B, W, H, Hkv, ps, positions, rotation, layout):
    g = torch.Generator().manual_seed(B + W)
    half = {"halves": D // 2, "pairs": D // 2, "part": 8, "part_pairs": 12, "none": 0}[rotation]
    q, k, v = (torch.randn(B, W, h, D, generator=g).to(dtype).cuda() for h in (H, Hkv, Hkv))
    angles = torch.rand(300, half, generator=g) * 6.3
    cos, sin = angles.cos().cuda(), angles.sin().cuda()
    count = (B * W + ps - 1) // ps + 1
    slots = torch.randperm(count * ps, generator=g)[:B * W].view(B, W).int()
    slots[-1, -1] = -1
    if W > 1:
        slots[0, 0] = count * ps
    pages = [lay(packed(torch.randn(count, ps, Hkv, D, generator=g)), layout) for _ in "kv"]
    pages = [lay(Pages(*(t.cuda() for t in p)), layout) for p in pages]
    before = [Pages(*(t.clone() for t in p)) for p in pages]
    positions = torch.tensor(positions).cuda()
    slots = slots.cuda()
    got = ops.paged_int4.append(q, k, v, positions, cos, sin, *pages, slots, interleaved=rotation.endswith("pairs"))
    check_append(q, k, v, positions, cos, sin, slots, pages, got, before, rotation.endswith("pairs"))
    for dt in (BF16, FP16, F32):
        for x, p in zip(ops.paged_int4.gather(*pages, slots, dt), pages):
            at = slots.long().clamp(0, count * ps - 1)
            want = values(p)[at // ps, at % ps] * ((slots >= 0) & (slots < count * ps))[:, :, None, None]
            assert x.dtype == dt and x.is_contiguous()
            assert bool(((x.double() - want).abs() <= (torch.finfo(dt).eps / 2 + 2.0 ** -24) * want.abs() + 2.0 ** -25).all())


def test_append_borders():
    """Numbers on, and in 32 bits next to, the borders between two codes; ranges of nothing; numbers that are not finite."""
    D, ps = 32, 16
    x = torch.linspace(0, 15, 32)                            # m = 0, s = 1
    rows = [x.clone() for _ in range(16)]
    for i, r in enumerate(rows):
        r[1:31] = torch.arange(30) / 2 + torch.tensor([0.0, 2.0 ** -22, -2.0 ** -22, 2.0 ** -20])[i % 4] * (torch.arange(30) / 2 + (i >= 4))
    rows[8][:] = 3.25
    rows[9][:] = 0.0
    rows[10][7] = float("nan")
    rows[11][7] = float("inf")
    rows[12][7] = -1e6
    rows[13] *= 1e-7
    rows[14] *= 2.0 ** -24
    rows[15] = rows[15] * 1000 - 20000
    k = torch.stack(rows).view(1, 16, 1, D).cuda()
    pages = [ops.paged_int4.new_pages(1, ps, 1, D, "cuda") for _ in "kv"]
    slots = torch.arange(16, dtype=torch.int32, device="cuda").view(1, 16)
    none = torch.zeros(20, 0, device="cuda")
    ops.paged_int4.append(k, k, k, torch.zeros(1, dtype=torch.long, device="cuda"), none, none, *pages, slots)
    want = packed(k[0].cpu())
    for p in pages:
        assert torch.equal(p.codes[0].cpu(), want.codes)
        assert torch.equal(p.steps[0].cpu().nan_to_num(7.0, 8.0, 9.0), want.steps.nan_to_num(7.0, 8.0, 9.0))


def test_append_takes_sections_and_odd_views():
    """Sections of a projection's output, views that begin at no packet, tables and slots of other kinds."""
    B, W, H, Hkv, D = 2, 3, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    cos, sin = ops.rope.rope_tables(64, D, device="cuda")
    flat = torch.randn(W, B, (H + 2 * Hkv) * D + 3, generator=g, device="cuda").to(BF16)
    positions = torch.tensor([5, 14], device="cuda")
    slots = torch.randperm(64, device="cuda")[:6].view(B, W)
    for qkv in (flat[..., :-3], flat[..., 3:]):
        for c, s, sl, pos in ((cos, sin, slots, positions), (cos.t().contiguous().t(), sin, slots.t().contiguous().t().int(), positions.int())):
            q, k, v = (t.unflatten(-1, (-1, D)).transpose(0, 1) for t in qkv.split([H * D, Hkv * D, Hkv * D], -1))
            pages = [ops.paged_int4.new_pages(4, 16, Hkv, D, "cuda") for _ in "kv"]
            before = [Pages(*(t.clone() for t in p)) for p in pages]
            got = ops.paged_int4.append(q, k, v, pos, c, s, *pages, sl)
            check_append(q, k, v, positions, cos, sin, slots, pages, got, before, False)


def test_append_outside_the_rotation_tables():
    pages = [ops.paged_int4.new_pages(2, 16, 1, 64, "cuda") for _ in "kv"]
    x = torch.ones(3, 4, 1, 64, device="cuda", dtype=BF16)
    cos, sin = ops.rope.rope_tables(10, 64, device="cuda")
    slots = torch.arange(12, dtype=torch.int32, device="cuda").view(3, 4)
    lost = torch.zeros(1, dtype=torch.int32, device="cuda")
    positions = torch.tensor([0, 8, -2], device="cuda")
    ops.paged_int4.append(x, x, x, torch.tensor([0, 6, 3], device="cuda"), cos, sin, *pages, slots, lost=lost)
    assert int(lost) == 0
    for p in pages:
        p.codes.zero_(), p.steps.zero_()
    q = ops.paged_int4.append(x, x, x, positions, cos, sin, *pages, slots, lost=lost)
    there = torch.tensor([[1, 1, 1, 1], [1, 1, 0, 0], [0, 0, 1, 1]], dtype=torch.bool, device="cuda")
    assert int(lost) == 1 and torch.equal(q.ne(0).any(-1).any(-1), there)
    assert torch.equal(pages[1].steps[0, :12].ne(0).flatten(1).any(-1), there.flatten())


# --------------------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("B, W, H, Hkv, ps, positions, lens", [
    (1, 1, 1, 1, 16, [0], None),
    (1, 1, 8, 1, 16, [1], None),
    (3, 1, 4, 4, 16, [-1, 15, 16], None),
    (4, 1, 8, 2, 48, [63, 64, 65, 200], [1, 1, 0, 1]),
    (2, 1, 16, 1, 32, [300, 5], None),
    (2, 1, 32, 1, 16, [130, 5], None),                      # more rows than a tile of 16
    (3, 5, 8, 1, 16, [0, 70, 255], [5, 3, 5]),
    (2, 3, 6, 2, 128, [600, 100], None),
    (3, 33, 4, 2, 64, [0, 17, 400], [33, 0, 20]),
    (2, 90, 3, 1, 16, [-1, 37], None),
    (2, 300, 8, 2, 64, [500, 30], [300, 111]),             # enough for the tensor memory
    (1, 4, 4, 4, 16, [700], None),
])
@pytest.mark.parametrize("layout", ["heads", "rows", "slice"])
def test_attention(dtype, D, B, W, H, Hkv, ps, positions, lens, layout):
    d = make(B * W + H, "cuda", dtype, B, W, H, Hkv, D, ps, positions, lens, layout=layout)
    got = attend(d)
    check(d, got)
    assert got.transpose(0, 1).is_contiguous()
    assert torch.equal(got, attend(d))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("W, G, positions, cols", [(1, 4, [1500, 40], None), (1, 1, [2100], 1000), (2, 8, [5000, 900, 33], 400), (1, 8, [40000], None), (1, 16, [33000, 10], None),
                                                   (3, 8, [9000], 4200)])
def test_attention_of_long_sequences(dtype, W, G, positions, cols):
    """Pairs that clusters share, and pairs that are dealt out over the GPU, some of them cut."""
    d = make(4, "cuda", dtype, len(positions), W, G, 1, 128, 16 if cols else 128, positions, cols=cols)
    check(d, attend(d))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("k_factor, v_factor, v_add", [(1, 1000, 0), (1, 1e-4, 0), (1, 1, 300), (6, 1, 0), (0, 1, 0), (1, 0, 0), (1, 0, 5), (1, 4000, -20000)])
def test_attention_of_other_sizes(dtype, k_factor, v_factor, v_add):
    for B, W, H, Hkv, D, positions in ((2, 1, 8, 2, 128, [400, 70]), (1, 6, 4, 1, 64, [500])):
        d = make(6, "cuda", dtype, B, W, H, Hkv, D, 16, positions, k_factor=k_factor, v_factor=v_factor, v_add=v_add)
        check(d, attend(d), None)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_attention_of_steps_that_grow(dtype):
    """Values whose steps get larger from token to token, and scores that do: weights are taken relative to ever other references."""
    d = make(7, "cuda", dtype, 1, 2, 8, 1, 128, 16, [800])
    at = d["table"][0].long()
    grow = (2.0 ** (torch.arange(at.numel() * 16, device="cuda") / 60)).half().view(-1, 16, 1, 1)
    steps = d["v_pages"].steps
    steps[at] = torch.where(steps[at].isnan(), steps[at], (steps[at].float() * grow[..., None].float()).half())
    steps = d["k_pages"].steps
    steps[at] = torch.where(steps[at].isnan(), steps[at], (steps[at].float() * grow[..., None].float() ** 0.3).half())
    check(d, attend(d))


@pytest.mark.parametrize("factor", [1e-30, 1e-8, 0.0, 1e4, 1e6])
def test_attention_of_other_queries(factor):
    """Queries far below and above half precision: a scale that brings the scores back."""
    d = make(8, "cuda", BF16, 2, 1, 8, 2, 128, 16, [100, 37])
    d["q"] = d["q"] * factor
    check(d, attend(d, scale=0.1 / max(factor, 1e-28)), 0.1 / max(factor, 1e-28))


def test_a_query_of_nan_is_its_own():
    d = make(9, "cuda", BF16, 2, 3, 8, 2, 128, 16, [100, 37])
    clean = attend(d)
    d["q"] = d["q"].clone()
    d["q"][0, 1, 3] = float("nan")
    got = attend(d)
    assert bool(got[0, 1, 3].isnan().all())
    got[0, 1, 3] = clean[0, 1, 3]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("W, positions, lens", [(1, [64, 200, -1], None), (3, [64, 90, 33], [3, 1, 0]), (40, [100, 40, 64], None)])
def test_shared_pages_and_holes(W, positions, lens):
    d = make(10, "cuda", BF16, 3, W, 8, 2, 128, 16, positions, lens, shared=2)
    check(d, attend(d))
    d["table"][0, :2] = 1 << 30                              # not looked at
    check(d, attend(d))
    d["table"][1, 3] = -7
    d["shared_pages"][1] = d["k_pages"].codes.shape[0]
    check(d, attend(d))
    assert not bool(attend({**d, "table": torch.full_like(d["table"], -1), "shared_pages": None}).any())


def test_other_scales_and_integers():
    d = make(11, "cuda", FP16, 2, 2, 8, 2, 128, 32, [70, 31], [2, 1])
    for scale in (0.01, 1.0):
        check(d, attend(d, scale=scale), scale)
    want = attend(d)
    odd = {**d, "table": d["table"].long(), "positions": d["positions"].int(), "lens": d["lens"].int()}
    assert torch.equal(attend(odd), want)
    base = torch.zeros(d["q"].numel() + 1, dtype=FP16, device="cuda")
    base[1:] = d["q"].reshape(-1)
    assert torch.equal(attend({**d, "q": base[1:].view(d["q"].shape)}), want)


def test_heads_of_other_sizes_and_types():
    for dtype, D in ((BF16, 32), (FP16, 96), (F32, 128), (F32, 64), (BF16, 256)):
        d = make(12, "cuda", dtype, 2, 2, 4, 2, D, 16, [40, 3])
        check(d, attend(d))


# ----------------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype, interleaved", [(BF16, False), (FP16, True)])
def test_a_server(dtype, interleaved):
    """Prompts, tokens and a drafted window of three sequences, one of which ends and begins anew: tables, append, attention, captured for the tokens."""
    B, H, Hkv, D, ps, n, P = 3, 8, 2, 64, 16, 6, 14
    g = torch.Generator(device="cuda").manual_seed(3)
    angles = torch.rand(n * ps, 16, generator=g, device="cuda") * 6
    cos, sin = angles.cos(), angles.sin()
    pages = [ops.paged_int4.new_pages(P, ps, Hkv, D, "cuda") for _ in "kv"]
    table, held = torch.full((B, n), -1, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    free, span = torch.randperm(P, generator=g, device="cuda").int(), torch.tensor([0, P], device="cuda")
    short = torch.zeros(1, dtype=torch.int32, device="cuda")
    keys = [[] for _ in range(B)]                            # what each row has been given: (key, value) as held

    def ask(positions, new, lens=None, lengths=None):
        return ops.page_tables.assign(table, held, free, span, positions, new, ps, lens=lens, lengths=lengths, short=short, in_place=True).slots

    def whole(q, k, v, positions, slots, lens):
        turned = ops.paged_int4.append(q, k, v, positions, cos, sin, *pages, slots, interleaved=interleaved)
        return turned, ops.paged_int4.attention(turned, *pages, table, positions, lens=lens)

    def fresh(W):
        return [torch.randn(W, B, h, D, generator=g, device="cuda").to(dtype).transpose(0, 1) for h in (H, Hkv, Hkv)]

    def compare(turned, out, positions, W, lens):
        d = {"q": turned, "k_pages": pages[0], "v_pages": pages[1], "table": table, "positions": positions, "lens": lens, "shared_pages": None}
        check(d, out)
        for b in range(B):
            p, m = int(positions[b]), W if lens is None else int(lens[b])
            if p < 0:
                continue
            assert len(keys[b]) >= p
            del keys[b][p:]
            for w in range(m):
                at = int(table[b, (p + w) // ps]), (p + w) % ps
                keys[b].append([Pages(x.codes[at], x.steps[at]) for x in pages])
            for j, kept in enumerate(keys[b]):               # nobody has written over what a row holds
                at = int(table[b, j // ps]), j % ps
                for x, old in zip(pages, kept):
                    assert torch.equal(x.codes[at], old.codes) and torch.equal(x.steps[at], old.steps)
        for b in range(B):
            keys[b] = [[Pages(x.codes.clone(), x.steps.clone()) for x in pair] for pair in keys[b]]

    # prompts
    positions, lens = torch.tensor([0, 0, 0], device="cuda"), torch.tensor([20, 33, 5], device="cuda")
    compare(*whole(*fresh(33), positions, ask(positions, 33, lens), lens), positions, 33, lens)
    # tokens, captured once
    positions = lens.clone()
    q, k, v = fresh(1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        turned, out = whole(q, k, v, positions, ask(positions, 1), None)
    for i in range(14):
        for a, b in zip((q, k, v), fresh(1)):
            a.copy_(b)
        graph.replay()
        compare(turned, out, positions, 1, None)
        positions += 1
    # a drafted window; then the second row ends, and begins anew with a prompt, and the others stay
    compare(*whole(*fresh(4), positions, ask(positions, 4), None), positions, 4, None)
    ask(torch.tensor([-1, -1, -1], device="cuda"), 0, lengths=torch.tensor([-1, 0, -1], device="cuda"))
    keys[1] = []
    assert held.tolist()[1] == 0 and int(span[1] - span[0]) == P - int(held.sum())
    positions, lens = torch.tensor([-1, 0, -1], device="cuda"), torch.tensor([0, 40, 0], device="cuda")
    compare(*whole(*fresh(40), positions, ask(positions, 40, lens), lens), positions, 40, lens)
    assert int(short) == 0


def test_on_another_stream_and_captured_twice():
    """Two captured graphs of one pool, replayed after each other on a stream of their own, give what the calls give."""
    a = make(13, "cuda", BF16, 2, 1, 8, 2, 128, 16, [100, 50], cols=2600)              # dealt out: with a workspace
    b = make(14, "cuda", BF16, 3, 20, 4, 2, 128, 32, [0, 64, 200])
    want = attend(a), attend(b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphs, outs = [], []
        for d in (a, b):
            attend(d)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(attend(d))
            graphs.append(graph)
        for _ in range(3):
            for o in outs:
                o.fill_(float("nan"))
            for graph in graphs:
                graph.replay()
            assert all(torch.equal(o, w) for o, w in zip(outs, want))
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("B, H, shared", [(1, 3, 0), (3, 1, 0), (3, 1, 1)])
def test_portions_whose_pages_are_unpacked_in_unlike_turns(B, H, shared):
    """Tables of 200,000 tokens, of which a few hundred are there: two heads, or two sequences, are unpacked in the first turn, and one in the second."""
    d = make(5, "cuda", BF16, B, 48, H, H, 128, 128, [300, 17, 411][:B])
    d["table"] = torch.cat([d["table"], torch.full((B, 200000 // 128 - d["table"].shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
    if shared:
        d["shared_pages"] = d["table"][0, :1].contiguous()
        d["table"][1:, 0] = -1
    check(d, attend(d))


@pytest.mark.parametrize("B, W, H, Hkv, D, positions", [(2, 1, 8, 8, 128, [26930, 20000]), (1, 1, 8, 2, 64, [60000]), (1, 2, 8, 1, 128, [30000]), (1, 8, 4, 4, 128, [9000])])
def test_half_precision_over_many_keys(B, W, H, Hkv, D, positions):
    """Averages of thousands of values are a hundredth of them.  What rounding the result leaves is at most 2^-11 of each number, evenly spread, in the 2-norm 2^-11 / sqrt(3)
    of all at most (and 0.75 of that, because numbers lie all over between two powers of two): with everything else the error stays below that."""
    d = make(3, "cuda", FP16, B, W, H, Hkv, D, 64, positions)
    got, want = attend(d), attention(d)[0]
    assert float((got.double() - want).norm() / want.norm()) < 2.0 ** -11 / 3 ** 0.5


@pytest.mark.parametrize("W", [1, 5, 200])
def test_pages_behind_4_gigabytes(W):
    """The last pages of a pool of 4.3 GB of codes: written, read back and attended to as the same pages of a small pool, bit by bit (200 tokens: unpacked)."""
    ps, H, Hkv, D, n = 16, 16, 2, 128, 2 ** 21 + 64
    d = make(7, "cuda", BF16, 1, W, H, Hkv, D, ps, [700])
    used, at = d["k_pages"].codes.shape[0], n - d["k_pages"].codes.shape[0]
    assert at * ps * Hkv * D // 2 > 2 ** 32 and used <= 64
    d["table"] = torch.cat([d["table"], torch.full((1, 4000 - d["table"].shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
    slots = (d["table"][:, 700 // ps:].repeat_interleave(ps, 1) * ps + torch.arange(ps, device="cuda").repeat(4000 - 700 // ps))[:, 700 % ps:][:, :W].int()
    small = [Pages(*(t.clone() for t in p)) for p in (d["k_pages"], d["v_pages"])]
    large = [ops.paged_int4.new_pages(n, ps, Hkv, D, device="cuda") for _ in "kv"]
    for p, from_ in zip(large, small):
        for t, x in zip(p, from_):
            t[at:] = x
    angles = torch.rand(1000, D // 2, device="cuda")
    out = []
    for pages, off in ((small, 0), (large, at)):
        table = torch.where(d["table"] >= 0, d["table"] + off, -1)
        q = ops.paged_int4.append(d["q"], d["k"], d["v"], d["positions"], angles.cos(), angles.sin(), *pages, slots + off * ps)
        out.append([q, *ops.paged_int4.gather(*pages, slots + off * ps, F32), ops.paged_int4.attention(q, *pages, table, d["positions"])])
    assert all(torch.equal(a, b) for a, b in zip(*out)) and bool(out[0][3].isfinite().all())
    for p, from_ in zip(large, small):
        for t, x in zip(p, from_):
            assert torch.equal(t[at:].nan_to_num(), x.nan_to_num()) and not bool(t[:64].any())


@pytest.mark.parametrize("n, Hkv, D", [(30000, 1, 32), (20011, 1, 64), (9001, 3, 96), (4003, 9, 128), (2500, 40, 64), (130, 1100, 128)])
def test_gather_of_many_tokens(n, Hkv, D):
    g = torch.Generator(device="cuda").manual_seed(n)
    pages = [ops.paged_int4.new_pages(24, 16, Hkv, D, device="cuda") for _ in "kv"]
    for p in pages:
        p.codes.copy_(torch.randint(0, 256, p.codes.shape, generator=g, device="cuda", dtype=torch.uint8))
        p.steps.copy_(torch.randn(p.steps.shape, generator=g, device="cuda"))
    slots = torch.randint(-1, 24 * 16 + 1, (1, n), generator=g, device="cuda", dtype=torch.int32)
    at, there = slots.long().clamp(0, 24 * 16 - 1), (slots >= 0) & (slots < 24 * 16)
    for x, p in zip(ops.paged_int4.gather(*pages, slots, BF16), pages):
        assert x.shape == (1, n, Hkv, D)
        for lo in range(0, n, 4000):
            a = at[:, lo:lo + 4000]
            want = values(Pages(*(t[a // 16, a % 16] for t in p))) * there[:, lo:lo + 4000, None, None]
            assert bool(((x[:, lo:lo + 4000].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -24) * want.abs() + 2.0 ** -25).all())


def test_refusals():
    refusals("cuda")
    d = make(1, "cuda", BF16, 2, 3, 4, 2, 64, 16, [3, 20])
    with pytest.raises(ValueError):
        ops.paged_int4.attention(d["q"], d["k_pages"], d["v_pages"], d["table"].cpu(), d["positions"])
    with pytest.raises(ValueError):
        ops.paged_int4.attention(d["q"], d["k_pages"], Pages(*(t.cpu() for t in d["v_pages"])), d["table"], d["positions"])
