"""Attention over 4-bit pages by the kernels of many rows: pages unpacked to halves for the tensor memory, and row tiles beside them."""
import pytest
import torch

from paged_cases import make as make16
from paged_int4_cases import attention, bound, make, values
from paged_oracle import attention as oracle16

from neuronx_distributed_b200 import ops
from neuronx_distributed_b200.ops import _ext

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def wide(d, tokens):
    """A table of so many tokens, behind the last page of which there is none: from some width on portions of prompts are unpacked."""
    B, n = d["table"].shape
    cols = -(-tokens // d["k_pages"].codes.shape[1])
    return {**d, "table": torch.cat([d["table"], torch.full((B, max(0, cols - n)), -1, dtype=torch.int32, device="cuda")], 1)}


def attend(d, unpacked=None, **kw):
    """``unpacked``: whether the pages are, by the launches: queries, pages, attention, and often the joining of its parts, for one or two."""
    n = _ext.launches()
    out = ops.paged_int4.attention(d["q"], d["k_pages"], d["v_pages"], d["table"], d["positions"], lens=d["lens"], shared_pages=d["shared_pages"], **kw)
    assert unpacked is None or unpacked == (_ext.launches() - n > 2)
    return out


def check(d, got, scale=None, more=0.0):
    want, size = attention(d, scale)
    off = (got.double() - want).abs() - bound(d["q"].dtype, want, size) - more * size
    assert bool((off <= 0).all()), (float(off.max()), (~(off <= 0)).nonzero()[:4].tolist())


@pytest.mark.parametrize("scale", [None, 1 / 128, 1e-8, 1e-25, 1e-39])
@pytest.mark.parametrize("B, W, H, Hkv, tokens, unpacked", [(2, 80, 8, 2, 8192, True), (2, 6, 8, 2, 0, False), (2, 1, 8, 2, 0, False)])
def test_rows_of_zeros(scale, B, W, H, Hkv, tokens, unpacked):
    """Rows of zeros, as append leaves them for tokens without a slot, and rows of the smallest numbers see the average of the values; so does everybody where the scale is next to
    nothing."""
    d = wide(make(21, "cuda", BF16, B, W, H, Hkv, 128, 16, [100, 37]), tokens)
    d["q"] = d["q"].clone()
    d["q"][0, 0, 1:3] = 0.0
    d["q"][1] = 0.0
    d["q"][0, -1, :2] *= 1e-37
    check(d, attend(d, unpacked, scale=scale), scale)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("W", [1, 60])
def test_scales_below_the_normal_numbers_over_16_bit_pages(dtype, W):
    d = make16(22, "cuda", dtype, 2, W, 8, 2, 128, 16, [100, 37])
    got = ops.paged.attention(d["q"], d["k_cache"], d["v_cache"], d["table"], d["positions"], scale=1e-39)
    want, size = oracle16(d["q"], d["k_cache"], d["v_cache"], d["table"], d["positions"], 1e-39)
    assert bool(((got.double() - want).abs() <= torch.finfo(dtype).eps / 2 * (want.abs() + size) + 2.0 ** -13 * size + 1e-7).all())


def key_roundings(d, scale=None):
    """What unpacked keys, rounded to halves, do to the weights.  Each number is off by 2^-11 of itself at most, evenly spread and for itself, a score by six standard deviations of their
    sum; by that a weight, and by that the sum of all."""
    D = d["q"].shape[-1]
    scale = D ** -0.5 if scale is None else scale
    k, most = values(d["k_pages"]), 0.0
    for b in range(d["q"].shape[0]):
        table = d["table"][b].clone()
        if d["shared_pages"] is not None:
            table[:len(d["shared_pages"])] = d["shared_pages"]
        keys = k[table[(table >= 0) & (table < k.shape[0])].long()].flatten(0, 1).nan_to_num(0.0)
        q = d["q"][b].double().unflatten(1, (keys.shape[1], -1))
        most = max([most, *(float(torch.einsum("wgd,nd->wgn", q[:, h] ** 2, keys[:, h] ** 2).amax()) for h in range(keys.shape[1]))])
    return 2 * 6 * 2.0 ** -11 / 3 ** 0.5 * scale * most ** 0.5


@pytest.mark.parametrize("layout", ["heads", "rows", "slice"])
@pytest.mark.parametrize("D, B, W, H, Hkv, ps, positions, lens", [
    (64, 2, 300, 8, 2, 64, [500, 30], [300, 111]),
    (128, 2, 300, 8, 2, 64, [500, 30], [300, 111]),
    (64, 3, 128, 6, 1, 16, [-1, 0, 700], None),
    (128, 3, 100, 4, 4, 48, [64, -1, 511], [100, 50, 0]),
    (64, 1, 257, 24, 8, 128, [1000], None),
    (128, 4, 33, 32, 4, 32, [0, 1, 127, 900], [1, 33, 32, 7]),
])
def test_portions(D, B, W, H, Hkv, ps, positions, lens, layout):
    """Heads of either size, in groups and alone, rows that are idle or count in part, pages laid out in every way."""
    d = wide(make(B * W + H, "cuda", BF16, B, W, H, Hkv, D, ps, positions, lens, layout=layout), 40000)
    got = attend(d, True)
    check(d, got, more=key_roundings(d))
    assert torch.equal(got, attend(d, True))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("k_factor, v_factor, v_add, scale", [(6, 1, 0, None), (0, 1, 0, None), (1, 1000, 0, None), (1, 1e-3, 0, None), (1, 1, 300, None), (1, 0, 0, None), (1, 4000, -20000, None),
                                                              (1, 1, 0, 0.01), (1, 1, 0, 0.5), (30, 1, 0, 0.003)])
def test_portions_of_other_sizes(D, k_factor, v_factor, v_add, scale):
    d = wide(make(6, "cuda", BF16, 2, 70, 8, 2, D, 16, [400, 37], k_factor=k_factor, v_factor=v_factor, v_add=v_add), 20000)
    check(d, attend(d, True, scale=scale), scale, key_roundings(d, scale))


@pytest.mark.parametrize("D", [64, 128])
def test_shared_pages_and_holes_in_portions(D):
    d = wide(make(10, "cuda", BF16, 3, 70, 8, 2, D, 16, [64, 90, 33], [70, 1, 0], shared=2), 20000)
    check(d, attend(d, True), more=key_roundings(d))
    d["table"][0, :2] = 1 << 30                              # not looked at
    check(d, attend(d, True), more=key_roundings(d))
    d["table"][1, 3] = -7
    d["table"][0, 4:6] = -1
    d["shared_pages"][1] = d["k_pages"].codes.shape[0]
    check(d, attend(d, True), more=key_roundings(d))
    assert not bool(attend({**d, "table": torch.full_like(d["table"], -1), "shared_pages": None}, True).any())


@pytest.mark.parametrize("factor", [1e-30, 1e-8, 1e4, 1e6])
def test_portions_of_other_queries(factor):
    d = wide(make(8, "cuda", BF16, 2, 80, 8, 2, 128, 16, [100, 37]), 20000)
    d["q"] = d["q"] * factor
    check(d, attend(d, True, scale=0.1 / factor), 0.1 / factor, key_roundings(d, 0.1 / factor))


def test_a_query_of_nan_is_its_own_in_portions():
    d = wide(make(9, "cuda", BF16, 2, 80, 8, 2, 128, 16, [100, 37]), 20000)
    clean = attend(d, True)
    d["q"] = d["q"].clone()
    d["q"][0, 11, 3] = float("nan")
    got = attend(d, True)
    assert bool(got[0, 11, 3].isnan().all())
    got[0, 11, 3] = clean[0, 11, 3]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("W, H, Hkv, cols", [(1, 8, 8, 2100), (3, 8, 8, 2100), (2, 8, 1, 2100), (5, 16, 8, 2100)])
def test_many_pairs_behind_wide_tables(W, H, Hkv, cols):
    """More pairs than blocks, dealt out because the table is wide: cut pairs are joined by the block in front of whose share they are cut."""
    B = 300 // Hkv + 1
    positions = [(37 * i) % 900 for i in range(B)]
    positions[3], positions[7], positions[11] = -1, 33000, 0
    d = make(W + H, "cuda", BF16, B, W, H, Hkv, 64, 16, [p if p < 5000 else 900 for p in positions])
    d["table"] = torch.cat([d["table"], torch.full((B, cols - d["table"].shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
    long = d["table"][7, :50].repeat(cols // 50 + 1)[:cols]                    # a long sequence, whose pages stand in its table again and again
    d["table"][7] = long
    d["positions"][7] = 33000
    n = _ext.launches()
    got = attend(d)
    assert _ext.launches() == n + 2
    check(d, got)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("W, tokens, unpacked", [(1, 0, False), (6, 0, False), (70, 20000, True)])
def test_numbers_next_to_and_beyond_the_largest_half(D, W, tokens, unpacked):
    """Groups from 0 to the largest half, whose last code stands for more than that, and groups that reach beyond it: finite, and what they are, however many rows there are."""
    d = wide(make(31, "cuda", BF16, 2, W, 8, 2, D, 16, [300, 37]), tokens)
    for n in ("k_pages", "v_pages"):
        steps = d[n].steps
        s, m = steps[..., 0, :].float(), steps[..., 1, :].float()
        far = torch.arange(s.shape[-1], device="cuda") % 2 == 1
        # of 2.2 below and above: 0 to 65520, and 40000 to 75000 and more
        steps[..., 0, :] = torch.where(s.isnan(), s, torch.where(far, s * 8000, 4368.0)).half()
        steps[..., 1, :] = torch.where(m.isnan(), m, torch.where(far, m * 8000 + 56000, 0.0)).half()
    most = float(values(d["v_pages"]).nan_to_num(0.0).max())
    assert 70000 < most < 131008
    got = attend(d, unpacked, scale=1e-5)
    # scores are sums of up to 128 products whose magnitudes add up to 100 here: off by 128 * 2^-24 * 100 < 2^-10 of the weights at most
    check(d, got, 1e-5, key_roundings(d, 1e-5) + 2.0 ** -10)


@pytest.mark.parametrize("tokens, unpacked", [(1 << 21, True), ((1 << 21) + 16, False), (1 << 28, False)])
def test_portions_behind_tables_of_millions_of_tokens(tokens, unpacked):
    """Unpacked heads take 1 GB at most, however wide the table is."""
    d = wide(make(41, "cuda", BF16, 1, 60, 4, 1, 128, 16, [100]), tokens)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = attend(d, unpacked)
    assert torch.cuda.max_memory_allocated() - before < 1.1 * 2 ** 30
    check(d, got, more=key_roundings(d))


def test_portions_captured_twice_on_another_stream():
    """Two captured portions whose pages are unpacked, one in several turns, replayed after each other on a stream of their own, give what the calls give."""
    a = wide(make(51, "cuda", BF16, 2, 70, 8, 2, 64, 16, [100, 50]), 20000)
    b = wide(make(52, "cuda", BF16, 3, 48, 2, 1, 128, 128, [300, 17, 411]), 200000)
    want = attend(a, True), attend(b, True)
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
