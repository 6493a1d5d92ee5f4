"""The cache in 4 bits (``ops.paged_int4``) in plain torch against its definition in 64 bits, and what it refuses."""
import pytest
import torch

from paged_int4_cases import append, attention, bound, make, packed, rotate, values

from neuronx_distributed_b200 import ops
from neuronx_distributed_b200.ops.paged_int4 import Pages

F32, BF16 = torch.float32, torch.bfloat16


def test_pack_and_unpack():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 3, 96, generator=g) * torch.logspace(-6, 4, 5)[:, None, None]
    x[0, 0, :32] = 0.25                                      # no range at all
    x[1, 1, 5] = float("nan")
    x[2, 2, 40] = 1e6                                        # beyond half precision
    got, want = ops.paged_int4.pack(x), packed(x)
    assert torch.equal(got.codes, want.codes) and torch.equal(got.steps.view(torch.int16), want.steps.view(torch.int16))
    v = ops.paged_int4.unpack(got, torch.float64)
    assert torch.equal(v.nan_to_num(), values(got).nan_to_num())
    assert torch.equal(ops.paged_int4.unpack(got, BF16).nan_to_num(), v.float().to(BF16).nan_to_num())
    assert bool((v[0, 0, :32] == 0.25).all()) and bool(v[1, 1, :32].isnan().all()) and bool(v[1, 1, 32:].isfinite().all())
    assert not bool(v[2, 2, 32:64].isfinite().any())
    # half a step, and what the roundings of m and s (2^-11 each, and 2^-25 where they are denormal) move the ends by
    s, m = got.steps.double()[..., 0, :].repeat_interleave(32, -1), got.steps.double()[..., 1, :].repeat_interleave(32, -1)
    off = (v - x.double()).abs()
    ok = v.isfinite()
    assert bool((off <= s / 2 + 2.0 ** -11 * (15 * s + m.abs()) + 16 * 2.0 ** -25)[ok].all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("half", [0, 1, 8, 16, 32])
def test_append_and_gather(half, interleaved):
    B, W, H, Hkv, D, ps = 3, 5, 4, 2, 64, 16
    g = torch.Generator().manual_seed(half)
    q, k, v = (torch.randn(B, W, h, D, generator=g) for h in (H, Hkv, Hkv))
    cos, sin = torch.rand(40, half, generator=g), torch.rand(40, half, generator=g)
    positions = torch.tensor([0, 33, 37])                    # the last row runs out of the rotation tables
    slots = torch.randperm(4 * ps, generator=g)[:B * W].view(B, W).int()
    slots[1, 2], slots[0, 0] = -1, 4 * ps
    pages = [ops.paged_int4.new_pages(4, ps, Hkv, D) for _ in "kv"]
    for p in pages:
        p.codes.fill_(7)
    want_q, written = append(q, k, v, positions, cos, sin, slots, 4 * ps, interleaved)
    lost = torch.zeros(1, dtype=torch.int32)
    got = ops.paged_int4.append(q, k, v, positions, cos, sin, *pages, slots, interleaved=interleaved, lost=lost)
    assert int(lost) == 1
    torch.testing.assert_close(got.double(), want_q, rtol=2.0 ** -24, atol=1e-12)
    for i, p in enumerate(pages):
        for slot in range(4 * ps):
            here = Pages(p.codes[slot // ps, slot % ps], p.steps[slot // ps, slot % ps])
            if slot in written:
                want = packed(written[slot][i])
                assert torch.equal(here.codes, want.codes) and torch.equal(here.steps, want.steps)
            else:
                assert bool((here.codes == 7).all()) and bool((here.steps == 0).all())
    back = ops.paged_int4.gather(*pages, slots, F32)
    for x, p in zip(back, pages):
        want = values(p)
        for b in range(B):
            for w in range(W):
                slot = int(slots[b, w])
                assert torch.equal(x[b, w], want[slot // ps, slot % ps].float() if 0 <= slot < 4 * ps else torch.zeros(Hkv, D))


@pytest.mark.parametrize("B, W, H, Hkv, D, ps, positions, lens, kw", [
    (1, 1, 2, 1, 64, 16, [0], None, {}),
    (3, 2, 4, 2, 32, 16, [-1, 14, 40], None, {"garbage": float("nan")}),
    (2, 9, 6, 2, 64, 48, [100, 0], [9, 4], {"layout": "rows"}),
    (3, 3, 4, 4, 32, 16, [40, 33, 50], [3, 0, 2], {"shared": 2, "layout": "slice"}),
])
def test_attention(B, W, H, Hkv, D, ps, positions, lens, kw):
    d = make(3, "cpu", F32, B, W, H, Hkv, D, ps, positions, lens, **kw)
    d["table"][0, 0] = -5 if B == 2 else d["table"][0, 0]
    got = ops.paged_int4.attention(d["q"], d["k_pages"], d["v_pages"], d["table"], d["positions"], lens=d["lens"], shared_pages=d["shared_pages"])
    want, size = attention(d)
    assert bool(((got.double() - want).abs() <= bound(F32, want, size)).all())
    assert got.transpose(0, 1).is_contiguous()


def refusals(device):
    d = make(1, device, BF16, 2, 3, 4, 2, 64, 16, [3, 20])
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
    kp, vp = d["k_pages"], d["v_pages"]
    tables = z(64, 32), z(64, 32)
    slots = torch.arange(6, dtype=torch.int32, device=device).view(2, 3)
    bad_pages = [Pages(kp.codes.int(), kp.steps), Pages(kp.codes, kp.steps.float()), Pages(kp.codes[:, :, :1], kp.steps), Pages(kp.codes[..., :16], kp.steps),
                 Pages(kp.codes[:, :8], kp.steps[:, :8]), Pages(kp.codes[0], kp.steps[0]), Pages(kp.codes[:0], kp.steps[:0])]
    good = dict(q=d["q"], k=d["k"], v=d["v"], positions=d["positions"], cos=tables[0], sin=tables[1], k_pages=kp, v_pages=vp, slots=slots)
    bad = [("q", d["q"][..., :32]), ("q", d["q"][:, :, :3]), ("q", d["q"][0]), ("q", d["q"].float()), ("k", d["k"][:, :2]), ("v", d["v"].half()), ("positions", d["positions"][:1]),
           ("cos", z(64, 16)), ("cos", z(64, 32, dtype=BF16)), ("slots", slots[:, :2]), ("slots", slots.float()), ("lost", z(1)), ("lost", z(2, dtype=torch.int32))]
    for name, value in bad + [("k_pages", p) for p in bad_pages] + [("v_pages", p) for p in bad_pages]:
        with pytest.raises(ValueError):
            ops.paged_int4.append(**{**good, name: value})
    with pytest.raises(ValueError):
        ops.paged_int4.append(**{**good, "cos": z(64, 40), "sin": z(64, 40)})
    ops.paged_int4.append(**good)
    for args in ((kp, vp, slots[0]), (kp, vp, slots.float()), (kp, vp, slots, torch.int32), *((p, vp, slots) for p in bad_pages), *((kp, p, slots) for p in bad_pages)):
        with pytest.raises(ValueError):
            ops.paged_int4.gather(*args)
    good = dict(q=d["q"], k_pages=kp, v_pages=vp, page_table=d["table"], positions=d["positions"])
    bad = [("q", d["q"][..., :32]), ("q", d["q"][:, :, :3]), ("q", d["q"][0]), ("q", d["q"][:, :, :0]), ("page_table", d["table"][:1]), ("page_table", d["table"][0]),
           ("positions", d["positions"][:1]), ("lens", d["positions"][:1]), ("scale", 0.0), ("scale", -1.0), ("scale", float("nan")), ("scale", float("inf")),
           ("shared_pages", d["table"]), ("shared_pages", torch.zeros(d["table"].shape[1] + 1, dtype=torch.int32, device=device))]
    for name, value in bad + [("k_pages", p) for p in bad_pages] + [("v_pages", p) for p in bad_pages]:
        with pytest.raises(ValueError):
            ops.paged_int4.attention(**{**good, name: value})
    ops.paged_int4.attention(**good)
    for name in ("q", "k", "v"):
        x = {**dict(q=d["q"], k=d["k"], v=d["v"]), name: d[name].detach().clone().requires_grad_()}
        with pytest.raises(RuntimeError):
            ops.paged_int4.append(x["q"], x["k"], x["v"], d["positions"], *tables, kp, vp, slots)
    with pytest.raises(RuntimeError):
        ops.paged_int4.attention(d["q"].detach().clone().requires_grad_(), kp, vp, d["table"], d["positions"])


def test_refusals():
    refusals("cpu")
    for args in ((4, 24, 2, 64), (4, 0, 2, 64), (4, 16, 2, 48), (4, 16, 2, 0), (0, 16, 2, 64), (4, 16, 0, 64)):
        with pytest.raises(ValueError):
            ops.paged_int4.new_pages(*args)
    with pytest.raises(ValueError):
        ops.paged_int4.pack(torch.zeros(4, 40))


def test_empty_calls():
    d = make(1, "cpu", F32, 2, 3, 4, 2, 64, 16, [3, 20])
    none = torch.zeros(2, 0, dtype=torch.int32)
    got = ops.paged_int4.attention(d["q"], d["k_pages"], d["v_pages"], none, d["positions"])
    assert got.shape == d["q"].shape and not bool(got.any())
    assert ops.paged_int4.attention(d["q"][:, :0], d["k_pages"], d["v_pages"], d["table"], d["positions"]).shape == (2, 0, 4, 64)
    k, v = ops.paged_int4.gather(d["k_pages"], d["v_pages"], none)
    assert k.shape == v.shape == (2, 0, 2, 64)
    q = ops.paged_int4.append(d["q"][:, :0], d["k"][:, :0], d["v"][:, :0], d["positions"], torch.ones(9, 32), torch.zeros(9, 32), d["k_pages"], d["v_pages"], none)
    assert q.shape == (2, 0, 4, 64)


@pytest.mark.skipif(ops._ext._load() is None, reason="extension not built")
@pytest.mark.parametrize("heads_outside", [False, True])
def test_pools_whose_places_pass_32_bits(heads_outside):
    """The kernels count packets of 16 bytes and rows of steps in 32 bits, heads among them: a pool of 2^32 packets is refused, one of a page less is not."""
    q, table, positions = torch.empty(1, 1, 8, 128, dtype=BF16, device="meta"), torch.empty(1, 4, dtype=torch.int32, device="meta"), torch.empty(1, dtype=torch.long, device="meta")

    def pages(n):
        shape = (8, n, 16) if heads_outside else (n, 8, 16)
        to = (1, 2, 0, 3) if heads_outside else (0, 2, 1, 3)
        codes = torch.empty(*shape, 64, dtype=torch.uint8, device="meta").permute(*to)
        return codes, torch.empty(*shape, 2, 4, dtype=torch.float16, device="meta").permute(*to, 4)

    small, large = pages(2 ** 23 - 1), pages(2 ** 23)
    one = tuple(t[:1].expand(2 ** 23, *t.shape[1:]) for t in small)
    apart = one[0], torch.empty_strided(one[1].shape, (8 * 513, 0, 0, 4, 1), dtype=torch.float16, device="meta")
    for k, v in ((large, one), (one, large), (apart, one), (one, apart)):
        with pytest.raises(ValueError, match="span"):
            ops._ext._load().int4_attention(q, *k, *v, table, positions, None, None, None)
    with pytest.raises(ValueError, match="on a GPU"):
        ops._ext._load().int4_attention(q, *small, *small, table, positions, None, None, None)
    with pytest.raises(ValueError, match="2.31 tokens"):
        ops._ext._load().int4_attention(q, *small, *small, table[:, :1].expand(1, 2 ** 28), positions, None, None, None)
