"""A cache in pages on the CPU path: against the definitions in 64 bits, and what is refused."""
import pytest
import torch

import paged_oracle as oracle
from paged_cases import bound, make

from neuronx_distributed_b200 import ops

CASES = [
    # B, W, H, Hkv, D, ps, positions, lens, shared
    (1, 1, 4, 4, 16, 16, [0], None, 0),
    (3, 1, 4, 2, 16, 16, [0, 15, 40], None, 0),
    (3, 4, 6, 1, 8, 48, [0, 47, 90], [4, 1, 0], 0),
    (4, 3, 4, 2, 16, 16, [-1, 33, 32, 5], None, 2),
    (2, 20, 4, 2, 16, 16, [0, 7], [20, 11], 0),
]


@pytest.mark.parametrize("case", CASES)
def test_append_and_attention(case):
    B, W, H, Hkv, D, ps, positions, lens, shared = case
    d = make(1, "cpu", torch.float32, B, W, H, Hkv, D, ps, positions, lens, shared)
    cos, sin = ops.rope.rope_tables(256, D)
    want_q, want_k, want_v, written = oracle.append(d["q"], d["k"], d["v"], d["positions"], cos, sin, d["k_cache"], d["v_cache"], d["table"], d["lens"])
    before = d["k_cache"].clone(), d["v_cache"].clone()
    q = ops.paged.rope_append(d["q"], d["k"], d["v"], d["positions"], cos, sin, d["k_cache"], d["v_cache"], d["table"], lens=d["lens"])
    # products and their sum in 32 bits: three roundings of numbers below 6
    assert torch.allclose(q.double(), want_q, rtol=0, atol=6 * 3 * 2.0 ** -24)
    for got, want, old in ((d["k_cache"], want_k, before[0]), (d["v_cache"], want_v, before[1])):
        assert torch.allclose(got[written].double(), want[written], rtol=0, atol=6 * 3 * 2.0 ** -24)
        assert torch.equal(got[~written].nan_to_num(), old[~written].nan_to_num())
    out = ops.paged.attention(q, d["k_cache"], d["v_cache"], d["table"], d["positions"], lens=d["lens"], shared_pages=d["shared_pages"])
    want, size = oracle.attention(q, d["k_cache"], d["v_cache"], d["table"], d["positions"], lens=d["lens"], shared_pages=d["shared_pages"])
    assert (out.double() - want).abs().le(bound(torch.float32, want, size)).all()


def test_tokens_outside_tables_and_pool():
    d = make(2, "cpu", torch.float32, 3, 4, 2, 2, 8, 16, [14, 30, 2], None, 0)
    d["table"][0, 1], d["table"][1, 0], d["table"][2, 0] = -1, 10 ** 6, -7
    table = d["table"][:, :2].contiguous()                         # row 1's last tokens stand behind the table's end
    cos, sin = ops.rope.rope_tables(33, 8)                         # and its last one behind the rotation tables'
    want_q, want_k, want_v, written = oracle.append(d["q"], d["k"], d["v"], d["positions"], cos, sin, d["k_cache"], d["v_cache"], table)
    old = d["k_cache"].clone()
    q = ops.paged.rope_append(d["q"], d["k"], d["v"], d["positions"], cos, sin, d["k_cache"], d["v_cache"], table)
    assert int(written.sum()) == 4 and not bool(q[1, 3].any())
    assert torch.allclose(q.double(), want_q, atol=1e-5) and torch.allclose(d["k_cache"][written].double(), want_k[written], atol=1e-5)
    assert torch.equal(d["k_cache"][~written].nan_to_num(), old[~written].nan_to_num())
    out = ops.paged.attention(q, d["k_cache"], d["v_cache"], table, d["positions"])
    want, _ = oracle.attention(q, d["k_cache"], d["v_cache"], table, d["positions"])
    assert torch.allclose(out.double(), want, atol=1e-5) and not bool(out[2].any())


def _good():
    d = make(3, "cpu", torch.float32, 2, 2, 4, 2, 16, 16, [3, 20])
    cos, sin = ops.rope.rope_tables(64, 16)
    append = [d[n] for n in ("q", "k", "v", "positions")] + [cos, sin] + [d[n] for n in ("k_cache", "v_cache", "table")]
    attention = [d[n] for n in ("q", "k_cache", "v_cache", "table", "positions")]
    return append, attention


@pytest.mark.parametrize("which, change", [
    (0, lambda t: t[0]), (0, lambda t: t[..., :8]), (0, lambda t: t[:, :, :3]), (0, lambda t: t.half()),
    (1, lambda t: t[:, :1]), (1, lambda t: t.half()), (2, lambda t: t[:1]), (3, lambda t: t[:1]), (3, lambda t: t[None]),
    (4, lambda t: t[:, :4]), (4, lambda t: t.half()), (5, lambda t: t[:3]), (6, lambda t: t[:, :8]), (6, lambda t: t[:1]), (7, lambda t: t[:, :, :1]),
    (6, lambda t: t.half()), (8, lambda t: t[:1]), (8, lambda t: t[0]),
])
def test_append_refuses(which, change):
    args, _ = _good()
    ops.paged.rope_append(*args)
    args[which] = change(args[which])
    with pytest.raises(ValueError):
        ops.paged.rope_append(*args)


@pytest.mark.parametrize("which, change", [
    (0, lambda t: t[0]), (0, lambda t: t[..., :8]), (0, lambda t: t.double()), (1, lambda t: t[:, :8]), (1, lambda t: t[:, :, :1]), (2, lambda t: t[:1]),
    (3, lambda t: t[:1]), (3, lambda t: t[0]), (4, lambda t: t[:1]),
])
def test_attention_refuses(which, change):
    _, args = _good()
    ops.paged.attention(*args)
    args[which] = change(args[which])
    with pytest.raises(ValueError):
        ops.paged.attention(*args)


def test_refuses_gradients_lens_and_shared_pages():
    append, attention = _good()
    with pytest.raises(ValueError):
        ops.paged.attention(*attention, lens=torch.ones(3, dtype=torch.long))
    with pytest.raises(ValueError):
        ops.paged.attention(*attention, shared_pages=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.paged.attention(*attention, shared_pages=torch.zeros(1, 1, dtype=torch.int32))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            ops.paged.attention(*attention, scale=scale)
    for args, call in ((append, ops.paged.rope_append), (attention, ops.paged.attention)):
        args[0] = args[0].clone().requires_grad_(True)
        with pytest.raises(RuntimeError):
            call(*args)
        with torch.no_grad():
            call(*args)


def test_empty_batches():
    d = make(4, "cpu", torch.float32, 2, 2, 4, 2, 16, 16, [3, 20])
    cos, sin = ops.rope.rope_tables(64, 16)
    for q, k, v, p, t in ((d["q"][:0], d["k"][:0], d["v"][:0], d["positions"][:0], d["table"][:0]), (d["q"][:, :0], d["k"][:, :0], d["v"][:, :0], d["positions"], d["table"]),
                          (d["q"], d["k"], d["v"], d["positions"], d["table"][:, :0])):
        old = d["k_cache"].clone()
        r = ops.paged.rope_append(q, k, v, p, cos, sin, d["k_cache"], d["v_cache"], t)
        assert r.shape == q.shape and torch.equal(old.nan_to_num(), d["k_cache"].nan_to_num())
        o = ops.paged.attention(q, d["k_cache"], d["v_cache"], t, p)
        assert o.shape == q.shape and not bool(o.any())


def test_verify_against_the_definition():
    g = torch.Generator().manual_seed(5)
    B, K, V = 12, 3, 17
    target = torch.softmax(torch.randn(B, K + 1, V, generator=g) * 2, -1)
    draft = torch.softmax(target[:, :K].log() + torch.randn(B, K, V, generator=g) * 0.7, -1)
    tokens = torch.multinomial(draft.view(-1, V), 1, generator=g).view(B, K)
    accept, sample = torch.rand(B, K, generator=g), torch.rand(B, generator=g)
    tokens[0, 1] = -1
    tokens[1] = V
    draft[2] = target[2, :K]                                        # nothing left of p - q: drawn from p
    accept[2] = 1.0
    target[3] = 0.0
    target[4, :, 5] = float("nan")
    target[5, 0] = -1.0
    got, n = ops.select.verify_drafts(tokens, draft, target, accept, sample)
    want, m = oracle.verify(tokens, draft, target, accept, sample)
    assert torch.equal(got, want) and torch.equal(n, m)
    assert 0 < int((n == K).sum()) < B and int(got[3, 0]) == -1
    got, n = ops.select.verify_drafts(tokens[:, :0], draft[:, :0], target[:, :1], accept[:, :0], sample)
    want, m = oracle.verify(tokens[:, :0], draft[:, :0], target[:, :1], accept[:, :0], sample)
    assert torch.equal(got, want) and torch.equal(n, m)


@pytest.mark.parametrize("which, change", [
    (0, lambda t: t.int()), (0, lambda t: t[0]), (1, lambda t: t[:, :1]), (1, lambda t: t[..., :4]), (1, lambda t: t.half()), (2, lambda t: t[:, :2]),
    (2, lambda t: t.double()), (3, lambda t: t[:, :1]), (3, lambda t: t.double()), (4, lambda t: t[:1]), (4, lambda t: t.double()),
])
def test_verify_refuses(which, change):
    args = [torch.zeros(2, 2, dtype=torch.long), torch.full((2, 2, 8), 0.125), torch.full((2, 3, 8), 0.125), torch.rand(2, 2), torch.rand(2)]
    ops.select.verify_drafts(*args)
    args[which] = change(args[which])
    with pytest.raises(ValueError):
        ops.select.verify_drafts(*args)


def test_verify_draws_what_the_target_would():
    """The token behind a window is distributed as the target's own: counts of 40000 first tokens lie within five standard deviations."""
    g = torch.Generator().manual_seed(6)
    V, N = 6, 40000
    p, q = torch.tensor([0.3, 0.05, 0.25, 0.2, 0.15, 0.05]), torch.tensor([0.1, 0.3, 0.2, 0.1, 0.2, 0.1])
    tokens = torch.multinomial(q, N, replacement=True, generator=g).view(N, 1)
    out, _ = ops.select.verify_drafts(tokens, q.expand(N, 1, V).contiguous(), p.expand(N, 2, V).contiguous(), torch.rand(N, 1, generator=g),
                                      torch.rand(N, generator=g))
    counts = torch.bincount(out[:, 0], minlength=V).double()
    assert ((counts - N * p).abs() <= 5 * (N * p * (1 - p)).sqrt()).all()


@pytest.mark.skipif(ops._ext._load() is None, reason="extension not built")
def test_refusals_of_the_extension():
    """The extension's own checks come before anything on a device, with a message each."""
    e = ops._ext._load()
    append, attention = _good()
    bf16 = lambda args: [t.bfloat16() if t.dtype == torch.float32 and t.dim() == 4 else t for t in args]
    for args, call in ((bf16(append), lambda a: e.paged_append(*a, None)), (bf16(attention), lambda a: e.paged_attention(*a, 1.0, None, None))):
        for i, t in enumerate(args):
            changes = [t[:1], t[None]]
            if t.dim() == 2 and t.dtype == torch.float32:                  # rotation tables: of any length
                changes = [t[:, :3], t[None]]
            for x in changes:
                with pytest.raises(ValueError, match=r"[a-z]{4}"):
                    call(args[:i] + [x] + args[i + 1:])
    with pytest.raises(ValueError, match="lens"):
        e.paged_attention(*bf16(attention), 1.0, torch.ones(3, dtype=torch.long), None)
    with pytest.raises(ValueError, match="probabilities"):
        e.verify_drafts(torch.zeros(2, 2, dtype=torch.long), torch.zeros(2, 2, 8), torch.zeros(2, 2, 8), torch.rand(2, 2), torch.rand(2))
