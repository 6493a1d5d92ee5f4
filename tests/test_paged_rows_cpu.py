"""Rows of a paged cache as a model's callers use them: what has no page, or lies behind ``max_seq_len``, is refused and never left out quietly."""
import pytest
import torch

from dist_utils import run_distributed


def _model(pages=None, batch=2, length=128, logits=False, **kw):
    from neuronx_distributed_b200.models.llama import LlamaConfig
    from neuronx_distributed_b200.models.llama_inference import LlamaForInference

    torch.manual_seed(1)
    cfg = LlamaConfig(vocab_size=96, hidden_size=32, intermediate_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      dtype=torch.float32, max_position_embeddings=128)
    return LlamaForInference(cfg, batch_size=batch, max_seq_len=length, page_size=pages, on_device_sampling=not logits, **kw).eval()


def _start(world=1):
    from neuronx_distributed_b200.parallel_layers import parallel_state as ps

    ps.initialize_model_parallel(tensor_model_parallel_size=world)


def _ids(seed, *shape):
    return torch.randint(0, 96, shape, generator=torch.Generator().manual_seed(seed))


def _longest_sequence(rank, world):
    from neuronx_distributed_b200.utils.speculative import speculative_generate

    _start()
    prompts = _ids(3, 2, 40)
    rows, pages = _model(length=50), _model(48, length=50)       # two pages of 48 would hold 96 tokens, the rotation tables end at 50
    assert torch.equal(rows.generate(prompts, 11), pages.generate(prompts, 11))          # the last token of the eleven has no place of its own
    for call in (lambda: pages.generate(prompts, 12), lambda: pages.context_encoding(_ids(4, 2, 60)), lambda: pages.share_prefix(_ids(5, 96))):
        with pytest.raises(ValueError, match="max_seq_len 50"):
            call()
    for tokens in (51, 96):
        with pytest.raises(ValueError):
            pages.kv.reserve(0, tokens)
        with pytest.raises(ValueError):
            pages.kv.reserve_rows(2, tokens)
    one = _model(48, batch=1, length=50)
    with pytest.raises(ValueError):
        speculative_generate(one, _model(48, batch=1, length=50), prompts[:1], 24, 4)
    want = _model(batch=1, length=50).generate(prompts[:1], 10)
    assert torch.equal(speculative_generate(one, _model(48, batch=1, length=50), prompts[:1], 10, 4)[0], want)


def _steps_over_page_borders(rank, world):
    """Prompt, then single tokens and windows, over several page borders, with nobody reserving: as contiguous rows."""
    _start()
    ids, lens = _ids(6, 2, 14), torch.tensor([14, 5])
    rows, pages = _model(logits=True), _model(16, logits=True)
    steps = []
    for m in (rows, pages):
        out, pos = [m.context_encoding(ids, lens - 1)], lens.clone()
        for i in range(40):                                     # every fourth step a window of five, of which two stay
            w = 5 if i % 4 == 3 else 1
            step = m.speculation_forward if w > 1 else m.token_generation
            out.append(step(_ids(50 + i, 2, w), pos).reshape(2, w, -1))
            pos = pos + (2 if w > 1 else 1)
        steps.append(out)
    for a, b in zip(*steps):
        torch.testing.assert_close(b, a, rtol=1e-5, atol=1e-5)
    assert pages.kv.free_pages == 16 - 5 - 4                   # rows end at 14 + 50 (windows reach 3 further: 67) and 5 + 50 (58)
    # a row that stands at -1 is idle and takes no pages, whatever its number of tokens before
    pages.kv.release(1)
    free = pages.kv.free_pages
    a = rows.token_generation(ids[:, :1], torch.tensor([64, 0]))[0]
    b = pages.token_generation(ids[:, :1], torch.tensor([64, -1]))[0]
    torch.testing.assert_close(b, a, rtol=1e-5, atol=1e-5)
    assert pages.kv.free_pages == free
    # steps behind the longest sequence are refused, as contiguous rows refuse them; so are steps for which the pool has no page
    for m in (rows, pages):
        with pytest.raises((ValueError, IndexError)):
            m.token_generation(ids[:, :1], torch.tensor([128, 3]))
    with pytest.raises(ValueError):
        pages.speculation_forward(_ids(7, 2, 5), torch.tensor([124, 3]))
    small = _model(16, num_pages=3)
    small.context_encoding(ids, lens - 1)
    small.token_generation(ids[:, :1], torch.tensor([14, 5]))
    small.token_generation(ids[:, :1], torch.tensor([15, 6]))
    small.token_generation(ids[:, :1], torch.tensor([16, 7]))  # the third page
    with pytest.raises(RuntimeError, match="pool"):
        small.token_generation(ids[:, :1], torch.tensor([17, 16]))
    # a row that starts over reserves anew
    small.kv.release(0)
    small.token_generation(ids[:, :1], torch.tensor([-1, 16]))
    assert small.kv.free_pages == 1 and int((small.kv.page_table[0] >= 0).sum()) == 0


def _adapter(rank, world):
    """The transformers-like generate over pages: as over contiguous rows, behind a shared prefix too, which it keeps."""
    from neuronx_distributed_b200.inference.hf_adapter import HuggingFaceGenerationAdapter

    _start()
    ids, mask = _ids(8, 2, 14), torch.ones(2, 14, dtype=torch.long)
    mask[1, :6] = 0                                             # left-padded
    rows, pages = HuggingFaceGenerationAdapter(_model()), HuggingFaceGenerationAdapter(_model(16))
    want = rows.generate(ids, mask, max_new_tokens=40)
    for _ in range(2):
        assert torch.equal(pages.generate(ids, mask, max_new_tokens=40), want)
    drawn = [a.generate(ids, mask, max_new_tokens=20, do_sample=True, top_k=5, generator=torch.Generator().manual_seed(2)) for a in (rows, pages)]
    assert torch.equal(*drawn)
    assert torch.equal(pages.generate(ids, mask), rows.generate(ids, mask))              # as far as max_seq_len goes
    # steps that wait for nothing: the same when the model's steps may not reserve
    m = _model(16)
    m.kv.cover = lambda positions, tokens: (_ for _ in ()).throw(AssertionError()) if not m.kv._ahead else None
    assert torch.equal(HuggingFaceGenerationAdapter(m).generate(ids, mask, max_new_tokens=40), want)
    # behind a prefix
    prefix = _ids(9, 32)
    whole, lens = torch.zeros(2, 46, dtype=torch.long), [14, 8]
    long_mask = torch.zeros(2, 46, dtype=torch.long)
    for b, n in enumerate(lens):
        whole[b, 46 - 32 - n:] = torch.cat([prefix, ids[b, 14 - n:]])
        long_mask[b, 46 - 32 - n:] = 1
    want = rows.generate(whole, long_mask, max_new_tokens=30)[:, 46:]
    shared = _model(16)
    shared.share_prefix(prefix)
    adapter = HuggingFaceGenerationAdapter(shared)
    for _ in range(2):
        assert torch.equal(adapter.generate(ids, mask, max_new_tokens=30)[:, 14:], want)
        assert shared.kv.shared_tokens == 32
    full = adapter.generate(ids, mask)
    assert full.shape[1] == 14 + 128 - 32 - 14 and torch.equal(full[:, 14:], rows.generate(whole, long_mask)[:, 46:])
    # prompts as wide as they come go to the programs, which were captured for that width
    seen = []
    adapter.use_programs(lambda i, last: seen.append(tuple(i.shape)) or shared.context_encoding(i, last), shared.token_generation)
    wide, wide_mask = torch.cat([ids, ids[:, :4]], 1), torch.cat([mask, torch.zeros(2, 4, dtype=torch.long)], 1)
    assert torch.equal(adapter.generate(wide, wide_mask, max_new_tokens=30)[:, 18:], want) and seen == [(2, 18)]
    # a pool with just enough pages for one call at a time
    small = _model(16, num_pages=2 + 2 * 3)
    small.share_prefix(prefix)
    for _ in range(2):
        assert torch.equal(HuggingFaceGenerationAdapter(small).generate(ids, mask, max_new_tokens=30)[:, 14:], want)
    with pytest.raises(RuntimeError, match="pool"):
        HuggingFaceGenerationAdapter(small).generate(ids, mask, max_new_tokens=40)
    assert small.kv.shared_tokens == 32 and not small.kv._ahead


def _record(call, *inputs):
    from neuronx_distributed_b200.inference import launch_plan

    return launch_plan.record(call, inputs)


def _programs_and_prefixes(rank, world):
    """A recorded program reads the pages of the prefix there is when it runs; a prefix of another length, which it cannot know, is refused."""
    _start()
    ids, lens = _ids(10, 2, 10), torch.tensor([10, 4])
    x, pos = ids[:, :1].contiguous(), lens + 48
    m = _model(16, logits=True, num_pages=12)
    m.share_prefix(_ids(11, 48))
    m.context_encoding(ids, lens - 1)
    m.kv.reserve_rows(2, 64)
    at = m.kv.shared_pages.data_ptr()
    step = _record(m.token_generation, x, pos)
    torch.testing.assert_close(step(x, pos), m.token_generation(x, pos), rtol=0, atol=0)
    # another prefix, in other pages
    m.kv.release(0)
    m.share_prefix(_ids(12, 48))
    m.context_encoding(ids, lens - 1)
    m.kv.reserve_rows(2, 64)
    assert m.kv.shared_pages.data_ptr() == at
    fresh = _model(16, logits=True)
    fresh.share_prefix(_ids(12, 48))
    fresh.context_encoding(ids, lens - 1)
    want = fresh.token_generation(x, pos)
    torch.testing.assert_close(step(x, pos), want, rtol=0, atol=0)
    torch.testing.assert_close(m.token_generation(x, pos), want, rtol=0, atol=0)
    held, free = m.kv.shared_pages.tolist(), m.kv.free_pages
    for n in (0, 32, 64):
        with pytest.raises(RuntimeError, match="captured"):
            m.share_prefix(_ids(13, n))
    with pytest.raises(RuntimeError, match="captured"):
        m.kv.reset()
    assert m.kv.shared_pages.tolist() == held and m.kv.free_pages == free
    torch.testing.assert_close(step(x, pos), want, rtol=0, atol=0)
    m.kv.forget_programs()                                      # the step above is not run any more
    m.share_prefix(_ids(13, 32))
    assert m.kv.shared_tokens == 32
    m.kv.reset()
    assert m.kv.shared_pages is None and m.kv.free_pages == 12
    # pages are handed out on the host: a program cannot take any, nor keep a prefix
    with pytest.raises(RuntimeError, match="captured"):
        _record(m.context_encoding, ids, lens - 1)
    with pytest.raises(RuntimeError, match="captured"):
        _record(m.share_prefix, _ids(13, 32))
    m.kv.reserve(0, 16)
    with pytest.raises(RuntimeError, match="captured"):
        _record(lambda t: m.kv.release(0) or t, ids)
    m.kv.release(0)
    assert m.kv.free_pages == 12 and not bool((m.kv.page_table >= 0).any())


def _programs_without_pages(rank, world):
    """A program that runs for tokens without a page says so at the next look: after a release, past the reserved pages, past max_seq_len."""
    _start()
    ids, lens = _ids(14, 2, 10), torch.tensor([10, 4])
    x = ids[:, :1].contiguous()
    m = _model(16, logits=True, length=50)
    m.kv.reserve_rows(2, 16)
    prompt, step = _record(m.context_encoding, ids, lens - 1), _record(m.token_generation, x, lens)
    want = [m.context_encoding(ids, lens - 1), m.token_generation(x, lens)]

    def run(at):
        torch.testing.assert_close(prompt(ids, lens - 1), want[0], rtol=0, atol=0)
        got = step(x, at)
        if torch.equal(at, lens):
            torch.testing.assert_close(got, want[1], rtol=0, atol=0)

    run(lens)
    m.kv.check()
    run(torch.tensor([15, -1]))
    m.kv.check()
    m.kv.release(0)
    m.kv.reserve(0, 16)
    run(lens)
    m.kv.check()
    step(x, torch.tensor([16, 4]))                              # behind its one page
    with pytest.raises(RuntimeError, match="without a page"):
        m.kv.check()
    m.kv.check()                                                # said once
    m.kv.release(1)
    step(x, torch.tensor([-1, 4]))
    with pytest.raises(RuntimeError, match="without a page"):
        m.kv.release(0)
    prompt(ids, lens - 1)
    with pytest.raises(RuntimeError, match="without a page"):
        m.kv.reset()
    m.kv.reserve_rows(2, 50)
    run(torch.tensor([49, 49]))
    m.kv.check()
    step(x, torch.tensor([50, 3]))                              # its last page has room, the rotation tables end
    with pytest.raises(RuntimeError, match="without a page"):
        m.kv.reset()
    run(lens)
    m.kv.reset()
    m.kv.reset()
    prompt(ids, lens - 1)
    m.kv.forget_programs()
    m.kv.check()


def _plans_without_their_weights_part(rank, world):
    """A launch plan whose weight-only part has been taken out goes by the tables as they are, not as they were then."""
    from neuronx_distributed_b200.inference.launch_plan import LaunchPlan

    _start()
    ids, lens = _ids(15, 2, 10), torch.tensor([10, 4])
    x = ids[:, :1].contiguous()
    for prefix in (0, 32):
        m, pos = _model(16, logits=True), lens + prefix
        m.share_prefix(_ids(16, prefix))
        m.context_encoding(ids, lens - 1)
        plan = _record(m.token_generation, x, pos)
        transformer, main, _ = plan.hoist_weight_only()
        assert transformer.nodes
        main.apply_transformer(transformer)
        stored = LaunchPlan.from_json(plan.to_json()).bind(plan.named_constants())
        again, rest, _ = stored.hoist_weight_only()
        rest.apply_transformer(again)
        before = m.kv.page_table.clone()
        for turn in range(2):
            want = m.token_generation(x, pos)
            for p in (plan, main, rest):
                torch.testing.assert_close(p(x, pos), want, rtol=0, atol=0)
            if turn == 0:                                       # rows change their pages, and the prefix its own
                m.kv.release(0)
                m.share_prefix(_ids(17, prefix))
                m.kv.reserve(1, prefix + 30)
                m.context_encoding(ids, lens - 1)
                assert not torch.equal(m.kv.page_table, before)


def _prefix_that_fails(rank, world):
    """A prefix whose encoding fails is not kept: its pages hold nothing that a row may begin with."""
    _start()
    m, ids = _model(16, logits=True), _ids(18, 2, 10)
    want = m.context_encoding(ids)
    body = m._body
    m._body = lambda *a: (_ for _ in ()).throw(MemoryError("no room"))
    with pytest.raises(MemoryError):
        m.share_prefix(_ids(19, 32))
    m._body = body
    assert m.kv.shared_tokens == 0 and m.kv.shared_pages is None and m.kv.free_pages == 16
    torch.testing.assert_close(m.context_encoding(ids), want, rtol=0, atol=0)
    # behind a prefix that programs count on: they are not run without one, and another of its length can be shared
    m.kv.reset()
    m.share_prefix(_ids(19, 32))
    m.context_encoding(ids)
    x = ids[:, :1].contiguous()
    pos = torch.tensor([42, 42])
    step = _record(m.token_generation, x, pos)
    m._body = lambda *a: (_ for _ in ()).throw(MemoryError("no room"))
    with pytest.raises(MemoryError):
        m.share_prefix(_ids(20, 32))
    m._body = body
    assert m.kv.shared_tokens == 0 and m.kv.free_pages == 16
    step(x, pos)
    with pytest.raises(RuntimeError, match="without a page"):
        m.kv.check()
    m.share_prefix(_ids(20, 32))
    m.context_encoding(ids)
    torch.testing.assert_close(step(x, pos), m.token_generation(x, pos), rtol=0, atol=0)
    m.kv.check()


def _rows_keep_out_of_the_prefix(rank, world):
    """A token of one row inside the shared prefix would change it for all rows: refused, and the prefix is as it was."""
    _start()
    m, ids, lens = _model(16, logits=True), _ids(23, 2, 10), torch.tensor([10, 4])
    m.share_prefix(_ids(24, 32))
    m.context_encoding(ids, lens - 1)
    pool = [t.clone() for t in m.kv.k + m.kv.v]
    for pos in ([10, 4], [42, 31], [0, -1]):                    # positions that do not count the prefix, or all of it
        with pytest.raises(ValueError, match="shared prefix"):
            m.token_generation(ids[:, :1], torch.tensor(pos))
        with pytest.raises(ValueError, match="shared prefix"):
            m.speculation_forward(ids[:, :3], torch.tensor(pos))
    assert all(torch.equal(a, b) for a, b in zip(pool, m.kv.k + m.kv.v))
    m.token_generation(ids[:, :1], torch.tensor([32, -1]))      # the first token behind it


def _kv_len_and_experts(rank, world):
    """kv_len, which contiguous rows read no further than, changes nothing over pages; a model of routed experts goes by them as well."""
    from neuronx_distributed_b200.models.llama_inference import LlamaForInference
    from neuronx_distributed_b200.models.mixtral import MixtralConfig, MixtralForCausalLM

    _start()
    ids, lens = _ids(21, 2, 14), torch.tensor([14, 5])
    rows, pages = _model(logits=True), _model(16, logits=True)
    for m in (rows, pages):
        m.context_encoding(ids, lens - 1)
    pos = lens                                                  # no position is left out: keys that nobody wrote are whatever a cache held before
    for i in range(6):
        w = 1 + 3 * (i % 2)
        call = "speculation_forward" if w > 1 else "token_generation"
        a, b, c = (getattr(m, call)(_ids(30 + i, 2, w), pos, **kw) for m, kw in ((rows, {"kv_len": 48}), (pages, {"kv_len": 48}), (pages, {})))
        torch.testing.assert_close(b.reshape(a.shape), a, rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(b, c, rtol=0, atol=0)
        pos = pos + w
    out = []
    for page in (None, 16):
        torch.manual_seed(3)
        cfg = MixtralConfig(vocab_size=64, hidden_size=32, intermediate_size=48, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                            num_local_experts=4, num_experts_per_tok=2, dtype=torch.float32, max_position_embeddings=64)
        m = LlamaForInference(cfg, batch_size=2, max_seq_len=64, lm_cls=MixtralForCausalLM, page_size=page).eval()
        out.append(m.generate(_ids(22, 2, 9) % 64, 30, torch.tensor([9, 4])))
    assert torch.equal(*out)


@pytest.mark.parametrize("part", [_longest_sequence, _steps_over_page_borders, _adapter, _programs_and_prefixes, _programs_without_pages,
                                  _plans_without_their_weights_part, _prefix_that_fails, _kv_len_and_experts, _rows_keep_out_of_the_prefix])
def test_rows(part):
    run_distributed(part, 1, timeout=240)


# first positions, lens, whether a token that counts has no place: tables of three pages of 16 tokens (-1, 9: no page), rotation tables of 40 rows
LOST = [([0, 14, 30], None, False), ([0, 14, 30], [2, 2, 3], False), ([31, 0, 0], None, True), ([31, 0, 0], [1, 2, 2], False),
        ([0, 15, 0], None, True), ([0, 15, 0], [2, 1, 2], False), ([0, -1, 30], None, False), ([0, 0, 32], None, True), ([0, 0, 39], None, True),
        ([0, 0, 38], [2, 2, 0], False), ([40, 0, 0], None, True), ([40, 0, 0], [0, 2, 2], False), ([1 << 40, 0, 0], None, True), ([-5, -1, -9], None, False)]


def append_notes(device, dtype, first, lens, noted):
    from neuronx_distributed_b200 import ops

    B, W, H, D, ps = 3, 2, 2, 16, 16
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(B, W, H, D, generator=g).to(device, dtype) for _ in range(3))
    cos, sin = (t.to(device) for t in ops.rope.rope_tables(40, D))
    table = torch.tensor([[0, 1, -1], [2, -1, -1], [3, 4, 9]], dtype=torch.int32, device=device)         # of six pages
    lost = torch.zeros(1, dtype=torch.int32, device=device)
    kc, vc = (torch.zeros(6, ps, H, D, device=device, dtype=dtype) for _ in range(2))
    args = (q, k, v, torch.tensor(first, device=device), cos, sin, kc, vc, table)
    lens = None if lens is None else torch.tensor(lens, device=device)
    ops.paged.rope_append(*args, lens=lens, lost=lost)
    assert int(lost) == noted
    lost.fill_(1)
    out = ops.paged.rope_append(*args, lens=lens, lost=lost)                     # it is never taken back
    assert int(lost) == 1 and torch.equal(out, ops.paged.rope_append(*args, lens=lens))
    for bad in (torch.zeros(1), torch.zeros(2, dtype=torch.int32), torch.zeros((), dtype=torch.int32)):
        with pytest.raises(ValueError, match="lost"):
            ops.paged.rope_append(*args, lost=bad.to(device))


@pytest.mark.parametrize("first, lens, noted", LOST)
def test_append_notes_tokens_without_a_place(first, lens, noted):
    # the second row's second page is missing, the third row's third page lies outside the pool
    append_notes("cpu", torch.float32, first, lens, noted)


def test_manager_ends_at_max_seq_len():
    from neuronx_distributed_b200.inference.paged_cache import PagedKVCacheManager

    kv = PagedKVCacheManager(1, 2, 100, 1, 8, page_size=32, dtype=torch.float32)
    kv.reserve(0, 100)
    assert kv.free_pages == 4
    for call in (lambda: kv.reserve(1, 101), lambda: kv.reserve_rows(2, 128), lambda: kv.take_shared(128)):
        with pytest.raises(ValueError, match="max_seq_len 100"):
            call()
    assert kv.free_pages == 4 and kv.shared_pages is None and int((kv.page_table[0] >= 0).sum()) == 4
    kv.take_shared(96)
    assert kv.shared_tokens == 96


def test_example_refuses_sampling_on_tensor_parallel_ranks():
    """Before any model is built: the whole rows of logits that sampled speculation goes by are not there."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, "examples", "inference", "run_llama_speculative.py"), "--temperature", "0.8", "--tp_degree", "2"],
                       capture_output=True, text=True, timeout=240)
    assert r.returncode == 2 and "--tp_degree 1" in r.stderr, r.stderr[-500:]
