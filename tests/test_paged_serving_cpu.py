"""A Llama model served from a cache in pages: against the same model with contiguous rows, prefixes that all rows share, sampled speculation."""
import pytest
import torch

from dist_utils import run_distributed


def _model(seed, layers=2, pages=None, batch=2, logits=False, **kw):
    from neuronx_distributed_b200.models.llama import LlamaConfig
    from neuronx_distributed_b200.models.llama_inference import LlamaForInference

    torch.manual_seed(seed)
    cfg = LlamaConfig(vocab_size=96, hidden_size=32, intermediate_size=64, num_hidden_layers=layers, num_attention_heads=4, num_key_value_heads=2,
                      dtype=torch.float32, max_position_embeddings=128)
    return LlamaForInference(cfg, batch_size=batch, max_seq_len=128, page_size=pages, on_device_sampling=not logits, **kw).eval()


def _same_as_contiguous(rank, world):
    from neuronx_distributed_b200.parallel_layers import parallel_state as ps

    ps.initialize_model_parallel(tensor_model_parallel_size=world)
    g = torch.Generator().manual_seed(3)
    prompts, lens = torch.randint(0, 96, (2, 21), generator=g), torch.tensor([21, 9])
    rows, pages = _model(1), _model(1, pages=16)
    want, got = rows.generate(prompts, 30, lens), pages.generate(prompts, 30, lens)
    assert torch.equal(want, got)
    # windows of drafted tokens, and logits
    rows, pages = _model(1, logits=True), _model(1, pages=32, logits=True)
    for m in (rows, pages):
        m.context_encoding(prompts, lens - 1)
    pages.kv.reserve_rows(2, 40)
    window = torch.randint(0, 96, (2, 5), generator=g)
    a, b = rows.speculation_forward(window, lens), pages.speculation_forward(window, lens)
    torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
    a, b = rows.token_generation(window[:, :1], lens), pages.token_generation(window[:, :1], lens)
    torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
    with pytest.raises(ValueError):
        pages.speculation_forward(window, lens, tree_mask=torch.ones(5, 5), tree_depth=torch.arange(5))


def _shared_prefix(rank, world):
    from neuronx_distributed_b200.parallel_layers import parallel_state as ps

    ps.initialize_model_parallel(tensor_model_parallel_size=world)
    g = torch.Generator().manual_seed(4)
    prefix, prompts, lens = torch.randint(0, 96, (48,), generator=g), torch.randint(0, 96, (2, 10), generator=g), torch.tensor([10, 4])
    whole, want = _model(2, batch=1), []
    for b in range(2):
        ids = torch.cat([prefix, prompts[b, :lens[b]]])[None]
        want.append(whole.generate(ids, 12)[0])
        whole.kv.reset()
    m = _model(2, pages=16, num_pages=3 + 2 * 2)                # the prefix once, two pages for each row
    m.share_prefix(prefix)
    assert m.kv.shared_tokens == 48 and m.kv.free_pages == 4
    assert torch.equal(m.generate(prompts, 12, lens), torch.stack(want))
    with pytest.raises(RuntimeError):
        m.generate(prompts, 40, lens)                           # no room, and nothing was taken
    m.kv.release(0)
    m.kv.release(1)
    assert m.kv.free_pages == 4
    assert torch.equal(m.generate(prompts, 12, lens), torch.stack(want))
    with pytest.raises(ValueError):
        m.share_prefix(prefix[:20])
    m.share_prefix(prefix[:0])
    assert m.kv.shared_pages is None and m.kv.free_pages == 7
    with pytest.raises(ValueError):
        whole.share_prefix(prefix)


def _sampled_speculation(rank, world):
    from neuronx_distributed_b200.parallel_layers import parallel_state as ps
    from neuronx_distributed_b200.utils.speculative import speculative_generate, speculative_sample

    ps.initialize_model_parallel(tensor_model_parallel_size=world)
    g = torch.Generator().manual_seed(6)
    prompt = torch.randint(0, 96, (1, 7), generator=g)
    for pages in ((16, None), (None, 32), (32, 16)):             # greedy, in pages too
        target = _model(1, batch=1, pages=pages[0])
        want = target.generate(prompt, 12)
        target.kv.reset()
        assert torch.equal(speculative_generate(target, _model(1, batch=1, pages=pages[1]), prompt, 12, 3)[0], want)
    g = torch.Generator().manual_seed(5)
    prompts, lens = torch.randint(0, 96, (2, 9), generator=g), torch.tensor([9, 5])
    want = _model(1).generate(prompts, 14, lens)
    # a temperature at which one token has all the probability: the target's greedy decoding, whatever the draft says
    for draft, pages in ((_model(1, logits=True, pages=16), 16), (_model(7, 1, logits=True), None), (_model(7, 1, logits=True, pages=32), 16)):
        target = _model(1, logits=True, pages=pages)
        got, accepted = speculative_sample(target, draft, prompts, 14, 3, temperature=1e-5, generator=torch.Generator().manual_seed(0), prompt_lens=lens)
        assert torch.equal(got, want), (got, want)
        assert 0 <= accepted <= 3 and (draft.cfg.num_hidden_layers == 1 or accepted > 2)
    # the same random numbers draw the same tokens
    runs = [speculative_sample(_model(1, logits=True, pages=16), _model(7, 1, logits=True, pages=16), prompts, 10, 4,
                               generator=torch.Generator().manual_seed(11), prompt_lens=lens)[0] for _ in range(2)]
    assert torch.equal(*runs) and runs[0].shape == (2, 10) and int(runs[0].min()) >= 0
    with pytest.raises(ValueError):
        speculative_sample(_model(1, logits=True), _model(1, logits=True), prompts, 4, temperature=0.0)
    with pytest.raises(ValueError):
        speculative_sample(_model(1), _model(1, logits=True), prompts, 4)
    with pytest.raises(ValueError):
        speculative_sample(_model(1, logits=True), _model(1, logits=True), prompts, 120)


def _first_tokens(rank, world):
    """What comes out is distributed as the target's own samples, whatever the draft: the token behind the first, over 4000 rows, within five
    standard deviations of its probability (of the ones that are not rare)."""
    from neuronx_distributed_b200.parallel_layers import parallel_state as ps
    from neuronx_distributed_b200.utils.speculative import speculative_sample

    ps.initialize_model_parallel(tensor_model_parallel_size=world)
    N = 4000
    prompts = torch.tensor([[5, 17, 3]]).expand(N, 3).contiguous()
    target, draft = _model(1, 1, batch=N, logits=True, pages=16, num_pages=N), _model(2, 1, batch=N, logits=True, pages=16, num_pages=N)
    out, _ = speculative_sample(target, draft, prompts, 2, 2, temperature=0.5, generator=torch.Generator().manual_seed(1))
    one = _model(1, 1, batch=1, logits=True)
    p0 = torch.softmax(one.context_encoding(prompts[:1]) / 0.5, -1)[0]
    first = torch.bincount(out[:, 0], minlength=96)
    assert ((first - N * p0).abs() <= 5 * (N * p0 * (1 - p0)).sqrt() + 1).all()
    common = int(first.argmax())
    p1 = torch.softmax(one.token_generation(torch.tensor([[common]]), torch.tensor([3])) / 0.5, -1)[0]
    n = int(first[common])
    second = torch.bincount(out[out[:, 0] == common, 1], minlength=96)
    assert ((second - n * p1).abs() <= 5 * (n * p1 * (1 - p1)).sqrt() + 1).all()


@pytest.mark.parametrize("part", [_same_as_contiguous, _shared_prefix, _sampled_speculation, _first_tokens])
def test_served_from_pages(part):
    run_distributed(part, 1, timeout=240)


def test_tensor_parallel_ranks_keep_pages_of_their_heads():
    run_distributed(_same_as_contiguous, 2, timeout=240)


def test_manager():
    from neuronx_distributed_b200.inference.paged_cache import PagedKVCacheManager

    kv = PagedKVCacheManager(1, 3, 100, 2, 8, page_size=16, num_pages=10, dtype=torch.float32)
    assert kv.columns == 7 and kv.k[0].shape == (10, 16, 2, 8) and kv.free_pages == 10
    kv.reserve(0, 1)
    kv.reserve(0, 33)
    kv.reserve(0, 20)
    assert (kv.page_table[0] >= 0).tolist() == [True] * 3 + [False] * 4 and kv.free_pages == 7
    with pytest.raises(RuntimeError):
        kv.reserve_rows(3, 100)
    assert kv.free_pages == 7
    kv.take_shared(64)
    assert kv.free_pages == 6 and kv.shared_pages.tolist() == kv.page_table[2, :4].tolist()
    kv.reserve(1, 65)
    kv.reserve(2, 64)
    used = [p for row in kv.page_table.tolist() for p in row[4:] if p >= 0] + kv.shared_pages.tolist()
    assert len(used) == len(set(used)) == 5
    with pytest.raises(ValueError):
        kv.reserve(1, 113)
    with pytest.raises(ValueError):
        kv.take_shared(8)
    with pytest.raises(ValueError):
        PagedKVCacheManager(1, 1, 64, 1, 8, page_size=8)
    kv.reset()
    assert kv.free_pages == 10 and kv.shared_pages is None and not bool((kv.page_table >= 0).any())
