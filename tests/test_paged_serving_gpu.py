"""Append, attention and verification together, as a served Llama model calls them: prompts, shared prefixes, windows, captured single tokens."""
import pytest
import torch

pytestmark = pytest.mark.gpu
SIZES = dict(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
             max_position_embeddings=512)


@pytest.fixture(scope="module", autouse=True)
def groups():
    import torch.distributed as dist

    from neuronx_distributed_b200.parallel_layers import parallel_state as ps

    if not dist.is_initialized():
        torch.cuda.set_device(0)
        dist.init_process_group("nccl", store=dist.HashStore(), rank=0, world_size=1, device_id=torch.device("cuda", 0))
    if not ps.model_parallel_is_initialized():
        ps.initialize_model_parallel(tensor_model_parallel_size=1)


def model(dtype=torch.bfloat16, device="cuda", batch=3, seed=1, layers=None, **kw):
    from neuronx_distributed_b200.models.llama import LlamaConfig
    from neuronx_distributed_b200.models.llama_inference import LlamaForInference

    sizes = dict(SIZES, **({} if layers is None else {"num_hidden_layers": layers}))
    m = LlamaForInference(LlamaConfig(dtype=dtype, device=torch.device(device), **sizes), batch_size=batch, max_seq_len=512, on_device_sampling=False, **kw).eval()
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for p in m.lm.parameters():
            p.copy_(torch.randn(p.shape, generator=g) * (0.05 if p.dim() > 1 else 0.1) + (0 if p.dim() > 1 else 1))
            p.copy_(p.to(torch.bfloat16))                    # the same numbers in every type
    return m


def error(a, exact):
    return float((a.double().cpu() - exact.double().cpu()).norm() / exact.double().cpu().norm())


def test_logits_are_as_near_as_contiguous_rows():
    """Prompt, window and single token: as far from the model in 32 bits as contiguous rows are, within half as much again (another order of the same
    roundings)."""
    g = torch.Generator().manual_seed(2)
    ids, lens, window = torch.randint(0, 512, (3, 150), generator=g), torch.tensor([150, 33, 90]), torch.randint(0, 512, (3, 5), generator=g)
    wide, rows, pages = model(torch.float32), model(), model(page_size=48)
    pages.kv.reserve_rows(3, 200)
    out = []
    for m in (wide, rows, pages):
        steps = [m.context_encoding(ids.cuda(), lens.cuda() - 1), m.speculation_forward(window.cuda(), lens.cuda()),
                 m.token_generation(window[:, :1].cuda(), lens.cuda() + 5)]
        out.append(steps)
    for exact, a, b in zip(*out):
        assert error(b, exact) <= 1.5 * error(a, exact) + 1e-4, (error(a, exact), error(b, exact))


def test_shared_prefix_with_windows_and_captured_tokens():
    """Rows behind a shared prefix give what they give with the prefix in every row's own pages; single tokens as a captured program."""
    g = torch.Generator().manual_seed(3)
    prefix, ids = torch.randint(0, 512, (128,), generator=g).cuda(), torch.randint(0, 512, (3, 40), generator=g).cuda()
    lens, window = torch.tensor([40, 7, 21]).cuda(), torch.randint(0, 512, (3, 4), generator=g).cuda()
    whole = torch.zeros(3, 168, dtype=torch.long, device="cuda")
    for b, n in enumerate(lens.tolist()):
        whole[b, :128], whole[b, 128:128 + n] = prefix, ids[b, :n]
    wide, own, shared = model(torch.float32), model(page_size=32), model(page_size=32)
    shared.share_prefix(prefix)
    for m in (own, shared):
        m.kv.reserve_rows(3, 256)
    assert shared.kv.free_pages == own.kv.free_pages + 2 * 4
    x, position = window[:, :1].clone(), lens + 128 + 4
    results = []
    for m in (wide, own, shared):
        p = [m.context_encoding(ids, lens - 1) if m is shared else m.context_encoding(whole, lens + 127), m.speculation_forward(window, lens + 128)]
        m.token_generation(x, position)
        if m is not wide:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = m.token_generation(x, position)
            for step in range(3):
                graph.replay()
                p.append(out.clone())
                position += 1
            position -= 3
        else:
            for step in range(3):
                p.append(m.token_generation(x, position + step))
        results.append(p)
    for exact, a, b in zip(*results):
        assert error(b, exact) <= 1.5 * error(a, exact) + 1e-4, (error(a, exact), error(b, exact))


def test_sampled_speculation():
    """A draft that is the target itself: almost everything is accepted (what is not: roundings of a window against single tokens).  The same
    random numbers give the same tokens."""
    from neuronx_distributed_b200.utils.speculative import speculative_sample

    ids, lens = torch.randint(0, 512, (3, 30), generator=torch.Generator().manual_seed(4)).cuda(), torch.tensor([30, 12, 1]).cuda()
    runs = []
    for _ in range(2):
        g = torch.Generator(device="cuda").manual_seed(5)
        runs.append(speculative_sample(model(page_size=16), model(page_size=16), ids, 40, 4, 0.7, g, lens))
    assert torch.equal(runs[0][0], runs[1][0]) and runs[0][0].shape == (3, 40) and runs[0][1] > 3.0
    assert int(runs[0][0].min()) >= 0 and int(runs[0][0].max()) < 512
    out, accepted = speculative_sample(model(page_size=16), model(seed=9, layers=1), ids, 20, 3, 1.0, torch.Generator(device="cuda").manual_seed(6), lens)
    assert out.shape == (3, 20) and 0 <= accepted <= 3
