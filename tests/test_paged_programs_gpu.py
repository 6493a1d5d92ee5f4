"""Captured programs over a paged cache: they read the tables as they are when they run."""
import pytest
import torch

from test_paged_serving_gpu import groups, model  # noqa: F401

pytestmark = pytest.mark.gpu


def capture(call, *inputs):
    """One warm-up call, then the captured one, as a program that gives its results anew."""
    call(*inputs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(*inputs)

    def run():
        graph.replay()
        return out.clone()

    return run


def ids(seed, *shape):
    return torch.randint(0, 512, shape, generator=torch.Generator().manual_seed(seed)).cuda()


def test_another_prefix_of_the_same_length():
    m, fresh = model(page_size=32), model(page_size=32)
    prompts, lens = ids(1, 3, 40), torch.tensor([40, 7, 21]).cuda()
    x, pos = ids(2, 3, 1), lens + 128
    m.share_prefix(ids(3, 128))
    m.context_encoding(prompts, lens - 1)
    m.kv.reserve_rows(3, 256)
    step = capture(m.token_generation, x, pos)
    assert torch.equal(step(), m.token_generation(x, pos))
    m.kv.release(1)                                             # so that the next prefix lies elsewhere
    m.share_prefix(ids(4, 128))
    m.context_encoding(prompts, lens - 1)
    m.kv.reserve_rows(3, 256)
    filler = torch.full((1 << 16,), 1 << 20, dtype=torch.int32, device="cuda")         # over whatever has been given back
    fresh.share_prefix(ids(4, 128))
    fresh.context_encoding(prompts, lens - 1)
    want = fresh.token_generation(x, pos)
    assert torch.equal(step(), want) and torch.equal(m.token_generation(x, pos), want)
    with pytest.raises(RuntimeError, match="captured"):
        m.share_prefix(ids(5, 64))
    assert torch.equal(step(), want) and filler.numel()
