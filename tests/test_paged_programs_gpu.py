"""Captured programs over a paged cache: they read the tables as they are when they run."""
import pytest
import torch

from test_paged_rows_cpu import LOST, append_notes
from test_paged_serving_gpu import groups, model  # noqa: F401

pytestmark = pytest.mark.gpu


def capture(call, *inputs):
    """One warm-up call, then the captured one, as a program that gives its results anew and keeps its inputs."""
    call(*inputs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(*inputs)

    def run(held=inputs):
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first, lens, noted", LOST)
def test_append_notes_tokens_without_a_place(first, lens, noted, dtype):
    append_notes("cuda", dtype, first, lens, noted)


def test_captured_prompts_and_pages_that_come_and_go():
    """A captured prompt and step go on with whatever pages the rows hold; tokens without a page are said at the next look."""
    m, fresh = model(page_size=16, num_pages=3 * 16), model(page_size=16)
    prompts, lens = ids(6, 3, 40), torch.tensor([40, 7, 21]).cuda()
    x, pos = ids(7, 3, 1), lens.clone()
    with pytest.raises(RuntimeError, match="captured"):          # no pages yet, and none are handed out inside
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            m.context_encoding(prompts, lens - 1)
    torch.cuda.synchronize()
    assert m.kv.free_pages == 48
    prompt = capture(m.context_encoding, prompts, lens - 1)
    m.kv.reserve_rows(3, 64)
    step = capture(m.token_generation, x, pos)
    for seed in (8, 9):
        m.kv.reset()
        m.kv.reserve(2, 64)
        m.kv.reserve(1, 64)                                     # other pages than before
        m.kv.reserve(0, 64)
        prompts.copy_(ids(seed, 3, 40))
        fresh.kv.reset()
        want = [fresh.context_encoding(prompts, lens - 1), fresh.token_generation(x, pos)]
        assert torch.equal(prompt(), want[0]) and torch.equal(step(), want[1])
        m.kv.check()
    m.kv.release(0)
    prompt()
    with pytest.raises(RuntimeError, match="without a page"):
        m.kv.check()
    m.kv.reserve(0, 64)
    prompt()
    step()
    m.kv.check()
    pos.fill_(64)
    step()
    with pytest.raises(RuntimeError, match="without a page"):
        m.kv.reset()
    m.kv.reset()
    assert m.kv.free_pages == 48


@pytest.mark.parametrize("prefix", [0, 64])
def test_recorded_plans(prefix):
    """Append, attention over own and shared pages, and verification as nodes of a launch plan: run at other positions and over other pages than it was
    recorded with, with and without its weight-only part, and captured."""
    from neuronx_distributed_b200 import ops
    from neuronx_distributed_b200.inference.launch_plan import record

    m = model(page_size=32)
    prompts, lens = ids(10, 3, 40), torch.tensor([40, 7, 21]).cuda()

    def begin(seed):
        m.share_prefix(ids(seed, prefix))
        m.context_encoding(prompts, lens - 1)
        m.kv.reserve_rows(3, prefix + 100)

    def step(window, pos, drafted, draft, accept, sample):
        judged = torch.softmax(m.speculation_forward(window, pos), -1)
        new, n = ops.select.verify_drafts(drafted, draft, judged, accept, sample)
        return judged, new, n

    def inputs(seed, shift):
        g = torch.Generator(device="cuda").manual_seed(seed)
        draft = torch.softmax(torch.randn(3, 4, 512, generator=g, device="cuda"), -1)
        drafted = ids(seed, 3, 4)
        return [torch.cat([ids(seed + 1, 3, 1), drafted], 1), lens + prefix + shift, drafted, draft, torch.rand(3, 4, generator=g, device="cuda"),
                torch.rand(3, generator=g, device="cuda")]

    begin(11)
    plan = record(step, inputs(20, 0))
    targets = plan.summary()["top_targets"] and {n.target for n in plan.nodes}
    assert {"paged_append", "paged_attention", "verify_drafts"} <= targets, targets
    transformer, main, _ = plan.hoist_weight_only()
    main.apply_transformer(transformer)
    live = [t.clone() for t in inputs(20, 0)]
    captured = capture(lambda *a: torch.cat([main(*a)[0].flatten(), main(*a)[1].flatten().float()]), *live)
    for turn in range(2):
        for shift in (0, 9, 30):
            x = inputs(21 + shift, shift)
            want = step(*x)
            for p in (plan, main):
                for a, b in zip(p(*x), want):
                    assert torch.equal(a, b)
            for a, b in zip(live, x):
                a.copy_(b)
            assert torch.equal(captured(), torch.cat([want[0].flatten(), want[1].flatten().float()]))
        m.kv.check()
        if turn == 0:
            before = m.kv.page_table.clone()
            m.kv.release(0)
            m.kv.reserve(2, prefix + 100)
            begin(12)
            m.kv.release(0)
            m.kv.release(1)
            m.kv.reserve(1, prefix + 100)
            m.context_encoding(prompts, lens - 1)
            m.kv.reserve_rows(3, prefix + 100)
            assert not torch.equal(before, m.kv.page_table)


@pytest.mark.parametrize("prefix", [0, 64])
def test_adapter_over_captured_programs(prefix):
    """Prompt and step of a paged model captured by the builder, called by the generation adapter, over several calls: the tokens of eager steps."""
    from neuronx_distributed_b200.inference.hf_adapter import HuggingFaceGenerationAdapter
    from neuronx_distributed_b200.trace.model_builder import ModelBuilder

    def served():
        m = model(page_size=16, num_pages=prefix // 16 + 3 * 8)
        m.on_device_sampling = True
        m.share_prefix(ids(30, prefix))
        return m

    eager, m = served(), served()
    prompts, mask = ids(31, 3, 40), torch.ones(3, 40, dtype=torch.long, device="cuda")
    mask[1, :33], mask[2, :19] = 0, 0
    builder = ModelBuilder(use_cuda_graphs=True)
    builder.add("prompt", m, [(torch.zeros(3, 40, dtype=torch.long, device="cuda"), torch.full((3,), 39, device="cuda"))],
                step_fn=lambda m, i, last: m.context_encoding(i, last))
    builder.add("step", m, [(torch.zeros(3, 1, dtype=torch.long, device="cuda"), torch.full((3,), prefix + 40, device="cuda"))],
                step_fn=lambda m, i, pos: m.token_generation(i, pos))
    programs = builder.trace()
    by_steps = HuggingFaceGenerationAdapter(eager)
    captured = HuggingFaceGenerationAdapter(m).use_programs(programs, programs)
    for seed in (31, 32):
        for new in (60, 20, 88):
            prompts = ids(seed, 3, 40)
            assert torch.equal(captured.generate(prompts, mask, max_new_tokens=new), by_steps.generate(prompts, mask, max_new_tokens=new))
            assert m.kv.shared_tokens == prefix
    with pytest.raises(RuntimeError, match="pool"):
        captured.generate(prompts, mask, max_new_tokens=100)
