"""A served Llama over pages of 4 bits on the GPU, captured and recorded, with page tables that are handed out on the host or on the device."""
import pytest
import torch

from test_paged_programs_gpu import capture, ids
from test_paged_serving_gpu import error, groups, model  # noqa: F401

pytestmark = pytest.mark.gpu


def steps(m, prompts, lens, window):
    return [m.context_encoding(prompts, lens - 1), m.speculation_forward(window, lens), m.token_generation(window[:, :1], lens + window.shape[1])]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("device_tables", [False, True])
def test_logits_are_near_the_model_without_codes(device_tables, dtype):
    """A number is off by up to half a step, a step is a fifteenth of the range of 32 numbers, about 4.1 of their deviations: 4.1 / 15 / sqrt(12) = 0.079 of them, for
    keys and for values, in two layers: 0.079 * 2 of what the attention adds to the logits; half as much again, and what the type leaves."""
    prompts, lens, window = ids(2, 3, 150), torch.tensor([150, 33, 90]).cuda(), ids(3, 3, 5)
    exact, rows = steps(model(torch.float32), prompts, lens, window), steps(model(dtype), prompts, lens, window)
    m = model(dtype, page_size=48, kv_bits=4, device_tables=device_tables)
    for e, a, b in zip(exact, rows, steps(m, prompts, lens, window)):
        assert error(b, e) <= 1.5 * 2 * 0.079 + 2 * error(a, e), (error(a, e), error(b, e))
    m.kv.check()


@pytest.mark.parametrize("bits", [None, 4])
def test_captured_programs_take_pages(bits):
    """A prompt and a token captured once, with tables on the device: rows grow, end and begin anew, and the programs take pages for them."""
    m, fresh = model(page_size=16, num_pages=20, kv_bits=bits, device_tables=True), model(page_size=16, kv_bits=bits)
    prompts, last, x = ids(6, 3, 40), torch.tensor([39, 6, 20]).cuda(), ids(7, 3, 1)
    pos = last + 1
    prompt = capture(m.context_encoding, prompts, last)
    step = capture(m.token_generation, x, pos)
    for seed in (8, 9):
        for row in range(3):
            m.kv.release(row)
        prompts.copy_(ids(seed, 3, 40))
        fresh.kv.reset()
        pos.copy_(last + 1)
        assert torch.equal(prompt(), fresh.context_encoding(prompts, last))
        for i in range(40):
            x.copy_(ids(100 * seed + i, 3, 1))
            assert torch.equal(step(), fresh.token_generation(x, pos)), i
            pos += 1
        assert m.kv.held.tolist() == [5, 3, 4] and m.kv.free_pages == 8
        m.kv.check()
    pos.fill_(480)
    step()
    with pytest.raises(RuntimeError, match="without a page"):
        m.kv.check()


@pytest.mark.parametrize("device_tables", [False, True])
@pytest.mark.parametrize("prefix", [0, 64])
def test_recorded_plans(prefix, device_tables):
    """Tables, append and attention as nodes of a launch plan, run at other positions and over other pages than it was recorded with."""
    from neuronx_distributed_b200.inference.launch_plan import record

    m, fresh = (model(page_size=32, kv_bits=4, device_tables=device_tables) for _ in range(2))
    prompts, lens = ids(10, 3, 40), torch.tensor([40, 7, 21]).cuda()
    x, pos = ids(11, 3, 4), lens + prefix

    def begin(k, seed):
        k.share_prefix(ids(seed, prefix))
        k.context_encoding(prompts, lens - 1)
        if not device_tables:
            k.kv.reserve_rows(3, prefix + 100)

    begin(m, 12)
    plan = record(lambda a, b: m.speculation_forward(a, b), [x, pos])
    assert {"assign_pages", "int4_append", "int4_attention"} <= {n.target for n in plan.nodes}
    transformer, main, _ = plan.hoist_weight_only()
    main.apply_transformer(transformer)
    for seed, shift in ((13, 0), (14, 9), (15, 40)):
        begin(m, seed)
        begin(fresh, seed)
        a, b = ids(seed, 3, 4), pos + shift
        want = fresh.speculation_forward(a, b)
        for p in (plan, main):
            assert torch.equal(p(a, b), want)
        m.kv.check()
        for k in (m, fresh):
            for row in range(3):
                k.kv.release(row)


def test_shared_prefix():
    """Rows behind a shared prefix write the codes that they write with it in their own pages, as far as the first layer's numbers, which no attention has
    entered, go; and the logits are as near as two halves' roundings of the rest leave them (see above)."""
    prefix, prompts, lens, window = ids(3, 128), ids(4, 3, 40), torch.tensor([40, 7, 21]).cuda(), ids(5, 3, 4)
    whole, m = model(page_size=64, kv_bits=4), model(page_size=64, kv_bits=4, device_tables=True)
    want = steps(whole, torch.cat([prefix.expand(3, 128), prompts], 1), lens + 128, window)
    m.share_prefix(prefix)
    got = [m.context_encoding(prompts, lens - 1), m.speculation_forward(window, lens + 128), m.token_generation(window[:, :1], lens + 132)]
    for a, b in zip(want, got):
        assert error(b, a) <= 1.5 * 2 * 0.079, error(b, a)
    for row in range(3):
        n = int(lens[row]) + 128 + 5
        for x, y in ((whole.kv.k[0], m.kv.k[0]), (whole.kv.v[0], m.kv.v[0])):
            a, b = (torch.cat([p.codes[t[row].long()].flatten(0, 1)[:n], p.steps[t[row].long()].flatten(0, 1)[:n].flatten(2).view(torch.uint8)], -1)
                    for p, t in ((x, whole.kv.page_table.clamp(min=0)), (y, m.kv.page_table.clamp(min=0))))
            assert float((a != b).float().mean()) < 0.05     # products of other row counts round elsewhere now and then
    m.kv.check()
