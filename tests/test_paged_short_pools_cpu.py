"""A pool that runs short under tables on the device: whoever generates with it says so, and does not answer with tokens over keys that are missing."""
import pytest
import torch

from test_paged_int4_serving_cpu import _model
from test_paged_serving_cpu import run_distributed


def _loops(logits):
    from neuronx_distributed_b200.utils.speculative import speculative_generate, speculative_sample

    if logits:
        return [lambda t, d, ids: speculative_sample(t, d, ids, 10, 3, generator=torch.Generator().manual_seed(1))[0]]
    return [lambda t, d, ids: t.generate(ids, 10), lambda t, d, ids: speculative_generate(t, d, ids, 10, 3)[0]]


def _all(rank, world):
    from neuronx_distributed_b200.parallel_layers import parallel_state as ps

    ps.initialize_model_parallel(tensor_model_parallel_size=world)
    prompts = torch.randint(0, 96, (1, 30), generator=torch.Generator().manual_seed(6))          # with 10 tokens more: three pages
    for bits in (None, 4):
        for logits in (False, True):
            for loop in _loops(logits):
                host, device = (dict(batch=1, logits=logits, kv_bits=bits, device_tables=d) for d in (False, True))
                want = loop(_model(**host), _model(**host), prompts)
                target, draft = _model(num_pages=3, **device), _model(num_pages=3, **device)
                assert torch.equal(loop(target, draft, prompts), want)
                short = _model(num_pages=2, **device)
                with pytest.raises(RuntimeError, match="without a page"):
                    loop(short, draft, prompts)
                short.kv.check()                             # said once
                with pytest.raises(RuntimeError, match="pages left"):
                    loop(_model(num_pages=2, **host), _model(**host), prompts)
                # what was lost before is not this call's, and is said before it begins
                target.kv.lost.fill_(1)
                with pytest.raises(RuntimeError, match="without a page"):
                    loop(target, draft, prompts)
                assert torch.equal(loop(target, draft, prompts), want)
    draft = _model(1, logits=False, kv_bits=4, device_tables=True, num_pages=2)
    with pytest.raises(RuntimeError, match="without a page"):
        _loops(False)[1](_model(1, logits=False, kv_bits=4, device_tables=True), draft, prompts)
    # an error of the caller's own stays what it is
    m = _model(1, logits=False, device_tables=True)
    with pytest.raises(ZeroDivisionError):
        with m.kv.reserved_ahead(1, 10):
            m.kv.lost.fill_(1)
            1 / 0


def test_loops_say_that_a_pool_is_short():
    run_distributed(_all, 1, timeout=240)
