"""A served Llama over pages of 4 bits, and over page tables that are handed out on the device (here in plain torch)."""
import os
import subprocess
import sys

import pytest
import torch

from test_paged_serving_cpu import run_distributed

SIZES = dict(vocab_size=96, hidden_size=128, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
             max_position_embeddings=128, dtype=torch.float32, device=torch.device("cpu"))


def _model(batch=2, seed=1, logits=True, page_size=16, **kw):
    from neuronx_distributed_b200.models.llama import LlamaConfig
    from neuronx_distributed_b200.models.llama_inference import LlamaForInference

    torch.manual_seed(seed)
    return LlamaForInference(LlamaConfig(**SIZES), batch_size=batch, max_seq_len=100, on_device_sampling=not logits, page_size=page_size, **kw).eval()


def _steps(m, ids, lens, window):
    return [m.context_encoding(ids, lens - 1), m.speculation_forward(window, lens), m.token_generation(window[:, :1], lens + window.shape[1])]


def _same_whoever_hands_out_pages(rank, world):
    from neuronx_distributed_b200.parallel_layers import parallel_state as ps

    ps.initialize_model_parallel(tensor_model_parallel_size=world)
    g = torch.Generator().manual_seed(3)
    ids, lens, window = torch.randint(0, 96, (2, 40), generator=g), torch.tensor([40, 17]), torch.randint(0, 96, (2, 4), generator=g)
    for bits in (None, 4):
        host, device = _model(kv_bits=bits), _model(kv_bits=bits, device_tables=True)
        for a, b in zip(_steps(host, ids, lens, window), _steps(device, ids, lens, window)):
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
        assert device.kv.held.tolist() == [3, 2] and device.kv.free_pages == 2 * 7 - 5          # 45 and 22 tokens: what counts, and no padding
        device.kv.release(0)
        assert device.kv.held.tolist() == [0, 2] and device.kv.free_pages == 12
        device.kv.check()


def _prompt_and_tokens_agree(rank, world):
    """A token behind a prompt sees the codes that a longer prompt writes: the same logits, within sums in another order."""
    from neuronx_distributed_b200.parallel_layers import parallel_state as ps

    ps.initialize_model_parallel(tensor_model_parallel_size=world)
    ids = torch.randint(0, 96, (1, 50), generator=torch.Generator().manual_seed(4))
    whole, parts = _model(1, kv_bits=4), _model(1, kv_bits=4, device_tables=True)
    parts.context_encoding(ids[:, :30])
    for n in range(30, 50):
        got = parts.token_generation(ids[:, n:n + 1], torch.tensor([n]))
        if n % 7 == 0 or n == 49:
            torch.testing.assert_close(got, whole.context_encoding(ids[:, :n + 1]), rtol=1e-3, atol=1e-3)
            whole.kv.reset()
    assert all(type(p).__name__ == "Pages" and p.codes.dtype == torch.uint8 for p in (*parts.kv.k, *parts.kv.v))


def _shared_prefix(rank, world):
    from neuronx_distributed_b200.parallel_layers import parallel_state as ps

    ps.initialize_model_parallel(tensor_model_parallel_size=world)
    g = torch.Generator().manual_seed(5)
    prefix, prompts, lens = torch.randint(0, 96, (32,), generator=g), torch.randint(0, 96, (2, 10), generator=g), torch.tensor([10, 4])
    for bits in (None, 4):
        want = []
        for b in range(2):
            one = _model(1, logits=False, kv_bits=bits)
            want.append(one.generate(torch.cat([prefix, prompts[b, :lens[b]]])[None], 12)[0])
        for device in (False, True):
            m = _model(2, logits=False, kv_bits=bits, device_tables=device, num_pages=2 + 2 * 2)
            m.share_prefix(prefix)
            assert m.kv.shared_tokens == 32 and m.kv.free_pages == 4
            assert torch.equal(m.generate(prompts, 12, lens), torch.stack(want))
            for row in range(2):
                m.kv.release(row)
            assert m.kv.free_pages == 4
            m.kv.check()
            m.share_prefix(prefix[:0])
            assert m.kv.shared_pages is None and m.kv.free_pages == 6


def _short_pools(rank, world):
    from neuronx_distributed_b200.inference.hf_adapter import HuggingFaceGenerationAdapter
    from neuronx_distributed_b200.parallel_layers import parallel_state as ps

    ps.initialize_model_parallel(tensor_model_parallel_size=world)
    prompts = torch.randint(0, 96, (2, 30), generator=torch.Generator().manual_seed(6))
    m = _model(2, logits=False, kv_bits=4, device_tables=True, num_pages=5)
    want = _model(2, logits=False, kv_bits=4).generate(prompts, 10)
    a = HuggingFaceGenerationAdapter(m)
    got = a.generate(prompts, attention_mask=torch.tensor([[1] * 30, [0] * 20 + [1] * 10]), max_new_tokens=10)     # 39 and 19 tokens: five pages
    assert torch.equal(got[0, 30:], want[0])
    with pytest.raises(RuntimeError, match="without a page"):
        a.generate(prompts, max_new_tokens=10)               # six would be needed
    m.kv.reset()
    assert m.kv.free_pages == 5
    m.kv.reserve(0, 70)
    assert m.kv.held.tolist() == [5, 0] and m.kv.free_pages == 0
    m.kv.check()
    m.kv.reserve(1, 1)
    with pytest.raises(RuntimeError, match="without a page"):
        m.kv.check()
    m.kv.reserve_rows(2, 20)
    with pytest.raises(RuntimeError, match="without a page"):
        m.kv.reset()
    m.kv.reset()
    for call in (lambda: m.kv.reserve(0, 101), lambda: m.kv.reserve_rows(2, 101), lambda: m.context_encoding(torch.zeros(2, 101, dtype=torch.long))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("part", [_same_whoever_hands_out_pages, _prompt_and_tokens_agree, _shared_prefix, _short_pools])
def test_served(part):
    run_distributed(part, 1, timeout=240)


def test_tensor_parallel_ranks_hold_codes_of_their_heads():
    run_distributed(_same_whoever_hands_out_pages, 2, timeout=240)


def test_example_runs():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, os.path.join(root, "examples", "inference", "run_llama_speculative.py"), "--model", "tiny", "--page_size", "16", "--kv_bits",
                          "4", "--device_tables", "--prompt_length", "8", "--max_new_tokens", "6"],
                         env={**os.environ, "CUDA_VISIBLE_DEVICES": "", "MASTER_ADDR": "127.0.0.1", "MASTER_PORT": "29617"}, capture_output=True, text=True, timeout=240)
    assert out.returncode == 0 and "identical to greedy: True" in out.stdout, out.stdout[-500:] + out.stderr[-2000:]


def test_refusals():
    from neuronx_distributed_b200.inference.paged_cache import PagedKVCacheManager

    with pytest.raises(ValueError):
        PagedKVCacheManager(1, 2, 64, 2, 64, bits=8)
    with pytest.raises(ValueError):
        PagedKVCacheManager(1, 2, 64, 2, 48, bits=4)
    for kw in (dict(kv_bits=4), dict(device_tables=True)):
        with pytest.raises(ValueError):
            _model(page_size=None, **kw)
