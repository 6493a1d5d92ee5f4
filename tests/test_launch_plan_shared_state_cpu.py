"""Buckets that were recorded over one key/value cache share it after they have been stored and loaded, too."""
import pytest
import torch

from test_paged_serving_cpu import run_distributed


def _served(rank, world, path, kw):
    from torch import nn

    from neuronx_distributed_b200.models.llama import LlamaConfig
    from neuronx_distributed_b200.models.llama_inference import LlamaForInference
    from neuronx_distributed_b200.parallel_layers import parallel_state as ps
    from neuronx_distributed_b200.trace.functions import compile as compile_bucket, compile_wlo, trace
    from neuronx_distributed_b200.trace.nxd_model import NxDModel
    from neuronx_distributed_b200.utils import safetensors_utils

    class Bucket(nn.Module):
        def __init__(self, model, name):
            super().__init__()
            self.model, self.name = model, name

        def forward(self, input_ids, aux):
            return self.model.context_encoding(input_ids, aux) if self.name == "prompt" else self.model.token_generation(input_ids, aux)

    ps.initialize_model_parallel(1)
    torch.manual_seed(0)
    model = LlamaForInference(LlamaConfig(vocab_size=256, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=2,
                                          dtype=torch.float32, device=torch.device("cpu"), max_position_embeddings=64), batch_size=2, max_seq_len=48, **kw).eval()
    prompts, last = [torch.randint(0, 256, (2, 24), generator=torch.Generator().manual_seed(s)) for s in (1, 2)], torch.tensor([23, 15])
    want = [model.generate(p, 8, prompt_lens=last + 1) for p in prompts]
    buckets = {n: trace(Bucket(model, n), a) for n, a in (("prompt", (prompts[0], last)), ("token", (torch.zeros(2, 1, dtype=torch.long), last + 1)))}
    nxd = NxDModel(world_size=1)
    nxd.add("prompt", buckets["prompt"], compile_bucket(buckets["prompt"], None, None, "--plan", "prompt"))
    nxd.add("token", buckets["token"], compile_wlo(buckets["token"], None, None, None, "token"))
    nxd.to_neuron()

    def generate(m, ids):
        tok, out, pos = m(ids, last, model_name="prompt"), [], last + 1
        for _ in range(7):
            out.append(tok.clone())
            tok, pos = m(tok.view(2, 1), pos, model_name="token"), pos + 1
        return torch.stack(out + [tok], 1)

    assert torch.equal(generate(nxd, prompts[0]), want[0])
    nxd.save(path, save_weights=True, portable=True)
    load = safetensors_utils.load_state_dict_safetensors
    safetensors_utils.load_state_dict_safetensors = lambda p: {n: t.clone() for n, t in load(p).items()}          # as a copy to another device does
    loaded = NxDModel.load(path)
    loaded.to_neuron()
    for i in (1, 0):                                         # the caches that were stored hold the first prompts' keys
        assert torch.equal(generate(loaded, prompts[i]), want[i])
        assert torch.equal(generate(nxd, prompts[i]), want[i])          # and the model they come from has its own


@pytest.mark.parametrize("kw", [{}, {"page_size": 16}, {"page_size": 16, "kv_bits": 4}, {"page_size": 16, "device_tables": True}, {"page_size": 16, "kv_bits": 4, "device_tables": True}])
def test_stored_buckets_share_their_cache(tmp_path, kw):
    run_distributed(_served, 1, str(tmp_path / "served"), kw, timeout=240)
