"""CPU tests of what ``LlamaForCausalLM`` does around the model calls of a served batch: refusals that come before any of
them, and the loop of ``generate`` over a model that only records what it is called with."""
from types import SimpleNamespace

import pytest
import torch


@pytest.fixture(scope="module")
def pkg():
    import __graft_entry__
    __graft_entry__._load_builder().build()
    import fourierattention_b200 as p
    return p


def small(pkg):
    cfg = pkg.modeling_llama_fourier.LlamaConfig(vocab_size=11, hidden_size=64, intermediate_size=64, num_hidden_layers=1,
                                                 num_attention_heads=1, num_key_value_heads=1, head_dim=64)
    return pkg.modeling_llama_fourier.LlamaForCausalLM(cfg)


def paged(pkg, batch=3):
    return pkg.PagedCache(1, 1, 64, batch, 40, page_size=16, device="cpu")


@pytest.mark.parametrize("plan", [[5, 0, 3], [0, 8, 0]])
def test_generate_refuses_idle_sequences(pkg, plan):
    """A sequence without new tokens in the prompt would be drawn from another one's logits."""
    cache = paged(pkg)
    cache.plan(plan)
    with pytest.raises(ValueError, match="without new tokens"):
        small(pkg).generate(torch.zeros(1, 8, dtype=torch.int64), cache, 2)
    assert cache.lengths == [0, 0, 0] and cache.planned == plan
