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


@pytest.mark.parametrize("keep", [2, 7])
def test_packed_logits_are_not_cut_across_sequences(pkg, keep):
    """The last rows of packed tokens are those of the last sequences, not the last ones of each."""
    cache, ids = paged(pkg), torch.zeros(1, 8, dtype=torch.int64)
    cache.plan([4, 1, 3])
    with pytest.raises(ValueError, match="num_logits_to_keep"):
        small(pkg)(ids, past_key_values=cache, num_logits_to_keep=keep)
    assert cache.lengths == [0, 0, 0] and cache.planned == [4, 1, 3]


@pytest.mark.parametrize("keep,rows", [(0, 8), (1, 3), (8, 8), (20, 8)])
def test_packed_logits(pkg, keep, rows, monkeypatch):
    """All rows, or the last one of every sequence."""
    model, cache = small(pkg), paged(pkg)
    cache.plan([4, 1, 3])
    hidden = torch.randn(1, 8, 64)

    def layers(ids, past_key_values):
        past_key_values.begin_step(*ids.shape)
        return hidden
    monkeypatch.setattr(model.model, "forward", layers)
    logits = model(torch.zeros(1, 8, dtype=torch.int64), past_key_values=cache, num_logits_to_keep=keep).logits
    want = model.lm_head(hidden[0] if rows == 8 else hidden[0, [3, 4, 7]])
    torch.testing.assert_close(logits.reshape(rows, -1), want)


def test_generate_needs_a_cache(pkg):
    """Without one, every token after the first would be drawn without its context."""
    with pytest.raises(ValueError, match="cache"):
        small(pkg).generate(torch.zeros(1, 4, dtype=torch.int64), None, 2)


class Recorder:
    """Stands for the model's forward and for the sampler: what the model is called with, and the given tokens in turn."""

    def __init__(self, pkg, monkeypatch, tokens):
        self.model, self.seen, self.tokens = small(pkg), [], [torch.tensor(t) for t in tokens]
        monkeypatch.setattr(self.model, "forward", self.forward)
        monkeypatch.setattr(pkg.ops, "sample", lambda logits, u, **kw: self.tokens[len(self.seen) - 1])

    def forward(self, input_ids, past_key_values):
        self.seen.append(input_ids.tolist())
        return SimpleNamespace(logits=torch.zeros(input_ids.shape[0], 1, 11))


@pytest.mark.parametrize("eos", [None, 5, -1])
def test_generate_never_embeds_what_was_not_drawn(pkg, monkeypatch, eos):
    """-1, for a row without anything to draw from, is returned and not looked up."""
    r = Recorder(pkg, monkeypatch, [[3, -1], [5, -1], [-1, 2], [4, 4]])
    got = r.model.generate(torch.tensor([[1, 2], [3, 4]]), paged(pkg, 2), 4, eos_token_id=eos)
    assert tuple(got.shape) == (2, 4) and got[:, 0].tolist() == [3, -1]
    assert r.seen[0] == [[1, 2], [3, 4]] and all(t >= 0 for step in r.seen for row in step for t in row)
    if eos is None:
        assert got.tolist() == [[3, 5, -1, 4], [-1, -1, 2, 4]] and r.seen[1:] == [[[3], [0]], [[5], [0]], [[0], [2]]]
    if eos == 5:
        assert got[0].tolist() == [3, 5, 5, 5]


def test_generate_nothing(pkg):
    """No token for each sequence, a packed prompt's too; the cache stays as it is."""
    model, cache = small(pkg), paged(pkg)
    cache.plan([4, 1, 3])
    assert tuple(model.generate(torch.zeros(1, 8, dtype=torch.int64), cache, 0).shape) == (3, 0)
    assert tuple(model.generate(torch.zeros(2, 8, dtype=torch.int64), None, 0).shape) == (2, 0)
    assert cache.planned == [4, 1, 3] and cache.lengths == [0, 0, 0]
    with pytest.raises(ValueError):
        model.generate(torch.zeros(2, 8, dtype=torch.int64), None, -1)


def test_a_failed_forward_leaves_the_cache(pkg):
    """Here the cache's type is not the model's; the lengths must not count keys that were never stored."""
    model, cache = small(pkg), paged(pkg)                        # float32 model, bfloat16 cache
    for plan, shape in (([4, 1, 3], (1, 8)), (None, (3, 2))):
        if plan:
            cache.plan(plan)
        with torch.no_grad(), pytest.raises((ValueError, RuntimeError)):
            model(torch.zeros(shape, dtype=torch.int64), past_key_values=cache)
        assert cache.lengths == [0, 0, 0] and cache.kv_lens.tolist() == [0, 0, 0] and cache.planned == plan
        assert len(cache._free) == cache.num_pages
        cache._plan = None


def test_padded_batches_are_refused(pkg, monkeypatch):
    """Padding would be stored and attended like tokens; a mask that hides nothing is taken."""
    model, cache, ids = small(pkg), paged(pkg), torch.zeros(3, 4, dtype=torch.int64)
    mask = torch.ones(3, 4, dtype=torch.int64)
    mask[1, :2] = 0
    with pytest.raises(ValueError, match="padded"):
        model(ids, past_key_values=cache, attention_mask=mask)
    assert cache.lengths == [0, 0, 0]
    monkeypatch.setattr(model.model, "forward", lambda ids, past_key_values: past_key_values.begin_step(*ids.shape) or torch.zeros(3, 4, 64))
    assert model(ids, past_key_values=cache, attention_mask=torch.ones_like(mask)).logits.shape == (3, 1, 11)


def test_given_positions_reach_the_layers(pkg, monkeypatch):
    model, cache, seen = small(pkg), paged(pkg), []

    def layers(ids, past_key_values, position_ids=None):
        seen.append(position_ids)
        past_key_values.begin_step(*ids.shape)
        return torch.zeros(3, ids.shape[1], 64)
    monkeypatch.setattr(model.model, "forward", layers)
    at = torch.arange(4).expand(3, 4) + 7
    model(torch.zeros(3, 4, dtype=torch.int64), past_key_values=cache, position_ids=at)
    model(torch.zeros(3, 1, dtype=torch.int64), past_key_values=cache)
    assert seen[0] is at and seen[1] is None


def test_a_causal_mask_is_no_padding(pkg, monkeypatch):
    """One of four dimensions, 0 where a token sees another, says what the attention does anyway."""
    model, cache, ids = small(pkg), paged(pkg), torch.zeros(3, 4, dtype=torch.int64)
    monkeypatch.setattr(model.model, "forward", lambda ids, past_key_values: past_key_values.begin_step(*ids.shape) or torch.zeros(3, 4, 64))
    causal = torch.full((4, 4), float("-inf")).triu(1).expand(3, 1, 4, 4)
    assert model(ids, past_key_values=cache, attention_mask=causal).logits.shape == (3, 1, 11)
