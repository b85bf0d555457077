"""GPU tests of the operators of a served batch together, as the model calls them: ``PagedCache`` under the Llama of this
package (ragged prompts behind a shared prefix, decode steps, sampling), per-head norms in front of the Fourier cache.

The references are float64 evaluations of the same weights.  Tolerance of a logit or of a hidden state, in float16: a
layer rounds about ten tensors, each by at most 2^-11 of its largest value, and its products pass an error on at most
about fourfold (weights of spectral norm near one, residual stream): 2 layers x 10 x 4 x 2^-11 = 4 % of the largest
magnitude.
"""
import math
import os

import pytest
import torch

from oracle import fourier_oracle as fo
from tests.gpu_util import make_config, write_tables

pytestmark = pytest.mark.gpu
TOL = 2 * 10 * 4 * 2.0 ** -11


def small_model(qk_norm, head_dim=64, seed=0, dtype=torch.float16):
    from fourierattention_b200.modeling_llama_fourier import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(seed)
    cfg = LlamaConfig(vocab_size=211, hidden_size=256, intermediate_size=384, num_hidden_layers=2, num_attention_heads=6,
                      num_key_value_heads=2, head_dim=head_dim, max_position_embeddings=4096, qk_norm=qk_norm, rope_theta=10000.0)
    model = LlamaForCausalLM(cfg)
    for name, p in model.named_parameters():
        if p.dim() > 1:
            p.data.normal_(0.0, 1.0 / math.sqrt(p.shape[1]) if "embed" not in name else 1.0)
        else:
            p.data.add_(0.2 * torch.randn_like(p))
    return model.to("cuda", dtype).eval()


def reference_logits(model, ids):
    """Logits of every position of one sequence, (len, vocab), in float64."""
    cfg, w = model.config, {k: v.double() for k, v in model.state_dict().items()}
    rms = lambda x, g: x * (x.square().mean(-1, keepdim=True) + cfg.rms_norm_eps).rsqrt() * g
    h = w["model.embed_tokens.weight"][ids]
    n, d, hq, hkv = len(ids), cfg.head_dim, cfg.num_attention_heads, cfg.num_key_value_heads
    ang = torch.arange(n, device="cuda").double()[:, None] * model.model.rotary_emb.inv_freq.double()
    c, s = ang.cos()[:, None], ang.sin()[:, None]

    def rot(x):
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    late = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
    for i in range(cfg.num_hidden_layers):
        L = f"model.layers.{i}."
        x = rms(h, w[L + "input_layernorm.weight"])
        q, k, v = ((x @ w[L + f"self_attn.{t}_proj.weight"].T).view(n, -1, d) for t in "qkv")
        if cfg.qk_norm:
            q, k = rms(q, w[L + "self_attn.q_norm.weight"]), rms(k, w[L + "self_attn.k_norm.weight"])
        q, k = rot(q), rot(k)
        k, v = k.repeat_interleave(hq // hkv, 1), v.repeat_interleave(hq // hkv, 1)
        p = (torch.einsum("nhd,khd->hnk", q, k) / math.sqrt(d)).masked_fill(late, -math.inf).softmax(-1)
        h = h + torch.einsum("hnk,khd->nhd", p, v).reshape(n, -1) @ w[L + "self_attn.o_proj.weight"].T
        x = rms(h, w[L + "post_attention_layernorm.weight"])
        g = x @ w[L + "mlp.gate_proj.weight"].T
        h = h + (g * g.sigmoid() * (x @ w[L + "mlp.up_proj.weight"].T)) @ w[L + "mlp.down_proj.weight"].T
    return rms(h, w["model.norm.weight"]) @ w["lm_head.weight"].T


def check_last(logits, model, sequences):
    for b, ids in enumerate(sequences):
        if not len(ids):
            continue
        ref = reference_logits(model, torch.tensor(ids, device="cuda"))[-1]
        err = float((logits[b, -1].double() - ref).abs().max())
        assert err <= TOL * float(ref.abs().max()), (b, err)


@pytest.mark.parametrize("qk_norm,head_dim", [(False, 64), (True, 128)])
@pytest.mark.parametrize("prefix", [0, 37, 300])
def test_paged_model(qk_norm, head_dim, prefix):
    """A shared prefix, prompts of ragged lengths (one sequence idle), decode steps, a sequence that ends and whose place
    another one takes."""
    from fourierattention_b200 import PagedCache
    model = small_model(qk_norm, head_dim)
    g = torch.Generator().manual_seed(1)
    draw = lambda n: torch.randint(211, (n,), generator=g).tolist()
    B = 4
    cache = PagedCache(2, 2, head_dim, B, 400, page_size=16, dtype=torch.float16)
    for t in cache.k_pages + cache.v_pages:
        t.fill_(float("nan"))                       # what no key was written to is never read
    with torch.no_grad():
        pre = draw(prefix)
        if prefix:
            cache.plan([prefix, 0, 0, 0])
            out = model(torch.tensor([pre], device="cuda"), past_key_values=cache).logits
            check_last(out, model, [pre])
            cache.share_prefix(0)
            assert cache.prefix_len == prefix and cache.lengths == [0] * B
        seqs = [pre + draw(n) for n in (5, 70, 0, 16)]
        new = [len(s) - prefix for s in seqs]
        cache.plan(new)
        packed = torch.tensor([sum((s[prefix:] for s in seqs), [])], device="cuda")
        out = model(packed, past_key_values=cache).logits
        assert tuple(out.shape) == (B, 1, 211)
        check_last(out, model, [s if n else [] for s, n in zip(seqs, new)])
        for step in range(3):
            tok = draw(B)
            seqs = [s + [t] for s, t in zip(seqs, tok)]
            out = model(torch.tensor(tok, device="cuda")[:, None], past_key_values=cache).logits
            check_last(out, model, seqs)
        assert cache.get_seq_length() == max(len(s) for s in seqs)
        free = len(cache._free)
        cache.truncate(1)                           # ends; its pages go back
        assert len(cache._free) == free + 5
        seqs[1] = pre + draw(33)
        cache.plan([1, 33, 0, 2])
        more = [draw(1), seqs[1][prefix:], [], draw(2)]
        for b in (0, 3):
            seqs[b] = seqs[b] + more[b]
        out = model(torch.tensor([sum(more, [])], device="cuda"), past_key_values=cache).logits
        check_last(out, model, [seqs[0], seqs[1], [], seqs[3]])
        cache.reset()
        assert cache.lengths == [0] * B and len(cache._free) == cache.num_pages and cache.prefix_len == 0


def test_generate_is_forward_and_sample():
    from fourierattention_b200 import PagedCache, ops
    model = small_model(True)
    ids = torch.randint(211, (3, 21), device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    kw = dict(temperature=torch.tensor([0.8, 0.0, 1.3], device="cuda"), top_k=40, top_p=0.9, min_p=0.01)
    u = torch.rand(3, 6, device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    mk = lambda: PagedCache(2, 2, 64, 3, 64, page_size=16, dtype=torch.float16)
    got = model.generate(ids, mk(), 6, uniform=u, **kw)
    cache, x, want = mk(), ids, []
    with torch.no_grad():
        for i in range(6):
            t = ops.sample(model(x, past_key_values=cache).logits[:, -1], u[:, i].contiguous(), **kw)
            want.append(t)
            x = t[:, None]
    assert torch.equal(got, torch.stack(want, 1))
    # the greedy sequence takes the largest logit of the float64 model wherever that one is clear
    seq = ids[1].tolist()
    for t in got[1].tolist():
        top = reference_logits(model, torch.tensor(seq, device="cuda"))[-1].topk(2).values
        if float(top[0] - top[1]) > 2 * TOL * float(top.abs().max()):
            assert t == int(reference_logits(model, torch.tensor(seq, device="cuda"))[-1].argmax())
        seq.append(t)
    eos = int(got[0, 2])
    cut = model.generate(ids, mk(), 6, uniform=u, eos_token_id=eos, **kw)
    first = got[0].tolist().index(eos)
    assert cut[0, first:].tolist() == [eos] * (6 - first) and torch.equal(cut[0, :first], got[0, :first])
    same = [model.generate(ids, mk(), 3, generator=torch.Generator("cuda").manual_seed(9)) for _ in range(2)]
    assert torch.equal(*same)


def test_generate_over_the_fourier_cache():
    from fourierattention_b200 import DynamicCache, ops
    model = small_model(False)
    ids = torch.randint(211, (2, 90), device="cuda", generator=torch.Generator("cuda").manual_seed(8))
    u = torch.rand(2, 4, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    path = write_tables(fo.make_splithead_tables(2, 2, 64, 48, seed=3))
    try:
        mk = lambda: DynamicCache(make_config(dict(S=4, W=24, M=16, mpe=4096, Hkv=2, steps=8), path))
        caches = mk(), mk()
    finally:
        os.unlink(path)
    got = model.generate(ids, caches[0], 4, uniform=u, top_k=20)
    x, want = ids, []
    with torch.no_grad():
        for i in range(4):
            t = ops.sample(model(x, past_key_values=caches[1]).logits[:, -1], u[:, i].contiguous(), top_k=20)
            want.append(t)
            x = t[:, None]
    assert torch.equal(got, torch.stack(want, 1))
    assert caches[0].get_seq_length(0) == 93


def test_paged_decode_step_in_a_graph():
    """A decode step captured once and replayed while lengths and pages move on."""
    from fourierattention_b200 import PagedCache
    model = small_model(False)
    ids = torch.randint(211, (2, 14), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    tok = torch.zeros(2, 1, dtype=torch.int64, device="cuda")
    cache = PagedCache(2, 2, 64, 2, 64, page_size=16, dtype=torch.float16)
    seqs = ids.tolist()
    with torch.no_grad():
        model(ids, past_key_values=cache)
        step = lambda: model.lm_head(model.model.norm(_layers(model, tok, cache)))

        def _layers(m, t, c):
            h = m.model.embed_tokens(t)
            for layer in m.model.layers:
                h = layer(h, past_key_value=c)
            return h
        graph = None
        for i in range(6):                          # crosses a page boundary at 16
            cache.begin_step(2, 1)
            tok.copy_(torch.tensor([[3 * i + 1], [5 * i + 2]]))
            seqs = [s + [t] for s, t in zip(seqs, tok[:, 0].tolist())]
            if graph is None:
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    step()
                torch.cuda.current_stream().wait_stream(side)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    out = step()
            graph.replay()
            check_last(out, model, seqs)


def test_qk_norm_in_front_of_the_fourier_cache():
    """Prefill through the attention module with per-head norms: its output against float64, and the same keys in the
    Fourier cache's verbatim window."""
    from fourierattention_b200 import DynamicCache
    model = small_model(True)
    B, P, S, W, M = 2, 120, 4, 24, 16
    path = write_tables(fo.make_splithead_tables(2, 2, 64, 48, seed=3))
    try:
        cache = DynamicCache(make_config(dict(S=S, W=W, M=M, mpe=4096, Hkv=2, steps=4), path))
    finally:
        os.unlink(path)
    ids = torch.randint(211, (B, P), device="cuda", generator=torch.Generator("cuda").manual_seed(6))
    with torch.no_grad():
        out = model(ids, past_key_values=cache, num_logits_to_keep=P).logits
        for b in range(B):
            ref = reference_logits(model, ids[b])
            assert float((out[b].double() - ref).abs().max()) <= TOL * float(ref.abs().max())
        assert cache.key_cache[0]["k_local"].shape[1] == W
        at = model.model.layers[0].self_attn
        x = model.model.layers[0].input_layernorm(model.model.embed_tokens(ids[0])).double()
        k = (x @ at.k_proj.weight.double().T).view(P, 2, 64)
        k = k * (k.square().mean(-1, keepdim=True) + at.k_norm.variance_epsilon).rsqrt() * at.k_norm.weight.double()
        ang = torch.arange(P, device="cuda").double()[:, None, None] * at.rotary_emb.inv_freq.double()
        a, c = k.chunk(2, -1)
        k = torch.cat([a * ang.cos() - c * ang.sin(), c * ang.cos() + a * ang.sin()], -1).reshape(P, -1)
        got = cache.key_cache[0]["k_local"][0].double()
        # the projection's rounding to float16 passes through the norm and the rotation, and one more follows
        assert float((got - k[P - W:]).abs().max()) <= 4 * 2.0 ** -11 * float(k.abs().max())
        step = model(ids[:, :1], past_key_values=cache).logits
        assert tuple(step.shape) == (B, 1, 211) and bool(torch.isfinite(step).all())
    with pytest.raises(RuntimeError, match="backward"):
        model(ids)


def test_paged_steps_of_several_tokens_in_a_graph():
    """A step of four tokens per sequence, then of four packed ones in changing shares, captured once and replayed while
    lengths, pages and shares move on."""
    from fourierattention_b200 import PagedCache
    model = small_model(True)
    draw = lambda n: torch.randint(211, (n,), generator=g).tolist()
    for packed in (False, True):
        g = torch.Generator().manual_seed(3)
        cache = PagedCache(2, 2, 64, 2, 64, page_size=16, dtype=torch.float16)
        seqs = [draw(9), draw(9)]
        tok = torch.zeros((1, 8) if packed else (2, 4), dtype=torch.int64, device="cuda")

        def step():
            h = model.model.embed_tokens(tok)
            for layer in model.model.layers:
                h = layer(h, past_key_value=cache)
            return model.lm_head(model.model.norm(h))
        with torch.no_grad():
            model(torch.tensor(seqs, device="cuda"), past_key_values=cache)
            graph = None
            for shares in ([4, 4], [3, 5], [7, 1], [2, 6], [0, 8]):
                shares = shares if packed else [4, 4]
                new = [draw(n) for n in shares]
                if packed:
                    cache.plan(shares)
                cache.begin_step(*tok.shape)
                tok.copy_(torch.tensor(sum(new, [])).view(tok.shape))
                other = torch.full((64,), -1, dtype=torch.int32, device="cuda")      # takes memory that a step let go of
                seqs = [s + n for s, n in zip(seqs, new)]
                if graph is None:
                    side = torch.cuda.Stream()
                    side.wait_stream(torch.cuda.current_stream())
                    with torch.cuda.stream(side):
                        step()
                    torch.cuda.current_stream().wait_stream(side)
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        out = step()
                graph.replay()
                at = 0
                for s, n in zip(seqs, shares):
                    at += n
                    if n:
                        check_last(out.view(1, 8, -1)[:, :at], model, [s])
                del other


def test_a_step_is_not_captured_with_its_bookkeeping():
    """A replay would lengthen the sequences on the device alone, past the pages they have."""
    from fourierattention_b200 import PagedCache
    model = small_model(False)
    cache = PagedCache(2, 2, 64, 2, 64, page_size=16, dtype=torch.float16)
    tok = torch.zeros(2, 1, dtype=torch.int64, device="cuda")
    with torch.no_grad():
        model(tok, past_key_values=cache)
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="captured"):
            with torch.cuda.graph(graph):
                model(tok, past_key_values=cache)
        assert cache.lengths == [1, 1] and cache.kv_lens.tolist() == [1, 1]
        assert bool(torch.isfinite(model(tok, past_key_values=cache).logits).all()) and cache.lengths == [2, 2]
