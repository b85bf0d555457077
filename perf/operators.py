"""The serving operators of this package as measured work: a decode or prompt step of a batch from the projections to
the next token.

``listed()`` / ``draw()`` give cases, ``prepare()`` what a program has in hand before the call, ``run()`` one pass.
With ``own`` false ``run`` computes the operator in elementary torch operations, with ``own`` true through
``fourierattention_b200.ops``.

Operators:
  qk_norm_rope     RMS norm of every query and key head and the rotation by position, in one pass
  paged_append     keys (rotated) and values of the new tokens into the pages of a cache, queries rotated alongside
  paged_attention  attention of the new tokens over their pages and over a prefix that the whole batch shares
  sample           temperature, top-k, top-p and min-p, the draw made by given random numbers
"""
import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA = 500000.0
EPS = 1e-5


# ---------------------------------------------------------------------------------------------- cases
def listed():
    h8b = dict(q_heads=32, kv_heads=8, head_dim=128)       # the 8B benchmark geometry
    h3b = dict(q_heads=24, kv_heads=8, head_dim=128)       # the 3B one
    toy = dict(q_heads=8, kv_heads=2, head_dim=64)         # the geometry of the small tests
    return [
        # one decode step of the benchmark's eight sequences: latency
        dict(name="norm rope decode 8", op="qk_norm_rope", tokens=8, norm=True, far=32768, dtype="bf16", **h8b),
        # a prompt of odd length, no norm weights, small heads
        dict(name="rope prompt 4099", op="qk_norm_rope", tokens=4099, norm=False, far=4099, dtype="fp16", **toy),
        # the benchmark's 32k prompt
        dict(name="norm rope prompt 32768", op="qk_norm_rope", tokens=32768, norm=True, far=32768, dtype="bf16", **h8b),
        # one decode step of 64 sequences of different lengths
        dict(name="append decode 64", op="paged_append", batch=64, new=1, past=8192, page=16, norm=False, dtype="bf16",
             **h8b),
        # prompts of eight sequences of ragged lengths, q and k normed on the way
        dict(name="append prompts 8x4000", op="paged_append", batch=8, new=4000, past=0, page=64, norm=True,
             dtype="fp16", **h3b),
        # one sequence, 8k context (the single-layer benchmark): latency of the split over the length
        dict(name="attend 1x8192", op="paged_attention", batch=1, new=1, own=8192, prefix=0, page=16, dtype="fp16",
             **h8b),
        # ragged decode batch at the 3B geometry, 16k contexts: streaming of the pages
        dict(name="attend 32x16384", op="paged_attention", batch=32, new=1, own=16384, prefix=0, page=32, dtype="bf16",
             **h3b),
        # decode of 64 sequences behind one 32k prefix: each prefix key read once for all of them
        dict(name="attend 64 prefix 32768", op="paged_attention", batch=64, new=1, own=700, prefix=32768, page=64,
             dtype="bf16", **h8b),
        # questions of up to 250 tokens behind one 16k prefix: bound by the matrix units
        dict(name="attend 8x250 prefix 16384", op="paged_attention", batch=8, new=250, own=250, prefix=16384, page=64,
             dtype="bf16", **h8b),
        # one row of logits: latency
        dict(name="sample 1", op="sample", batch=1, vocab=128256, dtype="bf16"),
        # an odd vocabulary and batch
        dict(name="sample 33x32003", op="sample", batch=33, vocab=32003, dtype="fp16"),
        # a large batch of float32 logits, every row with parameters of its own
        dict(name="sample 256", op="sample", batch=256, vocab=128256, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qk_norm_rope", "paged_append", "paged_attention", "paged_attention", "sample"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "sample":
        batch, vocab = _log(rng, 1, 256), _log(rng, 1000, 128256)
        return dict(op=op, batch=batch, vocab=vocab, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    kv = rng.choice([1, 2, 4, 8])
    heads = dict(q_heads=kv * rng.choice([1, 2, 3, 4, 5, 8] if kv < 8 else [1, 2, 3, 4]), kv_heads=kv,
                 head_dim=rng.choice([64, 128]), dtype=dtype)
    if op == "qk_norm_rope":
        return dict(op=op, tokens=_log(rng, 1, 32768), norm=rng.random() < 0.5, far=_log(rng, 16, 131072), **heads)
    page = rng.choice([16, 32, 64, 128])
    if op == "paged_append":
        new = rng.choice([1, _log(rng, 2, 4000)])
        return dict(op=op, batch=_log(rng, 1, 64 if new == 1 else 8), new=new, past=_log(rng, 1, 8192), page=page,
                    norm=rng.random() < 0.5, **heads)
    if rng.random() < 0.6:
        batch, new = _log(rng, 1, 48), 1
    else:
        batch, new = _log(rng, 1, 8), _log(rng, 2, 250)
    return dict(op=op, batch=batch, new=new, own=new - 1 + _log(rng, 1, 8192 if new == 1 else 512),
                prefix=rng.choice([0, _log(rng, 16, 16384)]), page=page, **heads)


def _spread(most, n):
    """n lengths from about half of `most` up to it, in mixed order, the same ones for every seed."""
    return [most - ((5 * i) % n) * (most // 2) // n for i in range(n)]


# ---------------------------------------------------------------------------------------------- inputs
def _inv_freq(head_dim, device):
    return 1.0 / (THETA ** (torch.arange(0, head_dim, 2, dtype=torch.float32, device=device) / head_dim))


def _page_layout(g, lens, extra_tokens, page, device):
    """Pages of the sequences (and of a prefix) scattered over the pool, as a server that hands pages out and takes
    them back leaves them: (number of pages, (B, most) table, prefix pages)."""
    need = [-(-n // page) for n in lens]
    pre = -(-extra_tokens // page)
    total = sum(need) + pre + 3
    perm = torch.randperm(total, generator=g, device=device).to(torch.int32)
    table = torch.zeros((len(lens), max(need)), dtype=torch.int32, device=device)
    at = pre
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return total, table, perm[:pre].contiguous()


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DT[case["dtype"]]
    randn = lambda *s: torch.randn(s, generator=g, device=dev).to(dt)  # noqa: E731
    if case["op"] == "sample":
        b, v = case["batch"], case["vocab"]
        rand = lambda: torch.rand((b,), generator=g, device=dev)  # noqa: E731
        pick = lambda values: torch.tensor(values, device=dev)[  # noqa: E731
            torch.randint(len(values), (b,), generator=g, device=dev)]
        # logits as a language model gives them: a broad body and a few tokens far above it
        x = 2.5 * torch.randn((b, v), generator=g, device=dev)
        lift = torch.randint(v, (b, 24), generator=g, device=dev)
        x.scatter_add_(1, lift, 9.0 * torch.rand((b, 24), generator=g, device=dev))
        temperature = 0.5 + 0.7 * rand()
        if b > 1:
            temperature = torch.where(rand() < 0.1, torch.zeros_like(temperature), temperature)   # some rows greedy
        return dict(case=case, logits=x.to(dt), u=rand(), temperature=temperature,
                    top_k=pick([0, 20, 50, 400]).to(torch.int32), top_p=pick([1.0, 0.95, 0.9, 0.7]),
                    min_p=pick([0.0, 0.0, 0.02, 0.1]))
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    s = dict(case=case, inv_freq=_inv_freq(d, dev))
    weight = lambda: (1.0 + 0.2 * torch.randn((d,), generator=g, device=dev)).to(dt)  # noqa: E731
    if case["op"] == "qk_norm_rope":
        t = case["tokens"]
        # q and k are views of one fused projection
        qkv = randn(t, (hq + 2 * hkv) * d).view(t, hq + 2 * hkv, d)
        s.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv],
                 positions=torch.randint(case["far"], (t,), generator=g, device=dev),
                 q_weight=weight() if case["norm"] else None, k_weight=weight() if case["norm"] else None)
        return s
    new, page, b = _spread(case["new"], case["batch"]), case["page"], case["batch"]
    if case["op"] == "paged_append":
        past = _spread(case["past"], b) if case["past"] else [0] * b
        lens, prefix = [x + y for x, y in zip(past, new)], 0
    else:
        lens, prefix = [max(x, y) for x, y in zip(_spread(case["own"], b), new)], case["prefix"]
    t = sum(new)
    total, table, prefix_pages = _page_layout(g, lens, prefix, page, dev)
    s.update(k_pages=randn(total, hkv, page, d), v_pages=randn(total, hkv, page, d), page_table=table,
             kv_lens=torch.tensor(lens, dtype=torch.int32, device=dev),
             cu_seqlens=None if case["new"] == 1 else torch.tensor(
                 [0] + np.cumsum(new).tolist(), dtype=torch.int32, device=dev), most_new=max(new))
    if case["op"] == "paged_append":
        s.update(q=randn(t, hq, d), k=randn(t, hkv, d), v=randn(t, hkv, d),
                 q_weight=weight() if case["norm"] else None, k_weight=weight() if case["norm"] else None)
    else:
        # scores of a standard deviation of about two, as trained heads have them
        s.update(q=(2.0 * torch.randn((t, hq, d), generator=g, device=dev)).to(dt),
                 prefix_pages=prefix_pages if prefix else None, prefix_len=prefix)
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _rotate(x, weight, cos, sin):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _cos_sin(positions, inv_freq):
    angle = positions.double()[:, None, None] * inv_freq.double()
    return angle.cos().float(), angle.sin().float()


def _plain_qk_norm_rope(s):
    cos, sin = _cos_sin(s["positions"], s["inv_freq"])
    return {"q": _rotate(s["q"], s["q_weight"], cos, sin).to(s["q"].dtype),
            "k": _rotate(s["k"], s["k_weight"], cos, sin).to(s["k"].dtype)}


def _token_owner(s):
    """(sequence, index within its new tokens, number of its new tokens) of every new token."""
    cu, t = s["cu_seqlens"], s["q"].shape[0]
    if cu is None:
        seq = torch.arange(t, device=s["q"].device)
        return seq, torch.zeros_like(seq), torch.ones_like(seq)
    at = torch.arange(t, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), at, right=True)
    return seq, at - cu[seq], (cu[1:] - cu[:-1])[seq].long()


def _plain_paged_append(s):
    page = s["k_pages"].shape[2]
    seq, i, n = _token_owner(s)
    at = s["kv_lens"].long()[seq] - n + i
    cos, sin = _cos_sin(at, s["inv_freq"])
    where = s["page_table"].long()[seq, at // page]
    s["k_pages"][where, :, at % page] = _rotate(s["k"], s["k_weight"], cos, sin).to(s["k"].dtype)
    s["v_pages"][where, :, at % page] = s["v"]
    return {"q": _rotate(s["q"], s["q_weight"], cos, sin).to(s["q"].dtype), "k_pages": s["k_pages"],
            "v_pages": s["v_pages"]}


def _plain_paged_attention(s):
    q, (_, hkv, page, d) = s["q"], s["k_pages"].shape
    t, hq, _ = q.shape
    b = s["page_table"].shape[0]
    seq, i, n = _token_owner(s)
    # queries padded to (sequence, kv head, new token x query head of the group)
    most, group = s["most_new"], hq // hkv
    padded = torch.zeros((b, most, hkv, group, d), device=q.device)
    padded[seq, i] = q.float().view(t, hkv, group, d)
    rows = padded.permute(0, 2, 1, 3, 4).reshape(b, hkv, most * group, d) / math.sqrt(d)
    sees = torch.zeros((b, most), dtype=torch.long, device=q.device)
    sees[seq, i] = s["kv_lens"].long()[seq] - n + i + 1
    pages = lambda x, at: x[at.long()].float().transpose(-4, -3).flatten(-3, -2)  # noqa: E731
    keys, values = pages(s["k_pages"], s["page_table"]), pages(s["v_pages"], s["page_table"])
    score = rows @ keys.transpose(-1, -2)
    hidden = torch.arange(keys.shape[2], device=q.device) >= sees[:, :, None]
    score = score.view(b, hkv, most, group, -1).masked_fill_(hidden[:, None, :, None], -math.inf).view_as(score)
    top = score.amax(-1, keepdim=True)
    if s["prefix_len"]:
        n_pre = s["prefix_len"]
        pre_keys = pages(s["k_pages"], s["prefix_pages"])[:, :n_pre]
        pre_values = pages(s["v_pages"], s["prefix_pages"])[:, :n_pre]
        pre_score = rows @ pre_keys.transpose(-1, -2)
        top = torch.maximum(top, pre_score.amax(-1, keepdim=True))
    safe = top.masked_fill(top == -math.inf, 0.0)
    p = score.sub_(safe).exp_()
    total, out = p.sum(-1, keepdim=True), p @ values
    if s["prefix_len"]:
        p = pre_score.sub_(safe).exp_()
        total, out = total + p.sum(-1, keepdim=True), out + p @ pre_values
    lse = safe + total.log()
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    back = lambda x: x.view(b, hkv, most, group, -1)[seq, :, i].reshape(t, hq, -1)  # noqa: E731
    return {"out": back(out).to(q.dtype), "lse": back(lse)[..., 0].contiguous()}


def _plain_sample(s):
    # in 64 bits: whether a token is in or out hangs on sums next to a border
    x = s["logits"].double()
    v = x.shape[1]
    ordered, index = x.sort(dim=1, descending=True, stable=True)
    greedy = s["temperature"] == 0
    temperature = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None]
    w = ((ordered - ordered[:, :1]) / temperature).exp()
    rank = torch.arange(v, device=x.device)
    k = torch.where(s["top_k"] <= 0, torch.full_like(s["top_k"], v), s["top_k"])
    k = torch.where(greedy, torch.ones_like(k), k).long()[:, None]
    w = w.masked_fill(rank >= k, 0.0)
    total = w.cumsum(1)
    keep = (rank < k) & (w >= s["min_p"].double()[:, None])
    keep &= (total - w < s["top_p"].double()[:, None] * total[:, -1:]) | (s["top_p"][:, None] >= 1)
    keep[:, 0] = True
    # the draw: kept weights summed in the order of the tokens
    kept = torch.zeros_like(x).scatter_(1, index, w.masked_fill(~keep, 0.0))
    total = kept.cumsum(1)
    token = (total <= s["u"].double()[:, None] * total[:, -1:]).sum(1)
    p = kept.gather(1, token[:, None])[:, 0] / total[:, -1]
    return {"token": token, "logprob": p.log().float()}


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if not own:
        return {"qk_norm_rope": _plain_qk_norm_rope, "paged_append": _plain_paged_append,
                "paged_attention": _plain_paged_attention, "sample": _plain_sample}[op](s)
    from fourierattention_b200 import ops
    if op == "qk_norm_rope":
        q, k = ops.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], q_weight=s["q_weight"],
                                k_weight=s["k_weight"], eps=EPS)
        return {"q": q, "k": k}
    if op == "paged_append":
        q = ops.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_lens"], s["inv_freq"],
                             cu_seqlens=s["cu_seqlens"], q=s["q"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                             eps=EPS)
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if op == "paged_attention":
        out, lse = ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_lens"],
                                       cu_seqlens=s["cu_seqlens"], prefix_pages=s["prefix_pages"],
                                       prefix_len=s["prefix_len"], return_lse=True)
        return {"out": out, "lse": lse}
    token, logprob = ops.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                min_p=s["min_p"], return_logprob=True)
    return {"token": token, "logprob": logprob}


# ---------------------------------------------------------------------------------------------- what it has to do
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "sample":
        n = case["batch"] * case["vocab"]
        return {"bytes": n * size + case["batch"] * (5 * 4 + 12), "flops": 4 * n}
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "qk_norm_rope":
        n = case["tokens"] * (hq + hkv) * d
        return {"bytes": 2 * n * size + 8 * case["tokens"] + 2 * d, "flops": n * (8 if case["norm"] else 4)}
    new = _spread(case["new"], case["batch"])
    if case["op"] == "paged_append":
        n = sum(new) * (hq + 2 * hkv) * d
        return {"bytes": 2 * n * size + 8 * case["batch"] + 4 * sum(new) // case["page"],
                "flops": n * (8 if case["norm"] else 4)}
    lens = [max(x, y) for x, y in zip(_spread(case["own"], case["batch"]), new)]
    pairs = sum(n * case["prefix"] + n * (l - n) + n * (n + 1) // 2 for l, n in zip(lens, new))
    keys = sum(lens) + case["prefix"]
    return {"bytes": 2 * keys * hkv * d * size + 2 * sum(new) * hq * d * size + 4 * sum(new) * hq
            + 4 * (keys // case["page"] + 2 * case["batch"]), "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_rotate(x, weight, positions, inv_freq):
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    z = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                    torch.outer(positions.double(), inv_freq.double()))
    half = x.shape[-1] // 2
    y = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * z[:, None]
    return torch.cat([y.real, y.imag], -1)


def _exact_sample(s):
    token, logprob = [], []
    rows = s["logits"].double().cpu().numpy()
    params = zip(rows, *(s[k].double().cpu().numpy() for k in ("u", "temperature", "top_k", "top_p", "min_p")))
    for x, u, temperature, top_k, top_p, min_p in params:
        order = np.argsort(-x, kind="stable")
        if temperature == 0:
            token.append(int(order[0]))
            logprob.append(0.0)
            continue
        order = order[:int(top_k)] if top_k > 0 else order
        w = np.exp((x[order] - x[order[0]]) / temperature)
        n = len(order)
        if top_p < 1:
            n = min(n, int(np.searchsorted(np.cumsum(w), top_p * math.fsum(w), side="left")) + 1)
        n = max(1, min(n, int(np.sum(w >= min_p))))
        chosen = np.argsort(order[:n])
        run_sum = np.cumsum(w[chosen])
        at = chosen[int(np.searchsorted(run_sum, u * run_sum[-1], side="right"))]
        token.append(int(order[at]))
        logprob.append(math.log(w[at] / math.fsum(w[:n])))
    return {"token": torch.tensor(token), "logprob": torch.tensor(logprob, dtype=torch.float64)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    if case["op"] == "qk_norm_rope":
        return {n: _exact_rotate(s[n], s[n + "_weight"], s["positions"], s["inv_freq"]) for n in ("q", "k")}
    b = case["batch"]
    new, lens, (_, hkv, page, d) = _spread(case["new"], b), s["kv_lens"].tolist(), s["k_pages"].shape
    if case["op"] == "paged_append":
        at = torch.cat([torch.arange(l - n, l) for l, n in zip(lens, new)]).to(s["q"].device)
        q = _exact_rotate(s["q"], s["q_weight"], at, s["inv_freq"])
        k = _exact_rotate(s["k"], s["k_weight"], at, s["inv_freq"])
        k_pages, v_pages, done = s["k_pages"].double(), s["v_pages"].double(), 0
        for row, l, n in zip(s["page_table"].tolist(), lens, new):
            for first in range((l - n) // page * page, l, page):
                lo, hi = max(first, l - n), min(first + page, l)
                t0 = done + lo - (l - n)
                k_pages[row[first // page], :, lo - first:hi - first] = k[t0:t0 + hi - lo].transpose(0, 1)
                v_pages[row[first // page], :, lo - first:hi - first] = s["v"][t0:t0 + hi - lo].double().transpose(0, 1)
            done += n
        return {"q": q, "k_pages": k_pages, "v_pages": v_pages}
    hq = case["q_heads"]
    read = lambda x, at, n: x[at.long()].permute(0, 2, 1, 3).reshape(-1, hkv, d)[:n].double()  # noqa: E731
    outs, lses, done = [], [], 0
    for x, l, n in zip(s["page_table"], lens, new):
        keys, values = read(s["k_pages"], x, l), read(s["v_pages"], x, l)
        if case["prefix"]:
            keys = torch.cat([read(s["k_pages"], s["prefix_pages"], case["prefix"]), keys])
            values = torch.cat([read(s["v_pages"], s["prefix_pages"], case["prefix"]), values])
        # the last of the new tokens sees every key, each earlier one a key less
        late = torch.arange(len(keys), device=keys.device)[None] > torch.arange(
            len(keys) - n, len(keys), device=keys.device)[:, None]
        out, lse = [], []
        for h in range(hq):
            score = s["q"][done:done + n, h].double() @ keys[:, h * hkv // hq].T / math.sqrt(d)
            score = score.masked_fill(late, -math.inf)
            lse.append(torch.logsumexp(score, -1))
            out.append(torch.softmax(score, -1) @ values[:, h * hkv // hq])
        outs.append(torch.stack(out, 1))
        lses.append(torch.stack(lse, 1))
        done += n
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
