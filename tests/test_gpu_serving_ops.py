"""GPU tests of the operators of a served batch (norm + rotation, paged append, paged attention with a shared prefix,
sampling) against plain implementations in 64 bits.

Tolerances.  A value rounded once to a type with half-step ``h`` (bf16 2^-9, fp16 2^-12 of the next power of two, so at
most ``finfo.eps / 2`` of the value) may be off by ``h |x|``.

* rotation: the float32 arithmetic before the rounding adds at most 2^-20 of the head's largest value (a rotated value
  is a sum of two products whose factors carry a handful of float32 roundings, cos and sin a few 2^-24 of one);
* attention: with s_j = scale q.k_j, a score is off by at most e_s = D 2^-23 scale sum_d |q_d k_jd| (float32
  accumulation of D products, each partial sum truncated) and each probability is rounded once to the cache's type, so
  |error| <= h |o| + (h + 2 e_s + 2^-18) sum_j p_j |v_j| / l; 2^-18 covers exp2, the denominator's and the output's
  float32 sums.  lse is off by at most e_s + 2^-18 + 2^-22 |lse|;
* tokens are equal, log-probabilities off by 2^-22 of themselves + 1e-7 (one rounding to float32).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from fourierattention_b200 import ops as o
    return o


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def excess(err, tol):
    """The most by which an error passes its tolerance (NaN counts as infinite); at most 0 when all is well."""
    d = torch.nan_to_num(err - tol, nan=math.inf)
    return float(d.max()) if d.numel() else 0.0


# ------------------------------------------------------------------------------------------------ norm + rotation
def rope_ref(x, weight, eps, positions, inv_freq):
    x = x.double()
    if weight is not None:
        x = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.double()
    r = inv_freq.numel()
    ang = positions.double()[:, None, None] * inv_freq.double()
    c, s = ang.cos(), ang.sin()
    a, b = x[..., :r], x[..., r:2 * r]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * r:]], -1)


def close(got, ref, dtype, scale):
    err = (got.double() - ref).abs()
    tol = half_step(dtype) * ref.abs() + 2.0 ** -20 * scale + 2.0 ** -24
    assert excess(err, tol) <= 0


def inv_freq(r, theta=500000.0):
    return (1.0 / theta ** (torch.arange(0, r, 2, dtype=torch.float32, device="cuda") / max(r, 1))).contiguous()


@pytest.mark.parametrize("tokens,hq,hkv,d,r,dtype,wtype", [
    (1, 32, 8, 128, 128, BF, BF), (7, 24, 8, 128, 128, HF, torch.float32), (33, 8, 2, 64, 64, BF, None),
    (5, 3, 1, 32, 32, HF, HF), (9, 4, 4, 256, 64, BF, BF), (3, 5, 5, 80, 48, HF, HF), (2, 1, 1, 16, 16, BF, None),
    (4, 2, 1, 96, 0, BF, BF), (2500, 8, 2, 64, 64, HF, HF), (2371, 40, 8, 128, 128, BF, BF)])
def test_norm_rope(ops, tokens, hq, hkv, d, r, dtype, wtype):
    torch.manual_seed(tokens + d)
    qkv = (3 * torch.randn(tokens, hq + 2 * hkv, d, device="cuda")).to(dtype)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hkv]
    w = [None if wtype is None else (1 + 0.3 * torch.randn(d, device="cuda")).to(wtype) for _ in range(2)]
    pos = torch.randint(0, 1 << 20, (tokens,), device="cuda")
    pos[0] = 0
    f = inv_freq(r)
    qo, ko = ops.qk_norm_rope(q, k, pos, f, q_weight=w[0], k_weight=w[1], eps=1e-5)
    for got, x, wt in ((qo, q, w[0]), (ko, k, w[1])):
        ref = rope_ref(x, wt, 1e-5, pos, f)
        close(got, ref, dtype, ref.abs().amax(-1, keepdim=True) + 1)
    # int32 positions and the inputs as outputs give the same bits
    qi, ki = q.clone(), k.clone()
    a, b = ops.qk_norm_rope(qi, ki, pos.int(), f, q_weight=w[0], k_weight=w[1], eps=1e-5, q_out=qi, k_out=ki)
    assert a is qi and b is ki and torch.equal(qi, qo) and torch.equal(ki, ko)


@pytest.mark.parametrize("shift,pitch", [(0, 200), (1, 129), (3, 131)])
def test_norm_rope_any_stride(ops, shift, pitch):
    """Rows that start anywhere and heads of an odd pitch take single-element accesses; neighbours stay untouched."""
    t, h, d = 6, 3, 128
    base = torch.randn(t * h * pitch + 8, device="cuda").to(BF)
    q = base[shift:].as_strided((t, h, d), (h * pitch, pitch, 1), base.storage_offset() + shift)
    k = torch.randn(t, 1, d, device="cuda").to(BF)
    pos, f = torch.arange(t, device="cuda"), inv_freq(d)
    out_base = torch.full_like(base, 7.0)
    out = out_base.as_strided((t, h, d), (h * pitch, pitch, 1), shift)
    ops.qk_norm_rope(q, k, pos, f, q_out=out)
    ref = rope_ref(q, None, 0, pos, f)
    close(out, ref, BF, ref.abs().amax(-1, keepdim=True) + 1)
    touched = torch.zeros_like(base, dtype=torch.bool)
    touched.as_strided((t, h, d), (h * pitch, pitch, 1), shift).fill_(True)
    assert bool((out_base[~touched] == 7.0).all())


def test_norm_rope_nothing_and_far(ops):
    f = inv_freq(64)
    q, k = torch.randn(0, 4, 64, device="cuda").to(BF), torch.randn(0, 2, 64, device="cuda").to(BF)
    qo, ko = ops.qk_norm_rope(q, k, torch.zeros(0, dtype=torch.int64, device="cuda"), f)
    assert qo.shape == q.shape and ko.shape == k.shape
    # a position past 32 bits: the angle is reduced in float64
    q, k = torch.randn(2, 4, 64, device="cuda").to(HF), torch.randn(2, 2, 64, device="cuda").to(HF)
    pos = torch.tensor([2 ** 33 + 5, 2 ** 31 - 1], device="cuda")
    qo, _ = ops.qk_norm_rope(q, k, pos, f)
    # the float64 product of the reference carries 2^-53 of 2^33 turns: 1e-6
    ref = rope_ref(q, None, 0, pos, f)
    assert float((qo.double() - ref).abs().max()) < half_step(HF) * 8 + 2e-5


# ------------------------------------------------------------------------------------------------ pages
def make_pages(lens, hkv, d, ps, dtype, extra=3, layout="heads", max_pages=None):
    """NaN-filled pages with a random table; every entry that no sequence needs names page 0."""
    need = [-(-n // ps) for n in lens]
    total = sum(need) + extra
    if layout == "heads":          # (pages, heads, rows, d)
        mk = lambda: torch.full((total, hkv, ps, d), float("nan"), dtype=dtype, device="cuda")
    elif layout == "rows":         # memory order (pages, rows, heads, d)
        mk = lambda: torch.full((total, ps, hkv, d), float("nan"), dtype=dtype, device="cuda").transpose(1, 2)
    else:                          # K and V interleaved by page
        both = torch.full((total, 2, hkv, ps, d), float("nan"), dtype=dtype, device="cuda")
        it = iter((both[:, 0], both[:, 1]))
        mk = lambda: next(it)
    perm = torch.randperm(total, device="cuda").int()
    table = torch.zeros((len(lens), max_pages or max(need + [1])), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return mk(), mk(), table, perm[at:]


def read_pages(pages, ids, n):
    return pages[ids.long()].transpose(1, 2).flatten(0, 1)[:n]


APPEND = [
    ([1, 1, 1], [0, 15, 47], 16, BF, "heads", True), ([5, 0, 70, 1], [0, 9, 31, 16], 16, HF, "rows", False),
    ([130, 3], [62, 0], 64, BF, "pairs", True), ([1], [4096], 128, HF, "heads", False),
    ([1000, 1500], [7, 0], 48, BF, "rows", True)]


@pytest.mark.parametrize("new,past,ps,dtype,layout,norm", APPEND)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (6, 3, 128)])
def test_append(ops, new, past, ps, dtype, layout, norm, hq, hkv, d):
    torch.manual_seed(len(new) + ps)
    lens = [a + b for a, b in zip(new, past)]
    kp, vp, table, _ = make_pages(lens, hkv, d, ps, dtype, layout=layout)
    before_k, before_v = kp.clone(), vp.clone()
    t = sum(new)
    pad = 2                                                     # tokens behind the last sequence
    one = all(n == 1 for n in new)
    rows = t if one else t + pad
    q, k, v = (torch.randn(rows, h, d, device="cuda").to(dtype) for h in (hq, hkv, hkv))
    w = [(1 + 0.3 * torch.randn(d, device="cuda")).to(dtype) if norm else None for _ in range(2)]
    f = inv_freq(d)
    cu = None if one else torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32, device="cuda")
    q_out = torch.full_like(q, 5.0)
    got = ops.paged_append(k, v, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), f, cu_seqlens=cu,
                           pos_offset=11, q=q, q_weight=w[0], k_weight=w[1], q_out=q_out)
    assert got is q_out and bool((q_out[t:] == 5.0).all())
    pos = torch.cat([torch.arange(p, p + n, device="cuda") for p, n in zip(past, new)]) + 11
    ref_q, ref_k = rope_ref(q[:t], w[0], 1e-6, pos, f), rope_ref(k[:t], w[1], 1e-6, pos, f)
    close(q_out[:t], ref_q, dtype, ref_q.abs().amax(-1, keepdim=True) + 1)
    at = 0
    for b, (n, p) in enumerate(zip(new, past)):
        ks, vs = read_pages(kp, table[b], p + n)[p:], read_pages(vp, table[b], p + n)[p:]
        if n:
            close(ks, ref_k[at:at + n], dtype, ref_k[at:at + n].abs().amax(-1, keepdim=True) + 1)
        assert torch.equal(vs, v[at:at + n])
        for j in range(p, p + n):                               # what was written, taken out again
            page, row = int(table[b, j // ps]), j % ps
            kp[page, :, row] = before_k[page, :, row]
            vp[page, :, row] = before_v[page, :, row]
        at += n
    assert bool(kp.isnan().all()) and bool(vp.isnan().all())    # and nothing else


def test_append_explicit_positions_and_no_queries(ops):
    kp, vp, table, _ = make_pages([40, 8], 2, 64, 16, BF)
    k, v = torch.randn(2, 2, 64, device="cuda").to(BF), torch.randn(2, 2, 64, device="cuda").to(BF)
    pos = torch.tensor([1000, 3], device="cuda", dtype=torch.int32)
    f = inv_freq(32)                                            # half of the head is rotated
    lens = torch.tensor([40, 8], dtype=torch.int32, device="cuda")
    assert ops.paged_append(k, v, kp, vp, table, lens, f, positions=pos) is None
    ref = rope_ref(k, None, 0, pos, f)
    got = torch.stack([read_pages(kp, table[0], 40)[39], read_pages(kp, table[1], 8)[7]])
    close(got, ref, BF, ref.abs().amax(-1, keepdim=True) + 1)


def test_append_where_no_key_is(ops):
    """An inactive sequence (length 0), an index outside the table and page ids that name no page write nothing."""
    kp, vp, table, _ = make_pages([16, 16, 16, 16, 16], 1, 64, 16, BF)
    table[2, 0], table[3, 0] = -1, kp.shape[0]
    k, v = torch.ones(5, 1, 64, device="cuda").to(BF), torch.ones(5, 1, 64, device="cuda").to(BF)
    lens = torch.tensor([0, 17, 4, 4, 4], dtype=torch.int32, device="cuda")
    q = torch.randn(5, 2, 64, device="cuda").to(BF)
    out = ops.paged_append(k, v, kp, vp, table, lens, inv_freq(64), q=q)
    assert not bool(out.isnan().any())
    assert int((~kp.isnan()).sum()) == 64 and int((~vp.isnan()).sum()) == 64      # the fifth one's row alone
    assert bool((vp[int(table[4, 0]), 0, 3] == 1).all())


# ------------------------------------------------------------------------------------------------ attention
def attend_ref(q, new, lens, keys, values, pre_k, pre_v, scale):
    """Per sequence, in float64: (out, lse, sum p |v| / l, score error bound)."""
    outs = []
    at = 0
    hkv = pre_k.shape[1]
    g = q.shape[1] // hkv
    d = q.shape[2]
    for n, l, k, v in zip(new, lens, keys, values):
        k, v = torch.cat([pre_k, k]).double(), torch.cat([pre_v, v]).double()
        np_ = len(pre_k)
        qq = q[at:at + n].double().view(n, hkv, g, d)
        s = torch.einsum("nhgd,khd->nhgk", qq, k) * scale
        e = torch.einsum("nhgd,khd->nhgk", qq.abs(), k.abs()).amax(-1) * scale * d * 2.0 ** -23 if len(k) else torch.zeros(n, hkv, g, device="cuda")
        sees = np_ + l - n + torch.arange(n, device="cuda") + 1
        hid = torch.arange(len(k), device="cuda")[None] >= sees.clamp(min=np_)[:, None]
        s = s.masked_fill(hid[:, None, None], -math.inf)
        lse = torch.logsumexp(s, -1) if len(k) else torch.full((n, hkv, g), -math.inf, device="cuda", dtype=torch.float64)
        p = (s - lse.masked_fill(lse == -math.inf, 0)[..., None]).exp()
        o = torch.einsum("nhgk,khd->nhgd", p, v)
        a = torch.einsum("nhgk,khd->nhgd", p, v.abs())
        outs.append([x.reshape(n, hkv * g, x.shape[3] if x.dim() == 4 else 1) for x in (o, lse, a, e)])
        at += n
    return [torch.cat(x) for x in zip(*outs)]


def check_attention(ops, new, own, prefix, hq, hkv, d, ps, dtype, layout="heads", amp=2.0, scale=None, seed=0, pad=0,
                    q_layout="plain"):
    torch.manual_seed(seed)
    new, own = list(new), list(own)
    kp, vp, table, free = make_pages(own + [prefix], hkv, d, ps, dtype, layout=layout)
    pre_ids, table = table[-1], table[:-1].contiguous()
    pre_ids = pre_ids[:-(-prefix // ps)].contiguous()
    keys, values = [], []
    for ids, n in [(pre_ids, prefix)] + list(zip(table, own)):
        k, v = torch.randn(n, hkv, d, device="cuda").to(dtype), torch.randn(n, hkv, d, device="cuda").to(dtype)
        for j0 in range(0, n, ps):
            m = min(ps, n - j0)
            kp[int(ids[j0 // ps]), :, :m] = k[j0:j0 + m].transpose(0, 1)
            vp[int(ids[j0 // ps]), :, :m] = v[j0:j0 + m].transpose(0, 1)
        keys.append(k)
        values.append(v)
    t = sum(new)
    if q_layout == "plain":
        q = (amp * torch.randn(t + pad, hq, d, device="cuda")).to(dtype)
    else:                       # heads outside, a wide token pitch
        q = (amp * torch.randn(hq, t + pad, d + 8, device="cuda")).to(dtype)[:, :, :d].transpose(0, 1)
    one = all(n == 1 for n in new) and not pad
    cu = None if one else torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32, device="cuda")
    out = torch.full((t + pad, hq, d), 9.0, dtype=dtype, device="cuda")
    got, lse = ops.paged_attention(q, kp, vp, table, torch.tensor(own, dtype=torch.int32, device="cuda"), cu_seqlens=cu,
                                   prefix_pages=pre_ids if prefix else None, prefix_len=prefix, sm_scale=scale, out=out,
                                   return_lse=True)
    assert got is out and bool((out[t:] == 9.0).all())
    sc = scale or 1 / math.sqrt(d)
    o, ref_lse, a, e = attend_ref(q, new, own, keys[1:], values[1:], keys[0], values[0], sc)
    h = half_step(dtype)
    err = (out[:t].double() - o).abs()
    tol = h * o.abs() + (h + 2 * e + 2.0 ** -18) * a + 2.0 ** -24
    assert excess(err, tol) <= 0
    ref_lse, e = ref_lse[..., 0], e[..., 0]
    empty = ref_lse == -math.inf
    assert bool((lse[:t][empty] == -math.inf).all()) and bool((out[:t][empty] == 0).all())
    assert excess((lse[:t].double() - ref_lse)[~empty].abs(), (e + 2.0 ** -18 + 2.0 ** -22 * ref_lse.abs())[~empty]) <= 0
    return q, kp, vp, table, pre_ids


@pytest.mark.parametrize("own", [[1], [15, 16, 17], [0, 3, 0, 127, 128, 129], [2000, 1, 700], [257] * 9])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 64, HF), (32, 8, 128, BF), (3, 1, 128, HF), (9, 1, 64, BF),
                                            (40, 2, 128, BF)])
def test_attention_one_token(ops, own, hq, hkv, d, dtype):
    check_attention(ops, [1] * len(own), own, 0, hq, hkv, d, 16, dtype, seed=len(own) + hq)


@pytest.mark.parametrize("ps", [16, 32, 48, 64, 128, 1024])
@pytest.mark.parametrize("layout", ["heads", "rows", "pairs"])
def test_attention_pages(ops, ps, layout):
    check_attention(ops, [1, 1, 1], [333, 47, 1025], 200, 8, 2, 128, ps, BF, layout=layout, seed=ps, q_layout="wide")


@pytest.mark.parametrize("new,own", [([1], [1]), ([5, 1, 9], [5, 40, 200]), ([130], [130]), ([3, 0, 64, 2], [3, 50, 64, 1]),
                                     ([300, 17], [1000, 17]), ([40, 200], [20, 150])])
@pytest.mark.parametrize("prefix", [0, 1, 129, 1000])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 64, BF), (12, 4, 128, HF)])
def test_attention_many_tokens(ops, new, own, prefix, hq, hkv, d, dtype):
    """Causal rows; more new tokens than keys leaves the first of them without any (own < new)."""
    check_attention(ops, new, own, prefix, hq, hkv, d, 32, dtype, seed=prefix + len(new), pad=3)


@pytest.mark.parametrize("batch,prefix,hq,hkv,d,dtype", [(1, 4096, 8, 2, 64, BF), (3, 777, 32, 8, 128, HF),
                                                       (33, 2050, 32, 8, 128, BF), (70, 640, 16, 1, 128, HF),
                                                       (130, 300, 4, 4, 64, BF), (64, 5000, 8, 2, 128, BF)])
def test_attention_shared_prefix(ops, batch, prefix, hq, hkv, d, dtype):
    own = [(37 * b) % 300 for b in range(batch)]
    check_attention(ops, [1] * batch, own, prefix, hq, hkv, d, 64, dtype, seed=batch)


@pytest.mark.parametrize("amp,scale", [(30.0, None), (1.0, 3.0), (0.0, None)])
def test_attention_score_ranges(ops, amp, scale):
    """Scores of hundreds, where the running maximum jumps, and scores that are all alike."""
    check_attention(ops, [1, 1, 20], [1500, 40, 300], 900, 8, 2, 128, 64, HF, amp=amp, scale=scale)


def test_attention_rising_scores(ops):
    """Scores that rise with every tile move the running maximum, and all that it scales, each time."""
    for dtype, new in ((BF, 1), (BF, 100)):
        d, n = 128, 3000
        kp, vp, table, _ = make_pages([n], 1, d, 64, dtype)
        k = torch.zeros(n, 1, d, device="cuda")
        k[:, 0, 0] = torch.arange(n, device="cuda") / 8.0
        k, v = k.to(dtype), torch.randn(n, 1, d, device="cuda").to(dtype)
        for j0 in range(0, n, 64):
            m = min(64, n - j0)
            kp[int(table[0, j0 // 64]), :, :m] = k[j0:j0 + m].transpose(0, 1)
            vp[int(table[0, j0 // 64]), :, :m] = v[j0:j0 + m].transpose(0, 1)
        q = torch.zeros(new, 4, d, device="cuda")
        q[:, :, 0] = torch.tensor([1.0, 4.0, -4.0, 0.25], device="cuda")
        q = q.to(dtype)
        cu = torch.tensor([0, new], dtype=torch.int32, device="cuda")
        lens = torch.tensor([n], dtype=torch.int32, device="cuda")
        out, lse = ops.paged_attention(q, kp, vp, table, lens, cu_seqlens=cu, sm_scale=1.0, return_lse=True)
        none = torch.zeros(0, 1, d, device="cuda", dtype=dtype)
        o, rl, a, e = attend_ref(q, [new], [n], [k], [v], none, none, 1.0)
        h = half_step(dtype)
        assert excess((out.double() - o).abs(), h * o.abs() + (h + 2 * e + 2.0 ** -18) * a + 2.0 ** -24) <= 0
        assert excess((lse.double() - rl[..., 0]).abs(), e[..., 0] + 2.0 ** -18 + 2.0 ** -22 * rl[..., 0].abs()) <= 0


def test_attention_page_ids_that_name_no_page(ops):
    """Their keys do not exist: the result is that of the other pages."""
    d, ps = 64, 16
    kp, vp, table, _ = make_pages([96], 2, d, ps, BF)
    k, v = torch.randn(96, 2, d, device="cuda").to(BF), torch.randn(96, 2, d, device="cuda").to(BF)
    for i in range(6):
        kp[int(table[0, i])], vp[int(table[0, i])] = k[16 * i:16 * i + 16].transpose(0, 1), v[16 * i:16 * i + 16].transpose(0, 1)
    table[0, 1], table[0, 4] = -7, kp.shape[0] + 100
    q = torch.randn(1, 4, d, device="cuda").to(BF)
    out, lse = ops.paged_attention(q, kp, vp, table, torch.tensor([96], dtype=torch.int32, device="cuda"), return_lse=True)
    keep = torch.tensor([i for i in range(96) if i // 16 not in (1, 4)], device="cuda")
    none = torch.zeros(0, 2, d, device="cuda", dtype=BF)
    o, rl, a, e = attend_ref(q, [1], [64], [k[keep]], [v[keep]], none, none, 1 / 8)
    assert excess((out.double() - o).abs(), 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2 * e + 2.0 ** -18) * a) <= 0
    assert float((lse.double() - rl[..., 0]).abs().max()) < 1e-4
    table[:] = -1
    out, lse = ops.paged_attention(q, kp, vp, table, torch.tensor([96], dtype=torch.int32, device="cuda"), return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_many_sequences(ops):
    """More sequences than a CTA has threads: every scan over them takes several per thread."""
    check_attention(ops, [1] * 1500, [(7 * b) % 40 for b in range(1500)], 0, 4, 1, 64, 16, BF)
    new = [(0, 1, 2, 9)[b % 4] for b in range(900)]
    check_attention(ops, new, [n + (5 * b) % 30 for b, n in enumerate(new)], 50, 8, 2, 64, 16, HF, pad=2)
    check_attention(ops, [3 * (b % 30) for b in range(400)], [3 * (b % 30) + b % 7 for b in range(400)], 70, 8, 2, 64, 32, BF)
    lens = [n + (5 * b) % 30 for b, n in enumerate(new)]
    kp, vp, table, _ = make_pages(lens, 1, 64, 16, BF)
    t = sum(new)
    k, v = torch.randn(t, 1, 64, device="cuda").to(BF), torch.randn(t, 1, 64, device="cuda").to(BF)
    f = inv_freq(64)
    ops.paged_append(k, v, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), f,
                     cu_seqlens=torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32, device="cuda"))
    at = torch.cat([torch.arange(l - n, l) for l, n in zip(lens, new)]).cuda()
    seq = torch.repeat_interleave(torch.arange(900), torch.tensor(new)).cuda()
    page = table[seq, at // 16].long()
    assert torch.equal(vp[page, 0, at % 16], v[:, 0])
    ref = rope_ref(k, None, 0, at, f)
    close(kp[page, 0, at % 16], ref[:, 0], BF, ref[:, 0].abs().amax(-1, keepdim=True) + 1)
    assert int((~vp.isnan()).sum()) == t * 64
    x, u = torch.randn(3000, 257, device="cuda"), torch.rand(3000, device="cuda")
    check_sample(ops, x, u, top_k=30, top_p=0.9)
    check_sample(ops, x, u, top_p=0.7, min_p=0.01)


def test_attention_without_pages(ops):
    """A table of no pages, and tokens without sequences."""
    kp, vp = torch.zeros(2, 2, 2, 16, 64, device="cuda").to(BF)
    q = torch.randn(3, 4, 64, device="cuda").to(BF)
    none = torch.zeros((3, 0), dtype=torch.int32, device="cuda")
    out, lse = ops.paged_attention(q, kp, vp, none, torch.tensor([5, 0, -3], dtype=torch.int32, device="cuda"), return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    kv = torch.randn(3, 2, 64, device="cuda").to(BF)
    ops.paged_append(kv, kv, kp, vp, none, torch.tensor([5, 0, -3], dtype=torch.int32, device="cuda"), inv_freq(64))
    assert bool((kp == 0).all()) and bool((vp == 0).all())
    got = ops.paged_attention(q[:0], kp, vp, none[:0], torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert got.shape == (0, 4, 64)
    out = torch.full_like(q, 3.0)
    ops.paged_attention(q, kp, vp, none[:0], torch.zeros(0, dtype=torch.int32, device="cuda"),
                        cu_seqlens=torch.zeros(1, dtype=torch.int32, device="cuda"), out=out)
    assert bool((out == 3).all())


def test_attention_shared_pages_and_strided_table(ops):
    """Sequences that name the same pages, a table that is a view of a wider one."""
    torch.manual_seed(2)
    d, ps, n = 128, 32, 90
    kp, vp, table, _ = make_pages([n], 2, d, ps, HF)
    k, v = torch.randn(n, 2, d, device="cuda").to(HF), torch.randn(n, 2, d, device="cuda").to(HF)
    for i in range(3):
        m = min(ps, n - ps * i)
        kp[int(table[0, i]), :, :m], vp[int(table[0, i]), :, :m] = k[ps * i:ps * i + m].transpose(0, 1), v[ps * i:ps * i + m].transpose(0, 1)
    wide = torch.full((4, 9), -5, dtype=torch.int32, device="cuda")
    wide[:, 2:5] = table[:, :3]
    q = torch.randn(4, 8, d, device="cuda").to(HF)
    lens = [90, 1, 64, 33]
    out = ops.paged_attention(q, kp, vp, wide[:, 2:6], torch.tensor(lens, dtype=torch.int32, device="cuda"))
    none = torch.zeros(0, 2, d, device="cuda", dtype=HF)
    o, _, a, e = attend_ref(q, [1] * 4, lens, [k[:x] for x in lens], [v[:x] for x in lens], none, none, d ** -0.5)
    h = half_step(HF)
    assert excess((out.double() - o).abs(), h * o.abs() + (h + 2 * e + 2.0 ** -18) * a + 2.0 ** -24) <= 0


def test_attention_far_offsets(ops):
    """Pages beyond 2^31 elements, lengths beyond the table."""
    d, ps, hkv = 128, 1024, 8
    n_pages = 2 ** 31 // (hkv * ps * d) + 40                  # 4.5 GB per tensor
    kp = torch.empty((n_pages, hkv, ps, d), dtype=BF, device="cuda")
    vp = torch.empty_like(kp)
    ids = torch.tensor([[n_pages - 1, 0, n_pages - 3]], dtype=torch.int32, device="cuda")
    f = inv_freq(d)
    k, v = torch.randn(3 * ps, hkv, d, device="cuda").to(BF), torch.randn(3 * ps, hkv, d, device="cuda").to(BF)
    cu = torch.tensor([0, 3 * ps], dtype=torch.int32, device="cuda")
    lens = torch.tensor([3 * ps], dtype=torch.int32, device="cuda")
    ops.paged_append(k, v, kp, vp, ids, lens, f, cu_seqlens=cu)
    q = (2 * torch.randn(1, 16, d, device="cuda")).to(BF)
    out, lse = ops.paged_attention(q, kp, vp, ids, lens + 500, return_lse=True)      # cut at the table's end
    none = torch.zeros(0, hkv, d, device="cuda", dtype=BF)
    kk, vv = read_pages(kp, ids[0], 3 * ps), read_pages(vp, ids[0], 3 * ps)
    ref = rope_ref(k, None, 0, torch.arange(3 * ps, device="cuda"), f)
    close(kk, ref, BF, ref.abs().amax(-1, keepdim=True) + 1)
    assert torch.equal(vv, v)
    o, rl, a, e = attend_ref(q, [1], [3 * ps], [kk], [vv], none, none, d ** -0.5)
    assert excess((out.double() - o).abs(), 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2 * e + 2.0 ** -18) * a) <= 0


def test_attention_repeats_and_replays(ops):
    """The same call gives the same bits, on another stream too; a captured step follows lengths, tables and pages that
    change between replays, and two graphs that live at once do not share scratch."""
    q, kp, vp, table, pre = check_attention(ops, [1] * 5, [100, 700, 0, 333, 16], 600, 8, 2, 128, 16, BF)
    lens = torch.tensor([100, 700, 0, 333, 16], dtype=torch.int32, device="cuda")
    call = lambda: ops.paged_attention(q, kp, vp, table, lens, prefix_pages=pre, prefix_len=600, return_lse=True)
    a, la = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b, lb = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b) and torch.equal(la, lb)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        c1, _ = call()
    with torch.cuda.graph(g2):
        c2 = ops.paged_attention(q, kp, vp, table, lens)
    lens.copy_(torch.tensor([64, 1, 0, 300, 9], dtype=torch.int32))
    table[1].fill_(int(table[0, 0]))
    g1.replay()
    g2.replay()
    g1.replay()
    torch.cuda.synchronize()
    e1, _ = call()
    e2 = ops.paged_attention(q, kp, vp, table, lens)
    assert torch.equal(c1, e1) and torch.equal(c2[lens > 0], e2[lens > 0]) and bool((c2[2] == 0).all())


# ------------------------------------------------------------------------------------------------ sampling
def sample_ref(x, u, temperature, top_k, top_p, min_p):
    x = x.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1, -np.inf
    order = np.argsort(-x, kind="stable")
    if not temperature > 0:
        return int(order[0]), 0.0
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / temperature))
    n = len(order) if top_k <= 0 else min(top_k, len(order))
    if top_p < 1:
        n = min(n, int(np.searchsorted(np.cumsum(w[:n]), top_p * math.fsum(w[:n]), side="left")) + 1)
    n = max(1, min(n, int(np.sum(w >= min_p))))
    chosen = np.argsort(order[:n])
    cum = np.cumsum(w[chosen])
    at = min(int(np.searchsorted(cum, u * cum[-1], side="right")), n - 1)
    while w[chosen[at]] == 0:
        at -= 1
    return int(order[chosen[at]]), math.log(w[chosen[at]] / math.fsum(w[:n]))


def check_sample(ops, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    B = x.shape[0]
    got, lp = ops.sample(x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, return_logprob=True)
    per = lambda v: v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(B, float(np.float32(v)))
    params = list(zip(x.double().cpu().numpy(), per(u), per(temperature), per(top_k).astype(int), per(top_p), per(min_p)))
    want = [sample_ref(*p) for p in params]
    assert got.tolist() == [w[0] for w in want]
    ref = torch.tensor([w[1] for w in want], dtype=torch.float64)
    fin = torch.isfinite(ref)
    assert bool((lp.cpu()[~fin] == -math.inf).all())
    assert float(((lp.cpu().double() - ref)[fin].abs() - 2.0 ** -22 * ref[fin].abs()).max()) < 1e-7
    assert torch.equal(ops.sample(x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p), got)
    return got


@pytest.mark.parametrize("B,V", [(1, 1), (2, 2), (3, 31), (4, 33), (5, 1000), (2, 16385), (3, 32003), (1, 128256),
                                 (150, 4099), (2, 200001), (1, 393216)])
@pytest.mark.parametrize("dtype", [torch.float32, BF, HF])
def test_sample_shapes(ops, B, V, dtype):
    torch.manual_seed(B * V)
    x = (3 * torch.randn(B, V, device="cuda")).to(dtype)
    u = torch.rand(B, device="cuda")
    check_sample(ops, x, u)
    check_sample(ops, x, u, temperature=0.7, top_k=50, top_p=0.9, min_p=0.01)
    check_sample(ops, x, u, temperature=0.0)


@pytest.mark.parametrize("kw", [dict(top_k=1), dict(top_k=2), dict(top_k=700), dict(top_k=10 ** 6), dict(top_p=0.0),
                                dict(top_p=1e-6), dict(top_p=0.5), dict(top_p=0.99), dict(top_p=0.9999), dict(min_p=0.2),
                                dict(min_p=1.0), dict(top_k=2000, top_p=0.97), dict(top_k=5, top_p=0.3, min_p=0.5),
                                dict(temperature=0.01, top_p=0.9), dict(temperature=50.0, top_p=0.9),
                                dict(temperature=50.0, top_k=5000)])
@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_sample_filters(ops, kw, dtype):
    torch.manual_seed(5)
    x = (2.5 * torch.randn(24, 20011, device="cuda")).to(dtype)
    check_sample(ops, x, torch.rand(24, device="cuda"), **kw)


def test_sample_per_row_parameters(ops):
    torch.manual_seed(6)
    B = 97
    x = 4 * torch.randn(B, 5000, device="cuda")
    kw = dict(temperature=torch.rand(B, device="cuda") * 2, top_k=torch.randint(-1, 300, (B,), device="cuda", dtype=torch.int32),
              top_p=torch.rand(B, device="cuda") * 1.2, min_p=torch.rand(B, device="cuda") * 0.2)
    kw["temperature"][::7] = 0
    check_sample(ops, x, torch.rand(B, device="cuda"), **kw)


def test_sample_ties_and_specials(ops):
    inf, nan = math.inf, math.nan
    # long rows of equal logits: ties go by index, counted across CTAs
    for V in (700, 20000, 128256):
        x = torch.zeros(6, V, device="cuda", dtype=BF)
        x[:, V // 2:] = -1.0
        u = torch.tensor([0.0, 0.1, 0.37, 0.61, 0.93, 1 - 2.0 ** -24], device="cuda")
        check_sample(ops, x, u, top_k=V // 3)
        check_sample(ops, x, u, top_p=0.33)
        check_sample(ops, x, u, top_p=0.83)
        check_sample(ops, x, u, top_k=V - 5, top_p=0.9)
        got = ops.sample(x, u, top_k=1)
        assert got.tolist() == [0] * 6
    rows = [[-inf, 2.0, -inf, 1.0], [inf, 1.0, inf, 0.0], [nan, 0.0, 1.0, nan], [-inf] * 4, [nan] * 4,
            [-3.4e38, 3.4e38, 0.0, 1.0], [0.0, -0.0, 0.0, -0.0], [inf, -inf, nan, 3.0]]
    x = torch.tensor(rows, device="cuda")
    for u0 in (0.0, 0.4, 0.6, 0.99):
        u = torch.full((len(rows),), u0, device="cuda")
        check_sample(ops, x, u)
        check_sample(ops, x, u, top_k=2)
        check_sample(ops, x, u, top_p=0.6)
        check_sample(ops, x, u, top_k=3, min_p=0.5, temperature=0.5)
    # logits far apart, of many magnitudes: the bins of a row are of very different fill
    torch.manual_seed(9)
    x = torch.randn(8, 50000, device="cuda") * 10.0 ** torch.randint(-30, 30, (8, 50000), device="cuda").float()
    u = torch.rand(8, device="cuda")
    check_sample(ops, x, u, top_k=30000)
    check_sample(ops, x, u, top_k=17, top_p=0.8)
    x = 1e-6 * torch.randn(8, 50000, device="cuda") + 5.0
    check_sample(ops, x, u, top_k=20000)
    check_sample(ops, x, u, top_p=0.5)
    x[:, 100] = -1e30                                            # one bin holds everything but one
    check_sample(ops, x, u, top_k=20000)
    check_sample(ops, x, u, top_p=0.5)


def test_sample_strides_streams_graphs(ops):
    torch.manual_seed(3)
    wide = torch.randn(6, 4000, device="cuda").to(HF)
    x, u = wide[::2, 7:3010], torch.rand(3, device="cuda")       # a view: odd start, odd pitch
    check_sample(ops, x, u, top_p=0.9)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = ops.sample(x, u, top_p=0.9)
    s.synchronize()
    assert torch.equal(b, ops.sample(x, u, top_p=0.9))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c = ops.sample(x, u, top_k=20, top_p=0.9)
    u.copy_(torch.rand(3, device="cuda"))
    wide.copy_(torch.randn(6, 4000, device="cuda").to(HF))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(c, ops.sample(x, u, top_k=20, top_p=0.9))
    assert ops.sample(x[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("B,V", [(1, 128256), (5, 128256), (20, 128256), (150, 20000), (3, 4100)])
@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("run", [300, 1000])
def test_sample_masked_to_neighbours(ops, B, V, dtype, run):
    """Long rows masked to a run of neighbouring tokens, as a grammar does: few threads hold a logit that can be drawn,
    fewer than top-k wants (a thread reads 4 or 8 neighbours at once), in clusters of 1 to 8 CTAs."""
    torch.manual_seed(B + run)
    x = torch.full((B, V), -math.inf, device="cuda", dtype=dtype)
    for b in range(B):
        at = (997 * b) % (V - run)
        x[b, at:at + run] = (2 * torch.randn(run, device="cuda")).to(dtype)
    u = torch.rand(B, device="cuda")
    for k in (run // 6, run // 3, run - 1, run, run + 1):
        if k <= 512:
            check_sample(ops, x, u, top_k=k)
        check_sample(ops, x, u, top_k=k, top_p=0.8, min_p=0.001)
    check_sample(ops, x, u, top_p=0.9)


@pytest.mark.parametrize("new", [2, 3, 40, 60])
@pytest.mark.parametrize("prefix", [0, 100])
@pytest.mark.parametrize("past", [0, 1, 35, 2 ** 31 - 1 - 112])
def test_attention_lengths_behind_the_table(ops, new, prefix, past):
    """Several new tokens whose sequence is longer than its table: the keys behind the table do not exist, and each token
    sees those before it that do, counted from the length as given."""
    torch.manual_seed(new + prefix)
    d, ps, hkv, hq, cap = 64, 16, 2, 8, 112
    kp, vp, table, _ = make_pages([cap, 30, prefix], hkv, d, ps, BF)
    pre, table = table[2, :-(-prefix // ps)].contiguous(), table[:2].contiguous()
    keys, values = [], []
    for ids, n in ((pre, prefix), (table[0], cap), (table[1], 30)):
        k, v = torch.randn(n, hkv, d, device="cuda").to(BF), torch.randn(n, hkv, d, device="cuda").to(BF)
        for j0 in range(0, n, ps):
            m = min(ps, n - j0)
            kp[int(ids[j0 // ps]), :, :m], vp[int(ids[j0 // ps]), :, :m] = k[j0:j0 + m].transpose(0, 1), v[j0:j0 + m].transpose(0, 1)
        keys.append(k)
        values.append(v)
    lens, news = [cap + past, 30], [new, new]
    q = (2 * torch.randn(2 * new, hq, d, device="cuda")).to(BF)
    cu = torch.tensor([0, new, 2 * new], dtype=torch.int32, device="cuda")
    out, lse = ops.paged_attention(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), cu_seqlens=cu,
                                   prefix_pages=pre if prefix else None, prefix_len=prefix, return_lse=True)
    o, rl, a, e = attend_ref(q, news, lens, keys[1:], values[1:], keys[0], values[0], d ** -0.5)
    h = half_step(BF)
    assert excess((out.double() - o).abs(), h * o.abs() + (h + 2 * e + 2.0 ** -18) * a + 2.0 ** -24) <= 0
    rl, e = rl[..., 0], e[..., 0]
    some = rl > -math.inf
    assert excess((lse.double() - rl)[some].abs(), (e + 2.0 ** -18 + 2.0 ** -22 * rl.abs())[some]) <= 0
    assert bool((lse[~some] == -math.inf).all()) and bool((out[~some] == 0).all())


def _time(f, n=5):
    best = math.inf
    for _ in range(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("V", [262144, 393216])
def test_sample_large_vocabulary_of_equal_logits(ops, V):
    """2^18 equal weights fill 32 bits of a bin's count.  The proposal of a bin still names the right one: a wrong one is
    put right bin by bin, over a thousand passes over the row, where a proposal takes a few."""
    u = torch.tensor([0.0, 0.37, 0.93], device="cuda")
    x = torch.zeros(3, V, device="cuda", dtype=BF)
    x[:, 262144:] = -9.0                                        # exactly 2^18 of the largest
    check_sample(ops, x, u, top_p=0.5)
    x[:, 5] = -1.0
    check_sample(ops, x, u, top_p=0.25)
    check_sample(ops, x, u, top_p=0.75, min_p=0.5)
    x[:, 5] = 0.0
    spread = torch.randn(3, V, device="cuda").to(BF)
    ops.sample(spread, u, top_p=0.5)
    # the same number of passes as any other row, within a factor that a thousand passes would exceed by far
    assert _time(lambda: ops.sample(x, u, top_p=0.5)) < 10 * _time(lambda: ops.sample(spread, u, top_p=0.5))


@pytest.mark.parametrize("V", [64, 30000, 128256])
@pytest.mark.parametrize("top_k", [0, 40, 20000])
def test_sample_odd_filter_values(ops, V, top_k):
    """NaN filters are off and min_p above 1 keeps the first of the largest logits, whichever way a row is searched."""
    torch.manual_seed(V)
    B = 6
    x = torch.randn(B, V, device="cuda").to(BF)
    x[:, V // 2:V // 2 + 9] = 8.0                               # nine largest
    u = torch.tensor([0.0, 0.2, 0.4, 0.6, 0.8, 0.99], device="cuda")
    full = lambda v: torch.full((B,), v, device="cuda")
    nan = math.nan
    off = ops.sample(x, u, top_k=top_k, return_logprob=True)
    for kw in (dict(top_p=full(nan)), dict(min_p=full(nan)), dict(top_p=full(nan), min_p=full(nan)), dict(min_p=full(-1.0)),
               dict(top_p=full(math.inf))):
        got = ops.sample(x, u, top_k=top_k, return_logprob=True, **kw)
        assert torch.equal(got[0], off[0]) and torch.equal(got[1], off[1]), kw
    assert torch.equal(ops.sample(x, u, top_k=top_k, top_p=full(-3.0)), ops.sample(x, u, top_k=top_k, top_p=0.0))
    for kw in (dict(min_p=1.5), dict(min_p=full(1.5)), dict(min_p=full(math.inf), top_p=0.9)):
        token, logprob = ops.sample(x, u, top_k=top_k, return_logprob=True, **kw)
        assert token.tolist() == [V // 2] * B and bool((logprob == 0).all()), kw
        check_sample(ops, x, u, top_k=top_k, **kw)
    check_sample(ops, x, u, top_k=top_k, min_p=1.0)             # all nine
    assert torch.equal(ops.sample(x, u, temperature=full(nan)), ops.sample(x, u, temperature=0.0))


def kernels_of(f):
    """Number of kernels that ``f`` puts into a captured graph."""
    rt = pytest.importorskip("cuda.bindings.runtime")
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        f()
    raw = rt.cudaGraph_t(init_value=g.raw_cuda_graph())
    n = rt.cudaGraphGetNodes(raw)[2]
    nodes = rt.cudaGraphGetNodes(raw, n)[1] if n else []
    return sum(rt.cudaGraphNodeGetType(x)[1] == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for x in nodes)


@pytest.mark.parametrize("new,prefix", [(None, 0), (None, 40), (1, 40), (30, 40), (30, 0), (47, 40), (48, 40), (200, 40), (0, 40),
                                        (0, 0)])
def test_launches_are_counted_as_they_are(ops, new, prefix):
    """Two kernels without a prefix, three with one, two again where it is read in front of the sequences' own keys; none
    for an empty call."""
    B, d, hkv, hq = 2, 64, 2, 8
    kp, vp, table, pre = make_pages([256, 256], hkv, d, 16, BF)
    kp.zero_(), vp.zero_()
    t = B if new is None else B * new
    q, kv = torch.zeros(t, hq, d, device="cuda", dtype=BF), torch.zeros(t, hkv, d, device="cuda", dtype=BF)
    lens = torch.tensor([256, 250], dtype=torch.int32, device="cuda")
    cu = None if new is None else torch.tensor([0, new, 2 * new], dtype=torch.int32, device="cuda")
    f, x, u, pos = inv_freq(d), torch.zeros(t, 50, device="cuda"), torch.zeros(t, device="cuda"), torch.arange(t, device="cuda")
    for call in (lambda: ops.paged_attention(q, kp, vp, table, lens, cu_seqlens=cu, prefix_pages=pre, prefix_len=prefix),
                 lambda: ops.paged_append(kv, kv, kp, vp, table, lens, f, cu_seqlens=cu),
                 lambda: ops.qk_norm_rope(q, kv, pos, f), lambda: ops.sample(x, u)):
        call()
        before = ops.launch_count
        n = kernels_of(call)
        assert ops.launch_count - before == n


@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("shared", [False, True])
def test_attention_many_small_probabilities(ops, new, dtype, shared):
    """Keys far behind a few dominant ones, whose values are zero, make up the output: each of their probabilities has to
    keep its bits.  They are 2^-20.6 of the largest; below 2^-21 of it a float16 probability is off by up to 2^-32 of the
    largest, so n keys add n 2^-32 max |v| / (weight of the dominant ones) to the tolerance."""
    d, ps, hkv, n, B = 64, 64, 8, 20000, 20
    kp, vp, table, _ = make_pages([n], hkv, d, ps, dtype)
    k, v = torch.zeros(n, hkv, d, device="cuda"), torch.rand(n, hkv, d, device="cuda") + 0.5
    far, near = -14.25, torch.arange(0, 128, 16, device="cuda")
    k[:, :, 0] = far
    k[near] = 0.0
    v[near] = 0.0
    k, v = k.to(dtype), v.to(dtype)
    for j0 in range(0, n, ps):
        m = min(ps, n - j0)
        kp[int(table[0, j0 // ps]), :, :m], vp[int(table[0, j0 // ps]), :, :m] = k[j0:j0 + m].transpose(0, 1), v[j0:j0 + m].transpose(0, 1)
    q = torch.zeros(B * new, hkv, d, device="cuda", dtype=dtype)
    q[:, :, 0] = 1.0
    cu = None if new == 1 else torch.arange(0, B * new + 1, new, dtype=torch.int32, device="cuda")
    if shared:
        out, lse = ops.paged_attention(q, kp, vp, torch.zeros((B, 1), dtype=torch.int32, device="cuda"),
                                       torch.zeros(B, dtype=torch.int32, device="cuda"), cu_seqlens=cu, prefix_pages=table[0],
                                       prefix_len=n, sm_scale=1.0, return_lse=True)
        own, args = 0, (k, v)
    else:
        out, lse = ops.paged_attention(q, kp, vp, table.expand(B, -1), torch.full((B,), n, dtype=torch.int32, device="cuda"),
                                       cu_seqlens=cu, sm_scale=1.0, return_lse=True)
        own, args = n, (k[:0], v[:0])
    one = (k[:own], v[:own])
    o, rl, a, e = attend_ref(q[:new], [new], [own], [one[0]], [one[1]], *args, 1.0)
    h = half_step(dtype)
    tol = h * o.abs() + (h + 2 * e + 2.0 ** -18) * a + n * 2.0 ** -32 * 1.5 / 8 + 2.0 ** -24
    assert excess((out.double().view(B, new, hkv, d) - o).abs(), tol.expand(B, new, hkv, d)) <= 0
    assert excess((lse.double().view(B, new, hkv) - rl[..., 0]).abs(), (e[..., 0] + 2.0 ** -18 + 2.0 ** -22 * rl[..., 0].abs()).expand(B, new, hkv)) <= 0


@pytest.mark.parametrize("ps", [16, 64, 256])
@pytest.mark.parametrize("new", [1, 3, 30, 60])
@pytest.mark.parametrize("where", ["own", "prefix", "both", "all"])
def test_page_ids_that_name_no_page_in_every_form(ops, ps, new, where):
    """Their keys do not exist, for both kernels, in the own pages and in a prefix (read for the batch or in front of the own
    keys), with pages smaller and larger than a tile.  The pages that the ids used to name hold NaN."""
    torch.manual_seed(ps + new)
    d, hkv, hq, B, dtype = 128, 2, 8, 2, BF
    own, prefix = [5 * ps + 3 + new, 2 * ps + new], 4 * ps - 5
    kp, vp, table, _ = make_pages(own + [prefix], hkv, d, ps, dtype)
    drop = {0: [0, 2], 1: [1], 2: [1, 3]}                       # pages of the two sequences and of the prefix
    if where == "all":
        drop = {i: list(range(table.shape[1])) for i in range(3)}
    elif where != "both":
        drop = {i: (p if (i == 2) == (where == "prefix") else []) for i, p in drop.items()}
    keys, values = [], []
    for i, n in enumerate(own + [prefix]):
        k, v = torch.randn(n, hkv, d, device="cuda").to(dtype), torch.randn(n, hkv, d, device="cuda").to(dtype)
        for j in range(-(-n // ps)):
            m = min(ps, n - j * ps)
            if j in drop[i]:
                table[i, j] = -1 - j if j % 2 else kp.shape[0] + 7 * j
            else:
                kp[int(table[i, j]), :, :m] = k[j * ps:j * ps + m].transpose(0, 1)
                vp[int(table[i, j]), :, :m] = v[j * ps:j * ps + m].transpose(0, 1)
        keys.append(k)
        values.append(v)
    q = (2 * torch.randn(B * new, hq, d, device="cuda")).to(dtype)
    cu = torch.arange(0, B * new + 1, new, dtype=torch.int32, device="cuda")
    out, lse = ops.paged_attention(q, kp, vp, table[:2], torch.tensor(own, dtype=torch.int32, device="cuda"), cu_seqlens=cu,
                                   prefix_pages=table[2, :4].contiguous(), prefix_len=prefix, return_lse=True)
    there = lambda i, n: torch.tensor([j // ps not in drop[i] for j in range(n)], device="cuda")
    pre_there = there(2, prefix)
    for b in range(B):
        for i in range(new):                                    # a token at a time: what it sees, less what is not there
            sees = own[b] - new + 1 + i
            keep = there(b, own[b])[:sees]
            k, v = torch.cat([keys[2][pre_there], keys[b][:sees][keep]]), torch.cat([values[2][pre_there], values[b][:sees][keep]])
            o, rl, a, e = attend_ref(q[b * new + i][None], [1], [len(k)], [k], [v], k[:0], v[:0], d ** -0.5)
            h, got = half_step(dtype), out[b * new + i]
            if not len(k):
                assert bool((got == 0).all()) and bool((lse[b * new + i] == -math.inf).all())
                continue
            assert excess((got.double() - o[0]).abs(), (h * o.abs() + (h + 2 * e + 2.0 ** -18) * a + 2.0 ** -24)[0]) <= 0
            assert excess((lse[b * new + i].double() - rl[0, :, 0]).abs(), e[0, :, 0] + 2.0 ** -18 + 2.0 ** -22 * rl[0, :, 0].abs()) <= 0


@pytest.mark.parametrize("V", [131073, 151936, 262145, 393215])
def test_sample_long_rows_of_any_alignment(ops, V):
    """Several rounds per CTA; rows that start off 16 bytes, with and without room for what leads them in."""
    torch.manual_seed(V)
    for dtype in (torch.float32, HF):
        x, u = (3 * torch.randn(3, V, device="cuda")).to(dtype), torch.rand(3, device="cuda")
        check_sample(ops, x, u)
        check_sample(ops, x, u, top_k=50, top_p=0.9)
        check_sample(ops, x, u, top_k=3000, min_p=1e-4)
        check_sample(ops, x, u, top_p=0.95, temperature=0.8)
        check_sample(ops, x, u, temperature=0.0)


@pytest.mark.parametrize("ps", [48, 80, 128, 1024])
@pytest.mark.parametrize("layout", ["heads", "rows", "pairs"])
def test_attention_pages_of_many_tokens(ops, ps, layout):
    """Page sizes and layouts under the tensor-core kernel: a prefix as a phase of its own, and in front of the own keys."""
    for new in ([70, 30], [20, 9, 30]):
        own = [n + 333 * i for i, n in enumerate(new)]
        for prefix in (0, 700):
            check_attention(ops, new, own, prefix, 8, 2, 128, ps, HF, layout=layout, seed=ps, q_layout="wide", pad=1)


@pytest.mark.parametrize("new,own,prefix,hq,hkv,d,dtype", [
    ([2500, 1, 700], [2500, 2500, 900], 0, 8, 2, 128, BF), ([4000], [4000], 0, 4, 1, 64, HF),
    ([512] + [1] * 255, [1500] + [100 + 3 * i for i in range(255)], 0, 8, 2, 128, BF),
    ([512] + [1] * 255, [512] + [1 + 3 * i for i in range(255)], 333, 16, 2, 64, HF),
    ([0] * 63 + [700], [40] * 63 + [900], 1000, 8, 2, 128, BF)])
def test_attention_prompts_and_mixed_batches(ops, new, own, prefix, hq, hkv, d, dtype):
    """Prompts of thousands of tokens without a prefix, one prompt among many sequences of a token each or idle ones."""
    check_attention(ops, new, own, prefix, hq, hkv, d, 64, dtype, pad=2)
