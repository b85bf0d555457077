"""CPU tests of what the operators of a served batch refuse, and of their argument blocks: checks run before a device is
touched, so they need none."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    import __graft_entry__
    __graft_entry__._load_builder().build()
    from fourierattention_b200 import ops as o
    return o


@pytest.mark.parametrize("ctype,pytype", [("fa_rope_args_t", "RopeArgs"), ("fa_paged_attn_args_t", "PagedAttnArgs")])
def test_argument_blocks_match_c(ops, ctype, pytype):
    mirror = getattr(ops._lib, pytype)
    fields = [f[0] for f in mirror._fields_]
    prog = f'#include <stdio.h>\n#include <stddef.h>\n#include "fourier_b200.h"\nint main(){{printf("%zu\\n", sizeof({ctype}));\n'
    prog += "".join(f'printf("%zu\\n", offsetof({ctype}, {f}));\n' for f in fields) + "return 0;}\n"
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(src, "w").write(prog)
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe])
        vals = [int(x) for x in subprocess.check_output([exe]).split()]
    assert vals == [C.sizeof(mirror)] + [getattr(mirror, f).offset for f in fields]
    # and packed at once it is the same bytes as filled in field by field
    block, values = mirror(), list(range(3, 3 + len(fields)))
    for name, v in zip(fields, values):
        setattr(block, name, v)
    assert ops._lib.packer(mirror).pack(*values) == bytes(block)


def _t(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def _i(*v):
    return torch.tensor(v, dtype=torch.int32)


def rope_args(**kw):
    d = dict(q=_t(4, 8, 64), k=_t(4, 2, 64), positions=torch.arange(4), inv_freq=_t(32, dtype=F32))
    d.update(kw)
    return d


@pytest.mark.parametrize("kw", [
    dict(q=_t(4, 8, 64, dtype=F32)), dict(q=_t(4, 512)), dict(k=_t(3, 2, 64)), dict(k=_t(4, 2, 32)), dict(k=_t(4, 2, 64, dtype=HF)),
    dict(q=_t(4, 64, 8).transpose(1, 2)), dict(positions=torch.arange(3)), dict(positions=torch.arange(4).float()),
    dict(positions=torch.arange(8)[::2]), dict(inv_freq=_t(32)), dict(inv_freq=_t(4, 8, dtype=F32)),
    dict(q_weight=_t(32)), dict(q_weight=_t(64, dtype=HF)), dict(q_weight=_t(64), k_weight=_t(64, dtype=F32)),
    dict(q_out=_t(4, 8, 32)), dict(q_out=_t(4, 8, 64, dtype=HF)), dict(k_out=_t(4, 8, 64))])
def test_qk_norm_rope_refuses(ops, kw):
    with pytest.raises(ValueError):
        ops.qk_norm_rope(**rope_args(**kw))


def append_args(**kw):
    d = dict(k=_t(2, 2, 64), v=_t(2, 2, 64), k_pages=_t(5, 2, 16, 64), v_pages=_t(5, 2, 16, 64), page_table=_t(2, 3, dtype=torch.int32),
             kv_lens=_i(1, 1), inv_freq=_t(32, dtype=F32))
    d.update(kw)
    return d


@pytest.mark.parametrize("kw", [
    dict(v=_t(2, 1, 64)), dict(v=_t(2, 2, 64, dtype=HF)), dict(k_pages=_t(5, 1, 16, 64)), dict(k_pages=_t(5, 2, 16, 32)),
    dict(v_pages=_t(5, 2, 16, 64, dtype=HF)), dict(v_pages=_t(4, 2, 16, 64)), dict(k_pages=_t(2, 16, 64)),
    dict(k_pages=_t(5, 2, 64, 16).transpose(2, 3)), dict(page_table=_t(2, 3, dtype=torch.int64)), dict(page_table=_i(1, 2)),
    dict(kv_lens=_i(1)), dict(kv_lens=torch.tensor([1, 1])), dict(k=_t(3, 2, 64), v=_t(3, 2, 64)),
    dict(cu_seqlens=_i(0, 2)), dict(cu_seqlens=torch.tensor([0, 1, 2])), dict(q=_t(3, 8, 64)), dict(q=_t(2, 8, 32)),
    dict(positions=torch.arange(3))])
def test_paged_append_refuses(ops, kw):
    with pytest.raises(ValueError):
        ops.paged_append(**append_args(**kw))


def attend_args(**kw):
    d = dict(q=_t(2, 8, 64), k_pages=_t(5, 2, 16, 64), v_pages=_t(5, 2, 16, 64), page_table=_t(2, 3, dtype=torch.int32),
             kv_lens=_i(1, 1))
    d.update(kw)
    return d


@pytest.mark.parametrize("kw", [
    dict(q=_t(2, 8, 64, dtype=F32)), dict(q=_t(2, 8, 64, dtype=HF)), dict(q=_t(3, 8, 64)), dict(q=_t(2, 512)), dict(q=_t(2, 8, 32)),
    dict(k_pages=_t(2, 16, 64)), dict(v_pages=_t(5, 2, 32, 64)), dict(prefix_len=5), dict(prefix_len=5, prefix_pages=_t(1, 1, dtype=torch.int32)),
    dict(prefix_len=5, prefix_pages=torch.tensor([1])), dict(out=_t(2, 8, 32)), dict(out=_t(2, 8, 64, dtype=HF)), dict(cu_seqlens=_i(0, 1, 2, 3)),
    dict(sm_scale=0.0), dict(sm_scale=-1.0), dict(prefix_len=-1)])
def test_paged_attention_refuses(ops, kw):
    with pytest.raises(ValueError):
        ops.paged_attention(**attend_args(**kw))


def sample_args(**kw):
    d = dict(logits=_t(3, 100), u=_t(3, dtype=F32))
    d.update(kw)
    return d


@pytest.mark.parametrize("kw", [
    dict(logits=_t(3, 100, dtype=torch.float64)), dict(logits=_t(100)), dict(logits=_t(100, 3).T), dict(u=_t(2, dtype=F32)),
    dict(u=_t(3)), dict(temperature=_t(2, dtype=F32)), dict(temperature=_t(3)), dict(top_k=torch.tensor([1, 2, 3])),
    dict(top_p=_t(3, 1, dtype=F32)), dict(min_p=_t(6, dtype=F32)[::2]),
    dict(temperature=None)])
def test_sample_refuses(ops, kw):
    with pytest.raises(ValueError):
        ops.sample(**sample_args(**kw))


def test_cpu_tensors_are_refused(ops):
    for f, kw in ((ops.qk_norm_rope, rope_args()), (ops.paged_append, append_args()), (ops.paged_attention, attend_args()),
                  (ops.sample, sample_args())):
        with pytest.raises(RuntimeError, match="CUDA"):
            f(**kw)


def test_inputs_that_need_a_gradient_are_refused(ops):
    """None of the four has a backward pass: nothing breaks a graph silently."""
    grad = lambda *s: torch.zeros(s, dtype=BF, requires_grad=True)
    calls = [(ops.qk_norm_rope, rope_args(q=grad(4, 8, 64))), (ops.qk_norm_rope, rope_args(k_weight=grad(64))),
             (ops.paged_append, append_args(v=grad(2, 2, 64))), (ops.paged_attention, attend_args(q=grad(2, 8, 64))),
             (ops.sample, sample_args(logits=grad(3, 100)))]
    for f, kw in calls:
        with pytest.raises(RuntimeError, match="backward"):
            f(**kw)


def test_library_refuses(ops):
    """The C entries check sizes, alignment and pointers themselves."""
    lib, L = ops.lib, ops._lib
    call = lambda f, a: f(bytes(a), None)

    def rope(**kw):
        a = L.RopeArgs()
        d = dict(tokens=2, Hq=4, Hkv=2, D=64, R=64, dtype=1, q=4096, k=4096, q_out=4096, k_out=4096, positions=4096, inv_freq=4096)
        d.update(kw)
        for k, v in d.items():
            setattr(a, k, v)
        return a
    for kw, rc in ((dict(dtype=2), -3), (dict(tokens=-1), -2), (dict(D=72), -2), (dict(D=512), -2), (dict(R=128), -2), (dict(R=24), -2),
                   (dict(Hq=0, Hkv=0), -2), (dict(q=None), -1), (dict(k_out=None), -1), (dict(positions=None), -1),
                   (dict(inv_freq=None), -1), (dict(tokens=0, q=None), 0), (dict(Hq=70000), -5)):
        assert call(lib.fa_qk_norm_rope, rope(**kw)) == rc, kw
    assert lib.fa_qk_norm_rope(None, None) == -1
    app = dict(B=2, page_size=16, max_pages=3, num_pages=4, v=4096, k_pages=4096, v_pages=4096, page_table=4096, kv_lens=4096)
    for kw, rc in ((dict(page_size=0), -2), (dict(B=3), -2), (dict(v=None), -1), (dict(kv_lens=None), -1), (dict(page_table=None), -1),
                   (dict(k_pages=None), -1), (dict(tokens=0, B=0), 0)):
        assert call(lib.fa_paged_append, rope(**{**app, **kw})) == rc, kw

    def attn(**kw):
        a = L.PagedAttnArgs()
        d = dict(tokens=2, B=2, Hq=8, Hkv=2, D=64, page_size=16, num_pages=4, max_pages=3, dtype=1, q=4096, out=4096, k_pages=4096,
                 v_pages=4096, page_table=4096, kv_lens=4096, q_st=512, q_sh=64, o_st=512, o_sh=64, kp_sp=2048, kp_sh=1024, kp_sr=64,
                 vp_sp=2048, vp_sh=1024, vp_sr=64, scratch=4096, scratch_bytes=1 << 40)
        d.update(kw)
        for k, v in d.items():
            setattr(a, k, v)
        return a
    for kw, rc in ((dict(dtype=2), -3), (dict(Hq=7), -2), (dict(D=96), -7), (dict(page_size=8), -2), (dict(page_size=40), -2),
                   (dict(num_pages=0), -2), (dict(B=3), -2), (dict(prefix_len=65, n_prefix_pages=4, prefix_pages=4096), -2),
                   (dict(prefix_len=64, n_prefix_pages=4), -1), (dict(max_pages=1 << 28), -5), (dict(q=None), -1), (dict(q=4098), -4),
                   (dict(q_st=513), -4), (dict(out=4104), -4), (dict(kp_sr=68), -4), (dict(v_pages=4100), -4), (dict(scratch=None), -5),
                   (dict(scratch_bytes=16), -5), (dict(scratch=4100), -5), (dict(tokens=0, B=0), 0)):
        assert call(lib.fa_paged_attn, attn(**kw)) == rc, kw
    assert lib.fa_paged_attn_scratch_bytes(bytes(attn())) > 0
    assert lib.fa_paged_attn_scratch_bytes(bytes(attn(D=96))) == 0
    for kw in (dict(tokens=0, B=0), dict(tokens=0, B=0, cu_seqlens=4096), dict(tokens=5, B=0, cu_seqlens=4096)):
        lib.fa_paged_attn_scratch_bytes(bytes(attn(**kw)))          # sizes of nothing: no fault
    one = lambda **kw: lib.fa_sample(*{**dict(x=4096, dt=1, B=2, V=10, sb=10, u=4096, t=None, t0=1.0, k=None, k0=0, p=None, p0=1.0, m=None,
                                              m0=0.0, tok=4096, lp=None, st=None), **kw}.values())
    assert one(dt=3) == -3 and one(V=0) == -2 and one(B=-1) == -2 and one(V=393217) == -5 and one(x=None) == -1
    assert one(u=None) == -1 and one(tok=None) == -1 and one(B=0, x=None) == 0


@pytest.mark.parametrize("kw", [dict(top_k=2 ** 31), dict(top_k=2 ** 32 + 5), dict(top_k=-2 ** 31 - 1), dict(top_k=2.5),
                                dict(temperature=float("nan")), dict(top_p=float("nan")), dict(min_p=float("nan"))])
def test_sample_refuses_numbers(ops, kw):
    """A top_k that does not fit its 32 bits would be another one, a NaN is no setting at all."""
    with pytest.raises(ValueError, match=next(iter(kw))):
        ops.sample(**sample_args(**kw))


def test_paged_append_refuses_an_output_without_queries(ops):
    """It would come back unwritten."""
    with pytest.raises(ValueError, match="q_out"):
        ops.paged_append(**append_args(q_out=_t(2, 8, 64)))
