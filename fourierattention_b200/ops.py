"""Tensor-level wrappers of the C ABI: pointer/stride marshalling only, no arithmetic.

Every function runs the sm_100a kernels on the current CUDA stream of the tensors' device.
PyTorch is used for device memory and streams.
"""
import ctypes as C

import torch

from . import _lib
from ._lib import DecodeArgs, check, lib

_DT = {torch.float16: _lib.FA_DTYPE_F16, torch.bfloat16: _lib.FA_DTYPE_BF16}
ANGLE_EXACT, ANGLE_KM57 = _lib.FA_ANGLE_EXACT, _lib.FA_ANGLE_KM57

_scratch = {}
launch_count = 0          # kernels-launching C-ABI calls made so far (for benchmark accounting)
last_decode_path = None   # fa_decode_path() of the most recent decode_attn call (0 exact, 1 tensor-core pass, 2 warp-specialised, 3 warp-specialised with the accumulator in tensor memory)


def _dt(t):
    try:
        return _DT[t.dtype]
    except KeyError:
        raise ValueError(f"unsupported dtype {t.dtype}: the cache stores float16 or bfloat16") from None


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("fourierattention_b200 kernels need CUDA tensors (there is no CPU path)")


def _stream(t):
    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _p(t):
    return C.c_void_p(t.data_ptr()) if t is not None else C.c_void_p(0)


def scratch(device, nbytes):
    """A grow-only byte buffer per (device, stream); kernels on one stream are ordered, so one
    buffer per stream is enough."""
    key = (device.index if device.index is not None else torch.cuda.current_device(),
           torch.cuda.current_stream(device).cuda_stream)
    buf = _scratch.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(int(nbytes), 1 << 20), dtype=torch.uint8, device=device)
        _scratch[key] = buf
    return buf


def _rows3(x):
    """(B, K, C) view parameters of a tensor whose last dim is contiguous."""
    if x.dim() != 3 or x.stride(2) != 1:
        raise ValueError("expected a (B, K, C) tensor with a contiguous last dimension")
    return x.shape[0], x.shape[1], x.stride(0), x.stride(1)


def gather_cols(x, idx32, out):
    _need_cuda(x, idx32, out)
    B, K, sb, sk = _rows3(x)
    with torch.cuda.device(x.device):
        check(lib.fa_gather_cols(_p(x), _dt(x), B, K, sb, sk, _p(idx32), idx32.numel(), _p(out), out.stride(0),
                                 out.stride(1), _stream(x)), "fa_gather_cols")
    _count(1)
    return out


def colstats(x, idx32=None):
    _need_cuda(x, idx32)
    B, K, sb, sk = _rows3(x)
    Mc = idx32.numel() if idx32 is not None else x.shape[2]
    avg = torch.empty((B, Mc), dtype=torch.float32, device=x.device)
    dev = torch.empty_like(avg)
    with torch.cuda.device(x.device):
        check(lib.fa_colstats(_p(x), _dt(x), B, K, sb, sk, _p(idx32), Mc, _p(avg), _p(dev), _stream(x)), "fa_colstats")
    _count(1)
    return avg, dev


def compress(x, idx32, N, T_c, k_start=0, coef=None, accumulate=False):
    _need_cuda(x, idx32, coef)
    B, K, sb, sk = _rows3(x)
    Mc = idx32.numel() if idx32 is not None else x.shape[2]
    if coef is None:
        coef = torch.empty((B, 2 * N, Mc), dtype=torch.float32, device=x.device)
        accumulate = False
    elif coef.shape != (B, 2 * N, Mc) or coef.dtype != torch.float32 or not coef.is_contiguous():
        raise ValueError("coef must be a contiguous float32 (B, 2N, Mc) tensor")
    with torch.cuda.device(x.device):
        nbytes = lib.fa_compress_scratch_bytes(B, K, N, Mc, x.shape[2])
        sc = scratch(x.device, nbytes) if nbytes else None
        check(lib.fa_compress(_p(x), _dt(x), B, K, sb, sk, x.shape[2], _p(idx32), Mc, N, int(T_c), int(k_start), _p(coef),
                              int(bool(accumulate)), _p(sc), nbytes, _stream(x)), "fa_compress")
    _count(2 if nbytes else 1)
    return coef


def evict_update(k_coef, k_row, k_idx32, v_coef, v_row, v_idx32, phase, T_c, angle_mode=ANGLE_KM57):
    """In place: coef += basis(phase) (x) row[idx] for K and V.  ``*_row``: (B, F) with contiguous rows."""
    _need_cuda(k_coef, k_row, v_coef, v_row)
    ref = k_coef if k_coef is not None else v_coef
    B, N2 = ref.shape[0], ref.shape[1]
    row = k_row if k_row is not None else v_row
    with torch.cuda.device(ref.device):
        check(lib.fa_evict_update(_p(k_coef), _p(k_row), k_row.stride(0) if k_row is not None else 0, _p(k_idx32),
                                  k_coef.shape[2] if k_coef is not None else 0,
                                  _p(v_coef), _p(v_row), v_row.stride(0) if v_row is not None else 0, _p(v_idx32),
                                  v_coef.shape[2] if v_coef is not None else 0,
                                  _dt(row), B, N2 // 2, int(phase), int(T_c), int(angle_mode), _stream(ref)),
              "fa_evict_update")
    _count(1)


def recon_stats(coef, K, T):
    _need_cuda(coef)
    if coef.dim() != 3 or coef.dtype != torch.float32 or not coef.is_contiguous():
        raise ValueError("coef must be a contiguous float32 (B, 2N, Mc) tensor")
    B, N2, Mc = coef.shape
    avg = torch.empty((B, Mc), dtype=torch.float32, device=coef.device)
    dev = torch.empty_like(avg)
    with torch.cuda.device(coef.device):
        nbytes = lib.fa_recon_stats_scratch_bytes(B, int(K), Mc)
        sc = scratch(coef.device, nbytes)
        check(lib.fa_recon_stats(_p(coef), B, N2 // 2, Mc, int(K), int(T), _p(avg), _p(dev), _p(sc), nbytes,
                                 _stream(coef)), "fa_recon_stats")
    _count(2)
    return avg, dev


def fourier_inverse(c, K, T):
    _need_cuda(c)
    if c.dim() != 2 or c.dtype != torch.float32 or not c.is_contiguous():
        raise ValueError("c must be a contiguous float32 (M, 2N) tensor")
    M, N2 = c.shape
    out = torch.empty((M, int(K)), dtype=torch.float32, device=c.device)
    with torch.cuda.device(c.device):
        check(lib.fa_fourier_inverse(_p(c), M, N2 // 2, int(K), int(T), _p(out), _stream(c)), "fa_fourier_inverse")
    _count(1)
    return out


def cache_step(k_evict, v_evict, kn32, vn32, k_unc_row, v_unc_row, k_new, v_new, k_dst, v_dst):
    """``*_evict``/``*_dst``: (B, F) row views; ``*_unc_row``: (B, Mn) row views of the verbatim stores;
    ``*_new``: (B, Hkv, 1, D) or (B, Hkv, D) with a contiguous last dim."""
    _need_cuda(k_evict, k_new, k_dst)
    B, F = k_evict.shape
    if k_new.dim() == 4:
        k_new, v_new = k_new[:, :, 0], v_new[:, :, 0]
    Hkv, D = k_new.shape[1], k_new.shape[2]
    if k_new.stride(2) != 1 or v_new.stride() != k_new.stride() or v_evict.stride() != k_evict.stride() \
            or v_dst.stride() != k_dst.stride():
        raise ValueError("fa_cache_step: K and V must share strides and have a contiguous last dimension")
    with torch.cuda.device(k_evict.device):
        check(lib.fa_cache_step(_p(k_evict), _p(v_evict), k_evict.stride(0), _p(kn32), kn32.numel(), _p(vn32),
                                vn32.numel(), _p(k_unc_row), k_unc_row.stride(0), _p(v_unc_row), v_unc_row.stride(0),
                                _p(k_new), _p(v_new), k_new.stride(0), k_new.stride(1), _p(k_dst), _p(v_dst),
                                k_dst.stride(0), _dt(k_evict), B, Hkv, D, _stream(k_evict)), "fa_cache_step")
    _count(1)


def evict_step(k_coef, k_idx32, v_coef, v_idx32, phase, T_c, angle_mode,
               k_evict, v_evict, kn32, vn32, k_unc_row, v_unc_row, k_new, v_new, k_dst, v_dst):
    """``evict_update`` of the evicted row followed by ``cache_step``, as one launch."""
    _need_cuda(k_evict, k_new, k_dst)
    B, F = k_evict.shape
    if k_new.dim() == 4:
        k_new, v_new = k_new[:, :, 0], v_new[:, :, 0]
    Hkv, D = k_new.shape[1], k_new.shape[2]
    if k_new.stride(2) != 1 or v_new.stride() != k_new.stride() or v_evict.stride() != k_evict.stride() \
            or v_dst.stride() != k_dst.stride():
        raise ValueError("fa_evict_step: K and V must share strides and have a contiguous last dimension")
    ref = k_coef if k_coef is not None else v_coef
    N = ref.shape[1] // 2 if ref is not None else 1
    with torch.cuda.device(k_evict.device):
        check(lib.fa_evict_step(_p(k_coef), _p(k_evict) if k_coef is not None else None, k_evict.stride(0),
                                _p(k_idx32), k_coef.shape[2] if k_coef is not None else 0,
                                _p(v_coef), _p(v_evict) if v_coef is not None else None, v_evict.stride(0),
                                _p(v_idx32), v_coef.shape[2] if v_coef is not None else 0,
                                N, int(phase), int(T_c), int(angle_mode),
                                _p(k_evict), _p(v_evict), k_evict.stride(0), _p(kn32), kn32.numel(), _p(vn32),
                                vn32.numel(), _p(k_unc_row), k_unc_row.stride(0), _p(v_unc_row), v_unc_row.stride(0),
                                _p(k_new), _p(v_new), k_new.stride(0), k_new.stride(1), _p(k_dst), _p(v_dst),
                                k_dst.stride(0), _dt(k_evict), B, Hkv, D, _stream(k_evict)), "fa_evict_step")
    _count(1)


class DecodeTables:
    """int32 device copies of the eight index vectors the attention kernel reads."""

    def __init__(self, kc_list, kc_h, kn_list, kn_h, vc_list, vc_h, vn_list, vn_h, device):
        def cv(t):
            return torch.as_tensor(t).to(device=device, dtype=torch.int32).contiguous()
        self.kc_list, self.kc_h, self.kn_list, self.kn_h = cv(kc_list), cv(kc_h), cv(kn_list), cv(kn_h)
        self.vc_list, self.vc_h, self.vn_list, self.vn_h = cv(vc_list), cv(vc_h), cv(vn_list), cv(vn_h)
        # host copies of the two verbatim offset tables: the planner reads them to choose the kernel
        kh, vh = self.kn_h.cpu().tolist(), self.vn_h.cpu().tolist()
        self.kn_h_host = (C.c_int32 * len(kh))(*kh)
        self.vn_h_host = (C.c_int32 * len(vh))(*vh)


def decode_attn(q, k_sink, v_sink, k_win, v_win, k_mn, v_mn, k_coef, v_coef,
                avg_k_u, avg_k_d, scale_k, avg_v_u, avg_v_d, scale_v, tables,
                num_head_q, num_head_kv, T, sm_scale=-1.0, mid_l0=0, out=None, return_lse=False, phase_events=None,
                static_scratch=False):
    """Fused decode attention.  q: (B, Hq*D) (or (B,1,Hq*D)); sinks/window: (B, n, F) or None;
    k_mn/v_mn: (B, n_mid, Mn) row-strided views; coefficients (B, 2N, Mc) float32; statistics
    (B, Mc) float32.  Returns (B, Hq, D) float32 (plus (m, l) if ``return_lse``).
    ``static_scratch=True`` goes through ``fa_decode_attn_static``: no scratch tensor is taken from
    PyTorch's allocator, the kernels use the fixed buffer inside the library (see fourier_b200.h)."""
    _need_cuda(q)
    if q.dim() == 3:
        q = q[:, 0]
    B = q.shape[0]
    D = q.shape[1] // num_head_q
    F = num_head_kv * D
    dev = q.device
    a = DecodeArgs()
    a.B, a.Hq, a.Hkv, a.D = B, num_head_q, num_head_kv, D
    a.n_sink = k_sink.shape[1] if k_sink is not None else 0
    a.n_win = k_win.shape[1] if k_win is not None else 0
    a.n_mid = k_mn.shape[1] if k_mn is not None else 0
    a.mid_l0 = int(mid_l0)
    a.N = k_coef.shape[1] // 2 if k_coef is not None else 0
    a.T = int(T)
    a.Mc_k = k_coef.shape[2] if k_coef is not None else 0
    a.Mc_v = v_coef.shape[2] if v_coef is not None else 0
    a.Mn_k, a.Mn_v = F - a.Mc_k, F - a.Mc_v
    a.dtype = _dt(q)
    a.sm_scale = float(sm_scale) if sm_scale is not None else -1.0
    if q.stride(1) != 1:
        raise ValueError("q must have a contiguous last dimension")
    a.q, a.q_sb = q.data_ptr(), q.stride(0)

    def rows(t, name):
        if t is None:
            return 0, 0
        if t.stride(2) != 1 or t.stride(1) != F or t.dtype != q.dtype:
            raise ValueError(f"{name}: expected dtype {q.dtype} and dense (B, n, {F}) rows")
        return t.data_ptr(), t.stride(0)
    a.k_sink, a.sink_sb = rows(k_sink, "k_sink")
    a.v_sink, sb2 = rows(v_sink, "v_sink")
    a.k_win, a.win_sb = rows(k_win, "k_win")
    a.v_win, wb2 = rows(v_win, "v_win")
    if (k_sink is not None and sb2 != a.sink_sb) or (k_win is not None and wb2 != a.win_sb):
        raise ValueError("K and V segments must share their batch stride")
    if a.n_mid > 0:
        for t, nm in ((k_mn, "k_mn"), (v_mn, "v_mn")):
            if (t.shape[2] > 0 and t.stride(2) != 1) or t.dtype != q.dtype:
                raise ValueError(f"{nm}: expected dtype {q.dtype} with a contiguous last dimension")
        for t in (k_coef, v_coef, avg_k_u, avg_k_d, scale_k, avg_v_u, avg_v_d, scale_v):
            if t.dtype != torch.float32 or not t.is_contiguous():
                raise ValueError("coefficients and statistics must be contiguous float32")
        a.k_mn, a.k_mn_sb, a.k_mn_sk = k_mn.data_ptr(), k_mn.stride(0), max(k_mn.stride(1), a.Mn_k)
        a.v_mn, a.v_mn_sb, a.v_mn_sk = v_mn.data_ptr(), v_mn.stride(0), max(v_mn.stride(1), a.Mn_v)
        a.k_coef, a.v_coef = k_coef.data_ptr(), v_coef.data_ptr()
        a.avg_k_u, a.avg_k_d, a.scale_k = avg_k_u.data_ptr(), avg_k_d.data_ptr(), scale_k.data_ptr()
        a.avg_v_u, a.avg_v_d, a.scale_v = avg_v_u.data_ptr(), avg_v_d.data_ptr(), scale_v.data_ptr()
        tb = tables
        a.kc_list, a.kc_h, a.kn_list, a.kn_h = (tb.kc_list.data_ptr(), tb.kc_h.data_ptr(), tb.kn_list.data_ptr(),
                                                tb.kn_h.data_ptr())
        a.vc_list, a.vc_h, a.vn_list, a.vn_h = (tb.vc_list.data_ptr(), tb.vc_h.data_ptr(), tb.vn_list.data_ptr(),
                                                tb.vn_h.data_ptr())
        a.kn_h_host = C.cast(tb.kn_h_host, C.c_void_p)
        a.vn_h_host = C.cast(tb.vn_h_host, C.c_void_p)
    if out is None:
        out = torch.empty((B, num_head_q, D), dtype=torch.float32, device=dev)
    a.out = out.data_ptr()
    m = l = None
    if return_lse:
        m = torch.empty((B, num_head_q), dtype=torch.float32, device=dev)
        l = torch.empty_like(m)
        a.m_out, a.l_out = m.data_ptr(), l.data_ptr()
    if phase_events is not None:       # five torch.cuda.Event(enable_timing=True), see fourier_b200.h
        ev = (C.c_void_p * 5)(*[(e.cuda_event if e is not None else None) for e in phase_events])
        a.phase_events_host = C.cast(ev, C.c_void_p)
    global last_decode_path
    last_decode_path = lib.fa_decode_path(C.byref(a))
    if static_scratch:
        with torch.cuda.device(dev):
            check(lib.fa_decode_attn_static(C.byref(a), _stream(q)), "fa_decode_attn_static")
        _count(3 if a.n_mid > 0 else 2)
        return (out, m, l) if return_lse else out
    with torch.cuda.device(dev):
        nbytes = lib.fa_decode_scratch_bytes(C.byref(a))
        if nbytes == 0:
            check(lib.fa_decode_attn(C.byref(a), _stream(q)), "fa_decode_attn")   # reports the plan error
            raise RuntimeError("fa_decode_attn: empty scratch plan")
        sc = scratch(dev, nbytes)
        a.scratch, a.scratch_bytes = sc.data_ptr(), sc.numel()
        check(lib.fa_decode_attn(C.byref(a), _stream(q)), "fa_decode_attn")
    _count(3 if a.n_mid > 0 else 2)
    return (out, m, l) if return_lse else out


class LayerCalls:
    """The two per-step calls of one cached layer behind a library-side handle (``fa_layer_*``): buffers,
    tables, statistics, planner switches and tensor maps are bound once when the layer is created, a decode
    step passes the window offset, the span length and the new tensors only."""

    def __init__(self, kbuf, vbuf, k_unc, v_unc, k_coef, v_coef, stats32, tables, S, W, num_head_kv, T, mid_l0,
                 T_c, angle_mode, with_il=True):
        self.dev = kbuf.device
        self.B, rows, self.F = kbuf.shape
        self.S, self.W, self.Hkv = int(S), int(W), int(num_head_kv)
        self.D = self.F // self.Hkv
        self.tables, self.stats32 = tables, stats32           # keep the tensors alive
        self.k_coef, self.v_coef = k_coef, v_coef
        self.kbuf, self.vbuf = kbuf, vbuf
        if vbuf.stride(0) != kbuf.stride(0) or kbuf.stride(1) != self.F or kbuf.stride(2) != 1 \
                or vbuf.stride(1) != self.F or vbuf.stride(2) != 1:
            raise ValueError("K and V window buffers must be dense (B, rows, F) with equal strides")
        for t in stats32:
            if t.dtype != torch.float32 or not t.is_contiguous():
                raise ValueError("statistics must be contiguous float32")
        self.with_il = with_il
        tb = tables
        d = self.desc = _lib.LayerDesc()
        d.B, d.Hkv, d.D, d.S, d.W = self.B, self.Hkv, self.D, self.S, self.W
        have = k_coef if k_coef is not None else v_coef
        d.N = have.shape[1] // 2 if have is not None else 1
        d.T, d.T_c, d.angle_mode, d.dtype, d.mid_l0 = int(T), int(T_c), int(angle_mode), _dt(kbuf), int(mid_l0)
        d.Mc_k, d.Mc_v = tb.kc_list.numel(), tb.vc_list.numel()
        d.Mn_k, d.Mn_v = tb.kn_list.numel(), tb.vn_list.numel()
        d.with_il = 1 if with_il else 0
        d.kbuf, d.vbuf, d.buf_sb, d.buf_rows = kbuf.data_ptr(), vbuf.data_ptr(), kbuf.stride(0), rows
        d.k_coef = k_coef.data_ptr() if k_coef is not None else None
        d.v_coef = v_coef.data_ptr() if v_coef is not None else None
        (d.avg_k_u, d.avg_k_d, d.scale_k, d.avg_v_u, d.avg_v_d, d.scale_v) = [t.data_ptr() for t in stats32]
        d.kc_list, d.kc_h, d.kn_list, d.kn_h = (tb.kc_list.data_ptr(), tb.kc_h.data_ptr(), tb.kn_list.data_ptr(),
                                                tb.kn_h.data_ptr())
        d.vc_list, d.vc_h, d.vn_list, d.vn_h = (tb.vc_list.data_ptr(), tb.vc_h.data_ptr(), tb.vn_list.data_ptr(),
                                                tb.vn_h.data_ptr())
        d.kn_h_host = C.cast(tb.kn_h_host, C.c_void_p)
        d.vn_h_host = C.cast(tb.vn_h_host, C.c_void_p)
        self._set_stores(k_unc, v_unc)
        h = C.c_void_p()
        with torch.cuda.device(self.dev):
            check(lib.fa_layer_create(C.byref(d), C.byref(h)), "fa_layer_create")
        self._h = h
        self._scratch_key = None
        self._scratch_bytes = 0

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            lib.fa_layer_destroy(h)
            self._h = None

    def _set_stores(self, k_unc, v_unc):
        self.k_unc, self.v_unc = k_unc, v_unc
        d = self.desc
        d.k_unc, d.v_unc = k_unc.data_ptr(), v_unc.data_ptr()
        d.k_unc_sb, d.v_unc_sb = k_unc.stride(0), v_unc.stride(0)
        d.k_unc_sk, d.v_unc_sk = max(k_unc.stride(1), d.Mn_k), max(v_unc.stride(1), d.Mn_v)
        d.unc_rows = k_unc.shape[1]

    def set_statistics(self, stats32):
        """Replace the six float32 statistics tensors (avg_k_u, avg_k_d, scale_k, avg_v_u, avg_v_d, scale_v);
        the handle is made anew around the same buffers."""
        for t in stats32:
            if t.dtype != torch.float32 or not t.is_contiguous():
                raise ValueError("statistics must be contiguous float32")
        self.stats32 = stats32
        d = self.desc
        (d.avg_k_u, d.avg_k_d, d.scale_k, d.avg_v_u, d.avg_v_d, d.scale_v) = [t.data_ptr() for t in stats32]
        lib.fa_layer_destroy(self._h)
        h = C.c_void_p()
        with torch.cuda.device(self.dev):
            check(lib.fa_layer_create(C.byref(d), C.byref(h)), "fa_layer_create")
        self._h = h
        self._scratch_key = None

    def rebind(self, k_unc, v_unc):
        """(Re)attach the verbatim stores (they are reallocated when they grow)."""
        self._set_stores(k_unc, v_unc)
        d = self.desc
        check(lib.fa_layer_rebind_stores(self._h, d.k_unc, d.v_unc, d.k_unc_sb, d.v_unc_sb, d.k_unc_sk, d.v_unc_sk,
                                         d.unc_rows), "fa_layer_rebind_stores")
        self._scratch_key = None

    def step(self, off, n_mid, phase, k_new, v_new, appends=True):
        """One steady-state cache step: the window row at offset ``off`` is evicted (its compressed dims go into
        the coefficients at ``phase``, its verbatim dims to row ``n_mid`` of the stores) and the new token is
        written behind the window."""
        if k_new.dim() == 4:
            k_new, v_new = k_new[:, :, 0], v_new[:, :, 0]
        if k_new.stride(2) != 1 or v_new.stride() != k_new.stride():
            raise ValueError("fa_layer_update: K and V must share strides and have a contiguous last dimension")
        if torch.cuda.current_device() != self.dev.index:
            torch.cuda.set_device(self.dev)
        rc = lib.fa_layer_update(self._h, off, n_mid, int(phase), 1 if appends else 0, k_new.data_ptr(),
                                 v_new.data_ptr(), k_new.stride(0), k_new.stride(1),
                                 torch.cuda.current_stream(self.dev).cuda_stream)
        if rc:
            check(rc, "fa_layer_update")
        _count(1)

    def attend(self, q, off, n_mid, num_head_q, sm_scale=-1.0, phase_events=None, return_lse=False):
        """Decode attention of one query token per sequence; ``q``: (B, Hq*D).  Returns (B, Hq, D) float32
        (plus the softmax statistics (m, l) with ``return_lse``)."""
        global last_decode_path
        if q.stride(1) != 1 or q.dtype != self.kbuf.dtype:
            raise ValueError("q must have the cache dtype and a contiguous last dimension")
        out = torch.empty((self.B, num_head_q, self.D), dtype=torch.float32, device=self.dev)
        m = l = None
        if return_lse:
            m = torch.empty((self.B, num_head_q), dtype=torch.float32, device=self.dev)
            l = torch.empty_like(m)
        if n_mid == 0 and not self.with_il:
            # this rank holds no key at all (a span slice with no rows): an empty partial result that the
            # log-sum-exp merge ignores (l = 0), so that the rank still takes part in the exchange
            out.zero_()
            if return_lse:
                m.fill_(-1.0e30)
                l.zero_()
            return (out, m, l) if return_lse else out
        if torch.cuda.current_device() != self.dev.index:
            torch.cuda.set_device(self.dev)
        stream = torch.cuda.current_stream(self.dev).cuda_stream
        # the plan (and with it the scratch need) is constant while n_mid stays inside one 128-token super-tile
        key = (num_head_q, (n_mid + 127) >> 7)
        if key != self._scratch_key:
            nbytes = lib.fa_layer_scratch_bytes(self._h, num_head_q, n_mid)
            if nbytes == 0:
                check(lib.fa_layer_attend(self._h, off, n_mid, num_head_q, q.data_ptr(), q.stride(0), -1.0,
                                          out.data_ptr(), None, None, None, 0, None, stream), "fa_layer_attend")
                raise RuntimeError("fa_layer_attend: empty scratch plan")
            self._scratch_bytes = 2 * int(nbytes)
            self._scratch_key = key
            last_decode_path = lib.fa_layer_decode_path(self._h)
        sc = scratch(self.dev, self._scratch_bytes)
        ev = None
        if phase_events is not None:
            ev = (C.c_void_p * 5)(*[(e.cuda_event if e is not None else None) for e in phase_events])
        rc = lib.fa_layer_attend(self._h, off, n_mid, num_head_q, q.data_ptr(), q.stride(0),
                                 float(sm_scale) if sm_scale is not None else -1.0, out.data_ptr(),
                                 m.data_ptr() if m is not None else None, l.data_ptr() if l is not None else None,
                                 sc.data_ptr(), sc.numel(), ev, stream)
        if rc:
            check(rc, "fa_layer_attend")
        _count(3 if n_mid > 0 else 2)
        return (out, m, l) if return_lse else out


def merge(o, m, l):
    """o: (P, rows, D) normalised partial outputs, m/l: (P, rows).  Returns (rows, D)."""
    _need_cuda(o, m, l)
    P, rows, D = o.shape
    o, m, l = o.contiguous(), m.contiguous(), l.contiguous()
    out = torch.empty((rows, D), dtype=torch.float32, device=o.device)
    with torch.cuda.device(o.device):
        check(lib.fa_merge(_p(o), _p(m), _p(l), P, rows, D, _p(out), _stream(o)), "fa_merge")
    _count(1)
    return out


# ---- a served batch outside the compressed span: norm + rotation, paged cache, shared prefix, sampling ------------------

_raw_stream, _device_index = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _on(index, *ts):
    """Every given tensor on CUDA device ``index`` (-1: a CPU tensor, which is refused)."""
    if index < 0:
        raise RuntimeError("fourierattention_b200 kernels need CUDA tensors (there is no CPU path)")
    for t in ts:
        if t is not None and t.get_device() != index:
            raise ValueError(f"tensors on different devices: {t.device} and cuda:{index}")


def _no_grad(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise RuntimeError("this operator has no backward pass: call it under torch.no_grad()")


def _heads3(t, name, dtype):
    """Shape and strides of a (tokens, heads, D) tensor with a contiguous last dimension."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or (stride[2] != 1 and shape[2] > 1):
        raise ValueError(f"{name}: expected (tokens, heads, head_dim) with a contiguous last dimension")
    if t.dtype != dtype:
        raise ValueError(f"{name}: expected dtype {dtype}, got {t.dtype}")
    return shape, stride


def _int32(t, name, shape):
    if t.dtype != torch.int32 or t.shape != shape or (t.dim() and t.stride(-1) != 1 and t.shape[-1] > 1):
        raise ValueError(f"{name}: expected int32 {shape} with a contiguous last dimension, "
                         f"got {t.dtype} {tuple(t.shape)}")


def _call(fn, name, index, *args):
    """One call of the library on the current stream of device ``index``."""
    if _device_index() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        check(rc, name)


def _like(out, name, shape, dtype):
    """A given output has the shape of its input."""
    if out is not None and _heads3(out, name, dtype)[0] != shape:
        raise ValueError(f"{name} must have the shape of its input")


def _out3(out, like, shape):
    """The output tensor (a new one if not given) and its strides."""
    if out is None:
        return like.new_empty(shape), (shape[1] * shape[2], shape[2])
    return out, out.stride()


def _norm_weights(q_weight, k_weight, D, dtype):
    """(w_f32, pointers) of the norm weights."""
    if q_weight is None and k_weight is None:
        return 0, 0, 0
    f32 = None
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is None:
            continue
        if w.shape != (D,) or not w.is_contiguous() or (w.dtype != dtype and w.dtype != torch.float32):
            raise ValueError(f"{name}: expected a contiguous ({D},) tensor of {dtype} or float32")
        if f32 is not None and f32 != (w.dtype == torch.float32):
            raise ValueError("q_weight and k_weight must share their dtype")
        f32 = w.dtype == torch.float32
    return (1 if f32 else 0, q_weight.data_ptr() if q_weight is not None else 0,
            k_weight.data_ptr() if k_weight is not None else 0)


def _rotary_width(inv_freq):
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq: expected a contiguous float32 vector")
    return 2 * inv_freq.shape[0]


def _positions64(positions, tokens):
    """1 for int64 positions, 0 for int32."""
    if positions.dtype not in (torch.int64, torch.int32) or positions.shape != (tokens,) or not positions.is_contiguous():
        raise ValueError(f"positions: expected a contiguous int64 or int32 ({tokens},) tensor")
    return 1 if positions.dtype == torch.int64 else 0


def qk_norm_rope(q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6, q_out=None, k_out=None):
    """RMS norm of every query and key head (where a weight is given) and the rotation by position, in one pass.
    q: (tokens, Hq, D), k: (tokens, Hkv, D), any strides with a contiguous last dimension (views of a fused projection);
    positions: (tokens,) int64 or int32; inv_freq: (R/2,) float32, R <= D a multiple of 16 (rotated pairs are
    ``(i, i + R/2)``, dims from R on are passed through); weights: (D,) of the model dtype or float32.  float32
    arithmetic with exact angles, one rounding.  Returns (q, k), written to ``q_out`` / ``k_out`` if given (the inputs
    themselves are allowed)."""
    _no_grad(q, k, q_weight, k_weight)
    code, dtype = _dt(q), q.dtype
    qs, qst = _heads3(q, "q", dtype)
    ks, kst = _heads3(k, "k", dtype)
    tokens, Hq, D = qs
    if ks[0] != tokens or ks[2] != D:
        raise ValueError("q and k must have the same tokens and head dimension")
    R, wide = _rotary_width(inv_freq), _positions64(positions, tokens)
    w_f32, qw, kw = _norm_weights(q_weight, k_weight, D, dtype)
    _like(q_out, "q_out", qs, dtype)
    _like(k_out, "k_out", ks, dtype)
    index = q.get_device()
    _on(index, k, positions, inv_freq, q_weight, k_weight, q_out, k_out)
    q_out, qost = _out3(q_out, q, qs)
    k_out, kost = _out3(k_out, k, ks)
    a = _lib.pack_rope(tokens, Hq, ks[1], D, R, code, w_f32, wide, q.data_ptr(), k.data_ptr(), 0, qst[0], qst[1], kst[0],
                       kst[1], 0, 0, q_out.data_ptr(), k_out.data_ptr(), qost[0], qost[1], kost[0], kost[1],
                       positions.data_ptr(), inv_freq.data_ptr(), qw, kw, eps, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0,
                       0, 0)
    _call(lib.fa_qk_norm_rope, "fa_qk_norm_rope", index, a)
    _count(1 if tokens else 0)
    return q_out, k_out


def _pages(k_pages, v_pages, dtype, Hkv, D):
    """Shape and strides of a cache of pages (num_pages, Hkv, page_size, D)."""
    shape, ks, vs = k_pages.shape, k_pages.stride(), v_pages.stride()
    if len(shape) != 4 or shape != v_pages.shape or k_pages.dtype != dtype or v_pages.dtype != dtype \
            or shape[1] != Hkv or shape[3] != D or ks[3] != 1 or vs[3] != 1:
        raise ValueError(f"k_pages, v_pages: expected {dtype} (num_pages, {Hkv}, page_size, {D}) with a contiguous last "
                         "dimension")
    return shape, ks, vs


def _sequences(page_table, kv_lens, cu_seqlens, tokens):
    """Shape of the page table."""
    if page_table.dim() != 2:
        raise ValueError("page_table: expected int32 (sequences, pages)")
    B, most = page_table.shape
    _int32(page_table, "page_table", (B, most))
    _int32(kv_lens, "kv_lens", (B,))
    if cu_seqlens is not None:
        _int32(cu_seqlens, "cu_seqlens", (B + 1,))
    elif tokens != B:
        raise ValueError(f"{tokens} tokens of {B} sequences: without cu_seqlens there is one token per sequence")
    return B, most


def paged_append(k, v, k_pages, v_pages, page_table, kv_lens, inv_freq, cu_seqlens=None, positions=None, pos_offset=0,
                 q=None, q_weight=None, k_weight=None, eps=1e-6, q_out=None):
    """Writes the keys (normed where ``k_weight`` is given, rotated) and values of new tokens into the pages of a cache;
    with ``q`` the query heads are normed and rotated in the same launch.  k, v: (tokens, Hkv, D), q: (tokens, Hq, D);
    pages: (num_pages, Hkv, page_size, D); page_table: (B, pages) int32; kv_lens: (B,) int32, the length of every
    sequence with its new tokens; cu_seqlens: (B + 1,) int32, the first token of every sequence (None: one token each).
    A token's position is ``pos_offset`` + its index in its sequence unless ``positions`` gives it.  Tokens behind the
    last sequence, indices outside the table and page ids that name no page write nothing.  Returns the rotated
    queries (``q_out`` if given; None without q)."""
    _no_grad(k, v, q, q_weight, k_weight)
    code, dtype = _dt(k), k.dtype
    ks, kst = _heads3(k, "k", dtype)
    vs, vst = _heads3(v, "v", dtype)
    if vs != ks:
        raise ValueError("k and v must have the same shape")
    tokens, Hkv, D = ks
    R = _rotary_width(inv_freq)
    w_f32, qw, kw = _norm_weights(q_weight, k_weight, D, dtype)
    pages, kp, vp = _pages(k_pages, v_pages, dtype, Hkv, D)
    B, most = _sequences(page_table, kv_lens, cu_seqlens, tokens)
    Hq, q_ptr, qo_ptr, qst, qost = 0, 0, 0, (0, 0), (0, 0)
    if q is not None:
        qs, qst = _heads3(q, "q", dtype)
        if qs[0] != tokens or qs[2] != D:
            raise ValueError("q and k must have the same tokens and head dimension")
        _like(q_out, "q_out", qs, dtype)
    elif q_out is not None:
        raise ValueError("q_out is given without q")
    pos_ptr, wide = 0, 0
    if positions is not None:
        wide, pos_ptr = _positions64(positions, tokens), positions.data_ptr()
    index = k.get_device()
    _on(index, v, q, q_out, k_pages, v_pages, page_table, kv_lens, cu_seqlens, positions, inv_freq, q_weight, k_weight)
    if q is not None:
        q_out, qost = _out3(q_out, q, qs)
        Hq, q_ptr, qo_ptr = qs[1], q.data_ptr(), q_out.data_ptr()
    a = _lib.pack_rope(tokens, Hq, Hkv, D, R, code, w_f32, wide, q_ptr, k.data_ptr(), v.data_ptr(), qst[0], qst[1], kst[0],
                       kst[1], vst[0], vst[1], qo_ptr, 0, qost[0], qost[1], 0, 0, pos_ptr, inv_freq.data_ptr(), qw, kw, eps,
                       B, pages[2], most, pages[0], k_pages.data_ptr(), v_pages.data_ptr(), kp[0], kp[1], kp[2], vp[0],
                       vp[1], vp[2], page_table.data_ptr(), page_table.stride(0), kv_lens.data_ptr(),
                       cu_seqlens.data_ptr() if cu_seqlens is not None else 0, pos_offset)
    _call(lib.fa_paged_append, "fa_paged_append", index, a)
    _count(1 if tokens and B else 0)
    return q_out


def paged_attention(q, k_pages, v_pages, page_table, kv_lens, cu_seqlens=None, prefix_pages=None, prefix_len=0,
                    sm_scale=None, out=None, return_lse=False):
    """Attention of new tokens over the pages of their sequences and over a prefix that the whole batch shares, which is
    read once for all of its rows.  q: (tokens, Hq, D), D 64 or 128, tokens packed as in :func:`paged_append`; the last
    new token of sequence b sees ``kv_lens[b]`` keys of its own, each one before it a key less, and every token sees the
    first ``prefix_len`` keys of ``prefix_pages`` (int32 page ids).  Returns (tokens, Hq, D) of q's dtype, with
    ``return_lse`` also the log-sum-exp of the scores, (tokens, Hq) float32.  A token without any key gets 0 and
    -infinity; tokens behind the last sequence are left as they were.  Sums are float32, but each probability is rounded
    to the pages' type before it meets its value (the tensor cores multiply equal types), so the error against exact
    arithmetic is about a third above that of rounding the output alone: 2.3e-3 for 1.7e-3 in bfloat16, 2.5e-4 for 2.1e-4
    in float16, relative.  A value that is not finite may make earlier new tokens of its sequence NaN.  Scratch comes from PyTorch's allocator, per
    call."""
    _no_grad(q, k_pages, v_pages)
    code, dtype = _dt(q), q.dtype
    qs, qst = _heads3(q, "q", dtype)
    tokens, Hq, D = qs
    if k_pages.dim() != 4:
        raise ValueError("k_pages: expected (num_pages, kv_heads, page_size, head_dim)")
    pages, kp, vp = _pages(k_pages, v_pages, dtype, k_pages.shape[1], D)
    B, most = _sequences(page_table, kv_lens, cu_seqlens, tokens)
    if sm_scale is not None and not sm_scale > 0:
        raise ValueError(f"sm_scale must be positive (got {sm_scale})")
    if prefix_len < 0:
        raise ValueError(f"prefix_len must not be negative (got {prefix_len})")
    pre_ptr, n_pre = 0, 0
    if prefix_len:
        if prefix_pages is None or prefix_pages.dim() != 1:
            raise ValueError("prefix_pages: expected an int32 vector of page ids")
        n_pre = prefix_pages.shape[0]
        _int32(prefix_pages, "prefix_pages", (n_pre,))
        pre_ptr = prefix_pages.data_ptr()
    _like(out, "out", qs, dtype)
    index = q.get_device()
    _on(index, k_pages, v_pages, page_table, kv_lens, cu_seqlens, prefix_pages if prefix_len else None, out)
    out, ost = _out3(out, q, qs)
    lse = q.new_empty((tokens, Hq), dtype=torch.float32) if return_lse else None
    block = bytearray(_lib.pack_paged_attn(
        tokens, B, Hq, pages[1], D, pages[2], pages[0], most, n_pre, prefix_len, code,
        -1.0 if sm_scale is None else sm_scale, q.data_ptr(), qst[0], qst[1], out.data_ptr(), ost[0], ost[1],
        lse.data_ptr() if return_lse else 0, k_pages.data_ptr(), v_pages.data_ptr(), kp[0], kp[1], kp[2], vp[0], vp[1],
        vp[2], page_table.data_ptr(), page_table.stride(0), kv_lens.data_ptr(),
        cu_seqlens.data_ptr() if cu_seqlens is not None else 0, pre_ptr, 0, 0))
    if _device_index() == index:
        rc = _paged_attention(block, q, index)
    else:
        with torch.cuda.device(index):
            rc = _paged_attention(block, q, index)
    if rc:
        check(rc, "fa_paged_attn")
    # (asked for only where it is not plain: a prefix under several new tokens)
    _count(lib.fa_paged_attn_launches(bytes(block)) if prefix_len and cu_seqlens is not None
           else (3 if prefix_len else 2) if tokens and B else 0)
    return (out, lse) if return_lse else out


def _paged_attention(block, q, index):
    nbytes = lib.fa_paged_attn_scratch_bytes(bytes(block))
    # of this call alone: a buffer kept between calls would be shared by captured graphs
    sc = q.new_empty((nbytes,), dtype=torch.uint8)
    block[-16:] = _lib.pack_scratch(sc.data_ptr(), nbytes)        # the last two fields
    return lib.fa_paged_attn(bytes(block), _raw_stream(index))


def _row_parameter(value, name, dtype, B, index):
    """(pointer, value) of a per-row tensor or of one number for all rows."""
    if value is None:
        raise ValueError(f"{name}: expected a number or a tensor")
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype or value.shape != (B,) or not value.is_contiguous():
            raise ValueError(f"{name}: expected a number or a contiguous {dtype} ({B},) tensor")
        _on(index, value)
        return value.data_ptr(), 0
    if value != value or (dtype == torch.int32 and not (hasattr(value, "__index__") and -2 ** 31 <= value < 2 ** 31)):
        raise ValueError(f"{name}: expected {'a 32-bit integer' if dtype == torch.int32 else 'a number'}, got {value!r}")
    return None, value


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_logprob=False):
    """Draws one token per row of ``logits`` (B, V), float32, float16 or bfloat16, V <= 393216, with the uniform numbers
    ``u`` (B,) float32 in [0, 1).  Temperature is applied first (0: the largest logit), then top-k (0: off), top-p on
    what top-k kept (1: off), min-p relative to the largest probability (0: off); each is a number or a (B,) tensor
    (float32, ``top_k`` int32).  A NaN in a tensor of filters turns that one off; as a number it is refused.  Among equal logits the lower index counts as larger.  The token is the first index at
    which the running sum of kept probabilities exceeds u.  Returns int64 tokens, with ``return_logprob`` also the
    float32 logarithm of the probability each had in the kept distribution.  NaN logits are never drawn; a row without a
    logit above -infinity gives token -1."""
    _no_grad(logits)
    shape, stride = logits.shape, logits.stride()
    if len(shape) != 2 or (stride[1] != 1 and shape[1] > 1):
        raise ValueError("logits: expected (B, V) with a contiguous last dimension")
    B, V = shape
    code = _lib.FA_DTYPE_F32 if logits.dtype == torch.float32 else _dt(logits)
    if u.dtype != torch.float32 or u.shape != (B,) or not u.is_contiguous():
        raise ValueError(f"u: expected a contiguous float32 ({B},) tensor")
    index = u.get_device()
    tp, tv = _row_parameter(temperature, "temperature", torch.float32, B, index)
    kp, kv = _row_parameter(top_k, "top_k", torch.int32, B, index)
    pp, pv = _row_parameter(top_p, "top_p", torch.float32, B, index)
    mp, mv = _row_parameter(min_p, "min_p", torch.float32, B, index)
    _on(index, logits)
    token = u.new_empty((B,), dtype=torch.int64)
    logprob = u.new_empty((B,)) if return_logprob else None
    _call(lib.fa_sample, "fa_sample", index, logits.data_ptr(), code, B, V, stride[0], u.data_ptr(), tp, tv, kp, kv, pp, pv,
          mp, mv, token.data_ptr(), logprob.data_ptr() if return_logprob else None)
    _count(1 if B else 0)
    return (token, logprob) if return_logprob else token


def _count(n):
    global launch_count
    launch_count += n
