// Norm and rotation of the query and key heads of a batch of tokens, written densely (fa_qk_norm_rope) or, with the
// values, into the pages of a cache (fa_paged_append).  Per head x[D] with rotary width R <= D:
//   y = x * rsqrt(mean(x^2) + eps) * w            (no weight: y = x)
//   z[i]       = y[i] cos a_i - y[i + R/2] sin a_i,   z[i + R/2] = y[i + R/2] cos a_i + y[i] sin a_i,   i < R/2
//   z[d]       = y[d],  d >= R;      a_i = position * inv_freq[i]
// All arithmetic in float32, one rounding at the store.
//
// Bound: HBM (every element is read and written once, ~10 flop each).  A CTA takes TOK tokens; their angles are
// reduced in float64 (a float32 product is off by 0.008 rad at position 131072), once per token, and shared by all of
// its heads through shared memory.  D/16 neighbouring lanes hold a head, 8 + 8 elements each (the two halves of eight
// rotation pairs), so that the mean square is a few shuffles and every access is 16 bytes.  Each thread requests its
// first elements before it computes angles.
#include "common.cuh"

namespace fa {

struct RopeParams {
  fa_rope_args_t a;
  int lph_log2;   // lanes per head, log2
  int append;
};

constexpr int RA_THREADS = 256;
constexpr int RA_MAX_TOK = 4;
constexpr int RA_MAX_PAIRS = 128;
constexpr int RA_BATCH = 4;   // heads in flight per thread

template <typename T, bool VEC>
__device__ __forceinline__ void ra_load(const T* p, float* f) {
  if (VEC) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    unpack8<T>(raw, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f32(p[i]);
  }
}
__device__ __forceinline__ void ra_cvt(float f, __half* o) { *o = __float2half_rn(f); }
__device__ __forceinline__ void ra_cvt(float f, __nv_bfloat16* o) { *o = __float2bfloat16_rn(f); }
template <typename T, bool VEC>
__device__ __forceinline__ void ra_store(T* p, const float* f) {
  alignas(16) T v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) ra_cvt(f[i], v + i);
  if (VEC) {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = v[i];
  }
}
template <typename T>
__device__ __forceinline__ void ra_weight(const void* w, int f32, int d, float* f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = f32 ? reinterpret_cast<const float*>(w)[d + i] : to_f32(reinterpret_cast<const T*>(w)[d + i]);
}

template <typename T, int TOK, bool VEC>
__global__ void __launch_bounds__(RA_THREADS) rope_kernel(const __grid_constant__ RopeParams prm) {
  const fa_rope_args_t& a = prm.a;
  __shared__ float s_cos[TOK][RA_MAX_PAIRS], s_sin[TOK][RA_MAX_PAIRS];
  __shared__ long long s_pos[TOK];     // position of the token
  __shared__ int s_live[TOK];          // the token belongs to a sequence
  __shared__ long long s_kdst[TOK], s_vdst[TOK];   // element offset of (page, head 0, row) or -1: not stored
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * TOK;
  const int lph = 1 << prm.lph_log2;
  const int heads = a.Hq + a.Hkv + (prm.append ? a.Hkv : 0);
  const int total = TOK * heads;                       // (token, head) pairs of this CTA
  const int c = tid & (lph - 1);                       // chunk of the head this lane holds
  const int first = tid >> prm.lph_log2, step = RA_THREADS >> prm.lph_log2;
  const bool lane_on = c * 16 < a.D;
  const int nrot = a.R / 16;
  // element offsets of the two halves of the chunk: a rotation pair, or 16 elements behind the rotary width
  const int lo = c < nrot ? 8 * c : a.R + 16 * (c - nrot);
  const int hi = c < nrot ? a.R / 2 + 8 * c : lo + 8;

  auto source = [&](int it, int& kind, int& tok, int& h) -> const T* {
    tok = it / heads;
    const int x = it - tok * heads;
    const int64_t t = t0 + tok;
    if (x < a.Hq) {
      kind = 0, h = x;
      return reinterpret_cast<const T*>(a.q) + t * a.q_st + (int64_t)h * a.q_sh;
    }
    if (x < a.Hq + a.Hkv) {
      kind = 1, h = x - a.Hq;
      return reinterpret_cast<const T*>(a.k) + t * a.k_st + (int64_t)h * a.k_sh;
    }
    kind = 2, h = x - a.Hq - a.Hkv;
    return reinterpret_cast<const T*>(a.v) + t * a.v_st + (int64_t)h * a.v_sh;
  };

  // ---- request the first batch of elements ---------------------------------------------------------------------
  float x[RA_BATCH][16];
  auto load_batch = [&](int base) {
#pragma unroll
    for (int u = 0; u < RA_BATCH; ++u) {
      const int it = base + u * step;
      int kind, tok, h;
      if (it < total && lane_on && t0 + it / heads < a.tokens) {
        const T* p = source(it, kind, tok, h);
        ra_load<T, VEC>(p + lo, x[u]);
        ra_load<T, VEC>(p + hi, x[u] + 8);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[u][i] = 0.f;
      }
    }
  };
  load_batch(first);

  // ---- where the tokens belong ---------------------------------------------------------------------------------
  int seq0 = 0;
  if (prm.append && a.cu_seqlens) {
    // sequences that end at or before token t0; rows of empty sequences are passed over
    int n = 0;
    for (int b = tid; b < a.B; b += RA_THREADS) n += a.cu_seqlens[b + 1] <= t0;
    __shared__ int s_n[RA_THREADS / 32];
    n = __reduce_add_sync(0xffffffffu, n);
    if ((tid & 31) == 0) s_n[tid >> 5] = n;
    __syncthreads();
    for (int w = 0; w < RA_THREADS / 32; ++w) seq0 += s_n[w];
  }
  if (tid < TOK) {
    const int t = t0 + tid;
    bool live = t < a.tokens;
    long long pos = 0, kdst = -1, vdst = -1;
    if (prm.append && live) {
      int b, i, n;
      if (a.cu_seqlens) {
        b = seq0;
        while (b < a.B && a.cu_seqlens[b + 1] <= t) ++b;
        live = b < a.B;
        if (live) {
          const int beg = a.cu_seqlens[b];
          i = t - beg;
          n = a.cu_seqlens[b + 1] - beg;
        }
      } else {
        b = t, i = 0, n = 1;
        live = b < a.B;
      }
      if (live) {
        const long long j = (long long)a.kv_lens[b] - n + i;   // index in its own sequence
        pos = a.pos_offset + j;
        const long long pg = j >= 0 ? j / a.page_size : -1;
        if (i >= 0 && pg >= 0 && pg < a.max_pages) {
          const int page = a.page_table[(int64_t)b * a.table_sb + pg];
          if (page >= 0 && page < a.num_pages) {
            const long long row = j - pg * a.page_size;
            kdst = (long long)page * a.kp_sp + row * a.kp_sr;
            vdst = (long long)page * a.vp_sp + row * a.vp_sr;
          }
        }
      }
    }
    if (live && a.positions)
      pos = a.pos_i64 ? reinterpret_cast<const long long*>(a.positions)[t] : (long long)reinterpret_cast<const int*>(a.positions)[t];
    s_pos[tid] = pos;
    s_live[tid] = live;
    s_kdst[tid] = kdst;
    s_vdst[tid] = vdst;
  }
  __syncthreads();
  // ---- angles: turns in float64, the fraction of a turn in float32 -----------------------------------------------
  for (int i = tid; i < TOK * (a.R / 2); i += RA_THREADS) {
    const int tok = i / (a.R / 2), p = i - tok * (a.R / 2);
    double turns = (double)s_pos[tok] * (double)a.inv_freq[p] * 0.15915494309189533577;   // 1 / (2 pi)
    turns -= rint(turns);
    float sn, cs;
    sincospif(2.0f * (float)turns, &sn, &cs);
    s_cos[tok][p] = cs;
    s_sin[tok][p] = sn;
  }
  __syncthreads();

  for (int base = first; base - first < total; base += RA_BATCH * step) {
    if (base != first) load_batch(base);
#pragma unroll
    for (int u = 0; u < RA_BATCH; ++u) {
      const int it = base + u * step;
      int kind = 2, tok = 0, h = 0;
      if (it < total) source(it, kind, tok, h);
      const bool on = it < total && lane_on && s_live[tok];
      const void* w = kind == 0 ? a.q_weight : kind == 1 ? a.k_weight : nullptr;
      // every lane of a warp takes part in the shuffles; heads without a weight drop the result
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) ss = fmaf(x[u][i], x[u][i], ss);
      for (int o = lph >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (!on) continue;
      if (w) {
        const float r = 1.0f / sqrtf(ss / (float)a.D + a.eps);
        float wl[8], wh[8];
        ra_weight<T>(w, a.w_f32, lo, wl);
        ra_weight<T>(w, a.w_f32, hi, wh);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[u][i] *= r * wl[i];
          x[u][8 + i] *= r * wh[i];
        }
      }
      if (kind != 2 && c < nrot) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float cs = s_cos[tok][8 * c + i], sn = s_sin[tok][8 * c + i];
          const float y0 = x[u][i], y1 = x[u][8 + i];
          x[u][i] = y0 * cs - y1 * sn;
          x[u][8 + i] = y1 * cs + y0 * sn;
        }
      }
      T* dst;
      if (kind == 0) {
        dst = reinterpret_cast<T*>(a.q_out) + (int64_t)(t0 + tok) * a.qo_st + (int64_t)h * a.qo_sh;
      } else if (!prm.append) {
        dst = reinterpret_cast<T*>(a.k_out) + (int64_t)(t0 + tok) * a.ko_st + (int64_t)h * a.ko_sh;
      } else {
        const long long at = kind == 1 ? s_kdst[tok] : s_vdst[tok];
        if (at < 0) continue;
        dst = kind == 1 ? reinterpret_cast<T*>(a.k_pages) + at + (int64_t)h * a.kp_sh
                        : reinterpret_cast<T*>(a.v_pages) + at + (int64_t)h * a.vp_sh;
      }
      ra_store<T, VEC>(dst + lo, x[u]);
      ra_store<T, VEC>(dst + hi, x[u] + 8);
    }
  }
}

static bool al16(const void* p, int64_t s0, int64_t s1) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s0 % 8 == 0 && s1 % 8 == 0;
}

template <typename T, int TOK, bool VEC>
static void rope_launch(const RopeParams& prm, cudaStream_t st) {
  rope_kernel<T, TOK, VEC><<<ceil_div(prm.a.tokens, TOK), RA_THREADS, 0, st>>>(prm);
}
template <typename T>
static void rope_launch_t(const RopeParams& prm, bool vec, cudaStream_t st) {
  // one token per CTA until every SM has several: a lone token's latency is the call's; from there on four tokens
  // share the set-up
  const bool many = prm.a.tokens >= 16 * sm_count();
  if (many) {
    if (vec) rope_launch<T, RA_MAX_TOK, true>(prm, st);
    else rope_launch<T, RA_MAX_TOK, false>(prm, st);
  } else {
    if (vec) rope_launch<T, 1, true>(prm, st);
    else rope_launch<T, 1, false>(prm, st);
  }
}

static int rope_run(const fa_rope_args_t* a, int append, const char* what, cudaStream_t st) {
  FA_REQUIRE(a, FA_ERR_NULL, "%s: null argument block", what);
  FA_REQUIRE(a->dtype == FA_DTYPE_F16 || a->dtype == FA_DTYPE_BF16, FA_ERR_DTYPE, "%s: bad dtype %d", what, a->dtype);
  FA_REQUIRE(a->tokens >= 0 && a->Hq >= 0 && a->Hkv >= 0 && a->Hq + a->Hkv > 0, FA_ERR_SHAPE,
             "%s: bad sizes (tokens %d, heads %d + %d)", what, a->tokens, a->Hq, a->Hkv);
  FA_REQUIRE(a->D >= 16 && a->D <= 256 && a->D % 16 == 0, FA_ERR_SHAPE,
             "%s: the head dimension must be a multiple of 16 up to 256 (got %d)", what, a->D);
  FA_REQUIRE(a->R >= 0 && a->R <= a->D && a->R % 16 == 0, FA_ERR_SHAPE,
             "%s: the rotary width must be a multiple of 16 up to the head dimension (got %d)", what, a->R);
  FA_REQUIRE(a->Hq + 2 * (int64_t)a->Hkv <= 65536, FA_ERR_CAPACITY, "%s: too many heads", what);
  if (append) {
    FA_REQUIRE(a->B >= 0 && a->page_size > 0 && a->max_pages >= 0 && a->num_pages >= 0, FA_ERR_SHAPE,
               "%s: bad cache sizes", what);
    FA_REQUIRE(a->cu_seqlens || a->tokens == a->B, FA_ERR_SHAPE,
               "%s: without cu_seqlens there is one token per sequence (%d tokens, %d sequences)", what, a->tokens, a->B);
  }
  if (a->tokens == 0 || (append && a->B == 0)) return FA_OK;
  FA_REQUIRE(a->R == 0 || a->inv_freq, FA_ERR_NULL, "%s: null inv_freq", what);
  FA_REQUIRE(a->Hq == 0 || (a->q && a->q_out), FA_ERR_NULL, "%s: null query tensor", what);
  FA_REQUIRE(a->Hkv == 0 || a->k, FA_ERR_NULL, "%s: null key tensor", what);
  if (append) {
    FA_REQUIRE(a->kv_lens && (a->page_table || a->max_pages == 0), FA_ERR_NULL, "%s: null page table or lengths", what);
    FA_REQUIRE(a->Hkv == 0 || (a->v && a->k_pages && a->v_pages), FA_ERR_NULL, "%s: null values or pages", what);
  } else {
    FA_REQUIRE(a->positions, FA_ERR_NULL, "%s: null positions", what);
    FA_REQUIRE(a->Hkv == 0 || a->k_out, FA_ERR_NULL, "%s: null key output", what);
  }
  RopeParams prm;
  prm.a = *a;
  prm.append = append;
  prm.lph_log2 = 0;
  while ((16 << prm.lph_log2) < a->D) ++prm.lph_log2;
  bool vec = a->Hq == 0 || (al16(a->q, a->q_st, a->q_sh) && al16(a->q_out, a->qo_st, a->qo_sh));
  if (a->Hkv) {
    vec = vec && al16(a->k, a->k_st, a->k_sh);
    if (append)
      vec = vec && al16(a->v, a->v_st, a->v_sh) && al16(a->k_pages, a->kp_sp, a->kp_sh) && a->kp_sr % 8 == 0 &&
            al16(a->v_pages, a->vp_sp, a->vp_sh) && a->vp_sr % 8 == 0;
    else
      vec = vec && al16(a->k_out, a->ko_st, a->ko_sh);
  }
  if (a->dtype == FA_DTYPE_F16) rope_launch_t<__half>(prm, vec, st);
  else rope_launch_t<__nv_bfloat16>(prm, vec, st);
  FA_CHECK_LAUNCH(what);
  return FA_OK;
}

}  // namespace fa

extern "C" int fa_qk_norm_rope(const fa_rope_args_t* args_host, fa_stream_t stream) {
  return fa::rope_run(args_host, 0, "fa_qk_norm_rope", (cudaStream_t)stream);
}

extern "C" int fa_paged_append(const fa_rope_args_t* args_host, fa_stream_t stream) {
  return fa::rope_run(args_host, 1, "fa_paged_append", (cudaStream_t)stream);
}
