// Norm and rotation of the query and key heads of a batch of tokens, written densely (fa_qk_norm_rope) or, with the
// values, into the pages of a cache (fa_paged_append).  Per head x[D] with rotary width R <= D:
//   y = x * rsqrt(mean(x^2) + eps) * w            (no weight: y = x)
//   z[i]       = y[i] cos a_i - y[i + R/2] sin a_i,   z[i + R/2] = y[i + R/2] cos a_i + y[i] sin a_i,   i < R/2
//   z[d]       = y[d],  d >= R;      a_i = position * inv_freq[i]
// All arithmetic in float32, one rounding at the store.
//
// Bound: HBM (every element is read and written once, ~10 flop each), and close behind it the issue of instructions.
// A warp takes a token (of few tokens: some of its heads; of many, one token after another) and walks its heads, D/16
// neighbouring lanes to a head, each with 8 + 8 elements: the two halves of eight rotation pairs.  So the mean square is a
// few shuffles, every access is 16 bytes, cosines, sines and weights stay in registers for all heads, and the arithmetic
// runs on pairs of floats (f32x2).  The next heads are requested across the token's end.  Angles are reduced in float64 (a
// float32 product is off by 0.008 rad at position 131072), once per warp and token, two pairs to a lane.  Measured: 32768
// tokens of 32 + 8 heads of 128 in 146 us (4.6 TB/s, 70 % of the copy rate); with weights from L1 instead of registers
// 185 us, with three CTAs per SM and spills 183 us.
#include "common.cuh"

namespace fa {

struct RopeParams {
  fa_rope_args_t a;
  int lph_log2;   // lanes per head, log2
  int chunks;     // warps per token
  int warps;      // of the grid
};

constexpr int RA_WARPS = 8;
constexpr int RA_MAX_PAIRS = 128;
constexpr int RA_AHEAD = 3;   // heads in flight per lane

template <typename T, bool VEC>
__device__ __forceinline__ uint4 ra_load(const T* p) {
  if (VEC) return *reinterpret_cast<const uint4*>(p);
  alignas(16) T v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = p[i];
  return *reinterpret_cast<const uint4*>(v);
}
template <typename T, bool VEC>
__device__ __forceinline__ void ra_store(T* p, const uint4& raw) {
  if (VEC) {
    *reinterpret_cast<uint4*>(p) = raw;
  } else {
    const T* v = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = v[i];
  }
}
// pairs of floats
__device__ __forceinline__ uint64_t ra_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 ra_split(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t ra_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t ra_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
template <typename T>
__device__ __forceinline__ void ra_unpack(const uint4& raw, uint64_t* x) {
  const typename Pack2<T>::type* p = reinterpret_cast<const typename Pack2<T>::type*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = Pack2<T>::cvt(p[i]);
    x[i] = ra_pair(v.x, v.y);
  }
}
__device__ __forceinline__ uint32_t ra_round(uint64_t v, __half) {
  const float2 f = ra_split(v);
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t ra_round(uint64_t v, __nv_bfloat16) {
  const float2 f = ra_split(v);
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, bool VEC, bool APPEND>
__global__ void __launch_bounds__(RA_WARPS * 32, 2) rope_kernel(const __grid_constant__ RopeParams prm) {
  const fa_rope_args_t& a = prm.a;
  __shared__ __align__(16) float s_cos[RA_WARPS][RA_MAX_PAIRS], s_sin[RA_WARPS][RA_MAX_PAIRS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int unit = blockIdx.x * RA_WARPS + warp;
  int t = unit / prm.chunks;                               // the token at work
  const int chunk = unit - t * prm.chunks, stride = prm.warps / prm.chunks;
  const int heads = a.Hq + a.Hkv + (APPEND ? a.Hkv : 0);
  const int per = 32 >> prm.lph_log2;                      // heads a warp holds at once
  const int groups = (heads + per - 1) / per;
  const int g0 = groups * chunk / prm.chunks, g1 = groups * (chunk + 1) / prm.chunks;
  const int c = lane & ((1 << prm.lph_log2) - 1);          // chunk of the head this lane holds
  const bool lane_on = c * 16 < a.D;
  const int nrot = a.R / 16;
  // the two halves of the chunk: a rotation pair, or 16 elements behind the rotary width
  const int lo = c < nrot ? 8 * c : a.R + 16 * (c - nrot);
  const int hi = c < nrot ? a.R / 2 + 8 * c : lo + 8;
  const int sub = lane >> prm.lph_log2;                    // which of the heads held at once
  const int h_end = min(heads, g1 * per);

  uint4 raw[RA_AHEAD][2];
  int rt = t, rg = g0;                                     // token and heads of the next request
  auto request = [&](uint4* r) {
    r[0] = r[1] = make_uint4(0, 0, 0, 0);
    const int head = rg * per + sub;
    if (lane_on && head < h_end && rt < a.tokens) {
      const T* p;
      if (head < a.Hq) p = reinterpret_cast<const T*>(a.q) + (int64_t)rt * a.q_st + (int64_t)head * a.q_sh;
      else if (head < a.Hq + a.Hkv) p = reinterpret_cast<const T*>(a.k) + (int64_t)rt * a.k_st + (int64_t)(head - a.Hq) * a.k_sh;
      else p = reinterpret_cast<const T*>(a.v) + (int64_t)rt * a.v_st + (int64_t)(head - a.Hq - a.Hkv) * a.v_sh;
      r[0] = ra_load<T, VEC>(p + lo);
      r[1] = ra_load<T, VEC>(p + hi);
    }
    if (++rg == g1) rg = g0, rt += stride;
  };
#pragma unroll
  for (int u = 0; u < RA_AHEAD; ++u) request(raw[u]);

  bool live = true;                                        // the token belongs to a sequence
  long long kdst = -1, vdst = -1;                          // element offset of (page, head 0, row); -1: not stored
  uint64_t cs[4], sn[4];                                   // elements behind the rotary width turn by nothing
  auto begin_token = [&]() {
    // ---- where the token belongs ---------------------------------------------------------------------------------
    long long pos = 0;
    if (APPEND) {
      int b = t, i = 0, n = 1;
      kdst = vdst = -1;
      if (a.cu_seqlens) {
        // sequences that end at or before the token; empty ones are passed over
        int before = 0;
        for (int x = lane; x < a.B; x += 32) before += a.cu_seqlens[x + 1] <= t;
        b = __reduce_add_sync(0xffffffffu, before);
        if (b < a.B) {
          const int beg = a.cu_seqlens[b];
          i = t - beg;
          n = a.cu_seqlens[b + 1] - beg;
        }
      }
      live = b < a.B;
      if (!live) return;                                   // behind the last sequence: left as it was
      const long long j = (long long)a.kv_lens[b] - n + i; // index in its own sequence
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
    if (a.positions)
      pos = a.pos_i64 ? reinterpret_cast<const long long*>(a.positions)[t] : (long long)reinterpret_cast<const int*>(a.positions)[t];
    // ---- angles: turns in float64, the fraction of a turn in float32 -----------------------------------------------
    __syncwarp();
    for (int p = lane; p < a.R / 2; p += 32) {
      double turns = (double)pos * (double)a.inv_freq[p] * 0.15915494309189533577;   // 1 / (2 pi)
      turns -= rint(turns);
      sincospif(2.0f * (float)turns, &s_sin[warp][p], &s_cos[warp][p]);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      cs[i] = c < nrot ? *reinterpret_cast<const uint64_t*>(&s_cos[warp][8 * c + 2 * i]) : ra_pair(1.f, 1.f);
      sn[i] = c < nrot ? *reinterpret_cast<const uint64_t*>(&s_sin[warp][8 * c + 2 * i]) : 0;
    }
  };

  uint64_t w[8];
  int w_kind = -1;
  const float inv_d = 1.0f / (float)a.D;
  auto work = [&](int h, uint4* r) {
    const int kind = h < a.Hq ? 0 : h < a.Hq + a.Hkv ? 1 : 2;
    const void* wp = kind == 0 ? a.q_weight : kind == 1 ? a.k_weight : nullptr;
    uint64_t x[8];
    ra_unpack<T>(r[0], x);
    ra_unpack<T>(r[1], x + 4);
    float ss = 0.f;
    if (a.q_weight || a.k_weight) {
      // every lane takes part in the shuffles; heads without a weight drop the result
      uint64_t acc = ra_mul(x[0], x[0]);
#pragma unroll
      for (int i = 1; i < 8; ++i) acc = ra_fma(x[i], x[i], acc);
      const float2 f = ra_split(acc);
      ss = f.x + f.y;
      for (int o = (1 << prm.lph_log2) >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    if (!lane_on || h >= h_end || !live) return;
    if (wp) {
      if (w_kind != kind) {
        w_kind = kind;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = (i < 4 ? lo : hi - 8) + 2 * i;
          w[i] = a.w_f32 ? ra_pair(reinterpret_cast<const float*>(wp)[d], reinterpret_cast<const float*>(wp)[d + 1])
                         : ra_pair(to_f32(reinterpret_cast<const T*>(wp)[d]), to_f32(reinterpret_cast<const T*>(wp)[d + 1]));
        }
      }
      const float q = rsqrtf(fmaf(ss, inv_d, a.eps));
      const uint64_t q2 = ra_pair(q, q);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = ra_mul(ra_mul(x[i], q2), w[i]);
    }
    if (kind != 2) {
      uint32_t out[8];
      const uint64_t minus = ra_pair(-1.f, -1.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        out[i] = ra_round(ra_fma(x[i], cs[i], ra_mul(ra_mul(x[4 + i], sn[i]), minus)), T());
        out[4 + i] = ra_round(ra_fma(x[4 + i], cs[i], ra_mul(x[i], sn[i])), T());
      }
      r[0] = make_uint4(out[0], out[1], out[2], out[3]);
      r[1] = make_uint4(out[4], out[5], out[6], out[7]);
    }
    T* dst;
    if (kind == 0) {
      dst = reinterpret_cast<T*>(a.q_out) + (int64_t)t * a.qo_st + (int64_t)h * a.qo_sh;
    } else if (!APPEND) {
      dst = reinterpret_cast<T*>(a.k_out) + (int64_t)t * a.ko_st + (int64_t)(h - a.Hq) * a.ko_sh;
    } else {
      if (kdst < 0) return;
      dst = kind == 1 ? reinterpret_cast<T*>(a.k_pages) + kdst + (int64_t)(h - a.Hq) * a.kp_sh
                      : reinterpret_cast<T*>(a.v_pages) + vdst + (int64_t)(h - a.Hq - a.Hkv) * a.vp_sh;
    }
    ra_store<T, VEC>(dst + lo, r[0]);
    ra_store<T, VEC>(dst + hi, r[1]);
  };
  int g = g0;
  while (t < a.tokens) {
#pragma unroll
    for (int u = 0; u < RA_AHEAD; ++u) {
      if (t >= a.tokens) break;
      if (g == g0) begin_token();
      work(g * per + sub, raw[u]);
      request(raw[u]);
      if (++g == g1) g = g0, t += stride;
    }
  }
}

static bool al16(const void* p, int64_t s0, int64_t s1) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s0 % 8 == 0 && s1 % 8 == 0;
}

template <typename T, bool APPEND>
static void rope_launch(const RopeParams& prm, bool vec, cudaStream_t st) {
  const unsigned grid = prm.warps / RA_WARPS;
  if (vec) rope_kernel<T, true, APPEND><<<grid, RA_WARPS * 32, 0, st>>>(prm);
  else rope_kernel<T, false, APPEND><<<grid, RA_WARPS * 32, 0, st>>>(prm);
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
  // Two CTAs of 8 warps fill an SM.  From 16 tokens per SM on a warp takes tokens of its own, one after another; fewer are
  // divided among more warps, down to one pass over the heads each, so that the walk's latency is not the call's.
  const int groups = ceil_div(a->Hq + a->Hkv * (append ? 2 : 1), 32 >> prm.lph_log2);
  const int full = 2 * RA_WARPS * sm_count();
  prm.chunks = 1;
  while (prm.chunks < groups && (int64_t)a->tokens * (prm.chunks + 1) <= full) ++prm.chunks;
  const int unit = RA_WARPS * prm.chunks;             // whole tokens, whole CTAs
  prm.warps = (int)(prm.chunks > 1 ? ceil_div64((int64_t)a->tokens * prm.chunks, unit) * unit
                                   : (int64_t)RA_WARPS * ceil_div64(a->tokens < full ? a->tokens : full, RA_WARPS));
  if (a->dtype == FA_DTYPE_F16) append ? rope_launch<__half, true>(prm, vec, st) : rope_launch<__half, false>(prm, vec, st);
  else append ? rope_launch<__nv_bfloat16, true>(prm, vec, st) : rope_launch<__nv_bfloat16, false>(prm, vec, st);
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
