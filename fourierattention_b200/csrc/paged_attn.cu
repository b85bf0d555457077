// Attention of new tokens over the pages of a cache and over a prefix the batch shares (fa_paged_attn).
//   row (token, query head):  s_j = scale q . k_j,  m = max s,  p_j = e^(s_j - m),  l = sum p,  o = sum p_j v_j / l,
//   lse = m + ln l;  the keys are all of the prefix and the sequence's own keys up to the token.  A row without keys
//   gives o = 0, lse = -inf.
#include "paged_tile.cuh"

namespace fa {

// ---- few rows per key: streaming ---------------------------------------------------------------------------------------
// Bound: HBM (each key and value is read once, ~G multiply-adds per byte).  Eight warps, each on its own: a warp takes
// 16 keys of every 128-key tile, fetched by TMA (one page's rows, 128-byte swizzle) into a ring of its own, so no warp
// waits for another while keys stream.  The products are turned round, keys as the 16 rows of mma.m16n8k16 and query
// rows as its 8 columns: a group of up to 8 query heads fills the instruction, where query rows as the 16 rows would
// leave half of it empty and twice the accumulator registers.  The running maximum moves only when a score passes it
// by 2^8 (one vote per 16 keys instead of three shuffle rounds); until then probabilities stay inside fp16's range (PaLift),
// and the denominator sums what was not rounded.  Measured: 6.1 TB/s (93 % of the copy rate) for 32 sequences
// of up to 16384 keys, 24 / 8 heads; ring of 24 KB per warp, 192 KB per SM in flight.  Probabilities are rounded to the cache's type for the
// second product (relative error up to 2^-9 in bf16 and, from 2^-21 of the largest up, 2^-12 in fp16; independent from key
// to key).
template <int D>
struct PaStream {
  static constexpr int WARPS = 8;
  static constexpr int BOX = 16 * 128;                     // 16 keys x 64 columns
  static constexpr int STAGE = 2 * (D / 64) * BOX;         // K and V
  static constexpr int ST = 24 * 1024 / STAGE;             // 24 KB per warp in flight
  static constexpr int RING = WARPS * ST * STAGE;
  static constexpr int OPITCH = D + 4;
  static constexpr int OBUF = WARPS * 8 * OPITCH * 4;
  struct Small {
    uint64_t bar[WARPS][ST];
    float m[WARPS][16], l[WARPS][16];
    PaLocate loc;
    int dead;
  };
  static constexpr int SMEM = RING + OBUF + 2048;          // all of the 227 KB at D = 128
};
static_assert(sizeof(PaStream<128>::Small) <= 2048 && sizeof(PaStream<64>::Small) <= 2048, "barriers and statistics");

struct PaStreamParams {
  alignas(64) CUtensorMap tm_k, tm_v;
  PaCommon c;
  PaPhase p;
};

template <typename T>
__device__ __forceinline__ void pa_mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void pa_mma<__half>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void pa_mma<__nv_bfloat16>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pa_ldsm(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pa_ldsm_t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t pa_turn(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(256, 1) paged_stream_kernel(const __grid_constant__ PaStreamParams prm) {
  using C = PaStream<D>;
  const PaCommon& c = prm.c;
  const PaPhase& p = prm.p;
  extern __shared__ __align__(1024) unsigned char pa_dyn[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ring = pa_smem(pa_dyn) + warp * (C::ST * C::STAGE);
  float* obuf = reinterpret_cast<float*>(pa_dyn + C::RING);
  typename C::Small& sh = *reinterpret_cast<typename C::Small*>(pa_dyn + C::RING + C::OBUF);
  const uint32_t bar0 = pa_smem(&sh.bar[warp][0]);
  constexpr float LIFT = PaLift<T>::STEPS;

  if (tid == 0) {
    sh.dead = 0;
    for (int w = 0; w < C::WARPS; ++w)
      for (int s = 0; s < C::ST; ++s) pa_bar_init(pa_smem(&sh.bar[w][s]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    if (pa_smem(pa_dyn) & 1023u) sh.dead = 1;      // the swizzle pattern goes by the address
  }
  pa_let_next_begin();
  PaUnit u;
  int t;
  const PaRange range = pa_locate<256>(c, p, blockIdx.x, sh.loc, u, t);   // (its barriers order the initialisation too)

  // ---- this warp's fetches: the same walk as below, ST groups of 16 keys ahead -----------------------------------------
  PaUnit fu = u;
  int ft = t, f_left = (int)(range.end - range.beg);
  struct Fetch {
    int tok, page, head;                  // tok < 0: nothing left
  };
  auto f_next = [&]() -> Fetch {
    while (f_left > 0) {
      if (ft >= fu.tiles) {
        fu.next(c, p);
        ft = 0;
        continue;
      }
      const int tok = ft * PA_TILE + warp * 16;
      ++ft, --f_left;
      if (tok < fu.limit)
        return Fetch{tok, p.table[(int64_t)fu.b * p.table_sb + (unsigned)tok / (unsigned)c.page_size], fu.h};
    }
    return Fetch{-1, 0, 0};
  };
  uint32_t bad = 0;                       // stages whose page id names no page
  auto issue = [&](const Fetch& f, int stage) {
    if (f.tok < 0) return;
    const bool ok = f.page >= 0 && f.page < c.num_pages;
    bad = ok ? bad & ~(1u << stage) : bad | (1u << stage);
    if (lane == 0) {
      const uint32_t bar = bar0 + 8 * stage, dst = ring + stage * C::STAGE;
      if (ok) {
        const int row = (int)((unsigned)f.tok % (unsigned)c.page_size);
        pa_bar_expect(bar, C::STAGE);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          pa_tma(dst + i * C::BOX, &prm.tm_k, 64 * i, row, f.head, f.page, bar);
          pa_tma(dst + C::STAGE / 2 + i * C::BOX, &prm.tm_v, 64 * i, row, f.head, f.page, bar);
        }
      } else {
        pa_bar_arrive(bar);
      }
    }
  };
  // the page ids of the first groups are requested together, later ones a group ahead
  Fetch ahead;
  {
    Fetch f[C::ST];
#pragma unroll
    for (int s = 0; s < C::ST; ++s) f[s] = f_next();
    ahead = f_next();
#pragma unroll
    for (int s = 0; s < C::ST; ++s) issue(f[s], s);
  }

  const int g = lane >> 2, c2 = 2 * (lane & 3);
  const int ld_row = lane & 15, ld_half = lane >> 4;                       // K: rows as they lie
  const int lt_row = (lane & 7) + ((lane >> 4) << 3), lt_half = (lane >> 3) & 1;   // V: turned
  int stage = 0;
  uint32_t parity = 0;
  long long done = range.beg;             // tiles before the current one

  while (done < range.end) {
    if (t >= u.tiles) {
      u.next(c, p);
      t = 0;
      continue;
    }
    const int t_end = (int)min((long long)u.tiles, t + (range.end - done));
    // ---- the block's query rows, as the second operand -------------------------------------------------------------
    const int row0 = u.rb << p.rows_log2, L = pa_keys(p, u.s);
    const int n_rows = min(1 << p.rows_log2, u.s.n * c.G - row0);
    uint32_t qf[NT][D / 16][2];
    int lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + g;
      const bool on = r < n_rows;
      const int tok = (row0 + r) / c.G, hg = (row0 + r) - tok * c.G;
      const T* q = reinterpret_cast<const T*>(c.q) + (int64_t)(u.s.t0 + tok) * c.q_st + (int64_t)(u.h * c.G + hg) * c.q_sh + c2;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[nt][kk][0] = on ? *reinterpret_cast<const uint32_t*>(q + 16 * kk) : 0u;
        qf[nt][kk][1] = on ? *reinterpret_cast<const uint32_t*>(q + 16 * kk + 8) : 0u;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int rr = min(nt * 8 + c2 + j, n_rows - 1);
        lim[nt][j] = p.prefix_len > 0 ? L : min(L, u.s.len - u.s.n + (row0 + rr) / c.G + 1);
      }
    }
    const int lim0 = p.prefix_len > 0 ? L : min(L, u.s.len - u.s.n + row0 / c.G + 1);     // the first row sees least
    float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
    }

    for (int tt = t; tt < t_end; ++tt) {
      const int tok = tt * PA_TILE + warp * 16;
      if (tok >= u.limit) break;
      pa_bar_wait(bar0 + 8 * stage, parity, &sh.dead);
      if (!((bad >> stage) & 1)) {
        const uint32_t kb = ring + stage * C::STAGE, vb = kb + C::STAGE / 2;
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t a[4];
          const int ch = 2 * kk + ld_half;
          pa_ldsm(a, kb + (ch >> 3) * C::BOX + ld_row * 128 + (((ch & 7) ^ (ld_row & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) pa_mma<T>(s[nt], a, qf[nt][kk][0], qf[nt][kk][1]);
        }
        const bool masked = tok + 16 > lim0;
        bool rise = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[nt][j] *= c.scale_log2;
            if (masked && tok + g + 8 * (j >> 1) >= lim[nt][j & 1]) s[nt][j] = -INFINITY;
          }
          rise |= fmaxf(s[nt][0], s[nt][2]) > m[nt][0] + (8.f + LIFT) || fmaxf(s[nt][1], s[nt][3]) > m[nt][1] + (8.f + LIFT);
        }
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float mx = fmaxf(s[nt][j], s[nt][j + 2]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              mx = fmaxf(mx - LIFT, m[nt][j]);
              const float f = m[nt][j] == -INFINITY ? 0.f : pa_ex2(m[nt][j] - mx);
              m[nt][j] = mx;
              l[nt][j] *= f;
#pragma unroll
              for (int i = 0; i < D / 16; ++i) o[nt][i][j] *= f, o[nt][i][j + 2] *= f;
            }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
          const float p0 = pa_ex2(s[nt][0] - m0), p1 = pa_ex2(s[nt][1] - m1);
          const float p2 = pa_ex2(s[nt][2] - m0), p3 = pa_ex2(s[nt][3] - m1);
          l[nt][0] += p0 + p2;
          l[nt][1] += p1 + p3;
          pb[nt][0] = pa_turn(pa_pack<T>(p0, p1));
          pb[nt][1] = pa_turn(pa_pack<T>(p2, p3));
        }
        if (tok + 16 > L) {
          // rows behind the sequence hold anything: 0 x NaN must not reach the sums
          for (int i = lane; i < 16 * (D / 8); i += 32) {
            const int r = i / (D / 8), ch = i % (D / 8);
            if (tok + r >= L)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(vb + (ch >> 3) * C::BOX + r * 128 + ((ch & 7) << 4)), "r"(0) : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");   // before the next fetch into this stage
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t a[4];
          const int ch = 2 * i + lt_half;
          pa_ldsm_t(a, vb + (ch >> 3) * C::BOX + lt_row * 128 + (((ch & 7) ^ (lt_row & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) pa_mma<T>(o[nt][i], a, pb[nt][0], pb[nt][1]);
        }
      }
      __syncwarp();                       // every lane has read the stage
      issue(ahead, stage);
      ahead = f_next();
      if (++stage == C::ST) stage = 0, parity ^= 1;
    }

    // ---- the eight warps' results of this unit ---------------------------------------------------------------------------
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = l[nt][j];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (g == 0) sh.m[warp][nt * 8 + c2 + j] = m[nt][j], sh.l[warp][nt * 8 + c2 + j] = x;
      }
    const bool first = t == 0, last = t_end == u.tiles;
    const bool whole = first && last;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float* dst = obuf + (warp * 8 + c2 + j) * C::OPITCH + g;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          dst[16 * i] = o[nt][i][j];
          dst[16 * i + 8] = o[nt][i][j + 2];
        }
      }
      __syncthreads();
      const float poison = sh.dead ? __int_as_float(0x7fc00000) : 0.f;
      for (int e = tid; e < 8 * (D / 4); e += 256) {
        const int col = e / (D / 4), d4 = (e % (D / 4)) * 4;
        const int r = nt * 8 + col;
        if (r >= n_rows) continue;
        float mx = -INFINITY, lsum = 0.f;
#pragma unroll
        for (int w = 0; w < C::WARPS; ++w) mx = fmaxf(mx, sh.m[w][r]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < C::WARPS; ++w) {
          const float f = sh.m[w][r] == -INFINITY ? 0.f : pa_ex2(sh.m[w][r] - mx);
          lsum = fmaf(sh.l[w][r], f, lsum);
          const float4 v = *reinterpret_cast<const float4*>(obuf + (w * 8 + col) * C::OPITCH + d4);
          acc.x = fmaf(v.x, f, acc.x), acc.y = fmaf(v.y, f, acc.y), acc.z = fmaf(v.z, f, acc.z), acc.w = fmaf(v.w, f, acc.w);
        }
        acc.x += poison, acc.y += poison, acc.z += poison, acc.w += poison;
        lsum += poison;
        const int tok = u.s.t0 + (row0 + r) / c.G, hq = u.h * c.G + (row0 + r) % c.G;
        if (whole && p.direct) {
          const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
          T* dst = reinterpret_cast<T*>(c.out) + (int64_t)tok * c.o_st + (int64_t)hq * c.o_sh + d4;
          *reinterpret_cast<uint2*>(dst) = make_uint2(pa_pack<T>(acc.x * inv, acc.y * inv), pa_pack<T>(acc.z * inv, acc.w * inv));
          if (c.lse && d4 == 0)
            c.lse[(int64_t)tok * c.Hq + hq] = lsum == 0.f ? -INFINITY : (mx + log2f(lsum)) * 0.6931471805599453f;
        } else {
          const int64_t at = whole ? (int64_t)tok * c.Hq + hq
                                   : ((int64_t)(2 * blockIdx.x + (first ? 1 : 0)) << p.rows_log2) + r;
          *reinterpret_cast<float4*>((whole ? p.row_o : p.slot_o) + at * D + d4) = acc;
          if (d4 == 0) (whole ? p.row_ml : p.slot_ml)[at] = make_float2(mx, lsum);
        }
      }
      __syncthreads();
    }
    if (last && tid == 0) {
      const long long first_tile = done - t;
      p.info[pa_unit_id(c, p, u.b, u.s, u.h, u.rb)] = make_int2(pa_owner(range, first_tile), blockIdx.x);
    }
    done += t_end - t;
    t = t_end;
  }
  pa_leave(&sh.dead);
  pa_wait_for_previous();
}

// ---- joining the parts ---------------------------------------------------------------------------------------------------
// A warp per row, or per four neighbouring rows: the parts of the prefix and of the sequence's own keys, in the order of
// their keys.  Bound by the chain of lookups (sequence, unit, parts), which four rows share.
struct PaMergeParams {
  PaCommon c;
  PaPhase own, prefix;       // prefix.prefix_len == 0: none
};

template <int D>
__device__ __forceinline__ void pa_load(const float* src, int lane, float* o) {
  if (D == 128) {
    const float4 v = *reinterpret_cast<const float4*>(src + 4 * lane);
    o[0] = v.x, o[1] = v.y, o[2] = v.z, o[D / 32 - 1] = v.w;
  } else {
    const float2 v = *reinterpret_cast<const float2*>(src + 2 * lane);
    o[0] = v.x, o[1] = v.y;
  }
}

template <typename T, int D, int RPW>
__global__ void __launch_bounds__(256) paged_merge_kernel(const __grid_constant__ PaMergeParams prm) {
  constexpr int PB = 8 / RPW;             // parts of a row requested before the first is used
  const PaCommon& c = prm.c;
  const int lane = threadIdx.x & 31;
  const int64_t row0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * RPW;
  if (row0 >= (int64_t)c.tokens * c.Hq) return;
  const int t = (int)((unsigned)row0 / (unsigned)c.Hq), hq0 = (int)row0 - t * c.Hq;
  int b = t;
  if (c.cu) {
    int n = 0;
    for (int i = lane; i < c.B; i += 32) n += c.cu[i + 1] <= t;
    b = __reduce_add_sync(0xffffffffu, n);
  }
  pa_wait_for_previous();
  if (b >= c.B) return;                   // behind the last sequence: left as it was
  // Where the parts of every row lie, in both phases at once: (first CTA, last); one part in the row arrays, or slots.
  int2 who[2][RPW];
  int in_block[2][RPW];
  PaSeq s[2];
#pragma unroll
  for (int ph = 0; ph < 2; ++ph) s[ph] = pa_seq(c, ph == 0 ? prm.prefix : prm.own, ph == 0 ? 0 : b);
#pragma unroll
  for (int ph = 0; ph < 2; ++ph) {
    const PaPhase& p = ph == 0 ? prm.prefix : prm.own;
    const bool on = (ph == 1 || p.prefix_len > 0) && t >= s[ph].t0 && t < s[ph].t0 + s[ph].n;
#pragma unroll
    for (int j = 0; j < RPW; ++j) {
      const int hq = hq0 + j, h = hq / c.G;
      const int r = (t - s[ph].t0) * c.G + hq - h * c.G, rb = r >> p.rows_log2;
      in_block[ph][j] = r - (rb << p.rows_log2);
      who[ph][j] = make_int2(0, -1);
      if (on && pa_unit_tiles(p, pa_limit(c, p, s[ph], rb)) > 0)
        who[ph][j] = p.info[pa_unit_id(c, p, ph == 0 ? 0 : b, s[ph], h, rb)];
    }
  }
  float m[RPW], l[RPW], acc[RPW][D / 32];
  bool skip[RPW];                         // written already
#pragma unroll
  for (int j = 0; j < RPW; ++j) {
    m[j] = -INFINITY, l[j] = 0.f;
    skip[j] = prm.own.direct && who[1][j].x == who[1][j].y;
    if (skip[j]) who[1][j].y = who[1][j].x - 1;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[j][i] = 0.f;
  }
#pragma unroll
  for (int ph = 0; ph < 2; ++ph) {
    const PaPhase& p = ph == 0 ? prm.prefix : prm.own;
    int most = 0;
#pragma unroll
    for (int j = 0; j < RPW; ++j) most = max(most, who[ph][j].y - who[ph][j].x + 1);
    for (int base = 0; base < most; base += 32) {
      // maximum and denominator of up to 32 parts, a part per lane; then the parts' weights
      auto place = [&](int j, int k) -> int64_t {
        const int2 w = who[ph][j];
        const int cta = w.x + k;
        return w.x == w.y ? row0 + j : ((int64_t)(2 * cta + (cta == w.x ? 1 : 0)) << p.rows_log2) + in_block[ph][j];
      };
      float2 ml[RPW];
#pragma unroll
      for (int j = 0; j < RPW; ++j) {
        ml[j] = make_float2(-INFINITY, 0.f);
        const int2 w = who[ph][j];
        if (w.x + base + lane <= w.y) ml[j] = (w.x == w.y ? p.row_ml : p.slot_ml)[place(j, base + lane)];
      }
      float weight[RPW];
#pragma unroll
      for (int j = 0; j < RPW; ++j) {
        const float mx = fmaxf(m[j], warp_max(ml[j].x));
        const float f = m[j] == -INFINITY ? 0.f : pa_ex2(m[j] - mx);
        weight[j] = ml[j].x == -INFINITY ? 0.f : pa_ex2(ml[j].x - mx);
        if (ml[j].x != ml[j].x) weight[j] = ml[j].x;                    // a part that gave up poisons its rows
        m[j] = mx;
        l[j] = l[j] * f + warp_sum(weight[j] * ml[j].y);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[j][i] *= f;
      }
      for (int k0 = base; k0 < min(most, base + 32); k0 += PB) {
        float o[RPW][PB][D / 32];
#pragma unroll
        for (int j = 0; j < RPW; ++j)
#pragma unroll
          for (int k = 0; k < PB; ++k)
            if (who[ph][j].x + k0 + k <= who[ph][j].y)
              pa_load<D>((who[ph][j].x == who[ph][j].y ? p.row_o : p.slot_o) + place(j, k0 + k) * D, lane, o[j][k]);
#pragma unroll
        for (int j = 0; j < RPW; ++j)
#pragma unroll
          for (int k = 0; k < PB; ++k) {
            const float w = __shfl_sync(0xffffffffu, weight[j], (k0 + k - base) & 31);
            if (who[ph][j].x + k0 + k <= who[ph][j].y)
#pragma unroll
              for (int i = 0; i < D / 32; ++i) acc[j][i] = fmaf(o[j][k][i], w, acc[j][i]);
          }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < RPW; ++j) {
    if (skip[j]) continue;
    const float inv = l[j] == 0.f ? 0.f : 1.f / l[j];
    T* dst = reinterpret_cast<T*>(c.out) + (int64_t)t * c.o_st + (int64_t)(hq0 + j) * c.o_sh + lane * (D / 32);
    const float* a = acc[j];
    if (D == 128)
      *reinterpret_cast<uint2*>(dst) = make_uint2(pa_pack<T>(a[0] * inv, a[1] * inv), pa_pack<T>(a[2] * inv, a[D / 32 - 1] * inv));
    else
      *reinterpret_cast<uint32_t*>(dst) = pa_pack<T>(a[0] * inv, a[1] * inv);
    if (c.lse && lane == 0) c.lse[row0 + j] = l[j] == 0.f ? -INFINITY : (m[j] + log2f(l[j])) * 0.6931471805599453f;
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------------
static int pa_map(CUtensorMap* m, const void* base, const fa_paged_attn_args_t* a, int64_t sp, int64_t sh, int64_t sr,
                  int box_rows) {
  return make_tensor_map_4d(m, base, a->dtype, a->D, a->page_size, sr, a->Hkv, sh, a->num_pages, sp, 64, box_rows);
}

static int pa_check(const fa_paged_attn_args_t* a) {
  const char* w = "fa_paged_attn";
  FA_REQUIRE(a, FA_ERR_NULL, "%s: null argument block", w);
  FA_REQUIRE(a->dtype == FA_DTYPE_F16 || a->dtype == FA_DTYPE_BF16, FA_ERR_DTYPE, "%s: bad dtype %d", w, a->dtype);
  FA_REQUIRE(a->tokens >= 0 && a->B >= 0 && a->Hq > 0 && a->Hkv > 0 && a->max_pages >= 0 && a->num_pages > 0 && a->prefix_len >= 0,
             FA_ERR_SHAPE, "%s: bad sizes", w);
  FA_REQUIRE(a->Hq % a->Hkv == 0, FA_ERR_SHAPE, "%s: Hq (%d) must be a multiple of Hkv (%d)", w, a->Hq, a->Hkv);
  FA_REQUIRE(a->D == 64 || a->D == 128, FA_ERR_UNSUPPORTED, "%s: the head dimension must be 64 or 128 (got %d)", w, a->D);
  FA_REQUIRE(a->page_size >= 16 && a->page_size % 16 == 0, FA_ERR_SHAPE,
             "%s: the page size must be a multiple of 16 (got %d)", w, a->page_size);
  FA_REQUIRE((int64_t)a->max_pages * a->page_size < (1ll << 31) - PA_TILE, FA_ERR_CAPACITY,
             "%s: a sequence of up to %lld keys", w, (long long)a->max_pages * a->page_size);
  FA_REQUIRE((int64_t)a->tokens * a->Hq < (1ll << 31) - 4096, FA_ERR_CAPACITY, "%s: too many query rows", w);
  FA_REQUIRE(a->cu_seqlens || a->tokens == a->B, FA_ERR_SHAPE,
             "%s: without cu_seqlens there is one token per sequence (%d tokens, %d sequences)", w, a->tokens, a->B);
  FA_REQUIRE((int64_t)a->prefix_len < (1ll << 31) - PA_TILE && (a->prefix_len == 0 || (int64_t)a->n_prefix_pages * a->page_size >= a->prefix_len),
             FA_ERR_SHAPE, "%s: %d prefix pages of %d do not hold %d keys", w, a->n_prefix_pages, a->page_size, a->prefix_len);
  return FA_OK;
}

struct PaPlan {
  int rows_own, rows_pre, ctas;
  bool lead;                  // the prefix in front of every sequence's own keys, not as a phase of its own
  size_t bytes, slot_o[2], slot_ml[2], row_o[2], row_ml[2], info[2];
};

static PaPlan pa_plan(const fa_paged_attn_args_t* a) {
  PaPlan pl;
  const int64_t G = a->Hq / a->Hkv;
  pl.ctas = sm_count();
  // Eight rows fill the streaming kernel's instruction; sixteen take a second one per key; more go to the tile kernel.  The
  // mean over the batch decides, since the lengths are on the device: one long prompt among many sequences of a token
  // each is read in blocks of 16 rows.
  const int64_t own = a->cu_seqlens && a->B > 0 ? (int64_t)a->tokens * G / a->B : G, pre = (int64_t)a->tokens * G;
  pl.rows_own = a->cu_seqlens && own > 16 ? PT_ROWS : own <= 8 ? 8 : 16;
  pl.rows_pre = pre > 16 ? PT_ROWS : pre <= 8 ? 8 : 16;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t r = at;
    at += (n + 255) / 256 * 256;
    return r;
  };
  // Blocks that a sequence's own rows fill read the prefix no more often by themselves than packed with others', and the
  // prefix in front of their own keys saves a launch and partial results (4 heads per group, whole calls in short loops:
  // 8 x up to 250 tokens over 16384 keys 423 us against 435 as two phases, 4 x up to 1000 over 8192 462 against 558);
  // emptier blocks are better packed across the batch.
  pl.lead = a->prefix_len > 0 && pl.rows_own == PT_ROWS && own >= 3 * PT_ROWS / 4;
  const bool shared = a->prefix_len > 0 && !pl.lead;
  for (int i = 0; i < (shared ? 2 : 1); ++i) {
    const int64_t rows = i == 0 ? pl.rows_own : pl.rows_pre;
    pl.slot_o[i] = take((size_t)2 * pl.ctas * rows * a->D * 4);
    pl.slot_ml[i] = take((size_t)2 * pl.ctas * rows * 8);
    pl.info[i] = take((size_t)pa_info_count(a->tokens, i == 0 ? a->B : 1, G, a->Hkv, rows) * 8);
    pl.row_o[i] = pl.row_ml[i] = 0;
    if (shared) {
      pl.row_o[i] = take((size_t)a->tokens * a->Hq * a->D * 4);
      pl.row_ml[i] = take((size_t)a->tokens * a->Hq * 8);
    }
  }
  pl.bytes = at;
  return pl;
}

// `after`: may begin while the launch before drains
template <typename P>
static int pa_launch(void (*kernel)(P), const P& prm, unsigned grid, int threads, int smem, bool after, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, prm);
  return e == cudaSuccess ? FA_OK : cuda_fail(e, "fa_paged_attn");
}

template <typename T, int D, int NT>
static int pa_stream_launch(const PaStreamParams& prm, bool second, cudaStream_t st) {
  constexpr int smem = PaStream<D>::SMEM;
  const int rc = allow_smem<paged_stream_kernel<T, D, NT>>(smem, "cudaFuncSetAttribute(paged_stream)");
  if (rc != FA_OK) return rc;
  return pa_launch(paged_stream_kernel<T, D, NT>, prm, prm.p.ctas, 256, smem, second, st);
}

template <typename T, int D>
static int pa_tile_launch(const PaTileParams& prm, bool second, cudaStream_t st) {
  constexpr int smem = PaTile<D>::SMEM;
  const int rc = allow_smem<paged_tile_kernel<T, D>>(smem, "cudaFuncSetAttribute(paged_tile)");
  if (rc != FA_OK) return rc;
  return pa_launch(paged_tile_kernel<T, D>, prm, prm.p.ctas, PT_THREADS, smem, second, st);
}

template <typename T, int D>
static int pa_run(const fa_paged_attn_args_t* a, cudaStream_t st) {
  const PaPlan pl = pa_plan(a);
  unsigned char* s = reinterpret_cast<unsigned char*>(a->scratch);
  PaStreamParams prm;
  PaCommon& c = prm.c;
  c.q = a->q, c.q_st = a->q_st, c.q_sh = a->q_sh;
  c.out = a->out, c.o_st = a->o_st, c.o_sh = a->o_sh;
  c.lse = a->lse;
  c.kv_lens = a->kv_lens, c.cu = a->cu_seqlens;
  c.tokens = a->tokens, c.B = a->B, c.Hq = a->Hq, c.Hkv = a->Hkv, c.G = a->Hq / a->Hkv;
  c.page_size = a->page_size, c.num_pages = a->num_pages;
  const float scale = a->sm_scale > 0.f ? a->sm_scale : 1.f / sqrtf((float)D);
  c.scale_log2 = scale * 1.4426950408889634f;
  const bool shared = a->prefix_len > 0 && !pl.lead;
  PaTileParams tile;
  tile.box_rows = 16;
  while (tile.box_rows < PA_TILE && a->page_size % (2 * tile.box_rows) == 0) tile.box_rows *= 2;
  int rc = FA_OK;
  if (pl.rows_own < PT_ROWS || (shared && pl.rows_pre < PT_ROWS)) {
    rc = pa_map(&prm.tm_k, a->k_pages, a, a->kp_sp, a->kp_sh, a->kp_sr, 16);
    if (rc == FA_OK) rc = pa_map(&prm.tm_v, a->v_pages, a, a->vp_sp, a->vp_sh, a->vp_sr, 16);
  }
  if (rc == FA_OK && (pl.rows_own == PT_ROWS || (shared && pl.rows_pre == PT_ROWS))) {
    rc = pa_map(&tile.tm_k, a->k_pages, a, a->kp_sp, a->kp_sh, a->kp_sr, tile.box_rows);
    if (rc == FA_OK) rc = pa_map(&tile.tm_v, a->v_pages, a, a->vp_sp, a->vp_sh, a->vp_sr, tile.box_rows);
  }
  if (rc != FA_OK) return rc;
  tile.c = c;
  PaMergeParams mg;
  mg.c = c;
  auto phase = [&](int i) {
    PaPhase p;
    p.table = i == 0 ? a->page_table : a->prefix_pages;
    p.table_sb = i == 0 ? a->table_sb : 0;
    // (checked to be below 2^31; a prefix has its pages)
    p.cap = i == 0 ? (int)((int64_t)a->max_pages * a->page_size) : a->prefix_len;
    p.prefix_len = i == 0 ? 0 : a->prefix_len;
    p.lead_table = a->prefix_pages;
    p.lead_len = i == 0 && pl.lead ? a->prefix_len : 0;
    const int rows = i == 0 ? pl.rows_own : pl.rows_pre;
    p.rows_log2 = rows == PT_ROWS ? 8 : rows == 16 ? 4 : 3;
    p.ctas = pl.ctas;
    p.direct = !shared;
    p.slot_o = reinterpret_cast<float*>(s + pl.slot_o[i]);
    p.slot_ml = reinterpret_cast<float2*>(s + pl.slot_ml[i]);
    p.row_o = reinterpret_cast<float*>(s + pl.row_o[i]);
    p.row_ml = reinterpret_cast<float2*>(s + pl.row_ml[i]);
    p.info = reinterpret_cast<int2*>(s + pl.info[i]);
    return p;
  };
  mg.prefix = PaPhase{};
  for (int i = shared ? 1 : 0; i >= 0; --i) {
    prm.p = tile.p = phase(i);
    (i == 0 ? mg.own : mg.prefix) = prm.p;
    const bool second = shared && i == 0;
    rc = prm.p.rows_log2 == 8   ? pa_tile_launch<T, D>(tile, second, st)
         : prm.p.rows_log2 == 3 ? pa_stream_launch<T, D, 1>(prm, second, st)
                                : pa_stream_launch<T, D, 2>(prm, second, st);
    if (rc != FA_OK) return rc;
  }
  const int64_t rows = (int64_t)a->tokens * a->Hq;
  // four rows per warp once every SM has work of that kind for all of its warps
  if (a->Hq % 4 == 0 && rows >= 4 * 32 * (int64_t)sm_count())
    return pa_launch(paged_merge_kernel<T, D, 4>, mg, (unsigned)ceil_div64(rows, 32), 256, 0, true, st);
  return pa_launch(paged_merge_kernel<T, D, 1>, mg, (unsigned)ceil_div64(rows, 8), 256, 0, true, st);
}

}  // namespace fa

using namespace fa;

extern "C" size_t fa_paged_attn_scratch_bytes(const fa_paged_attn_args_t* args_host) {
  if (pa_check(args_host) != FA_OK) return 0;
  return pa_plan(args_host).bytes;
}

extern "C" int fa_paged_attn_launches(const fa_paged_attn_args_t* a) {
  if (pa_check(a) != FA_OK || a->tokens == 0 || a->B == 0) return 0;
  return a->prefix_len > 0 && !pa_plan(a).lead ? 3 : 2;
}

extern "C" int fa_paged_attn(const fa_paged_attn_args_t* a, fa_stream_t stream) {
  const int rc = pa_check(a);
  if (rc != FA_OK) return rc;
  if (a->tokens == 0 || a->B == 0) return FA_OK;
  FA_REQUIRE(a->q && a->out && a->k_pages && a->v_pages && a->kv_lens && (a->page_table || a->max_pages == 0), FA_ERR_NULL,
             "fa_paged_attn: null pointer");
  FA_REQUIRE(a->prefix_len == 0 || a->prefix_pages, FA_ERR_NULL, "fa_paged_attn: null prefix pages");
  auto aligned = [](const void* p, int64_t s0, int64_t s1, int64_t s2) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s0 % 8 == 0 && s1 % 8 == 0 && s2 % 8 == 0;
  };
  FA_REQUIRE(aligned(a->q, a->q_st, a->q_sh, 0) && aligned(a->out, a->o_st, a->o_sh, 0), FA_ERR_ALIGN,
             "fa_paged_attn: q and out must start on 16 bytes with strides of multiples of 8 elements");
  FA_REQUIRE(aligned(a->k_pages, a->kp_sp, a->kp_sh, a->kp_sr) && aligned(a->v_pages, a->vp_sp, a->vp_sh, a->vp_sr), FA_ERR_ALIGN,
             "fa_paged_attn: the pages must start on 16 bytes with strides of multiples of 8 elements");
  const size_t need = pa_plan(a).bytes;
  FA_REQUIRE(a->scratch && a->scratch_bytes >= need && (reinterpret_cast<uintptr_t>(a->scratch) & 255) == 0, FA_ERR_CAPACITY,
             "fa_paged_attn: scratch too small or not on 256 bytes (%zu < %zu bytes)", a->scratch_bytes, need);
  cudaStream_t st = (cudaStream_t)stream;
  if (a->dtype == FA_DTYPE_F16) return a->D == 64 ? pa_run<__half, 64>(a, st) : pa_run<__half, 128>(a, st);
  return a->D == 64 ? pa_run<__nv_bfloat16, 64>(a, st) : pa_run<__nv_bfloat16, 128>(a, st);
}
