// Many query rows per key: the tensor-core form of the paged attention.
//
// A unit is up to 256 query rows (two tiles of 128) that read the same keys.  Per 128-key tile and query tile
//   S = Q K^T   (tcgen05.mma, both from shared memory, M = N = 128),  P = 2^(S - m) rounded to the cache's type,
//   O += P V    (tcgen05.mma, P from tensor memory, V as it lies in the page: the MN-major operand).
// Bound: the tensor pipe (2 x 512 cycles per query tile and key tile at D = 128) and the exponentials (16 per cycle and
// SM: 1024 cycles), which run side by side: the warps of one query tile work while the other's products run.  Reached is
// 57 % of either with full blocks (8 x 256 tokens over 16384 keys, 32 / 8 heads: 554 GFLOP in 493 us at 1.64 GHz, 1.12 PFLOP/s):
// a query tile's chain of scores, maximum, exponentials and product takes 3680 cycles per key tile, of which 2048 are the
// products of the two query tiles.
//   warps 0-7, 8-15  softmax of query tile 0 / 1: two threads per row, 64 keys each, which agree through one barrier with
//                    a vote.  Four warps per scheduler cover one another's latencies better than two with 128 keys per
//                    thread (8 x up to 250 rows of 4 heads over 16384 keys, whole calls in a long loop, at
//                    the power limit: 489 us against 517, otherwise alike).
//   warp 16          issues the MMAs and owns tensor memory.  The issuing lane is chosen by elect.sync, descriptors are
//                    made once: the operands then sit in uniform registers and an MMA takes ~20 cycles to issue; behind
//                    `lane == 0`, with descriptors made per MMA, it took 100 to 160 and bound the kernel (an MMA of
//                    128 x 128 x 16 runs 64)
//   warp 17          fetches K and V tiles by TMA, a page's rows at a time, into a ring of 32 KB slots
//   warp 18          walks ahead of the softmax warps and writes down what they work on next
//   warp 19          completes the warpgroup that gives its registers away
// Tensor memory (512 columns): S0, S1 (128 each; P overwrites the first half of its S), O0, O1.  MMAs execute in the order
// of their issue, so S of the next tile may be issued behind the product that still reads P.  The running maximum moves
// only when a row passes it by 2^8 (more in fp16: PaLift); then the row's thread rescales its accumulator in tensor memory, which nothing else
// touches at that point: the product before has completed (the commit that announced S covers it), the next one waits
// for P.  The second half of a row writes its P over scores of the first half, behind the vote, when those are read.
#pragma once

#include "paged_attn.cuh"

namespace fa {

constexpr int PT_THREADS = 640;                           // 96 registers each at launch, moved to where they are needed:
constexpr int PT_SOFTMAX_REGS = 104, PT_OTHER_REGS = 64;   // 512 x 104 + 128 x 64 = 640 x 96
// (the compiler reports 900 bytes of spill stores and 516 of loads at D = 128, 236 and 352 were the warps with 64 registers,
// each with a walk over the units, given 96)
constexpr int PT_ROWS = 256;                              // rows_log2 = 8

// a stretch of one unit's tiles, as the softmax warps need it; written ahead by a warp of its own, so that the walk and
// its loads are off their path and take none of their registers
struct PtSegment {
  int more, row0, t0, n, len, h, t, t_end, first, last;   // more = 0: done
};
constexpr int PT_SEGS = 4;

template <int D>
struct PaTile {
  static constexpr int HALF = 128 * 128;                  // 128 rows x 64 columns
  static constexpr int SLOT = (D / 64) * HALF;            // a K or V tile
  static constexpr int QBYTES = 2 * SLOT;
  static constexpr int ST = 160 * 1024 / SLOT;            // 5 slots at D = 128
  struct Small {
    uint64_t full[ST], empty[ST], q_full[2], s_full[2], p_full[2], o_full[2], tail;
    uint32_t bad[16];          // keys of a tile that no page holds, by groups of 16; the fetches are < 16 tiles ahead
    PaLocate loc;
    PtSegment seg[PT_SEGS];
    uint64_t seg_full[PT_SEGS], seg_empty[PT_SEGS];
    float half[2][2][128];     // what the two halves of a row tell each other
    uint32_t tmem;
    int dead;
  };
  static constexpr int SMEM = QBYTES + ST * SLOT + 3 * 1024;
  static_assert(sizeof(Small) <= 3 * 1024, "barriers");
};

struct PaTileParams {
  alignas(64) CUtensorMap tm_k, tm_v;
  PaCommon c;
  PaPhase p;
  int box_rows;                // rows of a TMA box: a power of two that divides the page
};

// shared-memory matrix descriptors, 128-byte swizzle: start address, leading and stride byte offsets in 16-byte units
__device__ __forceinline__ uint64_t pt_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFF) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void pt_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
__device__ __forceinline__ void pt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
// one lane of a converged warp; what it computes stays in uniform registers
__device__ __forceinline__ bool pt_elect() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void pt_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pt_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void pt_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
#define PT_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define PT_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 columns of this warp's 32 lanes; the values are there after pt_wait_ld()
__device__ __forceinline__ void pt_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : PT_R8(r, 0), PT_R8(r, 8), PT_R8(r, 16), PT_R8(r, 24) : "r"(taddr));
}
__device__ __forceinline__ void pt_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void pt_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n" ::"r"(taddr),
      PT_W8(r, 0), PT_W8(r, 8), PT_W8(r, 16), PT_W8(r, 24) : "memory");
}
__device__ __forceinline__ void pt_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      : PT_R8(r, 0), PT_R8(r, 8) : "r"(taddr));
}
__device__ __forceinline__ void pt_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n" ::"r"(taddr),
      PT_W8(r, 0), PT_W8(r, 8) : "memory");
}
// two float32 at a time
__device__ __forceinline__ uint64_t pt_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void pt_unpair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t pt_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t pt_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// barrier of the 256 threads of a query tile, and the same with a vote
__device__ __forceinline__ void pt_sync(int id) { asm volatile("bar.sync %0, 256;\n" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool pt_sync_any(int id, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbar.red.or.pred q, %1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r) : "r"(id), "r"((uint32_t)x) : "memory");
  return r != 0;
}
__device__ __forceinline__ float pt_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void pt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

template <typename T>
struct PtFormat;
template <>
struct PtFormat<__half> {
  static constexpr uint32_t F = 0;
};
template <>
struct PtFormat<__nv_bfloat16> {
  static constexpr uint32_t F = 1;
};

template <typename T, int D>
__global__ void __launch_bounds__(PT_THREADS, 1) paged_tile_kernel(const __grid_constant__ PaTileParams prm) {
  using C = PaTile<D>;
  const PaCommon& c = prm.c;
  const PaPhase& p = prm.p;
  extern __shared__ __align__(1024) unsigned char pa_dyn[];
  typename C::Small& sh = *reinterpret_cast<typename C::Small*>(pa_dyn + C::QBYTES + C::ST * C::SLOT);
  const uint32_t q_smem = pa_smem(pa_dyn), ring = q_smem + C::QBYTES;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  volatile int* dead = &sh.dead;

  if (tid == 0) {
    sh.dead = (q_smem & 1023u) ? 1 : 0;                   // the swizzle pattern goes by the address
    for (int s = 0; s < C::ST; ++s) {
      pa_bar_init(pa_smem(&sh.full[s]), 1);
      pa_bar_init(pa_smem(&sh.empty[s]), 1);
    }
    for (int w = 0; w < 2; ++w) {
      pa_bar_init(pa_smem(&sh.q_full[w]), 8);           // an arrival per warp: one per thread took as long as the exponentials
      pa_bar_init(pa_smem(&sh.s_full[w]), 1);
      pa_bar_init(pa_smem(&sh.p_full[w]), 8);
      pa_bar_init(pa_smem(&sh.o_full[w]), 1);
    }
    pa_bar_init(pa_smem(&sh.tail), 1);
    for (int s = 0; s < PT_SEGS; ++s) {
      pa_bar_init(pa_smem(&sh.seg_full[s]), 1);
      pa_bar_init(pa_smem(&sh.seg_empty[s]), 16);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(pa_smem(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  pt_before();
  pa_let_next_begin();
  PaUnit u;
  int t;
  const PaRange range = pa_locate<PT_THREADS>(c, p, blockIdx.x, sh.loc, u, t);   // two block barriers
  pt_after();
  const uint32_t tmem = sh.tmem;
  long long done = range.beg;

  if (warp < 16) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(PT_SOFTMAX_REGS));
    // ---- softmax ------------------------------------------------------------------------------------------------------
    const int w = warp >> 3, half = (warp >> 2) & 1, i = tid & 127;   // query tile, half of the keys, row
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + w * 128 + lanes, to = tmem + 256 + w * 128 + lanes;
    const uint32_t s_full = pa_smem(&sh.s_full[w]), p_full = pa_smem(&sh.p_full[w]);
    const float scale = c.scale_log2;
    constexpr float LIFT = PaLift<T>::STEPS;
    uint32_t s_par = 0, o_par = 0;
    int tile_no = 0;                                      // tiles since the start
    for (int seg_no = 0;; ++seg_no) {
      const PtSegment& seg = sh.seg[seg_no % PT_SEGS];
      pa_bar_wait(pa_smem(&sh.seg_full[seg_no % PT_SEGS]), (seg_no / PT_SEGS) & 1, dead);
      // (by vote: after a wait that gave up the threads may not see alike, and barriers follow)
      if (pt_sync_any(1 + w, *dead || !seg.more)) break;
      const int t_beg = seg.t, t_end = seg.t_end, row0 = seg.row0 + w * 128;
      const int n_rows = max(0, min(128, seg.n * c.G - row0));
      if (n_rows == 0) {
        tile_no += t_end - t_beg;
      } else {
        // the query tile, zeros behind the last row
        const uint32_t qb = q_smem + w * C::SLOT;
        {
          const T* q = reinterpret_cast<const T*>(c.q) + (int64_t)seg.t0 * c.q_st + (int64_t)seg.h * c.G * c.q_sh;
          // a thread takes a half of row i, all of it requested at once
          constexpr int NQ = D / 16;
          const int tok = (int)((unsigned)(row0 + i) / (unsigned)c.G), hg = row0 + i - tok * c.G;
          const uint4* src = reinterpret_cast<const uint4*>(q + (int64_t)tok * c.q_st + (int64_t)hg * c.q_sh) + half * NQ;
          uint4 v[NQ];
#pragma unroll
          for (int k = 0; k < NQ; ++k) v[k] = i < n_rows ? src[k] : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int k = 0; k < NQ; ++k) {
            const int ch = half * NQ + k;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(qb + (ch >> 3) * C::HALF + i * 128 + (((ch & 7) ^ (i & 7)) << 4)),
                         "r"(v[k].x), "r"(v[k].y), "r"(v[k].z), "r"(v[k].w) : "memory");
          }
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");   // generic writes -> MMA reads
        pt_before();
        __syncwarp();
        if (lane == 0) pa_bar_arrive(pa_smem(&sh.q_full[w]));

        const int lim = p.prefix_len > 0 ? seg.len : min(min(seg.len, p.cap), seg.len - seg.n + (row0 + min(i, n_rows - 1)) / c.G + 1);
        // keys of this half of the tile that the row sees, counted from the lead's or the sequence's first key
        const int lead = pa_tiles(p.lead_len);
        int tt = t_beg;
        float m = -INFINITY, l = 0.f;
#pragma unroll 1
        for (; tt < t_end; ++tt) {
          const int nv = (tt < lead ? p.lead_len - tt * PA_TILE : lim - (tt - lead) * PA_TILE) - 64 * half;
          pa_bar_wait(s_full, s_par, dead);
          s_par ^= 1;
          pt_after();
          uint32_t sr[64];
          pt_ld32(ts + 64 * half, sr);
          pt_ld32(ts + 64 * half + 32, sr + 32);
          pt_wait_ld();
          const uint32_t bad = sh.bad[tile_no++ & 15] >> (4 * half);
          if (__any_sync(0xffffffffu, nv < 64 || bad != 0)) {
#pragma unroll
            for (int j = 0; j < 64; ++j)
              if (j >= nv || ((bad >> (j / 16)) & 1)) sr[j] = 0xff800000u;
          }
          float mx[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) mx[k] = fmaxf(__uint_as_float(sr[k]), __uint_as_float(sr[4 + k]));
#pragma unroll
          for (int j = 8; j < 64; j += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k) mx[k] = pt_max3(mx[k], __uint_as_float(sr[j + k]), __uint_as_float(sr[j + 4 + k]));
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
          if (pt_sync_any(1 + w, top > m + (8.f + LIFT))) {
            sh.half[w][half][i] = top;
            pt_sync(1 + w);
            const float nm = fmaxf(m, fmaxf(top, sh.half[w][half ^ 1][i]) - LIFT);
            const float f = m == -INFINITY ? 0.f : pa_ex2(m - nm);
            m = nm;
            l *= f;
            if (tt > t_beg) {
#pragma unroll 1
              for (int j = half * (D / 2); j < (half + 1) * (D / 2); j += 16) {
                uint32_t o[16];
                pt_ld16(to + j, o);
                pt_wait_ld();
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                pt_st16(to + j, o);
              }
            }
            pt_sync(1 + w);                               // sh.half has been read
          }
          const float off = m == -INFINITY ? 0.f : -m;
          const uint64_t sc2 = pt_pair(scale, scale), off2 = pt_pair(off, off);
          uint64_t sum[2] = {0, 0};
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            float a, b;
            pt_unpair(pt_fma2(pt_pair(__uint_as_float(sr[2 * j]), __uint_as_float(sr[2 * j + 1])), sc2, off2), a, b);
            a = pa_ex2(a), b = pa_ex2(b);
            sum[j & 1] = pt_add2(sum[j & 1], pt_pair(a, b));
            sr[j] = pa_pack<T>(a, b);
          }
          pt_st32(ts + 32 * half, sr);
          {
            float a, b;
            pt_unpair(pt_add2(sum[0], sum[1]), a, b);
            l += a + b;
          }
          pt_wait_st();
          pt_before();
          __syncwarp();
          if (lane == 0) pa_bar_arrive(p_full);
        }
        // ---- this segment's result ------------------------------------------------------------------------------------
        pa_bar_wait(pa_smem(&sh.o_full[w]), o_par, dead);
        o_par ^= 1;
        pt_after();
        const bool whole = seg.first && seg.last;
        sh.half[w][half][i] = l;
        pt_sync(1 + w);
        l += sh.half[w][half ^ 1][i];
        if (*dead) l = __int_as_float(0x7fc00000);
        const int r = row0 + i;
        const int tok = seg.t0 + r / c.G, hq = seg.h * c.G + r % c.G;
        const int64_t at = whole ? (int64_t)tok * c.Hq + hq : (int64_t)(2 * blockIdx.x + (seg.first ? 1 : 0)) * PT_ROWS + w * 128 + i;
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int j = half * (D / 2); j < (half + 1) * (D / 2); j += 32) {
          uint32_t o[32];
          pt_ld32(to + j, o);
          pt_wait_ld();
          if (i >= n_rows) continue;
          if (whole && p.direct) {
            uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(c.out) + (int64_t)tok * c.o_st + (int64_t)hq * c.o_sh + j);
            uint32_t v[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = pa_pack<T>(__uint_as_float(o[2 * k]) * inv, __uint_as_float(o[2 * k + 1]) * inv);
#pragma unroll
            for (int k = 0; k < 4; ++k) dst[k] = make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
          } else {
            float* dst = (whole ? p.row_o : p.slot_o) + at * D + j;      // a whole 32-byte sector per lane and store
#pragma unroll
            for (int k = 0; k < 32; k += 8)
              asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(dst + k), PT_W8(o, k) : "memory");
          }
        }
        if (i < n_rows && half == 0) {
          if (whole && p.direct) {
            if (c.lse) c.lse[(int64_t)tok * c.Hq + hq] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
          } else {
            (whole ? p.row_ml : p.slot_ml)[at] = make_float2(m, l);
          }
        }
        pt_before();
      }
      __syncwarp();
      if (lane == 0) pa_bar_arrive(pa_smem(&sh.seg_empty[seg_no % PT_SEGS]));   // read
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(PT_OTHER_REGS));
  }
  if (warp == 16) {
    // ---- the MMAs -----------------------------------------------------------------------------------------------------
    constexpr uint32_t F = PtFormat<T>::F;
    constexpr uint32_t id_qk = (1u << 4) | (F << 7) | (F << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
    constexpr uint32_t id_pv = (1u << 4) | (F << 7) | (F << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
    const uint64_t q_desc = pt_desc(q_smem, 16, 1024), k_desc = pt_desc(ring, 16, 1024), v_desc = pt_desc(ring, C::HALF, 1024);
    int slot = 0;
    uint32_t par = 0, q_par = 0, p_par = 0;               // q_par, p_par: a bit per query tile
    const int lead = pa_tiles(p.lead_len);
    auto advance = [&]() {
      if (++slot == C::ST) slot = 0, par ^= 1;
    };
    auto scores = [&](int w, int k_slot) {
      if (pt_elect()) {
        const uint64_t qd = q_desc + w * (C::SLOT >> 4), kd = k_desc + k_slot * (C::SLOT >> 4);
        const uint32_t s_tm = tmem + w * 128;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t o = ((kk >> 2) * C::HALF + (kk & 3) * 32) >> 4;
          pt_mma_ss(s_tm, qd + o, kd + o, id_qk, kk > 0);
        }
        pt_commit(pa_smem(&sh.s_full[w]));
      }
      __syncwarp();
    };
    while (done < range.end) {
      if (t >= u.tiles) {
        u.next(c, p);
        t = 0;
        continue;
      }
      const int t_end = (int)min((long long)u.tiles, t + (range.end - done));
      const int nw = u.s.n * c.G - u.rb * PT_ROWS > 128 ? 2 : 1;
      // K of the first tile
      pa_bar_wait(pa_smem(&sh.full[slot]), par, dead);
      for (int w = 0; w < nw; ++w) {
        pa_bar_wait(pa_smem(&sh.q_full[w]), (q_par >> w) & 1, dead);
        q_par ^= 1u << w;
        pt_after();
        scores(w, slot);
      }
      if (pt_elect()) pt_commit(pa_smem(&sh.empty[slot]));
      __syncwarp();
      advance();
      for (int tt = t; tt < t_end; ++tt) {
        const bool more = tt + 1 < t_end;
        const int steps = (min(PA_TILE, tt < lead ? p.lead_len - tt * PA_TILE : u.limit - (tt - lead) * PA_TILE) + 15) / 16;
        const int v_slot = slot;
        pa_bar_wait(pa_smem(&sh.full[slot]), par, dead);
        advance();
        const int k_slot = slot;
        const uint32_t k_par = par;
        if (more) advance();
        for (int w = 0; w < nw; ++w) {
          pa_bar_wait(pa_smem(&sh.p_full[w]), (p_par >> w) & 1, dead);
          p_par ^= 1u << w;
          pt_after();
          if (pt_elect()) {
            const uint64_t vd = v_desc + v_slot * (C::SLOT >> 4);
            const uint32_t p_tm = tmem + w * 128, o_tm = tmem + 256 + w * 128;
            if (steps == PA_TILE / 16) {
#pragma unroll
              for (int kk = 0; kk < PA_TILE / 16; ++kk)
                pt_mma_ts(o_tm, p_tm + kk * 8, vd + kk * (2048 >> 4), id_pv, kk > 0 || tt > t);
            } else {
              for (int kk = 0; kk < steps; ++kk)
                pt_mma_ts(o_tm, p_tm + kk * 8, vd + kk * (2048 >> 4), id_pv, kk > 0 || tt > t);
            }
            if (!more) pt_commit(pa_smem(&sh.o_full[w]));
          }
          __syncwarp();
          if (more) {
            if (w == 0) pa_bar_wait(pa_smem(&sh.full[k_slot]), k_par, dead);
            scores(w, k_slot);
          }
        }
        if (pt_elect()) {
          pt_commit(pa_smem(&sh.empty[v_slot]));
          if (more) pt_commit(pa_smem(&sh.empty[k_slot]));
        }
        __syncwarp();
      }
      done += t_end - t;
      t = t_end;
    }
  } else if (warp == 17) {
    // ---- the fetches --------------------------------------------------------------------------------------------------
    int slot = 0, tile_no = 0;
    uint32_t par = 1, t_par = 0;                          // the first pass over the ring finds it empty
    const int box_keys = prm.box_rows, lead = pa_tiles(p.lead_len);
    const uint32_t box_bytes = box_keys * 128;
    // lane i holds the page id of box i of the tile to come, requested while the tile before is fetched
    auto page_id = [&]() -> int {
      const int key = (t < lead ? t : t - lead) * PA_TILE + lane * box_keys;
      if (lane * box_keys >= PA_TILE || key >= (t < lead ? p.lead_len : u.limit)) return 0;
      return (t < lead ? p.lead_table : p.table + (int64_t)u.b * p.table_sb)[key / c.page_size];
    };
    auto to_tile = [&]() {
      while (done < range.end && t >= u.tiles) u.next(c, p), t = 0;
    };
    to_tile();
    int next_id = done < range.end ? page_id() : 0;
    while (done < range.end) {
      const int key0 = (t < lead ? t : t - lead) * PA_TILE, nv = min(PA_TILE, (t < lead ? p.lead_len : u.limit) - key0);
      const int need = (nv + box_keys - 1) / box_keys;                // boxes with keys
      const int row = (key0 + lane * box_keys) % c.page_size, head = u.h, L = t < lead ? p.lead_len : pa_keys(p, u.s);
      int page = next_id;
      const bool ok = lane >= need || (page >= 0 && page < c.num_pages);
      if (!ok) page = c.num_pages;                        // out of the map's range: zeros arrive
      // groups of 16 keys whose page id names no page
      const uint32_t miss = __ballot_sync(0xffffffffu, !ok);
      uint32_t bad = 0;
      if (miss != 0)
        for (int g = 0; g < PA_TILE / 16; ++g) bad |= ((miss >> (g * 16 / box_keys)) & 1u) << g;
      const bool tail = key0 + PA_TILE > L && (L & 15);               // keys and leftovers in one group of 16
      ++done, ++t;
      to_tile();
      if (done < range.end) next_id = page_id();
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint32_t dst = ring + slot * C::SLOT, full = pa_smem(&sh.full[slot]);
        const uint32_t bar = kv == 1 && tail ? pa_smem(&sh.tail) : full;
        pa_bar_wait(pa_smem(&sh.empty[slot]), par, dead);
        if (lane == 0) {
          if (kv == 0) sh.bad[tile_no & 15] = bad;
          pa_bar_expect(bar, (uint32_t)need * box_bytes * (D / 64));
        }
        __syncwarp();
        if (lane < need)
          for (int hf = 0; hf < D / 64; ++hf)
            pa_tma(dst + hf * C::HALF + lane * box_bytes, kv == 0 ? &prm.tm_k : &prm.tm_v, 64 * hf, row, head, page, bar);
        if (kv == 1 && tail) {
          // rows behind the sequence hold anything, and 0 x NaN must not reach the sums: zeros up to the end of the
          // group of 16 (the product stops there)
          pa_bar_wait(bar, t_par, dead);
          t_par ^= 1;
          const int r0 = L - key0, r1 = (r0 + 15) & ~15;
          for (int e = lane; e < (r1 - r0) * (D / 8); e += 32) {
            const int r = r0 + e / (D / 8), ch = e % (D / 8);
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(dst + (ch >> 3) * C::HALF + r * 128 + ((ch & 7) << 4)), "r"(0) : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
          __syncwarp();
          if (lane == 0) pa_bar_arrive(full);
        }
        if (++slot == C::ST) slot = 0, par ^= 1;
      }
      ++tile_no;
    }
  }
  if (warp == 18 && lane == 0) {
    // ---- what the softmax warps work on --------------------------------------------------------------------------------
    for (int seg_no = 0;; ++seg_no) {
      const int x = seg_no % PT_SEGS;
      if (seg_no >= PT_SEGS) pa_bar_wait(pa_smem(&sh.seg_empty[x]), (seg_no / PT_SEGS - 1) & 1, dead);
      PtSegment seg;
      seg.more = done < range.end && !*dead;
      if (seg.more) {
        while (t >= u.tiles) u.next(c, p), t = 0;
        seg.t = t;
        seg.t_end = (int)min((long long)u.tiles, t + (range.end - done));
        seg.row0 = u.rb * PT_ROWS;
        seg.t0 = u.s.t0, seg.n = u.s.n, seg.len = u.s.len, seg.h = u.h;
        seg.first = seg.t == 0, seg.last = seg.t_end == u.tiles;
      }
      sh.seg[x] = seg;
      pa_bar_arrive(pa_smem(&sh.seg_full[x]));
      if (!seg.more) break;
      if (seg.last) p.info[pa_unit_id(c, p, u.b, u.s, u.h, u.rb)] = make_int2(pa_owner(range, done - t), blockIdx.x);
      done += seg.t_end - seg.t;
      t = seg.t_end;
    }
  }
  pa_leave(dead);
  pt_before();
  __syncthreads();
  if (warp == 16) {
    pt_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
  }
  pa_wait_for_previous();
}

}  // namespace fa
