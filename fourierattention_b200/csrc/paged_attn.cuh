// Shared parts of the paged attention kernels: the work split, the record of partial results, small PTX helpers.
//
// Work is counted in tiles of 128 keys.  A unit is one KV head and one block of query rows (a row is a new token and
// one of the query heads of the group) that read the same keys: rows of one sequence and its pages, or, over the
// shared prefix, rows of the whole batch.  The tiles of all units, laid end to end, are cut into equal ranges, one per
// CTA, so ragged lengths load every SM alike and nothing is planned on the host: lengths are read from device memory,
// a captured launch follows them.  A unit inside one range is finished there; one that is cut leaves partial results
// (unnormalised output, running maximum, denominator) in slots, two per CTA, that the merge kernel joins in order.
#pragma once

#include "serving.cuh"

namespace fa {

constexpr int PA_TILE = 128;

struct PaPhase {
  const int32_t* table;      // (B, max_pages), or the prefix's pages
  int64_t table_sb;
  int cap;                   // keys that the table has room for
  int prefix_len;            // > 0: the shared prefix, every row sees all of it; 0: each sequence's own pages, causal
  const int32_t* lead_table; // own pages only: the pages of `lead_len` keys that come before them (tile kernel)
  int lead_len;
  int rows_log2;             // rows of a block
  int ctas;
  int direct;                // finished units go straight to `out`
  float* slot_o;             // (2 ctas, rows, D)
  float2* slot_ml;           // (2 ctas, rows)
  float* row_o;              // (tokens, Hq, D): finished units, when `direct` is 0
  float2* row_ml;
  int2* info;                // first and last CTA of every unit that has tiles
};

struct PaCommon {
  const void* q;
  int64_t q_st, q_sh;
  void* out;
  int64_t o_st, o_sh;
  float* lse;
  const int32_t *kv_lens, *cu;
  int tokens, B, Hq, Hkv, G;
  int page_size, num_pages;
  float scale_log2;          // softmax scale x log2(e): scores live in the log2 domain
};

struct PaSeq {
  int t0, n, len;            // first new token, number of new tokens, length (which the table may not hold)
};

__device__ __forceinline__ PaSeq pa_seq(const PaCommon& c, const PaPhase& p, int b) {
  PaSeq s;
  if (p.prefix_len > 0) {
    s.t0 = 0;
    s.n = c.cu ? max(0, min(c.tokens, c.cu[c.B])) : c.tokens;
    s.len = p.prefix_len;
    return s;
  }
  int t0 = b, t1 = b + 1;
  if (c.cu) t0 = c.cu[b], t1 = c.cu[b + 1];
  s.t0 = max(0, min(t0, c.tokens));
  s.n = max(0, min(t1, c.tokens) - s.t0);
  s.len = max(0, c.kv_lens[b]);
  return s;
}
// keys that exist: those behind the table do not, but a token's place counts from the length as it is
__device__ __forceinline__ int pa_keys(const PaPhase& p, const PaSeq& s) { return min(s.len, p.cap); }
__device__ __forceinline__ int pa_seqs(const PaCommon& c, const PaPhase& p) { return p.prefix_len > 0 ? 1 : c.B; }
__device__ __forceinline__ int pa_blocks(const PaCommon& c, const PaPhase& p, const PaSeq& s) {
  return (s.n * c.G + (1 << p.rows_log2) - 1) >> p.rows_log2;      // (tokens x G and a block more fit into 31 bits)
}
// keys seen by the last row of a block (a later token sees more)
__device__ __forceinline__ int pa_limit(const PaCommon& c, const PaPhase& p, const PaSeq& s, int rb) {
  if (p.prefix_len > 0) return s.len;
  const int last = min(s.n * c.G, (rb + 1) << p.rows_log2) - 1;
  return max(0, min(pa_keys(p, s), s.len - s.n + (int)((unsigned)last / (unsigned)c.G) + 1));
}
__device__ __forceinline__ int pa_tiles(int limit) { return (limit + PA_TILE - 1) / PA_TILE; }
// tiles of a unit whose rows see `limit` keys; those of the lead come first, in tiles of their own
__device__ __forceinline__ int pa_unit_tiles(const PaPhase& p, int limit) { return pa_tiles(p.lead_len) + pa_tiles(limit); }
__device__ __forceinline__ long long pa_head_tiles(const PaCommon& c, const PaPhase& p, const PaSeq& s) {
  const int nb = pa_blocks(c, p, s);
  if (nb == 0) return 0;
  if (p.prefix_len > 0) return (long long)nb * pa_tiles(s.len);
  long long sum = 0;
  for (int rb = 0; rb < nb; ++rb) sum += pa_unit_tiles(p, pa_limit(c, p, s, rb));
  return sum;
}
// number of a unit for `info`: distinct, and below pa_info_count()
__device__ __forceinline__ long long pa_unit_id(const PaCommon& c, const PaPhase& p, int b, const PaSeq& s, int h, int rb) {
  const int f0 = ((s.t0 * c.G) >> p.rows_log2) + b, f1 = (((s.t0 + s.n) * c.G) >> p.rows_log2) + b + 1;
  return (long long)f0 * c.Hkv + h * (f1 - f0) + rb;
}
inline int64_t pa_info_count(int64_t tokens, int64_t B, int64_t G, int64_t Hkv, int64_t rows) {
  return (tokens * G / rows + B + 1) * Hkv;
}

// A unit and the walk over units in the order of their tiles.
struct PaUnit {
  int b, h, rb, nb, limit, tiles;
  PaSeq s;
  __device__ __forceinline__ void set(const PaCommon& c, const PaPhase& p) {
    limit = pa_limit(c, p, s, rb);
    tiles = pa_unit_tiles(p, limit);
  }
  __device__ __forceinline__ void next(const PaCommon& c, const PaPhase& p) {
    if (++rb >= nb) {
      rb = 0;
      if (++h >= c.Hkv) {
        h = 0;
        const int B = pa_seqs(c, p);
        nb = 0;
        while (nb == 0 && ++b < B) {
          s = pa_seq(c, p, b);
          nb = pa_blocks(c, p, s);
        }
        if (nb == 0) {
          tiles = 0;
          return;
        }
      }
    }
    set(c, p);
  }
};

struct PaRange {
  long long total, beg, end;   // tiles of all units; this CTA's
  int ctas;                    // CTAs that have one: no more than there are tiles
};

struct PaLocate {              // shared memory of pa_locate()
  long long sum[32], off;
  int b;
};

// a / b, b > 0: by the short division where both fit 32 bits
__device__ __forceinline__ long long pa_div(long long a, long long b) {
  return ((unsigned long long)a >> 32) == 0 && ((unsigned long long)b >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}

// Finds this CTA's range of tiles and the unit it begins in (tile `t` of it).  One block-wide scan over the sequences.
template <int THREADS>
__device__ __forceinline__ PaRange pa_locate(const PaCommon& c, const PaPhase& p, int cta, PaLocate& sh, PaUnit& u, int& t) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int B = pa_seqs(c, p);
  const int chunk = (B + THREADS - 1) / THREADS;
  const int b0 = min(B, tid * chunk), b1 = min(B, b0 + chunk);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += pa_head_tiles(c, p, pa_seq(c, p, b)) * c.Hkv;
  long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) sh.sum[warp] = inc;
  __syncthreads();
  PaRange r;
  r.total = 0;
  long long pre = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) pre += sh.sum[w];
    r.total += sh.sum[w];
  }
  pre += inc - mine;
  r.ctas = (int)min((long long)p.ctas, r.total);
  r.beg = r.end = 0;
  if (cta < r.ctas) r.beg = pa_div(r.total * cta, r.ctas), r.end = pa_div(r.total * (cta + 1), r.ctas);
  if (r.beg < r.end && pre <= r.beg && r.beg < pre + mine) {
    long long off = r.beg - pre;
    int b = b0;
    for (; b < b1; ++b) {
      const long long n = pa_head_tiles(c, p, pa_seq(c, p, b)) * c.Hkv;
      if (off < n) break;
      off -= n;
    }
    sh.b = b, sh.off = off;
  }
  __syncthreads();
  if (r.beg >= r.end) return r;
  u.b = sh.b;
  u.s = pa_seq(c, p, u.b);
  u.nb = pa_blocks(c, p, u.s);
  const long long per = pa_head_tiles(c, p, u.s);
  u.h = (int)pa_div(sh.off, per);
  long long off = sh.off - u.h * per;
  u.rb = 0;
  u.set(c, p);
  while (off >= u.tiles) {
    off -= u.tiles;
    ++u.rb;
    u.set(c, p);
  }
  t = (int)off;
  return r;
}
__device__ __forceinline__ int pa_owner(const PaRange& r, long long tile) {
  return (int)pa_div((tile + 1) * r.ctas - 1, r.total);
}

// ---- the launches of one call ----------------------------------------------------------------------------------------
// The kernel over the prefix, the one over the sequences' own keys and the merge are launched so that each may begin
// while the one before drains (programmatic stream serialization).  The first two share nothing but the output of
// earlier launches; the second waits for the first before it ends, so that the merge, which waits for the second,
// finds both results complete.
__device__ __forceinline__ void pa_let_next_begin() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
__device__ __forceinline__ void pa_wait_for_previous() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

// ---- PTX -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t pa_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void pa_bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void pa_bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pa_bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool pa_bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// A bounded wait (about a second).  One that gives up sets `dead`, every later wait of the CTA returns at once, and
// the CTA's results become NaN.
__device__ __forceinline__ void pa_bar_wait(uint32_t bar, uint32_t parity, volatile int* dead) {
  if (pa_bar_try(bar, parity)) return;
  const long long t0 = clock64();
  while (!pa_bar_try(bar, parity)) {
    if (*dead || clock64() - t0 > 2000000000LL) {
      *dead = 1;
      return;
    }
  }
}
// After a wait that gave up: time for what is still in flight, before shared memory is given back.
__device__ __forceinline__ void pa_leave(volatile int* dead) {
  if (!*dead) return;
  const long long t0 = clock64();
  while (clock64() - t0 < 20000000LL) __nanosleep(1000);
}
__device__ __forceinline__ void pa_tma(uint32_t dst, const CUtensorMap* map, int x, int row, int head, int page,
                                       uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(
          dst), "l"(map), "r"(x), "r"(row), "r"(head), "r"(page), "r"(bar) : "memory");
}
__device__ __forceinline__ float pa_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// Probabilities are 2^(s - m) with m the running maximum less this many steps.  In fp16 a probability 2^-14 below the
// largest would lose bits and one 2^-25 below it vanish, and many keys that far behind a dominant one (a first token that
// draws the attention to itself) add up to what counts; seven steps higher, the largest still fit (2^15: the maximum may
// lag by 2^8) and bits are lost from 2^-21 on.  bf16 has float32's range.
template <typename T>
struct PaLift {
  static constexpr float STEPS = 0.f;
};
template <>
struct PaLift<__half> {
  static constexpr float STEPS = 7.f;
};
template <typename T>
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pa_pack<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pa_pack<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

}  // namespace fa
