// Drawing one token per row of logits (fa_sample): temperature, top-k, top-p, min-p, and a given uniform number.
//
// With M the row's largest logit, w_i = exp((x_i - M) / temperature) and the order "larger logit first, lower index
// first among equals", every filter keeps a head of that order:
//   top-k: the first k;  top-p: the shortest head of those with sum >= p * (sum of the top-k head);  min-p: w_i >= min_p.
// The token is the first index i (ascending) whose running sum of kept weights exceeds u * (their sum).
//
// Nothing is sorted as a whole.  A head of the order is {x > t} plus the ties at t up to an index, so each of top-k and
// top-p is a search for one element.
//   Small top-k (up to LIST): the k-th largest of the threads' own maxima is no larger than the k-th largest logit, so
//   a histogram of those (one atomic per thread) gives a border above which all k are; what is above it, a little more
//   than k, is listed and ranked by one CTA, which then cuts the list by top-p and min-p and draws from it.
//   Else: a histogram of (largest - x) over 1024 equal bins finds the bin the element is in, the bin's elements (up to
//   LIST of them) are ranked against one another, and a fuller bin is split again, down to bins of one value whose ties
//   are counted in the order of their indices.
// Whether a token is in hangs on sums next to a border, and one token too many or too few changes the draw, so every
// weight and sum that decides is taken in float64, in a fixed order; the histogram of top-p (integers: the same whatever
// the order of the atomics) only proposes a bin, which the float64 sums then confirm or move.
//
// Layout: a cluster of 1 to 8 CTAs holds a row in shared memory (float32, read from HBM once; a thread owns up
// to 32 neighbouring elements, read four at a time, its groups of four turned by its number so that a walk meets no bank
// twice) and exchanges partial
// results through distributed shared memory: every CTA reads all of them and decides alike, one cluster barrier per
// step.  Bound: the latency of those steps (a cluster barrier is ~1500 cycles, a pass over the CTA's elements 4 to 12
// thousand).  Measured: one row of 128256 27 us, 256 float32 rows 215 us (the rows' bytes alone: 20 us).  Everything is inlined:
// with the state behind a pointer it lived in local memory, and a row took 34 us.
#include <cooperative_groups.h>

#include "sample_exp.cuh"
#include "serving.cuh"

namespace cg = cooperative_groups;

namespace fa {

constexpr int SA_THREADS = 512;
constexpr int SA_WARPS = SA_THREADS / 32;
constexpr int SA_EPT = 32;                         // most neighbouring elements of a thread, per round
constexpr int SA_ROUND = SA_THREADS * SA_EPT;      // elements of a CTA, per round
constexpr int SA_MAX_ROUNDS = 3;
constexpr int SA_MAX_CLUSTER = 8;
constexpr int SA_BINS = 1024;
constexpr int SA_LIST = 512;
constexpr int SA_MAX_VOCAB = SA_MAX_CLUSTER * SA_MAX_ROUNDS * SA_ROUND;
constexpr int SA_STEPS = 8192;                     // of the largest weight in a bin; a bin of all elements fits 32 bits
static_assert((unsigned long long)SA_MAX_VOCAB * SA_STEPS < 1ull << 32, "the bins of a histogram");

struct SampleParams {
  const void* logits;
  int64_t sb;
  int V, slice, ept_log2, rounds; // elements of a CTA, of a thread per round; rounds of 512 threads
  const float *u, *temperature, *top_p, *min_p;    // per row, or null: the value below
  const int32_t* top_k;
  float temperature0, top_p0, min_p0;
  int top_k0;
  int64_t* token;
  float* logprob;
};

struct SaXchg {
  double s[2];
  float f[2];
  int n[2];
};

struct SaShared {
  double exp2[SA_EXP_TABLE];
  uint32_t hist[SA_BINS];
  SaXchg x[2];
  float lx[SA_LIST];          // this CTA's part of a bin
  int li[SA_LIST];
  unsigned ln;
  unsigned long long key[SA_LIST];   // the bin of the whole cluster
  double gw[SA_LIST];
  double red_d[2][SA_WARPS];
  float red_f[2][SA_WARPS];
  int red_n[2][SA_WARPS];
  int pick;
  double pick_d;
  int pick_i;
};

__device__ __forceinline__ double shfl_up_d(double v, int o) { return __shfl_up_sync(0xffffffffu, v, o); }
// The bin of a distance from the largest logit: the nearest multiple of 1 / scale, by adding 2^23 (a conversion to an
// integer takes the slow pipe, which the exponentials need).  Monotone in d; 0 for d = 0 even where scale is infinite.
__device__ __forceinline__ int sa_bin(float d, float scale) {
  const float t = d > 0.f ? d * scale : 0.f;
  return min(SA_BINS - 1, __float_as_int(t + 8388608.f) - 0x4b000000);
}
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__device__ __forceinline__ float sa_value(T v) {
  const float f = to_f32(v);
  return f != f ? -INFINITY : f + 0.f;       // NaN: never drawn; the two zeros are equal
}
template <>
__device__ __forceinline__ float sa_value<float>(float f) {
  return f != f ? -INFINITY : f + 0.f;
}

template <typename T>
struct Sampler {
  const SampleParams& p;
  SaShared& sh;
  float* xs;
  cg::cluster_group cl;
  int rank, size, n, base, xb;         // CTA of the cluster; elements held, index of the first
  int tid, lane, warp;
  float M;
  double inv_t;
  // the head kept so far: x > kx, or x == kx and index <= ki
  float kx;
  int ki;
  bool left = false;                   // no CTA reads another's shared memory any more

  // element i of the CTA is element i mod ept of a thread; position of its group of four
  __device__ __forceinline__ int group_at(int t, int c) const {
    const int groups = 1 << (p.ept_log2 - 2);
    return t * groups + ((c + t) & (groups - 1));
  }
  __device__ __forceinline__ float& at(int i) {
    const int t = i >> p.ept_log2, e = i & ((1 << p.ept_log2) - 1);
    return xs[4 * group_at(t, e >> 2) + (e & 3)];
  }
  __device__ __forceinline__ float4 four(int t, int c) const { return reinterpret_cast<const float4*>(xs)[group_at(t, c)]; }
  __device__ __forceinline__ double weight(float x) const { return sa_exp(((double)x - (double)M) * inv_t, sh.exp2); }
  __device__ __forceinline__ bool kept(float x, int i) const { return x > kx || (x == kx && i <= ki); }

  // f(logit, index) for this thread's elements, in the order of the indices within a round; those that only fill up the
  // thread's share are -infinity
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    for (int r = 0; r < p.rounds; ++r) {
      const int t = r * SA_THREADS + tid;
      for (int c = 0; c < 1 << (p.ept_log2 - 2); ++c) {
        const float4 v = four(t, c);
        const int i = base + (t << p.ept_log2) + 4 * c;
        f(v.x, i), f(v.y, i + 1), f(v.z, i + 2), f(v.w, i + 3);
      }
    }
  }
  // f(logit, index, weight) for the elements that `want` takes: first which they are, then their weights, two at a time,
  // so that a warp computes as many as its busiest lane has, not one for every element that some lane has
  // (MANY: where most may be wanted).
  template <bool MANY, typename P, typename F>
  __device__ __forceinline__ void each_weight(P want, F f) {
    for (int r = 0; r < p.rounds; ++r) {
      const int t = r * SA_THREADS + tid, i0 = t << p.ept_log2;
      unsigned mask = 0;
      for (int c = 0; c < 1 << (p.ept_log2 - 2); ++c) {
        const float4 v = four(t, c);
        const int i = base + i0 + 4 * c;
        mask |= ((unsigned)want(v.x, i) | (unsigned)want(v.y, i + 1) << 1 | (unsigned)want(v.z, i + 2) << 2 |
                 (unsigned)want(v.w, i + 3) << 3) << (4 * c);
      }
      if (MANY && __reduce_add_sync(0xffffffffu, __popc(mask)) > 16 << p.ept_log2) {
        // more than half of the warp's elements: all weights, four at a time
        for (int c = 0; c < 1 << (p.ept_log2 - 2); ++c) {
          const float4 v = four(t, c);
          const int i = i0 + 4 * c;
          const double w0 = weight(v.x), w1 = weight(v.y), w2 = weight(v.z), w3 = weight(v.w);
          if ((mask >> (4 * c)) & 1) f(v.x, base + i, w0);
          if ((mask >> (4 * c)) & 2) f(v.y, base + i + 1, w1);
          if ((mask >> (4 * c)) & 4) f(v.z, base + i + 2, w2);
          if ((mask >> (4 * c)) & 8) f(v.w, base + i + 3, w3);
        }
        continue;
      }
      while (mask) {
        const int a = __ffs(mask) - 1;
        mask &= mask - 1;
        const int b = mask ? __ffs(mask) - 1 : -1;
        mask &= mask - 1;
        const float xa = at(i0 + a), xb = b >= 0 ? at(i0 + b) : xa;
        const double wa = weight(xa), wb = weight(xb);
        f(xa, base + i0 + a, wa);
        if (b >= 0) f(xb, base + i0 + b, wb);
      }
    }
  }

  // Sums over the cluster, in a fixed order: lanes, warps, CTAs.  Every CTA returns the same.
  __device__ __forceinline__ void exchange(double s0, double s1, float mn, float mx, int n0, int n1, SaXchg& out) {
    s0 = warp_sum_d(s0), s1 = warp_sum_d(s1);
    mn = -warp_max(-mn), mx = warp_max(mx);
    n0 = __reduce_add_sync(0xffffffffu, n0), n1 = __reduce_add_sync(0xffffffffu, n1);
    __syncthreads();
    if (lane == 0) {
      sh.red_d[0][warp] = s0, sh.red_d[1][warp] = s1;
      sh.red_f[0][warp] = mn, sh.red_f[1][warp] = mx;
      sh.red_n[0][warp] = n0, sh.red_n[1][warp] = n1;
    }
    __syncthreads();
    if (warp == 0) {
      const bool on = lane < SA_WARPS;
      s0 = warp_sum_d(on ? sh.red_d[0][lane] : 0.0), s1 = warp_sum_d(on ? sh.red_d[1][lane] : 0.0);
      mn = -warp_max(on ? -sh.red_f[0][lane] : -INFINITY), mx = warp_max(on ? sh.red_f[1][lane] : -INFINITY);
      n0 = __reduce_add_sync(0xffffffffu, on ? sh.red_n[0][lane] : 0);
      n1 = __reduce_add_sync(0xffffffffu, on ? sh.red_n[1][lane] : 0);
      if (lane == 0) sh.x[xb] = SaXchg{{s0, s1}, {mn, mx}, {n0, n1}};
    }
    cl.sync();
    // a lane per CTA
    out = SaXchg{{0.0, 0.0}, {INFINITY, -INFINITY}, {0, 0}};
    if (lane < size) out = *cl.map_shared_rank(&sh.x[xb], lane);
#pragma unroll
    for (int o = SA_MAX_CLUSTER / 2; o > 0; o >>= 1) {
      out.s[0] += __shfl_xor_sync(0xffffffffu, out.s[0], o), out.s[1] += __shfl_xor_sync(0xffffffffu, out.s[1], o);
      out.f[0] = fminf(out.f[0], __shfl_xor_sync(0xffffffffu, out.f[0], o));
      out.f[1] = fmaxf(out.f[1], __shfl_xor_sync(0xffffffffu, out.f[1], o));
      out.n[0] += __shfl_xor_sync(0xffffffffu, out.n[0], o), out.n[1] += __shfl_xor_sync(0xffffffffu, out.n[1], o);
    }
    out.s[0] = __shfl_sync(0xffffffffu, out.s[0], 0), out.s[1] = __shfl_sync(0xffffffffu, out.s[1], 0);
    out.f[0] = __shfl_sync(0xffffffffu, out.f[0], 0), out.f[1] = __shfl_sync(0xffffffffu, out.f[1], 0);
    out.n[0] = __shfl_sync(0xffffffffu, out.n[0], 0), out.n[1] = __shfl_sync(0xffffffffu, out.n[1], 0);
    xb ^= 1;
  }
  // this thread's two bins of the histogram, over the cluster (in 32 bits: SA_STEPS)
  __device__ __forceinline__ void read_bins(unsigned& a, unsigned& b) {
    uint2 h[SA_MAX_CLUSTER];
#pragma unroll
    for (int r = 0; r < SA_MAX_CLUSTER; ++r) {
      h[r] = make_uint2(0, 0);
      if (r < size) h[r] = *reinterpret_cast<const uint2*>(cl.map_shared_rank(&sh.hist[2 * tid], r));
    }
    a = b = 0;
#pragma unroll
    for (int r = 0; r < SA_MAX_CLUSTER; ++r) a += h[r].x, b += h[r].y;
  }

  // index of the m-th (from 0) element equal to x in the order of the indices
  __device__ __forceinline__ int nth_tie(float x, int m) {
    int mine = 0;
    each([&](float v, int i) { mine += kept(v, i) && v == x; });
    if (p.rounds == 1) {
      // counts by thread are in the order of the indices
      int inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      return tie_locate(x, m, inc - mine, mine, 0, __shfl_sync(0xffffffffu, inc, 31));
    }
    return tie_rounds(x, m);
  }
  __device__ __forceinline__ int tie_locate(float x, int m, int excl, int mine, int round, int wtotal) {
    __syncthreads();
    if (lane == 31) sh.red_n[0][warp] = wtotal;
    if (tid == 0) sh.pick_i = -1;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < SA_WARPS; ++w) {
      if (w < warp) before += sh.red_n[0][w];
      all += sh.red_n[0][w];
    }
    if (tid == 0) sh.x[xb].n[0] = all;
    cl.sync();
    int pre = 0;
    for (int r = 0; r < rank; ++r) pre += cl.map_shared_rank(&sh.x[xb], r)->n[0];
    int k = m - pre - before - excl;
    if (k >= 0 && k < mine) {
      const int i0 = (round * SA_THREADS + tid) << p.ept_log2, i1 = i0 + (1 << p.ept_log2);
      for (int i = i0; i < i1; ++i)
        if (kept(at(i), base + i) && at(i) == x && k-- == 0) sh.pick_i = base + i;
    }
    xb ^= 1;
    __syncthreads();
    return share_pick();
  }
  // the index found by one thread of the cluster, to all
  __device__ __forceinline__ int share_pick() {
    if (tid == 0) sh.x[xb].n[0] = sh.pick_i;
    cl.sync();
    int found = -1;
    for (int r = 0; r < size; ++r) found = max(found, cl.map_shared_rank(&sh.x[xb], r)->n[0]);
    xb ^= 1;
    return found;
  }
  // several rounds: CTAs hold whole ranges of indices, so the CTA first, then its rounds one by one
  __device__ __forceinline__ int tie_rounds(float x, int m) {
    int mine = 0;
    each([&](float v, int i) { mine += kept(v, i) && v == x; });
    mine = __reduce_add_sync(0xffffffffu, mine);
    __syncthreads();
    if (lane == 0) sh.red_n[0][warp] = mine;
    if (tid == 0) sh.pick_i = -1;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < SA_WARPS; ++w) all += sh.red_n[0][w];
    if (tid == 0) sh.x[xb].n[0] = all;
    cl.sync();
    int k = m;
    for (int r = 0; r < rank; ++r) k -= cl.map_shared_rank(&sh.x[xb], r)->n[0];
    xb ^= 1;
    if (k >= 0 && k < all) {
      for (int r = 0; r < p.rounds; ++r) {
        const int i0 = (r * SA_THREADS + tid) << p.ept_log2, i1 = i0 + (1 << p.ept_log2);
        int c = 0;
        for (int i = i0; i < i1; ++i) c += kept(at(i), base + i) && at(i) == x;
        int inc = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += v;
        }
        __syncthreads();
        if (lane == 31) sh.red_n[0][warp] = inc;
        __syncthreads();
        int before = 0, tot = 0;
        for (int w = 0; w < SA_WARPS; ++w) {
          if (w < warp) before += sh.red_n[0][w];
          tot += sh.red_n[0][w];
        }
        int j = k - before - (inc - c);
        if (j >= 0 && j < c)
          for (int i = i0; i < i1; ++i)
            if (kept(at(i), base + i) && at(i) == x && j-- == 0) sh.pick_i = base + i;
        k -= tot;
      }
    }
    __syncthreads();
    return share_pick();
  }

  // Shortens the kept head: to its first `k` elements (by_weight false), or to the shortest one whose weight reaches
  // `goal` (by_weight true).  The element it ends with is in [lo, hi].
  __device__ __forceinline__ void shorten(bool by_weight, int k, double goal, float lo, float hi) {
    double near = 0.0;                 // what lies above hi: a number of elements or a weight
    for (int level = 0; level < 256; ++level) {
      // a bin number that never falls with hi - x, whatever the rounding; 0 for hi and the last one for lo, so that
      // every level separates the two
      const float half = hi - lo < INFINITY ? 1.f : 0.5f;
      const float top = half * hi, range = top - half * lo, scale = (float)SA_BINS / range;
      auto bin_of = [&](float x) { return sa_bin(fmaf(-half, x, top), scale); };
      const float width = range / (float)SA_BINS / half, c_w = (float)inv_t;
      __syncthreads();
      for (int i = tid; i < SA_BINS; i += SA_THREADS) sh.hist[i] = 0;
      __syncthreads();
      each([&](float x, int i) {
        if (!kept(x, i) || x > hi || x < lo) return;
        const int b = bin_of(x);
        // weights relative to the bin's near edge, in steps of 1 / SA_STEPS
        const float rel = fminf(0.f, (x - hi + fmaxf(0.f, (float)b - 0.5f) * width) * c_w);
        atomicAdd(&sh.hist[b], by_weight ? max(1u, __float_as_uint(fmaf((float)SA_STEPS, __expf(rel), 8388608.f)) - 0x4b000000u) : 1u);
      });
      cl.sync();
      // two neighbouring bins per thread, over the cluster
      unsigned h0, h1;
      read_bins(h0, h1);
      double v0 = (double)h0, v1 = (double)h1;
      if (by_weight) {
        // relative to the weight at hi
        v0 *= sa_exp((double)fmaxf(0.f, ((float)(2 * tid) - 0.5f) * width) * -inv_t, sh.exp2);
        v1 *= sa_exp((double)(((float)(2 * tid) + 0.5f) * width) * -inv_t, sh.exp2);
      }
      double total, pre = block_scan(v0 + v1, total) - (v0 + v1);   // what lies before this thread's bins
      // the histogram counts weights in units of 1 / SA_STEPS of the weight at hi
      const double unit = by_weight ? (double)SA_STEPS / weight(hi) : 1.0;
      double target = by_weight ? fmin((goal - near) * unit, total) : (double)k - near;

      // ---- the bin's elements, and what lies before it --------------------------------------------------------
      int b_min = 0, b_max = SA_BINS - 1;
      bool split = false;
      while (b_min <= b_max) {
        __syncthreads();
        if (tid == 0) sh.pick = b_max, sh.ln = 0;
        __syncthreads();
        if (v0 > 0.0 && pre + v0 >= target) atomicMin(&sh.pick, 2 * tid);
        else if (v1 > 0.0 && pre + v0 + v1 >= target) atomicMin(&sh.pick, 2 * tid + 1);
        __syncthreads();
        const int b = max(sh.pick, b_min);
        if (2 * tid == (b & ~1)) sh.pick_d = (b & 1) ? pre + v0 : pre;
        double s_before = 0.0, s_in = 0.0;
        float mn = INFINITY, mx = -INFINITY;
        int n_in = 0, n_before = 0;
        auto take = [&](float x, int i, double w) {
          if (x > hi || bin_of(x) < b) {
            s_before += w;
            ++n_before;
          } else {
            s_in += w;
            ++n_in;
            mn = fminf(mn, x), mx = fmaxf(mx, x);
            const unsigned slot = atomicAdd(&sh.ln, 1u);
            if (slot < SA_LIST) sh.lx[slot] = x, sh.li[slot] = i;
          }
        };
        auto want = [&](float x, int i) { return kept(x, i) && x >= lo && (x > hi || bin_of(x) <= b); };
        if (by_weight) each_weight<false>(want, take);
        else each([&](float x, int i) {
          if (want(x, i)) take(x, i, 0.0);
        });
        SaXchg o;
        exchange(s_before, s_in, mn, mx, n_before, n_in, o);
        if (by_weight) {
          // the answer is in this bin if the exact sum passes the goal inside it; else the proposal is made again from
          // the sum as it is, among the bins not ruled out
          const int move = o.s[0] >= goal && o.n[0] > 0 ? -1 : o.s[0] + o.s[1] < goal ? 1 : 0;
          if (move < 0) b_max = b - 1;
          if (move > 0) b_min = b + 1;
          if (move != 0 && b_min <= b_max) {
            target = (goal - o.s[0]) * unit + sh.pick_d;
            cl.sync();                        // the lists are written anew
            continue;
          }
        }
        if (o.n[1] == 0) return;              // nothing to cut
        if (o.f[0] == o.f[1]) {
          cut_ties(o.f[0], by_weight, k, goal, o);
          return;
        }
        if (o.n[1] <= SA_LIST) {
          cut_list(o.n[1], by_weight, k - o.n[0], o.s[0], goal);
          return;
        }
        lo = o.f[0], hi = o.f[1];
        near = by_weight ? o.s[0] : (double)o.n[0];
        split = true;
        break;
      }
      if (!split) return;
      cl.sync();
    }
  }

  // the bin is one value: its first m ties are kept
  __device__ __forceinline__ void cut_ties(float x, bool by_weight, int k, double goal, const SaXchg& o) {
    int m = k - o.n[0];
    if (by_weight) {
      const double w = weight(x);
      m = (int)fmin((double)o.n[1], fmax(1.0, ceil((goal - o.s[0]) / w)));
      while (m > 1 && o.s[0] + (double)(m - 1) * w >= goal) --m;
      while (m < o.n[1] && o.s[0] + (double)m * w < goal) ++m;
    }
    m = max(1, min(m, o.n[1]));
    const int last = m == o.n[1] ? 0x7fffffff : nth_tie(x, m - 1);
    ki = x == kx ? min(ki, last) : last;
    kx = x;
  }

  // larger logits first, lower indices first among equals: ascending
  static __device__ __forceinline__ unsigned long long key_of(float x, int i) {
    const unsigned u = __float_as_uint(x);
    return ((unsigned long long)((u >> 31) ? u : ~(u | 0x80000000u)) << 32) | (unsigned)i;
  }
  static __device__ __forceinline__ float key_value(unsigned long long k) {
    const unsigned u = (unsigned)(k >> 32);
    return __uint_as_float((u >> 31) ? u : ~(u | 0x80000000u));
  }
  // ascending order of one key per thread, the first n of which count (a bitonic network: within warps by shuffles)
  __device__ __forceinline__ unsigned long long sort_keys(unsigned long long k, int n_all) {
    int n2 = 32;
    while (n2 < n_all) n2 *= 2;
    for (int len = 2; len <= n2; len *= 2)
      for (int o = len / 2; o > 0; o /= 2) {
        unsigned long long other;
        if (o >= 32) {
          __syncthreads();
          sh.key[tid] = k;
          __syncthreads();
          other = sh.key[tid ^ o];
        } else {
          other = __shfl_xor_sync(0xffffffffu, k, o);
        }
        const bool low = (tid & o) == 0, up = (tid & len) == 0 || len == n2;
        k = (low == up) == (other < k) ? other : k;
      }
    return k;
  }
  // the listed elements of the cluster, one per thread
  __device__ __forceinline__ unsigned long long gather_list() {
    static_assert(SA_LIST == SA_THREADS, "an element per thread");
    const int mine = lane < size ? (int)*cl.map_shared_rank(&sh.ln, lane) : 0;
    unsigned long long k = ~0ull;
    int off = 0;
#pragma unroll
    for (int r = 0; r < SA_MAX_CLUSTER; ++r) {
      const int c = __shfl_sync(0xffffffffu, mine, r);
      if (tid >= off && tid < off + c)
        k = key_of(*cl.map_shared_rank(&sh.lx[tid - off], r), *cl.map_shared_rank(&sh.li[tid - off], r));
      off += c;
    }
    return k;
  }
  // running sum of one value per thread, and the sum of all
  __device__ __forceinline__ double block_scan(double v, double& total) {
    double inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = shfl_up_d(inc, o);
      if (lane >= o) inc += x;
    }
    __syncthreads();
    if (lane == 31) sh.red_d[0][warp] = inc;
    __syncthreads();
    double pre = 0.0;
    total = 0.0;
#pragma unroll
    for (int w = 0; w < SA_WARPS; ++w) {
      const double x = sh.red_d[0][w];
      if (w < warp) pre += x;
      total += x;
    }
    return pre + inc;
  }
  // cuts the kept head at the k-th of the n listed elements, or at the first where the running sum reaches the goal
  __device__ __forceinline__ void cut_list(int n_all, bool by_weight, int k, double before, double goal) {
    const unsigned long long key = sort_keys(gather_list(), n_all);
    __syncthreads();
    if (tid == 0) sh.pick = n_all - 1;
    __syncthreads();
    if (by_weight) {
      double total;
      const double inc = block_scan(tid < n_all ? weight(key_value(key)) : 0.0, total);
      if (tid < n_all && before + inc >= goal) atomicMin(&sh.pick, tid);
    } else if (tid == 0) {
      sh.pick = max(0, min(k - 1, n_all - 1));
    }
    __syncthreads();
    if (tid == sh.pick) sh.key[0] = key;
    __syncthreads();
    kx = key_value(sh.key[0]);
    ki = (int)(unsigned)sh.key[0];
    __syncthreads();
  }

  // Small top-k: true if the token has been drawn.  `mine` is the largest of the logits this thread has read.
  __device__ __forceinline__ bool draw_short(int row, int k, float mine, float low, float top_p, double min_p, double u) {
    const float half = M - low < INFINITY ? 1.f : 0.5f;
    const float top = half * M, range = top - half * low, scale = (float)SA_BINS / range;
    auto bin_of = [&](float x) { return sa_bin(fmaf(-half, x, top), scale); };
    for (int i = tid; i < SA_BINS; i += SA_THREADS) sh.hist[i] = 0;
    if (tid == 0) sh.pick = SA_BINS, sh.ln = 0;
    __syncthreads();
    if (mine > -INFINITY) atomicAdd(&sh.hist[bin_of(mine)], 1u);
    cl.sync();
    unsigned h0, h1;
    read_bins(h0, h1);
    const int v0 = (int)h0, v1 = (int)h1;
    int pre = v0 + v1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, pre, o);
      if (lane >= o) pre += v;
    }
    if (lane == 31) sh.red_n[0][warp] = pre;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SA_WARPS; ++w)
      if (w < warp) pre += sh.red_n[0][w];
    pre -= v0 + v1;
    if (v0 > 0 && pre + v0 >= k) atomicMin(&sh.pick, 2 * tid);
    else if (v1 > 0 && pre + v0 + v1 >= k) atomicMin(&sh.pick, 2 * tid + 1);
    __syncthreads();
    const int b = sh.pick;
    if (b >= SA_BINS) {                  // fewer threads with logits than k
      cl.sync();                         // the histograms are written anew
      return false;
    }
    // a border a little below the bin's far edge, whatever the rounding: more elements on the list do no harm
    const float border = b == SA_BINS - 1 ? low : fmaxf(low, (top - ((float)b + 0.501f) / scale) / half);
    each([&](float x, int i) {
      if (x >= border) {
        const unsigned slot = atomicAdd(&sh.ln, 1u);
        if (slot < SA_LIST) sh.lx[slot] = x, sh.li[slot] = i;
      }
    });
    cl.sync();
    const int n_all = __reduce_add_sync(0xffffffffu, lane < size ? (int)*cl.map_shared_rank(&sh.ln, lane) : 0);
    if (n_all > SA_LIST || n_all < k) {
      cl.sync();                         // the lists are written anew
      return false;
    }
    unsigned long long key = rank == 0 ? gather_list() : 0;
    cl.sync();                           // the lists have been read: the other CTAs leave
    left = true;
    if (rank != 0) return true;
    // ---- the k largest, in order, one per thread -----------------------------------------------------------------------
    key = sort_keys(key, n_all);
    const int index = (int)(unsigned)key;
    const double w = tid < k ? weight(key_value(key)) : 0.0;
    double total, kept_sum;
    const double inc = block_scan(w, total);
    const bool keep = tid == 0 || (tid < k && w >= min_p && (top_p >= 1.f || inc - w < (double)top_p * total));
    const int n_keep = __syncthreads_count(keep);      // a head of the order, as each of the three is
    // the kept ones in the order of their indices
    sh.gw[tid] = tid < n_keep ? w : 0.0;
    const unsigned long long by_index = sort_keys(tid < n_keep ? ((unsigned long long)index << 32) | (unsigned)tid : ~0ull, n_keep);
    __syncthreads();
    const double wi = tid < n_keep ? sh.gw[(unsigned)by_index & (SA_LIST - 1)] : 0.0;
    const double run_sum = block_scan(wi, kept_sum);
    if (tid == 0) sh.pick = SA_LIST, sh.pick_i = -1;
    __syncthreads();
    if (wi > 0.0) {
      if (run_sum > u * kept_sum) atomicMin(&sh.pick, tid);
      atomicMax(&sh.pick_i, tid);        // the last one, for u -> 1
    }
    __syncthreads();
    if (tid == (sh.pick < SA_LIST ? sh.pick : sh.pick_i)) {
      p.token[row] = (int64_t)(by_index >> 32);
      if (p.logprob) p.logprob[row] = (float)log(wi / kept_sum);
    }
    return true;
  }

  __device__ __forceinline__ void run(int row) {
    const T* x = reinterpret_cast<const T*>(p.logits) + (int64_t)row * p.sb;
    xb = 0;
    // The CTA's elements begin on 16 bytes: the row is led in by up to 7 that do not exist (unless the last CTA has no
    // room for them; then it is read one by one).
    constexpr int VL = 16 / (int)sizeof(T);
    int lead = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const bool vec = lead == 0 || p.V + lead <= p.slice * size;
    if (!vec) lead = 0;
    base = rank * p.slice - lead;
    n = max(0, min(p.V - base, p.slice));
    if (tid < SA_EXP_TABLE) sh.exp2[tid] = exp2((double)tid / SA_EXP_TABLE);
    const float temperature = p.temperature ? p.temperature[row] : p.temperature0;
    // a NaN filter is off; min_p above 1 leaves the largest logit alone, as top_k = 1 does
    float top_p = p.top_p ? p.top_p[row] : p.top_p0;
    top_p = top_p < 1.f ? fmaxf(top_p, 0.f) : 1.f;
    float min_p = p.min_p ? p.min_p[row] : p.min_p0;
    min_p = min_p > 0.f ? min_p : 0.f;
    int top_k = p.top_k ? p.top_k[row] : p.top_k0;
    if (min_p > 1.f) top_k = 1;
    // ---- the row, once ------------------------------------------------------------------------------------------
    float mn = INFINITY, mx = -INFINITY;
    int fin = 0;
    auto look = [&](float v) -> float {
      mx = fmaxf(mx, v);
      if (v > -INFINITY) {
        ++fin;
        mn = fminf(mn, v);
      }
      return v;
    };
    const int held = p.rounds * (SA_THREADS << p.ept_log2);
    if (vec) {
      constexpr int U = 4;             // loads in flight per thread
      const T* src = x + base;
      for (int v0 = tid; v0 * VL < held; v0 += U * SA_THREADS) {
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = (v0 + u * SA_THREADS) * VL;
          raw[u] = make_uint4(0, 0, 0, 0);
          if (base + i >= 0 && i + VL <= n) raw[u] = __ldg(reinterpret_cast<const uint4*>(src + i));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = (v0 + u * SA_THREADS) * VL;
          if (i >= held) break;
          const bool whole = base + i >= 0 && i + VL <= n;
          const T* e = reinterpret_cast<const T*>(&raw[u]);
          float v[VL];
#pragma unroll
          for (int j = 0; j < VL; ++j) {
            if (whole) v[j] = sa_value<T>(e[j]);
            else v[j] = base + i + j >= 0 && i + j < n ? sa_value<T>(src[i + j]) : -INFINITY;
            look(v[j]);
          }
#pragma unroll
          for (int j = 0; j < VL; j += 4)
            reinterpret_cast<float4*>(xs)[group_at((i + j) >> p.ept_log2, ((i + j) & ((1 << p.ept_log2) - 1)) >> 2)] =
                make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        }
      }
    } else {
      for (int i = tid; i < held; i += SA_THREADS) at(i) = i < n ? look(sa_value<T>(x[base + i])) : -INFINITY;
    }
    SaXchg o;
    exchange(0.0, 0.0, mn, mx, fin, 0, o);
    M = o.f[1];
    int n_fin = o.n[0];
    float low = o.f[0];
    kx = -INFINITY, ki = -1;               // everything above -infinity
    if (n_fin == 0) {
      // no logit to draw from
      if (rank == 0 && tid == 0) {
        p.token[row] = -1;
        if (p.logprob) p.logprob[row] = -INFINITY;
      }
      return;
    }
    if (M == INFINITY) {
      // the limit of ever larger logits: those at +infinity share the probability
      int c = 0;
      for (int i = tid; i < held; i += SA_THREADS) {
        const float v = at(i) == INFINITY ? 0.f : -INFINITY;
        at(i) = v;
        c += v == 0.f;
      }
      exchange(0.0, 0.0, 0.f, 0.f, c, 0, o);
      M = 0.f, low = 0.f, n_fin = o.n[0];
    }
    inv_t = temperature > 0.f ? 1.0 / (double)temperature : 0.0;
    if (!(temperature > 0.f)) top_k = 1;
    const double u = (double)p.u[row];
    if (top_k == 1) {
      // the largest logit, lowest index
      const int first = nth_tie(M, 0);
      if (rank == 0 && tid == 0) {
        p.token[row] = first;
        if (p.logprob) p.logprob[row] = 0.f;
      }
      return;
    }
    if (top_k > 0 && top_k <= SA_LIST && top_k < n_fin && M > low && draw_short(row, top_k, mx, low, top_p, (double)min_p, u))
      return;
    if (top_k > 0 && top_k < n_fin) shorten(false, top_k, 0.0, low, M);
    if (top_p < 1.f) {
      double s = 0.0;
      each_weight<true>([&](float v, int i) { return kept(v, i); }, [&](float, int, double w) { s += w; });
      exchange(s, 0.0, 0.f, 0.f, 0, 0, o);
      // logits so low that all of them together weigh less than half of what top-p drops are not where it ends
      const double p0 = (double)top_p;
      const float from = (float)((double)M + log(0.5 * (1.0 - p0) * o.s[0] / (double)n_fin) / inv_t);
      shorten(true, 0, p0 * o.s[0], fmaxf(kx > -INFINITY ? kx : low, fminf(from, M)), M);
    }
    draw(row, u, (double)min_p);
  }

  __device__ __forceinline__ void draw(int row, double u, double min_p) {
    double W = 0.0;
    auto mass = [&](int i) -> double {
      const float v = at(i);
      if (!kept(v, base + i)) return 0.0;
      const double w = weight(v);
      return w >= min_p || v == M ? w : 0.0;
    };
    double mine[SA_MAX_ROUNDS] = {0.0, 0.0, 0.0}, s = 0.0;
    each_weight<true>([&](float v, int i) { return kept(v, i); },
                      [&](float v, int i, double w) {
                        const int r = (i - base) >> (p.ept_log2 + 9);
                        static_assert(SA_THREADS == 512, "2^9 threads");
                        const double x = w >= min_p || v == M ? w : 0.0;
                        mine[0] += r == 0 ? x : 0.0, mine[1] += r == 1 ? x : 0.0, mine[2] += r == 2 ? x : 0.0;
                      });
#pragma unroll
    for (int r = 0; r < SA_MAX_ROUNDS; ++r) s += mine[r];
    // the CTA's sum, and those of the CTAs before it
    s = warp_sum_d(s);
    __syncthreads();
    if (lane == 0) sh.red_d[0][warp] = s;
    if (tid == 0) sh.pick_i = -1;
    __syncthreads();
    if (tid == 0) {
      double t = 0.0;
      for (int w = 0; w < SA_WARPS; ++w) t += sh.red_d[0][w];
      sh.x[xb].s[0] = t;
    }
    cl.sync();
    const double share = lane < size ? cl.map_shared_rank(&sh.x[xb], lane)->s[0] : 0.0;
#pragma unroll
    for (int r = 0; r < SA_MAX_CLUSTER; ++r) W += __shfl_sync(0xffffffffu, share, r);
    const double goal = u * W;
    double pre = 0.0, own_pre = 0.0;
    int owner = 0;
    bool found = false;
#pragma unroll
    for (int r = 0; r < SA_MAX_CLUSTER; ++r) {
      const double c = __shfl_sync(0xffffffffu, share, r);
      if (c > 0.0 && !found) owner = r, own_pre = pre;   // the last CTA with weight, unless one before it passes the goal
      if (pre + c > goal) found = true;
      pre += c;
    }
    xb ^= 1;
    if (rank == owner) {
      double before = own_pre;
#pragma unroll
      for (int r = 0; r < SA_MAX_ROUNDS; ++r) {
        if (r >= p.rounds) break;
        double inc = mine[r];
#pragma unroll
        for (int of = 1; of < 32; of <<= 1) {
          const double v = shfl_up_d(inc, of);
          if (lane >= of) inc += v;
        }
        __syncthreads();
        if (lane == 31) sh.red_d[1][warp] = inc;
        __syncthreads();
        double at0 = before;
        for (int w = 0; w < warp; ++w) at0 += sh.red_d[1][w];
        const double hi_s = at0 + inc;
        // the first thread whose sum passes the goal; the last one with weight as a fallback for u -> 1
        if (mine[r] > 0.0) {
          const int key = r * SA_THREADS + tid;
          if (hi_s > goal) atomicMin(reinterpret_cast<unsigned*>(&sh.pick_i), (unsigned)key);
        }
        for (int w = warp; w < SA_WARPS; ++w) at0 += sh.red_d[1][w];
        before = at0;
      }
      __syncthreads();
      finish(row, goal, own_pre, W, mine, mass);
    }
  }

  template <typename F>
  __device__ __forceinline__ void finish(int row, double goal, double own_pre, double W, const double* mine, F mass) {
    unsigned key = (unsigned)sh.pick_i;
    if (key == 0xffffffffu) {
      // rounding at the very end: the last thread with weight
      __syncthreads();
      int last = -1;
#pragma unroll
      for (int r = 0; r < SA_MAX_ROUNDS; ++r)
        if (mine[r] > 0.0) last = r * SA_THREADS + tid;
      last = __reduce_max_sync(0xffffffffu, last);
      if (lane == 0) sh.red_n[1][warp] = last;
      __syncthreads();
      for (int w = 0; w < SA_WARPS; ++w) last = max(last, sh.red_n[1][w]);
      key = (unsigned)last;
    }
    // the sum before that thread, in the order of the indices
    const int kr = key / SA_THREADS, kt = key % SA_THREADS;
    double before = own_pre;
#pragma unroll
    for (int r = 0; r < SA_MAX_ROUNDS; ++r) {
      if (r > kr) break;
      double v = (r < kr || tid < kt) ? mine[r] : 0.0;
      v = warp_sum_d(v);
      __syncthreads();
      if (lane == 0) sh.red_d[0][warp] = v;
      __syncthreads();
      for (int w = 0; w < SA_WARPS; ++w) before += sh.red_d[0][w];
    }
    if (warp == 0) {
      // an element per lane
      const int i0 = (kr * SA_THREADS + kt) << p.ept_log2;
      const double w = lane < (1 << p.ept_log2) ? mass(i0 + lane) : 0.0;
      double inc = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = shfl_up_d(inc, o);
        if (lane >= o) inc += v;
      }
      const unsigned passed = __ballot_sync(0xffffffffu, w > 0.0 && before + inc > goal);
      const unsigned any = __ballot_sync(0xffffffffu, w > 0.0);
      if (lane == (passed ? __ffs(passed) - 1 : 31 - __clz(any))) {
        p.token[row] = base + i0 + lane;
        if (p.logprob) p.logprob[row] = (float)log(w / W);
      }
    }
  }
};

// CTAS: how many share an SM.  Alone a CTA keeps its values in registers (118 instead of 64) and is 7 % faster; two hide
// each other's waits (256 rows of 128256: 214 us against 306).  Above 131072 logits only one fits into an SM's shared memory,
// whatever was asked for; the compiler reports 32 to 52 bytes of spills for two.
template <typename T, int CTAS>
__global__ void __launch_bounds__(SA_THREADS, CTAS) sample_kernel(const SampleParams p) {
  extern __shared__ float sa_xs[];
  __shared__ SaShared sh;
  cg::cluster_group cl = cg::this_cluster();
  Sampler<T> s{p, sh, sa_xs, cl};
  s.rank = (int)cl.block_rank(), s.size = (int)cl.num_blocks();
  s.tid = threadIdx.x, s.lane = threadIdx.x & 31, s.warp = threadIdx.x >> 5;
  s.run(blockIdx.x / s.size);
  if (!s.left) cl.sync();       // no CTA leaves while another may still read its shared memory
}

template <typename T, int CTAS>
static int sample_launch_t(const SampleParams& prm, int B, int cluster, cudaStream_t st) {
  const int smem = prm.rounds * (SA_THREADS << prm.ept_log2) * 4;
  const int rc = allow_smem<sample_kernel<T, CTAS>>(SA_MAX_ROUNDS * SA_ROUND * 4, "cudaFuncSetAttribute(sample)");
  if (rc != FA_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(B * cluster);
  cfg.blockDim = dim3(SA_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T, CTAS>, prm);
  if (e != cudaSuccess) return cuda_fail(e, "fa_sample");
  return FA_OK;
}

template <typename T>
static int sample_launch(const SampleParams& prm, int B, int cluster, cudaStream_t st) {
  return (int64_t)B * cluster <= sm_count() ? sample_launch_t<T, 1>(prm, B, cluster, st) : sample_launch_t<T, 2>(prm, B, cluster, st);
}

}  // namespace fa

using namespace fa;

extern "C" int fa_sample(const void* logits, int dtype, int B, int V, int64_t logits_sb, const float* u,
                         const float* temperature, float temperature0, const int32_t* top_k, int top_k0,
                         const float* top_p, float top_p0, const float* min_p, float min_p0, int64_t* token,
                         float* logprob, fa_stream_t stream) {
  FA_REQUIRE(dtype == FA_DTYPE_F16 || dtype == FA_DTYPE_BF16 || dtype == FA_DTYPE_F32, FA_ERR_DTYPE,
             "fa_sample: bad dtype %d", dtype);
  FA_REQUIRE(B >= 0 && V > 0, FA_ERR_SHAPE, "fa_sample: bad sizes (%d rows of %d logits)", B, V);
  FA_REQUIRE(V <= SA_MAX_VOCAB, FA_ERR_CAPACITY, "fa_sample: %d logits in a row, at most %d are held", V, SA_MAX_VOCAB);
  if (B == 0) return FA_OK;
  FA_REQUIRE(logits && u && token, FA_ERR_NULL, "fa_sample: null pointer");
  // A row takes as many CTAs as it has rounds of 16384 elements to keep one round each; with rows enough for only a
  // part of the GPU it is spread further, down to 2048 elements per CTA.
  int cluster = 1;
  while (cluster < SA_MAX_CLUSTER && (ceil_div(V, cluster) > SA_ROUND ||
                                      ((int64_t)B * cluster * 2 <= sm_count() && ceil_div(V, 2 * cluster) >= 2048)))
    cluster *= 2;
  SampleParams prm;
  prm.logits = logits;
  prm.sb = logits_sb;
  prm.V = V;
  // room for the elements that lead a row in, as long as it is there
  const int lead = 16 / (dtype == FA_DTYPE_F32 ? 4 : 2) - 1;
  prm.slice = ceil_div(ceil_div(V + lead, cluster), 8) * 8;
  if (prm.slice > SA_MAX_ROUNDS * SA_ROUND || (prm.slice > SA_ROUND && ceil_div(V, cluster) <= SA_ROUND))
    prm.slice = ceil_div(ceil_div(V, cluster), 8) * 8;
  prm.rounds = ceil_div(prm.slice, SA_ROUND);
  prm.ept_log2 = 2;
  while (prm.rounds == 1 && (SA_THREADS << prm.ept_log2) < prm.slice) ++prm.ept_log2;
  if (prm.rounds > 1) prm.ept_log2 = 5;
  prm.u = u;
  prm.temperature = temperature, prm.temperature0 = temperature0;
  prm.top_k = top_k, prm.top_k0 = top_k0;
  prm.top_p = top_p, prm.top_p0 = top_p0;
  prm.min_p = min_p, prm.min_p0 = min_p0;
  prm.token = token;
  prm.logprob = logprob;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == FA_DTYPE_F32) return sample_launch<float>(prm, B, cluster, st);
  if (dtype == FA_DTYPE_F16) return sample_launch<__half>(prm, B, cluster, st);
  return sample_launch<__nv_bfloat16>(prm, B, cluster, st);
}
