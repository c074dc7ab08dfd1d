// sample.cu -- the draw of the next token of each row of logits: temperature, top-k, top-p, min-p, and a uniform number per row.
//
// w_i = exp((x_i - max) / temp). The tokens in the order (logit falling, index rising): the first k; of these the shortest run from the
// top whose mass reaches p times their mass; of these the ones with w_i >= min_p. Drawn is the first of them, by index, whose
// running sum exceeds u times the sum of all.
//
// A draw goes by which side of a sum a number falls, and a row has 10^5 such borders; sums that are off by 1e-7 would move a border
// past u once in some hundred draws. So weights are fixed-point integers, 2^F for the largest, F = 62 - log2 of the row's length (44 for 2^18
// tokens): their sums are exact and the same in any order, each weight is off by at most half a unit and the error of the exponential
// (2^-49: double, a table of 2^(j/128) and a polynomial of degree 4).
//
// One thread-block cluster per row, each CTA with its slice of the row in shared memory: the logits are read from HBM once, all
// further passes stay on chip, and what the CTAs find meets in each other's shared memory. A thread has a contiguous run of tokens, so that
// sums over threads are sums in index order. Bound: the chain of passes and cluster barriers (some 1000 cycles each; a row takes
// one to six of them), for many rows also the exponentials of those that need all of them.
//  - top-k up to 512: the row's 512 groups of threads exchange their maxima; the k-th largest of those (but for its low bits) is a lower
//    bound: at least k tokens reach it, and few more. They go to the first CTA, which ranks them and does the rest alone.
//  - everything else: the border of a run (by count or by mass) from a histogram over the cluster, bins of 1/48 of a power of two of
//    the weight. A bin's mass is two 32-bit words, the upper touched by a carry or a weight of more than 2^32 units only (64-bit
//    atomics took 150 us at 1 x 128256, 720 at 64 x 152064). A short run of top-p goes to the first CTA whole, as above; of a long one
//    the bin on the border does, or, where that holds too many, is split further by the bits of the logits until what is left are
//    equal ones, which are counted off by index.
// Measured (one row of 128256 / 64 rows of 152064, us): temp 0 3.8 / 13, top-k 50 7.3 / 23, no filter 8.2 / 32, min-p 6.4 / 20, top-p 0.9 15 / 57,
// top-k 1000 17 / 51, top-p 0.95 of a flat row 24 / 90, a batch with all kinds 39.
#include <cuda_pipeline_primitives.h>
#include <math.h>

#include "common.cuh"

namespace ieb {

constexpr int SM_THREADS = 512, SM_WARPS = SM_THREADS / 32, SM_PER = 3, SM_BINS = SM_PER * SM_THREADS, SM_LIST = 1024, SM_SHORT = 256, SM_MAX_CL = 8, SM_TABLE = 128;
constexpr uint32_t SM_MAX_SLICE = 45056;  // floats of a CTA's slice: 176 KB
static_assert(SM_MAX_SLICE / 4u / SM_THREADS < 32u, "a thread's run is no longer than a warp is wide");
constexpr uint32_t SM_NONE = 0xFFFFFFFFu;

struct SampleArgs {
  const float *x, *u, *temp, *top_p, *min_p;
  const uint32_t *top_k;
  uint32_t *idx;
  float *prob;
  uint32_t n, slice, cl, wide, sorted;
  int frac;  // F
  size_t x_stride;
};

// A CTA's shared memory in front of its slice (with the slice of 152064 logits over 8 CTAs: two CTAs on an SM).
struct SampleSmem {
  uint32_t low[SM_BINS], high[SM_BINS];  // this CTA's histogram
  union {
    uint64_t bins[SM_BINS];              // the cluster's
    struct {
      uint64_t mine[SM_LIST];            // this CTA's candidates (key, ~index); in the first CTA then the sorted ones of the row
      uint64_t w[SM_THREADS];            // their weights
    };
  };
  uint64_t list[SM_LIST];                // the row's candidates (first CTA)
  uint64_t part[SM_MAX_CL];              // sums of the CTAs
  uint64_t wsum[SM_WARPS];               // of the warps
  double pow2[SM_TABLE];                 // 2^(F + j / 128)
  float max_of[SM_THREADS];              // maxima of the row's 512 groups of threads
  uint32_t first[SM_MAX_CL];             // index of each CTA's maximum
  uint32_t n_list, n_mine, base, bin;
  uint64_t above, cut;                   // mass ahead of the bin; a new cut: key, ~index
};
extern __shared__ __align__(16) uint8_t smem_s[];  // SampleSmem, then the slice
constexpr size_t SM_FRONT = (sizeof(SampleSmem) + 15u) & ~(size_t)15u;
__device__ __forceinline__ SampleSmem &sm_front() { return *reinterpret_cast<SampleSmem *>(smem_s); }

// Floats in an order of unsigned integers.
__device__ __forceinline__ uint32_t sm_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // (-0 is 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sm_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

__device__ __forceinline__ void dsm_st64(uint32_t a, uint64_t v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory"); }
__device__ __forceinline__ void dsm_st32(uint32_t a, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ uint32_t dsm_ld32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t dsm_add32(uint32_t a, uint32_t v) {
  uint32_t old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(a), "r"(v) : "memory");
  return old;
}

__device__ __forceinline__ uint64_t warp_scan64(uint64_t v, uint32_t lane) {  // inclusive
  for (uint32_t o = 1; o < 32u; o <<= 1) {
    const uint64_t w = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += w;
  }
  return v;
}
// The sum of v over the CTA's threads ahead of this one (x), and of all of them (y). (Out of line: it is used in many places.)
__device__ __noinline__ ulonglong2 sm_before(uint64_t v, uint32_t tid) {
  SampleSmem &s = sm_front();
  const uint32_t warp = tid >> 5, lane = tid & 31u;
  const uint64_t incl = warp_scan64(v, lane);
  __syncthreads();
  if (lane == 31u) s.wsum[warp] = incl;
  __syncthreads();
  const uint64_t of_warp = lane < SM_WARPS ? s.wsum[lane] : 0u, scan = warp_scan64(of_warp, lane);
  return make_ulonglong2(__shfl_sync(0xFFFFFFFFu, scan - of_warp, warp) + incl - v, __shfl_sync(0xFFFFFFFFu, scan, 31));
}

// 2^F w as an integer: t = (x - max) 128 log2(e) / temp = k + f, k the nearest integer, w = 2^(k / 128) 2^(f / 128), each step for all N, so that
// they run together: a row of which every weight is wanted is bound by the number of instructions, some 25 for each.
template <int N>
__device__ __forceinline__ void sm_weights(const double (&diff)[N], double c128, uint64_t (&w)[N]) {
  constexpr double MAGIC = 6755399441055744.0, L = 0.0054152123481245725;  // 1.5 * 2^52; ln 2 / 128
  double m[N], f[N], p[N];
#pragma unroll
  for (int e = 0; e < N; e++) m[e] = fma(diff[e], c128, MAGIC);  // k in the low bits
#pragma unroll
  for (int e = 0; e < N; e++) f[e] = fma(diff[e], c128, MAGIC - m[e]);
#pragma unroll
  for (int e = 0; e < N; e++) p[e] = fma(f[e], L * L * L * L / 24.0, L * L * L / 6.0);
#pragma unroll
  for (int e = 0; e < N; e++) p[e] = fma(f[e], p[e], L * L / 2.0);
#pragma unroll
  for (int e = 0; e < N; e++) p[e] = fma(f[e], p[e], L);
#pragma unroll
  for (int e = 0; e < N; e++) p[e] = fma(f[e], p[e], 1.0);
#pragma unroll
  for (int e = 0; e < N; e++) p[e] *= sm_front().pow2[__double2loint(m[e]) & (SM_TABLE - 1)];
#pragma unroll
  for (int e = 0; e < N; e++)  // (2^52 more: rounded to an integer, in the low bits)
    p[e] = __hiloint2double(__double2hiint(p[e]) + ((__double2loint(m[e]) & -SM_TABLE) << 13), __double2loint(p[e])) + 4503599627370496.0;
#pragma unroll
  for (int e = 0; e < N; e++) w[e] = (uint64_t)__double_as_longlong(p[e]) & 0xFFFFFFFFFFFFFull;
}
__device__ __noinline__ uint64_t sm_weight(double diff, double c128) {
  const double d[1] = {diff};
  uint64_t w[1];
  sm_weights<1>(d, c128, w);
  return w[0];
}

__device__ __forceinline__ void sample_out(const SampleArgs &a, uint32_t row, uint32_t idx, float prob) {
  a.idx[row] = idx;
  if (a.prob) a.prob[row] = prob;
}
// What a running sum of integers has to exceed to exceed u times the sum, and what it has to reach to reach p times the sum.
__device__ __forceinline__ uint64_t sample_goal(float u, uint64_t all) {
  const double g = (double)u * (double)all;
  return g > 0.0 ? min((uint64_t)min(g, 9.2e18), all - 1u) : 0u;
}
__device__ __forceinline__ uint64_t run_goal(float p, uint64_t all) {
  const double g = ceil((double)p * (double)all);
  return g > 1.0 ? min(all, (uint64_t)g) : 1u;
}

// Where the rows are more than run at once: the i-th row of those that top_p makes long, then the i-th of the others (up to 512 rows).
__device__ __forceinline__ uint32_t sample_row(const SampleArgs &a, uint32_t i) {
  SampleSmem &s = sm_front();
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, T = gridDim.x / a.cl;
  const uint32_t k = tid < T && a.top_k ? a.top_k[tid] : 0u;
  const bool in = tid < T, is_long = in && a.top_p && a.top_p[tid] < 1.0f && (k == 0u || k > (uint32_t)SM_THREADS) && (!a.temp || a.temp[tid] > 0.0f);
  const uint32_t longs = __ballot_sync(0xFFFFFFFFu, is_long);
  if (lane == 0) s.wsum[warp] = __popc(longs);
  __syncthreads();
  uint32_t before = __popc(longs & ((1u << lane) - 1u)), all = 0u;
  for (uint32_t w = 0; w < SM_WARPS; w++) {
    const uint32_t n = (uint32_t)s.wsum[w];
    if (w < warp) before += n;
    all += n;
  }
  if (in && (is_long ? before : all + tid - before) == i) s.base = tid;
  __syncthreads();
  return s.base;
}

struct Sampler {
  const SampleArgs &a;
  SampleSmem &s;
  float *xs;                             // the slice
  uint32_t row, rank, cl, begin, quads, run;  // rank, cl: of the cluster; first token and groups of four tokens of the slice; groups of a thread (odd: no bank conflicts)
  float xmax, c32, none, reach;          // c32: log2(e) / temp; none: log2 distance from which weights are less than half a unit; reach: or below min_p
  double xmax_d, c128;                   // 128 log2(e) / temp
  uint64_t least;                        // what a weight has to have to be drawn: min_p in their units, 1
  float cut_x;                           // the last token of the run that is kept so far
  uint32_t cut_idx, tid, warp, lane;
  bool dense;                            // the run has a fifth of the row or more

  __device__ __forceinline__ uint32_t peer(const void *p, uint32_t cta) const { return cluster_map_shared(p, cta); }

  __device__ __forceinline__ float distance(float x) const { return (xmax - x) * c32; }  // in powers of two; never falls where x falls
  // bin of 1/48 of a power of two (a NaN, from an infinity times a zero c32, goes to the last one)
  __device__ __forceinline__ uint32_t bin_of(float x) const {
    const float d = distance(x) * 48.0f;
    return __float_as_uint((d < (float)(SM_BINS - 1) ? d : (float)(SM_BINS - 1)) + 8388608.0f) & 0xFFFFu;
  }
  __device__ __forceinline__ uint64_t weight(float x) const { return distance(x) <= none ? sm_weight((double)x - xmax_d, c128) : 0u; }
  __device__ __forceinline__ void weights(const float (&x)[4], uint64_t (&w)[4]) const {
    double diff[4];
#pragma unroll
    for (int e = 0; e < 4; e++) diff[e] = (double)x[e] - xmax_d;
    sm_weights(diff, c128, w);
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = distance(x[e]) <= none ? w[e] : 0u;
  }
  // (Here and in what the passes pick by: no && and ||, whose branches took longer than what they saved.)
  __device__ __forceinline__ bool kept(float x, uint32_t i) const { return (x > cut_x) | ((x == cut_x) & (i <= cut_idx)); }

  // f(four logits, index of the first) for the tokens of this thread, in rising order
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const uint32_t q1 = min((tid + 1u) * run, quads);
#pragma unroll 1
    for (uint32_t q = tid * run; q < q1; q++) {
      const float4 v = *reinterpret_cast<const float4 *>(xs + 4u * q);
      const float x[4] = {v.x, v.y, v.z, v.w};
      f(x, begin + 4u * q);
    }
  }
  // use(logit, index, weight) for this thread's tokens, in rising order
  template <typename C>
  __device__ __forceinline__ void weigh_all(C use) const {
    each([&](const float (&x)[4], uint32_t i) {
      uint64_t w[4];
      weights(x, w);
#pragma unroll
      for (uint32_t e = 0; e < 4; e++) use(x[e], i + e, w[e]);
    });
    __syncwarp();
  }
  // (Whole warps call it.) The same for those that pred(logit, index) picks: 32 looked at at a time, so that few of them cost few
  // exponentials, not one for every four tokens of which some lane wants one; where a lane has many, all 32 are weighed, four together, and
  // the others used with a weight of 0.
  // maybe(logit): false only where pred is false for it and every smaller one; it is asked of the largest of four.
  template <typename M, typename P, typename C>
  __device__ __forceinline__ void weigh(M maybe, P pred, C use) const {
    const uint32_t q1 = min((tid + 1u) * run, quads);
#pragma unroll 1
    for (uint32_t g = 0; g < run; g += 8u) {  // (as often in every lane: they meet at its end)
      const uint32_t qa = tid * run + g, n = qa < q1 ? min(min(8u, run - g), q1 - qa) : 0u;
      uint32_t mask = 0u;
#pragma unroll 1
      for (uint32_t j = 0; j < n; j++) {
        const float4 v = *reinterpret_cast<const float4 *>(xs + 4u * (qa + j));
        const uint32_t i = begin + 4u * (qa + j);
        if (maybe(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w))))
          mask |= ((pred(v.x, i) ? 1u : 0u) | (pred(v.y, i + 1u) ? 2u : 0u) | (pred(v.z, i + 2u) ? 4u : 0u) | (pred(v.w, i + 3u) ? 8u : 0u)) << (4u * j);
      }
      if (__any_sync(0xFFFFFFFFu, 2u * __popc(mask) > 3u * n)) {  // (four together take about as long as one and a half alone)
#pragma unroll 1
        for (uint32_t j = 0; j < n; j++) {
          const float4 v = *reinterpret_cast<const float4 *>(xs + 4u * (qa + j));
          const float x[4] = {v.x, v.y, v.z, v.w};
          uint64_t w[4];
          weights(x, w);
#pragma unroll
          for (uint32_t e = 0; e < 4; e++)
            use(x[e], begin + 4u * (qa + j) + e, mask >> (4u * j + e) & 1u ? w[e] : 0u);
        }
      } else {
#pragma unroll 1
        while (mask) {
          const uint32_t l = __ffs(mask) - 1u;
          mask &= mask - 1u;
          const float x = xs[4u * qa + l];
          use(x, begin + 4u * qa + l, weight(x));
        }
      }
      __syncwarp();  // (lanes that a branch has parted would go on apart: the dense pass behind a sparse one took three times as long)
    }
  }
  __device__ __forceinline__ uint64_t block_before(uint64_t v, uint64_t &all) const {
    const ulonglong2 r = sm_before(v, tid);
    all = r.y;
    return r.x;
  }

  __device__ __forceinline__ void count(uint32_t bin, uint64_t v) {
    const uint32_t lo = (uint32_t)v;
    uint32_t hi = (uint32_t)(v >> 32);
    if (lo) hi += atomicAdd(&s.low[bin], lo) > ~lo;  // (a carry)
    if (hi) atomicAdd(&s.high[bin], hi);
  }
  __device__ __forceinline__ void clear(uint32_t last) {
    for (uint32_t i = tid; i < SM_BINS; i += SM_THREADS) s.low[i] = s.high[i] = 0u;
    if (tid == 0) s.n_mine = 0u, s.n_list = 0u, s.bin = last, s.above = 0u;
    __syncthreads();
  }
  // The bin of v (three to a thread) at which the bins up to it reach goal_of(sum of all): s.bin, and s.above the mass ahead of it.
  template <typename G>
  __device__ __forceinline__ void bin_at(const uint64_t (&v)[SM_PER], G goal_of) {
    uint64_t all, before = block_before(v[0] + v[1] + v[2], all);
    const uint64_t goal = goal_of(all);
#pragma unroll
    for (uint32_t i = 0; i < SM_PER; i++) {
      if (before < goal && goal <= before + v[i]) s.bin = SM_PER * tid + i, s.above = before;  // one thread
      before += v[i];
    }
    __syncthreads();
  }
  // The same of the cluster's histogram, in every CTA.
  template <typename G>
  __device__ __forceinline__ void border(G goal_of) {
    cluster_sync_all();
    const uint32_t side = tid & 1u;
    for (uint32_t i = tid; i < 2u * (SM_BINS / cl); i += SM_THREADS) {  // this CTA's share of the bins, for all; two threads to a bin (whole warps: cl is at most 8)
      const uint32_t b = rank * (SM_BINS / cl) + i / 2u;
      uint32_t lo[SM_MAX_CL / 2], hi[SM_MAX_CL / 2];
#pragma unroll
      for (uint32_t c = 0; c < SM_MAX_CL / 2; c++) {
        const uint32_t from = 2u * c + side;
        lo[c] = from < cl ? dsm_ld32(peer(&s.low[b], from)) : 0u, hi[c] = from < cl ? dsm_ld32(peer(&s.high[b], from)) : 0u;
      }
      uint64_t v = 0u;
#pragma unroll
      for (uint32_t c = 0; c < SM_MAX_CL / 2; c++) v += (uint64_t)hi[c] << 32 | lo[c];
      v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
      for (uint32_t c = side; c < cl; c += 2u) dsm_st64(peer(&s.bins[b], c), v);
    }
    cluster_sync_all();
    const uint64_t v[SM_PER] = {s.bins[SM_PER * tid], s.bins[SM_PER * tid + 1u], s.bins[SM_PER * tid + 2u]};
    bin_at(v, goal_of);
  }

  // A candidate, into this CTA's list.
  __device__ __forceinline__ void add(float x, uint32_t i) {
    const uint32_t at = atomicAdd(&s.n_mine, 1u);
    if (at < SM_LIST) s.mine[at] = (uint64_t)sm_key(x) << 32 | (uint32_t)~i;
  }
  // The CTAs' lists into the first CTA's; how many there are (more than SM_LIST: it is not whole). s.n_mine and s.n_list are zeroed a cluster
  // barrier ahead of the first add().
  __device__ __forceinline__ uint32_t gather() {
    __syncthreads();
    const uint32_t n = s.n_mine;
    if (tid < cl && n) {  // every CTA counts them all (nobody looks into another CTA's memory behind the last barrier: it may have ended)
      const uint32_t at = dsm_add32(peer(&s.n_list, tid), n);
      if (tid == 0) s.base = at;
    }
    __syncthreads();
    for (uint32_t i = tid; i < n && s.base + i < SM_LIST && i < SM_LIST; i += SM_THREADS) dsm_st64(peer(&s.list[s.base + i], 0u), s.mine[i]);
    cluster_sync_all();
    return s.n_list;
  }

  // s.list[0 .. n - 1] falling into s.mine (one CTA; n at most SM_LIST).
  __device__ void sort_falling(uint32_t n) {
    if (n <= (uint32_t)SM_SHORT) {  // by counting, for each, those ahead of it, two threads each (100 .. 256 values: 500 .. 1800 cycles, below 2000 .. 4500)
      const uint32_t half = (n + 1u) / 2u, i = tid >> 1, j0 = tid & 1u ? half : 0u, j1 = tid & 1u ? n : half;
      const uint64_t v = i < n ? s.list[i] : 0u;
      uint32_t before = 0u;
      if (i < n) {
#pragma unroll 8
        for (uint32_t j = j0; j < j1; j++) before += s.list[j] > v;
      }
      before += __shfl_xor_sync(0xFFFFFFFFu, before, 1);
      if (i < n && !(tid & 1u)) s.mine[before] = v;
      __syncthreads();
      return;
    }
    uint32_t m = 2u;
    while (m < n) m <<= 1;
    for (uint32_t i = tid; i < m; i += SM_THREADS) s.mine[i] = i < n ? s.list[i] : 0u;  // (the fill sorts to the end)
    __syncthreads();
    for (uint32_t size = 2; size <= m; size <<= 1)
      for (uint32_t step = size >> 1; step; step >>= 1) {
        for (uint32_t t = tid; t < m / 2u; t += SM_THREADS) {
          const uint32_t i = 2u * t - (t & (step - 1u)), j = i + step;
          const uint64_t p = s.mine[i], q = s.mine[j];
          if ((p < q) == ((i & size) == 0u)) s.mine[i] = q, s.mine[j] = p;
        }
        // pairs up to 32 apart stay within the 64 values of a warp, this step and the next ones
        if (step > 32u || (step == 1u && size >= 64u)) __syncthreads();
        else __syncwarp();
      }
    __syncthreads();
  }

  // The rest of the row in the first CTA alone: of its n candidates, which are the row's first ones, the first k (at most one per thread), of
  // these the run that reaches goal_of(mass of the k), of these the ones of `least`, and the draw.
  template <typename G>
  __device__ __forceinline__ void finish(uint32_t n, uint32_t k, float u, G goal_of) {
    sort_falling(n);
    uint64_t all, v = tid < k ? weight(sm_unkey((uint32_t)(s.mine[tid] >> 32))) : 0u;
    const uint64_t before = block_before(v, all);
    const bool keep = tid < k && before < goal_of(all) && v >= least;
    if (keep) s.w[tid] = v;
    const uint32_t m = (uint32_t)__syncthreads_count(keep);  // a run from the top
    // by index: the sum of the kept ones ahead of each, four threads to one of them
#pragma unroll 1
    for (uint32_t i0 = 0; i0 < m; i0 += SM_THREADS / 4u) {
      const uint32_t i = i0 + tid / 4u;
      uint64_t ahead = 0u, sum = 0u;
      const uint32_t me = i < m ? ~(uint32_t)s.mine[i] : 0u;
      if (i < m) {
#pragma unroll 4
        for (uint32_t j = tid & 3u; j < m; j += 4u) {
          const uint64_t w = s.w[j];
          sum += w;
          if (~(uint32_t)s.mine[j] < me) ahead += w;
        }
      }
      ahead += __shfl_xor_sync(0xFFFFFFFFu, ahead, 1), sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
      ahead += __shfl_xor_sync(0xFFFFFFFFu, ahead, 2), sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
      if (i < m && (tid & 3u) == 0u) {
        const uint64_t goal = sample_goal(u, sum), w = s.w[i];
        if (ahead <= goal && goal < ahead + w) sample_out(a, row, me, (float)((double)w / (double)sum));  // one thread
      }
    }
  }

  // The cut (the last kept token of the run) at which the mass of the kept tokens, taken from the top, reaches a goal. MASS: weights, the
  // goal p times the mass of all kept; otherwise counts, the goal k. True: the first CTA has done the rest of the row (MASS, u).
  template <bool MASS>
  __device__ __forceinline__ bool cut_run(float p, uint32_t k, float u) {
    uint64_t goal = k, above = 0u;
    // round 0: bins of the weights; then 10, 10, 10 and 2 bits of the key
    uint32_t coarse = 0u, prefix = 0u, bits = 0u;  // the bin of round 0, the leading bits of the key so far
#pragma unroll 1
    for (int round = 0; round < 5; round++) {
      const uint32_t w = round == 0 ? 0u : round == 4 ? 2u : 10u, last = round == 0 ? SM_BINS - 1u : (1u << w) - 1u;
      auto member = [&](float x, uint32_t i) {
        return round == 0 ? kept(x, i) : kept(x, i) & (bin_of(x) == coarse) & ((uint32_t)((uint64_t)sm_key(x) >> (32u - bits)) == prefix);
      };
      auto bin = [&](float x) { return round == 0 ? bin_of(x) : last - ((sm_key(x) >> (32u - bits - w)) & last); };
      clear(last);
      if (!MASS)
        each([&](const float (&x)[4], uint32_t i) {
#pragma unroll
          for (uint32_t e = 0; e < 4; e++)
            if (member(x[e], i + e)) atomicAdd(&s.low[bin(x[e])], 1u);
        });
      else if (round == 0 && cut_idx == SM_NONE) weigh_all([&](float x, uint32_t, uint64_t v) { count(bin_of(x), v); });
      else weigh([](float) { return true; }, member, [&](float x, uint32_t, uint64_t v) { count(bin(x), v); });
      border([&](uint64_t all) {
        if (MASS && round == 0) goal = run_goal(p, all);
        return goal - above;
      });
      const uint32_t b = s.bin;
      const uint64_t ahead = s.above;
      if (MASS && round == 0) {
        // A run of few tokens goes to the first CTA whole. How many are in the bins up to b: their masses over their weights, 1 % off.
        float about = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < SM_PER; i++)
          if (SM_PER * tid + i <= b) about += (float)s.bins[SM_PER * tid + i] * exp2f((float)(SM_PER * tid + i) * (1.0f / 48.0f) - (float)a.frac);
        about = warp_sum_all(about);
        if (lane == 0) s.max_of[warp] = about;  // (no longer needed for what it is)
        __syncthreads();
        about = 0.0f;
        for (int i = 0; i < SM_WARPS; i++) about += s.max_of[i];
        dense = about * 5.0f > (float)a.n;
        if (about <= 400.0f) {
          each([&](const float (&x)[4], uint32_t i) {
            if (bin_of(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))) > b) return;
#pragma unroll
            for (uint32_t e = 0; e < 4; e++)
              if ((bin_of(x[e]) <= b) & kept(x[e], i + e)) add(x[e], i + e);
          });
          const uint32_t n = gather();
          if (n <= (uint32_t)SM_THREADS) {
            if (rank == 0u) finish(n, n, u, [&](uint64_t) { return goal; });
            return true;
          }
          __syncthreads();  // (everybody has read the count)
          if (tid == 0) s.n_mine = 0u, s.n_list = 0u;
          cluster_sync_all();
        }
      }
      __syncthreads();  // (everybody has read the bins: the lists lie there)
      each([&](const float (&x)[4], uint32_t i) {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++)
          if ((bin(x[e]) == b) & member(x[e], i + e)) add(x[e], i + e);
      });
      const uint32_t n = gather();
      above += ahead;
      if (round == 0) coarse = b;
      else prefix = prefix << w | (last - b), bits += w;
      if (n <= (uint32_t)SM_LIST) {
        if (rank == 0u) {
          uint64_t at = above;
          uint32_t m = n;
          if (m > (uint32_t)SM_SHORT) {  // a histogram of the list first (a sort of 1024 takes 8000 cycles)
            auto fine = [&](float x) {
              if (round == 0) return min((uint32_t)(SM_BINS - 1), (uint32_t)fmaxf((distance(x) * 48.0f - ((float)b - 0.5f)) * (float)SM_BINS, 0.0f));
              return 1023u - ((uint32_t)((uint64_t)sm_key(x) << bits) >> 22);  // (bits may be 32: all are equal)
            };
            auto mass = [&](float x) { return MASS ? weight(x) : 1u; };
            __syncthreads();
            clear(SM_BINS - 1u);
            for (uint32_t i = tid; i < m; i += SM_THREADS) {
              const float x = sm_unkey((uint32_t)(s.list[i] >> 32));
              count(fine(x), mass(x));
            }
            __syncthreads();
            uint64_t v[SM_PER];
#pragma unroll
            for (uint32_t i = 0; i < SM_PER; i++) v[i] = (uint64_t)s.high[SM_PER * tid + i] << 32 | s.low[SM_PER * tid + i];
            bin_at(v, [&](uint64_t) { return goal - above; });
            at += s.above;
            for (uint32_t i = tid; i < m; i += SM_THREADS)
              if (fine(sm_unkey((uint32_t)(s.list[i] >> 32))) == s.bin) s.mine[atomicAdd(&s.n_mine, 1u)] = s.list[i];
            __syncthreads();
            m = s.n_mine;
            if (m > 32u) {
              for (uint32_t i = tid; i < m; i += SM_THREADS) s.list[i] = s.mine[i];
              __syncthreads();
            }
          }
          if (n > (uint32_t)SM_SHORT && m <= 32u) {  // as a rule: one warp does it
            if (warp == 0u) {
              const uint64_t e = lane < m ? s.mine[lane] : 0u, v = lane < m ? (MASS ? weight(sm_unkey((uint32_t)(e >> 32))) : 1u) : 0u;
              uint64_t before = at;
              for (uint32_t j = 0; j < m; j++) {
                const uint64_t o = __shfl_sync(0xFFFFFFFFu, e, j), w = __shfl_sync(0xFFFFFFFFu, v, j);
                if (o > e) before += w;
              }
              if (lane < m && before < goal && goal <= before + v)  // one thread
                for (uint32_t c = 0; c < cl; c++) dsm_st64(peer(&s.cut, c), e);
            }
            m = 0u;
          }
          if (m) sort_falling(m);
#pragma unroll 1
          for (uint32_t i0 = 0; i0 < m; i0 += SM_THREADS) {  // at most two rounds
            uint64_t all;
            const uint32_t i = i0 + tid;
            const uint64_t e = i < m ? s.mine[i] : 0u;
            const uint64_t v = i < m ? (MASS ? weight(sm_unkey((uint32_t)(e >> 32))) : 1u) : 0u, before = at + block_before(v, all);
            if (i < m && before < goal && goal <= before + v)  // one thread
              for (uint32_t c = 0; c < cl; c++) dsm_st64(peer(&s.cut, c), e);
            at += all;
          }
        }
        cluster_sync_all();
        cut_x = sm_unkey((uint32_t)(s.cut >> 32)), cut_idx = ~(uint32_t)s.cut;
        return false;
      }
      __syncthreads();  // (everybody has read the count)
    }
    // what is left are equal logits: as many of them as the goal takes, by index
    const float x = sm_unkey(prefix);
    const uint64_t w = MASS ? weight(x) : 1u, need = (goal - above + w - 1u) / w;
    locate<false>([&](float y, uint32_t i) { return kept(y, i) & (y == x); }, [&](uint64_t) { return need - 1u; },
                  [&](uint32_t idx, uint64_t, uint64_t) {
                    for (uint32_t c = 0; c < cl; c++) dsm_st32(peer(&s.base, c), idx);
                  });
    cluster_sync_all();
    cut_x = x, cut_idx = s.base;
    return false;
  }

  // The first token, by index, at which the running sum over those that pred(logit, index) picks exceeds goal_of(sum of all): found(index, its
  // part, the sum) in one thread of the cluster (in none if there is no such token). MASS: the sum of their weights of `least` and more,
  // otherwise their number.
  template <bool MASS, typename P, typename G, typename H>
  __device__ __forceinline__ void locate(P pred, G goal_of, H found) {
    uint64_t sum = 0u, mine, all = 0u;
    if (MASS && cut_idx == SM_NONE && reach == none) {  // everything is in
      weigh_all([&](float, uint32_t, uint64_t w) { sum += w; });
    } else if (MASS && dense) {  // (picking first: 10900 cycles for 36 tokens to a thread, so 8900)
      weigh_all([&](float x, uint32_t i, uint64_t w) { sum += pred(x, i) & (w >= least) ? w : 0u; });
    } else if (MASS) {
      weigh([&](float x) { return cut_idx != SM_NONE || distance(x) <= reach; }, pred, [&](float, uint32_t, uint64_t w) { sum += w >= least ? w : 0u; });
    } else {
      each([&](const float (&x)[4], uint32_t i) {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) sum += pred(x[e], i + e);
      });
    }
    uint64_t before = block_before(sum, mine);
    if (tid < cl) dsm_st64(peer(&s.part[rank], tid), mine);
    cluster_sync_all();
    for (uint32_t c = 0; c < cl; c++) {
      if (c < rank) before += s.part[c];
      all += s.part[c];
    }
    const uint64_t goal = goal_of(all);
    const uint32_t at = __ballot_sync(0xFFFFFFFFu, before <= goal && goal < before + sum);  // one thread of the cluster; its warp takes its run
    if (!at) return;
    const int owner = __ffs(at) - 1;
    uint64_t base = __shfl_sync(0xFFFFFFFFu, before, owner);
    const uint32_t q0 = (warp * 32u + owner) * run, q1 = min(q0 + run, quads);
#pragma unroll 1
    for (uint32_t qa = q0; qa < q1; qa += 32u) {
      const uint32_t q = qa + lane;
      uint64_t v[4] = {0u, 0u, 0u, 0u};
      if (q < q1) {
        const float4 y = *reinterpret_cast<const float4 *>(xs + 4u * q);
        const float x[4] = {y.x, y.y, y.z, y.w};
        if (MASS) weights(x, v);
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
          const bool in = pred(x[e], begin + 4u * q + e);
          v[e] = MASS ? (in & (v[e] >= least) ? v[e] : 0u) : in;
        }
      }
      const uint64_t four = (v[0] + v[1]) + (v[2] + v[3]), incl = warp_scan64(four, lane);
      uint64_t at_sum = base + incl - four;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (at_sum <= goal && goal < at_sum + v[e]) found(begin + 4u * q + e, v[e], all);
        at_sum += v[e];
      }
      base += __shfl_sync(0xFFFFFFFFu, incl, 31);
    }
  }
};

__global__ void __launch_bounds__(SM_THREADS, 2) sample_kernel(const SampleArgs a) {
  SampleSmem &s = sm_front();
  float *xs = reinterpret_cast<float *>(smem_s + SM_FRONT);
  cluster_arrive();  // (waited for ahead of the first store into a peer, which has to run by then)
  pdl_prologue();
  const uint32_t rank = blockIdx.x % a.cl, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cl = a.cl;
  const uint32_t row = a.sorted ? sample_row(a, blockIdx.x / a.cl) : blockIdx.x / a.cl;
  const uint32_t begin = min(a.n, rank * a.slice), count = min(a.n, begin + a.slice) - begin, quads = (count + 3u) / 4u;

  // ---- the slice; meanwhile the settings
  const float *x = reinterpret_cast<const float *>(reinterpret_cast<const char *>(a.x) + a.x_stride * row) + begin;
  for (uint32_t q = tid; q < quads; q += SM_THREADS) {
    if (a.wide && q * 4u + 4u <= count) {
      __pipeline_memcpy_async(xs + 4u * q, x + 4u * q, 16);
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 4; e++) {
        if (q * 4u + e < count) __pipeline_memcpy_async(xs + 4u * q + e, x + 4u * q + e, 4);
        else xs[4u * q + e] = -INFINITY;
      }
    }
  }
  __pipeline_commit();
  const float temp = a.temp ? a.temp[row] : 1.0f, top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f, u = a.u[row];
  const uint32_t top_k = a.top_k ? a.top_k[row] : 0u;
  const bool greedy = !(temp > 0.0f), by_k = !greedy && top_k > 0u && top_k < a.n, by_p = top_p < 1.0f;  // (a NaN: off)
  const double c128 = greedy ? 0.0 : 184.6649652337873 / (double)fmaxf(temp, 1.17549435e-38f);  // 128 log2(e) / temp (below 2^-126: as that, so that it fits in 32 bits)
  const float mp = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f, none = (float)(a.frac + 1);
  Sampler S = {a, s, xs, row, rank, cl, begin, quads, ((quads + SM_THREADS - 1u) / SM_THREADS) | 1u, 0.0f, (float)(c128 / 128.0), none,
               fminf(none, mp > 0.0f ? 0.01f - log2f(mp) : none), 0.0, c128, max((uint64_t)1u, (uint64_t)ceil((double)mp * (double)(1ull << a.frac))), -INFINITY,
               SM_NONE, tid, warp, lane, false};
  if (tid < SM_TABLE && !greedy) s.pow2[tid] = scalbn(exp2((double)tid / SM_TABLE), a.frac);
  if (tid == 0) s.n_mine = 0u, s.n_list = 0u;
  __pipeline_wait_prior(0);
  __syncthreads();

  // ---- maxima: of groups of cl threads, 512 of them in the row, for everybody (greedy: of the CTAs, with the first index of each)
  float mx = -INFINITY;
  S.each([&](const float (&v)[4], uint32_t i) {
    if (v[0] != v[0] || v[1] != v[1] || v[2] != v[2] || v[3] != v[3]) {  // a NaN is never drawn
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (v[e] != v[e]) xs[i - begin + e] = -INFINITY;
    }
    mx = fmaxf(fmaxf(mx, fmaxf(v[0], v[1])), fmaxf(v[2], v[3]));  // (fmaxf passes over a NaN)
  });
  __syncwarp();
  if (greedy) {
    uint32_t at = SM_NONE;
    const float wm = warp_max(mx);
    if (mx == wm && wm > -INFINITY)
      S.each([&](const float (&v)[4], uint32_t i) {
#pragma unroll
        for (int e = 3; e >= 0; e--)
          if (v[e] == wm) at = min(at, i + e);
      });
    __syncwarp();
    at = __reduce_min_sync(0xFFFFFFFFu, at);
    if (lane == 0) s.wsum[warp] = (uint64_t)sm_key(wm) << 32 | (uint32_t)~at;
    __syncthreads();
    cluster_wait();
    if (tid == 0) {
      uint64_t b = 0u;
      for (int w = 0; w < SM_WARPS; w++) b = max(b, s.wsum[w]);
      dsm_st32(S.peer(&s.first[rank], 0u), ~(uint32_t)b), dsm_st32(S.peer(&s.max_of[rank], 0u), __float_as_uint(sm_unkey((uint32_t)(b >> 32))));
    }
    cluster_sync_all();
    if (rank == 0u && tid == 0u) {
      uint32_t first = SM_NONE;
      float best = -INFINITY;
      for (uint32_t c = 0; c < cl; c++)
        if (s.max_of[c] > best) best = s.max_of[c], first = s.first[c];
      sample_out(a, row, first, first == SM_NONE ? 0.0f : 1.0f);
    }
    return;
  }
  float own = mx;
  for (uint32_t o = 1; o < cl; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
  cluster_wait();
  dsm_st32(S.peer(&s.max_of[rank * (SM_THREADS / cl) + tid / cl], tid % cl), __float_as_uint(mx));  // (a thread of each group for each CTA)
  cluster_sync_all();
  mx = s.max_of[tid];
  const float wm = warp_max(mx);
  if (lane == 0) s.wsum[warp] = __float_as_uint(wm);
  __syncthreads();
  float xmax = warp_max(lane < SM_WARPS ? __uint_as_float((uint32_t)s.wsum[lane]) : -INFINITY);
  if (xmax == -INFINITY) {
    if (rank == 0u && tid == 0u) sample_out(a, row, SM_NONE, 0.0f);
    return;
  }
  if (xmax == INFINITY) {  // its tokens, equally likely, and no other
    S.each([&](const float (&v)[4], uint32_t i) {
#pragma unroll
      for (int e = 0; e < 4; e++) xs[i - begin + e] = v[e] == INFINITY ? 0.0f : -INFINITY;
    });
    xmax = 0.0f, mx = mx == INFINITY ? 0.0f : -INFINITY, own = own == INFINITY ? 0.0f : -INFINITY;
    __syncthreads();
  }
  S.xmax = xmax, S.xmax_d = xmax;

  if (by_k && top_k <= (uint32_t)SM_THREADS) {
    // a lower bound of the k-th largest of the 512 maxima, bit by bit from the top, until less than a quarter more of them reach it
    const uint32_t key = sm_key(mx);
    uint32_t low = 0u, bit = 1u << 31;
    if ((uint32_t)__syncthreads_count(mx > -INFINITY) >= top_k) {  // the leading bits that all but those of -inf have in common are settled (8.3 -> 7.9 us, k 50)
      const uint32_t wl = __reduce_min_sync(0xFFFFFFFFu, mx > -INFINITY ? key : 0xFFFFFFFFu);
      if (lane == 0) s.wsum[warp] = wl;
      __syncthreads();
      const uint32_t least = __reduce_min_sync(0xFFFFFFFFu, lane < SM_WARPS ? (uint32_t)s.wsum[lane] : 0xFFFFFFFFu), diff = least ^ sm_key(xmax);
      bit = diff ? 1u << (31 - __clz(diff)) : 0u;
      low = least & ~(2u * bit - 1u);
      if (!bit) low = least;
    }
#pragma unroll 1
    for (; bit >= 1u << 8; bit >>= 1) {
      const uint32_t reached = (uint32_t)__syncthreads_count(key >= (low | bit));
      if (reached >= top_k) {
        low |= bit;
        if (reached <= top_k + top_k / 4u) break;
      }
    }
    const float floor_x = sm_unkey(max(low, 0x00800000u));  // (the lowest finite float: -inf is none)
    const uint32_t hits = __ballot_sync(0xFFFFFFFFu, own >= floor_x);
    if (2u * __popc(hits) <= S.run) {  // the warp looks through the runs of the few threads that have some, a lane to a group of four (1 x 128256, k 50: 7.9 -> 7.3 us)
#pragma unroll 1
      for (uint32_t b = hits; b; b &= b - 1u) {
        const uint32_t q = (warp * 32u + __ffs(b) - 1u) * S.run + lane;
        if (lane < S.run && q < quads) {
          const float4 y = *reinterpret_cast<const float4 *>(xs + 4u * q);
          const float v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (v[e] >= floor_x) S.add(v[e], begin + 4u * q + e);
        }
      }
    } else if (own >= floor_x) {
      S.each([&](const float (&v)[4], uint32_t i) {
        if (fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= floor_x) {
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (v[e] >= floor_x) S.add(v[e], i + e);
        }
      });
    }
    const uint32_t n = S.gather();
    if (n <= (uint32_t)SM_LIST) {
      if (rank == 0u) S.finish(n, min(top_k, n), u, [&](uint64_t all) { return by_p ? run_goal(top_p, all) : all; });
      return;
    }
    __syncthreads();  // (everybody has read the count)
  }
  if (by_k) S.cut_run<false>(0.0f, top_k, u);
  if (by_p && S.cut_run<true>(top_p, 0u, u)) return;
  S.locate<true>([&](float v, uint32_t i) { return (S.distance(v) <= S.reach) & S.kept(v, i); }, [&](uint64_t sum) { return sample_goal(u, sum); },
                 [&](uint32_t idx, uint64_t w, uint64_t all) { sample_out(a, row, idx, (float)((double)w / (double)all)); });
}

// CTAs of a row: as many as leave each 2000 logits while the batch runs at once (clusters lie within a part of the GPU each, so that is about
// 7/4 of the SMs, not twice), 4000 up to two rounds of it, and as many as the slices need. 1 x 32003, all kinds mixed: 1 CTA 13.6 us, 4 8.5,
// 8 7.2; 28 rows 4 18.9, 8 15.7; 37 rows 4 19, 8 17 (of one kind, top-k 50, 11 and 13.5); 128 rows 1 37, 4 27, 8 40; 64 x 16000 4 14.8, 8 19.2;
// 64 x 100000 38 and 30; 32 x 4000 1 11.5, 4 9.3, 8 11.6.
static uint32_t sample_ctas(uint32_t n, uint32_t T) {
  const uint64_t sms = (uint64_t)sm_count();
  uint32_t c = 1u;
  auto more = [&] {  // twice as many?
    const uint64_t ctas = (uint64_t)T * c * 2u;
    return n > c * SM_MAX_SLICE || (ctas <= 4u * sms && n >= (4u * ctas <= 7u * sms ? 4000u : 8000u) * c);
  };
  while (c < (uint32_t)SM_MAX_CL && more()) c *= 2u;
  return c;
}

}  // namespace ieb

using namespace ieb;

extern "C" int ie_b200_sample(const float *d_x, uint32_t n, uint32_t *d_idx, float *d_prob, const float *d_u, const float *d_temp, const uint32_t *d_top_k,
                              const float *d_top_p, const float *d_min_p, uint32_t T, size_t x_stride, void *stream) {
  if (T == 0) return IE_B200_OK;  // (an empty tensor may have no address)
  if (!d_x || !d_idx || !d_u) return fail(IE_B200_E_ARG, "ie_b200_sample: NULL pointer");
  if (((uintptr_t)d_x | (uintptr_t)d_idx | (uintptr_t)d_prob | (uintptr_t)d_u | (uintptr_t)d_temp | (uintptr_t)d_top_k | (uintptr_t)d_top_p | (uintptr_t)d_min_p | x_stride) & 3u)
    return fail(IE_B200_E_ARG, "ie_b200_sample: pointers and strides must be 4-byte aligned");
  if (n == 0 || n > SM_MAX_SLICE * SM_MAX_CL) return fail(IE_B200_E_SIZE, "ie_b200_sample: rows of %u logits (1 .. %u)", n, SM_MAX_SLICE * SM_MAX_CL);
  if (T > (1u << 20) || (T > 1u && x_stride < (size_t)n * 4u)) return fail(IE_B200_E_SIZE, "ie_b200_sample: %u rows (at most 2^20) %zu bytes apart", T, x_stride);
  SampleArgs a = {d_x, d_u, d_temp, d_top_p, d_min_p, d_top_k, d_idx, d_prob, n, 0u, sample_ctas(n, T), 0u, 0u, 0, x_stride};
  a.sorted = d_top_p && T <= (uint32_t)SM_THREADS && T * a.cl > 2u * (uint32_t)sm_count();
  a.slice = ((n + a.cl - 1u) / a.cl + 3u) & ~3u;
  a.wide = (((uintptr_t)d_x | (T > 1u ? x_stride : 0u)) & 15u) == 0u;
  int log2n = 0;
  while ((1u << log2n) < n) log2n++;
  a.frac = 62 - log2n < 50 ? 62 - log2n : 50;
  const size_t smem = SM_FRONT + (size_t)a.slice * 4u;
  if (int r = ensure_dynamic_smem(reinterpret_cast<const void *>(sample_kernel), smem)) return r;
  const cudaError_t e = launch_pdl_cluster(sample_kernel, dim3(T * a.cl), dim3(SM_THREADS), smem, static_cast<cudaStream_t>(stream), a.cl, a);
  count_launch();
  return e == cudaSuccess ? IE_B200_OK : cuda_fail(e, "sample_kernel");
}
