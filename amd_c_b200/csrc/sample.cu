// sample.cu -- the draw of the next token of each row of logits: temperature, top-k, top-p, min-p, and a uniform number per row.
//
// w_i = exp((x_i - max) / temp). The tokens in the order (logit falling, index rising): the first k; of these the shortest run from the
// top whose mass reaches p times their mass; of these the ones with w_i >= min_p. Drawn is the first of them, by index, whose
// running sum exceeds u times the sum of all.
//
// A draw goes by which side of a sum a number falls, and a row has 10^5 such borders; sums that are off by 1e-7 would move a border
// past u once in some hundred draws. So weights are fixed-point integers, 2^F for the largest, F = 62 - log2 of the row's length (44 for 2^18
// tokens): their sums are exact and the same in any order, each weight is off by at most half a unit and the error of the exponential
// (2^-50: double, a table of 2^(j/64) and a polynomial of degree 5).
//
// One thread-block cluster per row, each CTA with its slice of the row in shared memory: the logits are read from HBM once, all
// further passes stay on chip, and what the CTAs find meets in each other's shared memory. Bound: 4 bytes per logit for many
// rows; for few the chain of passes and cluster barriers.
//  - top-k up to 1024: with j = ceil(k / CTAs), the j-th largest of the 512 threads' own maxima (rounded down to a bin of a histogram of
//    their leading bits) is a lower bound of each CTA; the smallest of the CTAs' is one for the row: at least k tokens reach it, and few
//    more. They go to the first CTA, which sorts them and does the rest alone.
//  - everything else: the border of a run (by count or by mass) from a histogram over the cluster, 2048 bins of 1/64 of a power of two of
//    the weight, whose bin on the border is sorted by the first CTA, or, where it holds too many, split further by the bits of the
//    logits until what is left are equal ones; those are counted off by index.
#include <float.h>
#include <math.h>

#include "common.cuh"

namespace ieb {

constexpr int SM_THREADS = 512, SM_WARPS = SM_THREADS / 32, SM_BINS = 2048, SM_LIST = 1024, SM_MAX_CL = 8;
constexpr uint32_t SM_MAX_SLICE = 45056;  // floats of a CTA's slice: 176 KB
constexpr uint32_t SM_NONE = 0xFFFFFFFFu;

struct SampleArgs {
  const float *x, *u, *temp, *top_p, *min_p;
  const uint32_t *top_k;
  uint32_t *out;
  uint32_t n, slice, cl, wide;
  int frac;  // F
  size_t x_stride, out_stride;
};

// A CTA's shared memory in front of its slice.
struct SampleSmem {
  uint64_t hist[SM_BINS];            // masses (or counts) of the bins; as u32: counts of the threads' maxima
  uint64_t list[SM_LIST];            // (key, ~index) of the row's candidates (first CTA)
  uint64_t mine[SM_LIST];            // this CTA's candidates
  uint64_t range[SM_MAX_CL];         // masses of the CTAs' ranges of bins, or of their slices
  uint64_t wsum[2 * SM_WARPS + 2];   // of the warps
  double pow2[64];                   // 2^(F + j / 64)
  float max_v[SM_MAX_CL];
  uint32_t max_i[SM_MAX_CL], floor_key[SM_MAX_CL];
  uint32_t n_list, n_mine, base, bin;
  uint64_t above;
  uint32_t cut_key, cut_idx;
};

// Floats in an order of unsigned integers; NaN has been taken for -inf.
__device__ __forceinline__ uint32_t sm_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // (-0 is 0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sm_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

__device__ __forceinline__ void dsm_st64(uint32_t a, uint64_t v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory"); }
__device__ __forceinline__ void dsm_st32(uint32_t a, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ uint64_t dsm_ld64(uint32_t a) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t dsm_add32(uint32_t a, uint32_t v) {
  uint32_t old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(a), "r"(v) : "memory");
  return old;
}

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ uint64_t warp_scan64(uint64_t v, int lane) {  // inclusive
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t w = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += w;
  }
  return v;
}

struct Sampler {
  const SampleArgs &a;
  SampleSmem &s;
  float *xs;  // the slice
  uint32_t rank, cl, begin, count;  // of the cluster; first token and tokens of the slice
  float xmax, c32;                  // c32: log2(e) / temp
  double c64, min_w;                // 64 log2(e) / temp; min_p in units of the weights
  float far;                        // log2 distance from which a weight is not needed (0, or below min_p)
  uint32_t tid, warp, lane;

  __device__ __forceinline__ uint32_t peer(const void *p, uint32_t cta) const { return cluster_map_shared(p, cta); }

  __device__ __forceinline__ float distance(float x) const { return (xmax - x) * c32; }  // in powers of two; never falls where x falls
  __device__ __forceinline__ uint64_t weight(float x) const {
    if (x == xmax) return 1ull << a.frac;
    const double t = ((double)x - (double)xmax) * c64;
    if (!(t > -64.0 * (a.frac + 1))) return 0u;
    const double m = t + 6755399441055744.0, f = t - (m - 6755399441055744.0);  // the nearest integer, in the low bits of m; the rest
    const int k = __double2loint(m);
    constexpr double L = 0.010830424696249145;  // ln 2 / 64
    double p = fma(f, L * L * L * L * L / 120.0, L * L * L * L / 24.0);
    p = fma(f, p, L * L * L / 6.0), p = fma(f, p, L * L / 2.0), p = fma(f, p, L), p = fma(f, p, 1.0);
    p *= s.pow2[k & 63];
    p = __hiloint2double(__double2hiint(p) + ((k >> 6) << 20), __double2loint(p));  // at least 2^-2: no underflow
    return (uint64_t)__double_as_longlong(p + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;  // rounded to an integer
  }

  // f(x, index) for every token of the slice, a thread's in rising order
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (uint32_t q = tid; q * 4u < count; q += SM_THREADS) {
      const float4 v = *reinterpret_cast<const float4 *>(xs + 4u * q);
      f(v.x, begin + 4u * q), f(v.y, begin + 4u * q + 1u), f(v.z, begin + 4u * q + 2u), f(v.w, begin + 4u * q + 3u);
    }
  }

  // The border of a run in the cluster's histogram: the first bin at which `above` and the bins up to it reach `goal`
  // (goal_of(mass of all bins)). In: this CTA's hist, complete after a __syncthreads. Out, in every CTA: s.bin and s.above, the mass
  // ahead of the bin.
  template <typename G>
  __device__ void border(uint64_t above, G goal_of) {
    cluster_sync_all();
    const uint32_t per_cta = SM_BINS / cl, per = per_cta > SM_THREADS ? per_cta / SM_THREADS : 1u, b0 = rank * per_cta + tid * per;
    uint64_t v[SM_BINS / SM_THREADS], sum = 0u;
    for (uint32_t i = 0; i < SM_BINS / SM_THREADS; i++) {
      v[i] = 0u;
      if (i < per && tid * per + i < per_cta)
        for (uint32_t c = 0; c < cl; c++) v[i] += dsm_ld64(peer(&s.hist[b0 + i], c));
      sum += v[i];
    }
    const uint64_t incl = warp_scan64(sum, lane);
    if (lane == 31) s.wsum[warp] = incl;
    __syncthreads();
    uint64_t before = incl - sum, mine = 0u;
    for (uint32_t w = 0; w < SM_WARPS; w++) {
      if (w < warp) before += s.wsum[w];
      mine += s.wsum[w];
    }
    if (tid < cl) dsm_st64(peer(&s.range[rank], tid), mine);
    cluster_sync_all();
    uint64_t all = 0u, ahead = above;
    for (uint32_t c = 0; c < cl; c++) {
      if (c < rank) ahead += s.range[c];
      all += s.range[c];
    }
    const uint64_t goal = goal_of(all);
    before += ahead;
    for (uint32_t i = 0; i < SM_BINS / SM_THREADS; i++) {
      if (before < goal && goal <= before + v[i])  // one thread of the cluster
        for (uint32_t c = 0; c < cl; c++) dsm_st32(peer(&s.bin, c), b0 + i), dsm_st64(peer(&s.above, c), before);
      before += v[i];
    }
    cluster_sync_all();
  }

  // The tokens that `in` picks into the first CTA's list; how many there are (more than SM_LIST: the list is not whole).
  template <typename F>
  __device__ uint32_t gather(F in) {
    if (tid == 0) s.n_mine = 0u, s.n_list = 0u;
    cluster_sync_all();
    each([&](float x, uint32_t i) {
      if (in(x, i)) {
        const uint32_t at = atomicAdd(&s.n_mine, 1u);
        if (at < SM_LIST) s.mine[at] = (uint64_t)sm_key(x) << 32 | (uint32_t)~i;
      }
    });
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

  // v[0 .. n - 1] falling (one CTA; n at most SM_LIST, room up to the next power of two; the fill sorts to the end)
  __device__ void sort_falling(uint64_t *v, uint32_t n) const {
    uint32_t m = 2u;
    while (m < n) m <<= 1;
    for (uint32_t i = n + tid; i < m; i += SM_THREADS) v[i] = 0u;
    __syncthreads();
    for (uint32_t size = 2; size <= m; size <<= 1)
      for (uint32_t step = size >> 1; step; step >>= 1) {
        for (uint32_t t = tid; t < m / 2u; t += SM_THREADS) {
          const uint32_t i = 2u * t - (t & (step - 1u)), j = i + step;
          const uint64_t p = v[i], q = v[j];
          if ((p < q) == ((i & size) == 0u)) v[i] = q, v[j] = p;
        }
        // pairs up to 32 apart stay within the 64 values of a warp, this step and the next ones
        if (step > 32u || (step == 1u && size >= 64u)) __syncthreads();
        else __syncwarp();
      }
    __syncthreads();
  }

  // The sum of f over the CTA's threads ahead of this one, and of all of them.
  __device__ uint64_t block_before(uint64_t v, uint64_t &all) {
    const uint64_t incl = warp_scan64(v, lane);
    __syncthreads();
    if (lane == 31) s.wsum[warp] = incl;
    __syncthreads();
    uint64_t before = incl - v;
    all = 0u;
    for (uint32_t w = 0; w < SM_WARPS; w++) {
      if (w < warp) before += s.wsum[w];
      all += s.wsum[w];
    }
    return before;
  }

  __device__ __forceinline__ bool kept(float x, uint32_t i) const {
    const uint32_t k = sm_key(x);
    return k > s.cut_key || (k == s.cut_key && i <= s.cut_idx);
  }

  // The cut (the last kept token of the run) at which the mass of the kept tokens, taken from the top, reaches a goal. MASS: weights, the
  // goal p times the mass of all kept; otherwise counts, the goal k.
  template <bool MASS>
  __device__ void cut_run(double p, uint32_t k) {
    auto mass = [&](float x) { return MASS ? weight(x) : (uint64_t)1u; };
    uint64_t goal = k;
    auto goal_of = [&](uint64_t all) {
      const double g = ceil(p * (double)all);
      return g < 1.0 ? (uint64_t)1u : min(all, (uint64_t)g);
    };
    // round 0: bins of the weights (MASS); then 11, 11 and 10 bits of the key
    uint32_t coarse = 0u, prefix = 0u, bits = 0u;  // the bin of round 0, the leading bits of the key so far
    auto in_prefix = [&](float x) {
      return (!MASS || min((uint32_t)(SM_BINS - 1), (uint32_t)(distance(x) * 64.0f)) == coarse) && (bits == 0u || sm_key(x) >> (32u - bits) == prefix);
    };
    uint64_t above = 0u;
    for (int round = MASS ? 0 : 1; round < 4; round++) {
      const uint32_t w = round == 3 ? 10u : 11u;
      for (uint32_t i = tid; i < SM_BINS; i += SM_THREADS) s.hist[i] = 0u;
      __syncthreads();
      if (MASS && round == 0) {
        each([&](float x, uint32_t i) {
          if (kept(x, i)) {
            const uint64_t v = weight(x);
            if (v) atomicAdd(reinterpret_cast<unsigned long long *>(&s.hist[min((uint32_t)(SM_BINS - 1), (uint32_t)(distance(x) * 64.0f))]), (unsigned long long)v);
          }
        });
        border(0u, [&](uint64_t all) { return goal = goal_of(all); });
        coarse = s.bin;
      } else {
        each([&](float x, uint32_t i) {
          if (kept(x, i) && in_prefix(x)) {
            const uint32_t digit = (sm_key(x) >> (32u - bits - w)) & ((1u << w) - 1u);
            atomicAdd(reinterpret_cast<unsigned long long *>(&s.hist[(1u << w) - 1u - digit]), (unsigned long long)mass(x));
          }
        });
        border(above, [&](uint64_t) { return goal; });
        prefix = prefix << w | ((1u << w) - 1u - s.bin), bits += w;
      }
      above = s.above;
      const uint32_t n = gather([&](float x, uint32_t i) { return kept(x, i) && in_prefix(x); });
      if (n <= (uint32_t)SM_LIST) {
        if (rank == 0u) {
          sort_falling(s.list, n);
          uint64_t at = above;
          for (uint32_t i0 = 0; i0 < n; i0 += SM_THREADS) {  // at most two rounds
            uint64_t all;
            const uint32_t i = i0 + tid;
            const uint64_t v = i < n ? mass(sm_unkey((uint32_t)(s.list[i] >> 32))) : 0u, before = at + block_before(v, all);
            if (i < n && before < goal && goal <= before + v)  // one thread
              for (uint32_t c = 0; c < cl; c++) dsm_st32(peer(&s.cut_key, c), (uint32_t)(s.list[i] >> 32)), dsm_st32(peer(&s.cut_idx, c), ~(uint32_t)s.list[i]);
            at += all;
          }
        }
        cluster_sync_all();
        return;
      }
    }
    // what is left are equal logits: as many of them as the goal takes, by index
    const float x = sm_unkey(prefix);
    const uint64_t w = mass(x), need = (goal - above + w - 1u) / w;
    uint32_t idx;
    uint64_t v, all;
    locate([&](float y, uint32_t i) { return (uint64_t)(kept(y, i) && sm_key(y) == prefix); }, [&](uint64_t) { return need - 1u; }, idx, v, all);
    cluster_sync_all();  // (everybody has read the old cut)
    if (tid == 0) s.cut_key = prefix, s.cut_idx = idx;
    __syncthreads();
  }

  // The first token, by index, at which the running sum of f exceeds goal_of(sum of all); its f and the sum. In every CTA (idx is SM_NONE if
  // there is none).
  template <typename F, typename G>
  __device__ void locate(F f, G goal_of, uint32_t &idx, uint64_t &value, uint64_t &all) {
    // sums of the 128 tokens that a warp takes at a time, in the order of the indices: [step][warp]
    uint64_t *part = s.hist;
    const uint32_t quads = (count + 3u) / 4u, steps = (quads + SM_THREADS - 1u) / SM_THREADS;
    __syncthreads();
    if (tid == 0) s.bin = SM_NONE;
    uint64_t mine = 0u;
    auto quad = [&](uint32_t q, uint64_t (&v)[4]) {
      v[0] = v[1] = v[2] = v[3] = 0u;
      if (q < quads) {
        const float4 x = *reinterpret_cast<const float4 *>(xs + 4u * q);
        v[0] = f(x.x, begin + 4u * q), v[1] = f(x.y, begin + 4u * q + 1u), v[2] = f(x.z, begin + 4u * q + 2u), v[3] = f(x.w, begin + 4u * q + 3u);
      }
    };
    for (uint32_t k = 0; k < steps; k++) {
      uint64_t v[4];
      quad(k * SM_THREADS + tid, v);
      const uint64_t sum = warp_sum64(v[0] + v[1] + v[2] + v[3]);
      if (lane == 0) part[k * SM_WARPS + warp] = sum;
      mine += sum;
    }
    if (lane == 0) s.wsum[warp] = mine;
    __syncthreads();
    mine = 0u;
    for (uint32_t w = 0; w < SM_WARPS; w++) mine += s.wsum[w];
    if (tid < cl) dsm_st64(peer(&s.range[rank], tid), mine);
    cluster_sync_all();
    uint64_t before = 0u;
    all = 0u;
    for (uint32_t c = 0; c < cl; c++) {
      if (c < rank) before += s.range[c];
      all += s.range[c];
    }
    const uint64_t goal = goal_of(all);
    if (warp == 0 && before <= goal && goal < before + mine) {  // one CTA: the step and warp, then the token
      uint32_t at = 0u;
      for (uint32_t p0 = 0; p0 < steps * SM_WARPS; p0 += 32u) {
        const uint64_t v = p0 + lane < steps * SM_WARPS ? part[p0 + lane] : 0u, incl = before + warp_scan64(v, lane);
        const uint32_t over = __ballot_sync(0xFFFFFFFFu, incl > goal);
        if (over) {
          const int l = __ffs(over) - 1;
          at = p0 + l, before = __shfl_sync(0xFFFFFFFFu, incl - v, l);
          break;
        }
        before = __shfl_sync(0xFFFFFFFFu, incl, 31);
      }
      const uint32_t q = (at / SM_WARPS) * SM_THREADS + (at % SM_WARPS) * 32u + lane;
      uint64_t v[4];
      quad(q, v);
      uint64_t run = before + warp_scan64(v[0] + v[1] + v[2] + v[3], lane) - (v[0] + v[1] + v[2] + v[3]);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (run <= goal && goal < run + v[e])  // one thread of the cluster
          for (uint32_t c = 0; c < cl; c++) dsm_st32(peer(&s.bin, c), begin + 4u * q + e), dsm_st64(peer(&s.above, c), v[e]);
        run += v[e];
      }
    }
    cluster_sync_all();
    idx = s.bin, value = s.above;
  }
};

// u times the sum as a running sum of integers is compared with: exceeded means at least one more
__device__ __forceinline__ uint64_t sample_goal(float u, uint64_t all) {
  const double g = (double)u * (double)all;
  return g > 0.0 ? min((uint64_t)min(g, 9.2e18), all - 1u) : 0u;
}

__device__ __forceinline__ void sample_out(const SampleArgs &a, uint32_t row, uint32_t idx, float prob) {
  uint32_t *o = reinterpret_cast<uint32_t *>(reinterpret_cast<char *>(a.out) + a.out_stride * row);
  o[0] = idx, o[1] = __float_as_uint(prob);
}

__global__ void __launch_bounds__(SM_THREADS) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem_s[];
  SampleSmem &s = *reinterpret_cast<SampleSmem *>(smem_s);
  cluster_arrive();  // (waited for ahead of the first store into a peer, which has to run by then)
  pdl_prologue();
  const uint32_t row = blockIdx.x / a.cl, rank = blockIdx.x % a.cl, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cl = a.cl;
  const uint32_t begin = min(a.n, rank * a.slice), count = min(a.n, begin + a.slice) - begin;
  float *xs = reinterpret_cast<float *>(smem_s + ((sizeof(SampleSmem) + 15u) & ~(size_t)15u));
  const float temp = a.temp ? a.temp[row] : 1.0f, top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p ? a.min_p[row] : 0.0f, u = a.u[row];
  const uint32_t top_k = a.top_k ? a.top_k[row] : 0u;
  const bool greedy = !(temp > 0.0f), by_k = !greedy && top_k > 0u && top_k < a.n;

  // ---- the slice, its maximum, and the threads' own maxima
  for (uint32_t i = tid; i < SM_BINS / 2u; i += SM_THREADS) s.hist[i] = 0u;  // 2048 counts of 32 bits
  const float *x = reinterpret_cast<const float *>(reinterpret_cast<const char *>(a.x) + a.x_stride * row) + begin;
  float mx = -INFINITY;
  uint32_t mi = SM_NONE;
  for (uint32_t q = tid; q * 4u < count; q += SM_THREADS) {
    float v[4];
    if (a.wide && q * 4u + 4u <= count) {
      const float4 f = *reinterpret_cast<const float4 *>(x + 4u * q);
      v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = q * 4u + e < count ? x[4u * q + e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (!(v[e] >= -INFINITY)) v[e] = -INFINITY;  // a NaN is never drawn
      if (v[e] > mx) mx = v[e], mi = begin + 4u * q + e;
    }
    *reinterpret_cast<float4 *>(xs + 4u * q) = make_float4(v[0], v[1], v[2], v[3]);
  }
  __syncthreads();
  uint32_t *counts = reinterpret_cast<uint32_t *>(s.hist);
  if (by_k) atomicAdd(&counts[SM_BINS - 1u - (sm_key(mx) >> 21)], 1u);
  {
    float bv = mx;
    uint32_t bi = mi;
    for (int o = 16; o; o >>= 1) {
      const float ov = __shfl_xor_sync(0xFFFFFFFFu, bv, o);
      const uint32_t oi = __shfl_xor_sync(0xFFFFFFFFu, bi, o);
      if (ov > bv || (ov == bv && oi < bi)) bv = ov, bi = oi;
    }
    if (lane == 0) s.wsum[warp] = (uint64_t)sm_key(bv) << 32 | (uint32_t)~bi;
  }
  if (tid < 64u) s.pow2[tid] = scalbn(exp2((double)tid / 64.0), a.frac);
  __syncthreads();
  cluster_wait();
  if (warp == 0) {
    uint64_t b = lane < SM_WARPS ? s.wsum[lane] : 0u;
    for (int o = 16; o; o >>= 1) b = max(b, (uint64_t)__shfl_xor_sync(0xFFFFFFFFu, b, o));
    if (lane < cl) {
      dsm_st32(cluster_map_shared(&s.max_v[rank], lane), __float_as_uint(sm_unkey((uint32_t)(b >> 32))));
      dsm_st32(cluster_map_shared(&s.max_i[rank], lane), ~(uint32_t)b);
    }
  }
  if (by_k) {  // the bin of the threads' maxima at which j of them are reached, its lower end
    const uint32_t j = (top_k + cl - 1u) / cl;
    uint32_t c4[4], sum = 0u;
#pragma unroll
    for (int e = 0; e < 4; e++) c4[e] = counts[4u * tid + e], sum += c4[e];
    uint32_t incl = sum;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if ((int)lane >= o) incl += v;
    }
    uint32_t *ws = reinterpret_cast<uint32_t *>(s.wsum + SM_WARPS);
    if (lane == 31) ws[warp] = incl;
    if (tid == 0) s.bin = SM_NONE;
    __syncthreads();
    uint32_t before = incl - sum;
    for (uint32_t w = 0; w < warp; w++) before += ws[w];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (before < j && j <= before + c4[e]) s.bin = 4u * tid + e;
      before += c4[e];
    }
    __syncthreads();
    if (tid < cl) dsm_st32(cluster_map_shared(&s.floor_key[rank], tid), s.bin == SM_NONE ? 0u : (SM_BINS - 1u - s.bin) << 21);
  }
  cluster_sync_all();
  float xmax = -INFINITY;
  uint32_t imax = SM_NONE, floor_key = SM_NONE;
  for (uint32_t c = 0; c < cl; c++) {
    if (s.max_v[c] > xmax) xmax = s.max_v[c], imax = s.max_i[c];
    if (by_k) floor_key = min(floor_key, s.floor_key[c]);
  }
  if (greedy || imax == SM_NONE) {
    if (rank == 0u && tid == 0u) sample_out(a, row, imax, imax == SM_NONE ? 0.0f : 1.0f);
    return;
  }

  Sampler S = {a, s, xs, rank, cl, begin, count, xmax, 0.0f, 0.0, 0.0, 0.0f, tid, warp, lane};
  S.c64 = 64.0 * 1.4426950408889634 / (double)temp, S.c32 = (float)(S.c64 / 64.0);
  const float mp = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;
  S.min_w = (double)mp * (double)(1ull << a.frac);
  S.far = fminf((float)(a.frac + 2), mp > 0.0f ? 0.01f - log2f(mp) : INFINITY);
  const bool by_p = top_p < 1.0f;  // (a NaN: off)
  auto heavy = [&](uint64_t w) { return w && (double)w >= S.min_w; };

  if (by_k && top_k <= (uint32_t)SM_LIST) {
    const uint32_t n = S.gather([&](float v, uint32_t) { return sm_key(v) >= floor_key && v > -INFINITY; });
    if (n <= (uint32_t)SM_LIST) {
      if (rank != 0u) return;
      S.sort_falling(s.list, n);
      const uint32_t k = min(top_k, n);
      uint64_t w[2], before[2], sums[2] = {0u, 0u};
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const uint32_t i = r * SM_THREADS + tid;
        w[r] = i < k ? S.weight(sm_unkey((uint32_t)(s.list[i] >> 32))) : 0u;
        before[r] = S.block_before(w[r], sums[r]);
      }
      before[1] += sums[0];
      const double g = by_p ? (double)top_p * (double)(sums[0] + sums[1]) : INFINITY;
#pragma unroll
      for (int r = 0; r < 2; r++) {  // what is kept, by index: (~index, place)
        const uint32_t i = r * SM_THREADS + tid;
        const bool keep = i < k && ((double)before[r] < g || i == 0u) && heavy(w[r]);
        if (i < k) s.mine[i] = keep ? (s.list[i] << 32 | i) : 0u;
        if (i < k) s.hist[i] = w[r];
      }
      __syncthreads();
      S.sort_falling(s.mine, k);  // (tokens left out go to the end; index 0xFFFFFFFF does not exist, so no kept one is 0)
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const uint32_t i = r * SM_THREADS + tid;
        const uint64_t e = i < k ? s.mine[i] : 0u;
        w[r] = e ? s.hist[(uint32_t)e] : 0u;
        before[r] = S.block_before(w[r], sums[r]);
      }
      before[1] += sums[0];
      const uint64_t all = sums[0] + sums[1], goal = sample_goal(u, all);
#pragma unroll
      for (int r = 0; r < 2; r++)
        if (before[r] <= goal && goal < before[r] + w[r])  // one thread
          sample_out(a, row, ~(uint32_t)(s.mine[r * SM_THREADS + tid] >> 32), (float)((double)w[r] / (double)all));
      return;
    }
  }
  if (tid == 0) s.cut_key = 0u, s.cut_idx = SM_NONE;
  __syncthreads();
  if (by_k) S.cut_run<false>(0.0, top_k);
  if (by_p) S.cut_run<true>((double)top_p, 0u);
  uint32_t idx;
  uint64_t w, all;
  S.locate(
      [&](float v, uint32_t i) {
        if (!(S.distance(v) <= S.far) && v != xmax) return (uint64_t)0u;
        if (!S.kept(v, i)) return (uint64_t)0u;
        const uint64_t r = S.weight(v);
        return heavy(r) ? r : (uint64_t)0u;
      },
      [&](uint64_t sum) { return sample_goal(u, sum); }, idx, w, all);
  if (rank == 0u && tid == 0u) sample_out(a, row, idx, (float)((double)w / (double)all));
}

// CTAs of a row
static uint32_t sample_ctas(uint32_t n) { return n <= 4096u ? 1u : n <= 16384u ? 2u : n <= 49152u ? 4u : 8u; }

}  // namespace ieb

using namespace ieb;

extern "C" int ie_b200_sample(const float *d_x, uint32_t n, uint32_t *d_out, const float *d_u, const float *d_temp, const uint32_t *d_top_k, const float *d_top_p,
                              const float *d_min_p, uint32_t T, size_t x_stride, size_t out_stride, void *stream) {
  if (T == 0) return IE_B200_OK;  // (an empty tensor may have no address)
  if (!d_x || !d_out || !d_u) return fail(IE_B200_E_ARG, "ie_b200_sample: NULL pointer");
  if (((uintptr_t)d_x | (uintptr_t)d_out | (uintptr_t)d_u | (uintptr_t)d_temp | (uintptr_t)d_top_k | (uintptr_t)d_top_p | (uintptr_t)d_min_p | x_stride | out_stride) & 3u)
    return fail(IE_B200_E_ARG, "ie_b200_sample: pointers and strides must be 4-byte aligned");
  if (n == 0 || n > SM_MAX_SLICE * SM_MAX_CL) return fail(IE_B200_E_SIZE, "ie_b200_sample: rows of %u logits (1 .. %u)", n, SM_MAX_SLICE * SM_MAX_CL);
  if (T > (1u << 20) || (T > 1u && (x_stride < (size_t)n * 4u || out_stride < 8u)))
    return fail(IE_B200_E_SIZE, "ie_b200_sample: %u rows (at most 2^20) %zu bytes apart, results %zu", T, x_stride, out_stride);
  SampleArgs a = {d_x, d_u, d_temp, d_top_p, d_min_p, d_top_k, d_out, n, 0u, sample_ctas(n), 0u, 0, x_stride, out_stride};
  a.slice = ((n + a.cl - 1u) / a.cl + 3u) & ~3u;
  a.wide = (((uintptr_t)d_x | (T > 1u ? x_stride : 0u)) & 15u) == 0u;
  int log2n = 0;
  while ((1u << log2n) < n) log2n++;
  a.frac = 62 - log2n < 50 ? 62 - log2n : 50;
  const size_t smem = ((sizeof(SampleSmem) + 15u) & ~(size_t)15u) + (size_t)a.slice * 4u;
  if (int r = ensure_dynamic_smem(reinterpret_cast<const void *>(sample_kernel), smem)) return r;
  const cudaError_t e = launch_pdl_cluster(sample_kernel, dim3(T * a.cl), dim3(SM_THREADS), smem, static_cast<cudaStream_t>(stream), a.cl, a);
  count_launch();
  return e == cudaSuccess ? IE_B200_OK : cuda_fail(e, "sample_kernel");
}
