// attn_paged.cu -- attention of one new token per row over a paged KV cache, for a batch of rows of any lengths.
//
// For row r and query head h of KV head g: out = sum_p w_p v_p / sum_p w_p with w_p = exp(q . k_p / sqrt(hd) - max), over the
// positions p < len[r] of its sequence. K and V of a KV head are read once for all its query heads (up to eight; more come in groups,
// the later of which find the rows in L2). Bound: HBM, 2 len n_kv hd sizeof(KV) bytes a row.
//
// Work. A chunk is CH positions of one (row, KV head, head group); pages hold whole chunks, so a chunk is one contiguous run of K and
// one of V. All chunks of the batch, in that order, are cut into even shares, one per CTA, wherever the cuts fall: the CTAs finish
// together whatever the lengths are. A CTA finds its share by a prefix sum over the rows' lengths. Its four or eight warps take the chunks of
// a unit (row, KV head, group) in turn; each warp has its own ring of buffers that it fills itself (cp.async, rows past the length
// zero-filled) and its own running maximum, sum and outputs, so nothing in the stream waits for another warp, and the ring runs on into
// the next unit while this one's records are merged. A unit that lies in one CTA is finished there; the parts of a cut one go to
// global memory as (outputs, max, sum) records, and the CTA that finishes last adds them in the order of the positions. Where units are
// many and short, each is one warp's instead, and nothing meets.
//
// Half cache: mma.sync m16n8k16, the positions on the 16-row side, the heads on the 8-column side (as attn_decode.cu). q and the
// weights are carried as two f16 terms; every accumulation takes few MMAs (what the tensor cores cut off grows with their number) and is
// added up in fp32: S in three chains (low terms, even and odd steps of the high ones), O per chunk. f16's subnormals end at 2^-24, so both are
// scaled before they are split, for the low terms to keep their bits: the weights by 2^15, a head's q by the power of two that takes its largest
// value to 2^14 .. 2^15 (22 bits of every value down to 2^-17 of the largest, 2^-39 of that below, whatever q's size is).
// Float cache: the same with fp32 FMAs, four lanes per position.
//
// Measured (half cache, heads of 128): 256 rows of 1000 positions, 32 x 8 heads, 164 .. 167 us = 6.3 TB/s, 97 % of the measured copy rate; 64 rows of 1 to
// 8192, 28 x 4, 91 us = 6.0 TB/s; 1 of 32768, 40 x 8, 29.3 us (the contiguous kernel of attn_decode.cu 34 us with 32 x 8), of which
// 4 us are the start (length, page number, first rows: dependent round trips) and 4 the merge of 18 parts; 1 of 500, 8.1 us. Float cache, heads of
// 128: 64 rows of up to 3001, 132 us = 6.3 TB/s; of 64: 253 rows of 868 141 us = 6.4 TB/s.
#include <cuda_pipeline_primitives.h>
#include <math.h>
#include <type_traits>

#include "paged.cuh"
#include "row_store.cuh"

namespace ieb {

constexpr int AP_HEADS = 8;
constexpr uint32_t AP_MAX_CTAS = 1024u;  // the counters at the front of the scratch

struct PagedAttnArgs {
  const float *q;
  float *out, *rec;
  uint8_t *oq;
  const uint32_t *len, *seq;
  uint32_t *count, *err;
  ie_b200_kv_pages kv;
  uint32_t n_head, G, groups, gw, R, wide, seq0;  // groups: head groups of a KV head, gw heads each (the last may have fewer); seq0: sequence of row 0 where seq is NULL
  uint32_t min_share, most, fill;  // most: rows of a launch; fill: outputs whose rows of padding are zeros (1: out, 2: oq)
  uint32_t cpp, step_col, step_off;  // chunks of a page; a warp's step from chunk to chunk, in pages and chunks
  size_t q_stride, out_stride, oq_stride;
  float scale_log2;  // log2(e) / sqrt(hd)
};

// W: warps of a CTA
template <typename KV, int HD, int W>
struct ApGeom {
  static constexpr bool F16 = sizeof(KV) == 2;
  static constexpr int STAGES = HD == 32 ? 5 : HD == 128 ? 3 : W == 4 ? 4 : F16 ? 3 : 5;  // buffers of a warp
  static constexpr int CH = F16 ? 16 : 8;                       // positions of a chunk
  static constexpr int ROWB = HD * (int)sizeof(KV), PIECES = ROWB / 16, PER_LANE = CH * PIECES / 32;
  static constexpr int STAGE = 2 * CH * ROWB;                   // K rows, then V rows
  static constexpr bool PAIRS = F16 && HD <= 64 && STAGES >= 4;  // two chunks worked on at once, where they are short (256 x 1000 of 16 x 16 heads of 64 167 -> 161 us, of 8 x 4 of 32 32.2 -> 30.3)
  static constexpr int REC_ROW = HD + 4;                        // floats between the heads of a record in global memory: outputs, max, sum
  static constexpr int RING_OFF = 0, RED_OFF = W * STAGES * STAGE, ML_OFF = RED_OFF + W * AP_HEADS * HD * 4,
                       VALID_OFF = ML_OFF + W * AP_HEADS * 8, MISC_OFF = (VALID_OFF + W * STAGES * 4 + 15) / 16 * 16, TOTAL = MISC_OFF + 128,
                       Q_OFF = RED_OFF;  // float cache: the unit's q, until its records are written
  static constexpr int FIT = 228 * 1024 / (TOTAL + 1024), MOST = F16 || W == 4 ? 16 / W : 1, CTAS = FIT < MOST ? FIT : MOST;  // on an SM: what its shared memory and 128 registers a thread allow
  // Output d of head h in a warp's record in shared memory: the four head pairs that a store of the MMA's layout meets lie in different banks.
  __device__ static __forceinline__ uint32_t red_at(uint32_t h, uint32_t d) { return h * HD + (d ^ (h >> 1 & 3u) * 8u); }
  // The 16-byte pieces of a row change places so that the reads of eight rows (ldmatrix), or of two rows by four lanes each, meet
  // eight different bank groups.
  __device__ static __forceinline__ uint32_t at(uint32_t row, uint32_t piece) {
    const uint32_t x = F16 ? (HD == 32 ? (row >> 1) & 3u : row & 7u) : (row & 1u) * 4u;
    return row * ROWB + ((piece ^ x) * 16u);
  }
  // A lane's i-th piece (512 bytes from one to the next), from where its first one goes: the rows between are a power of two, above the lane's own row.
  __device__ static __forceinline__ uint32_t step(uint32_t first, int i) {
    const int row = 32 / PIECES * i;
    return (first ^ (F16 ? (HD == 32 ? (row >> 1) & 3 : row & 7) : (row & 1) * 4) * 16u) + 512u * i;
  }
};

__device__ __forceinline__ void ap_ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ap_ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t ap_movm_t(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void ap_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ap_split2(float x, float y, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 hf = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - hf.x, y - hf.y);
  hi = *reinterpret_cast<const uint32_t *>(&h), lo = *reinterpret_cast<const uint32_t *>(&l);
}

// ---- a warp's part of the arithmetic: its running maximum (log2 units), sum and outputs of the unit's heads. log2(e) / sqrt(hd) is multiplied into q, so that a
// score is in powers of two as it is summed (half cache: but for a whole power of two). The difference of the largest one to the maximum is then 0 and its weight
// 1, however large scores are; a maximum rounded after such a factor is off by half a unit in its last place, a whole power of two from 2^25 on, and
// a weight above 1 leaves half's range.
template <typename KV, int HD, int W>
struct ApWarp;

template <int HD, int W>
struct ApWarp<__half, HD, W> {
  using Gm = ApGeom<__half, HD, W>;
  static constexpr int KS = HD / 16;
  float2 q[KS][2];                // the next unit's q, on its way
  uint32_t qh[KS][2], ql[KS][2];  // B fragments of Q^T[16 dims x heads]: column lane / 4
  float o[KS][4], m[2], l[2];     // o[u][j], o[u][2 + j]: head 2 (lane % 4) + j, dims 16 u + lane / 4, + 8
  float unit[2];                  // what a sum for head 2 (lane % 4) + j counts for, a power of two

  __device__ __forceinline__ void load(const float *src, uint32_t heads, uint32_t tid) {
    const uint32_t h = (tid & 31u) >> 2, tq = tid & 3u;
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
      for (int e = 0; e < 2; e++) q[k][e] = h < heads ? *reinterpret_cast<const float2 *>(src + h * HD + 16 * k + 2 * tq + 8 * e) : make_float2(0.f, 0.f);
  }
  __device__ __forceinline__ void start(float scale_log2, uint32_t lane) {
    float part[2 * KS];  // (fmaxf passes over a NaN)
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
      for (int e = 0; e < 2; e++) part[2 * k + e] = fmaxf(fabsf(q[k][e].x), fabsf(q[k][e].y));
#pragma unroll
    for (int n = KS; n; n >>= 1)
#pragma unroll
      for (int i = 0; i < n; i++) part[i] = fmaxf(part[i], part[i + n]);
    float big = fmaxf(part[0], __shfl_xor_sync(0xFFFFFFFFu, part[0], 1));  // of head lane / 4
    big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2)) * scale_log2;
    // The power of two, times 2^127, that takes it to 2^14 .. 2^15; at most 2^100 (a q that small leaves all weights alike). A score takes it back, up to 2^88 of
    // what can be 2^38: above that a head has all its weight on its largest scores either way, and nothing passes fp32's end.
    const uint32_t up = min(268u - (__float_as_uint(big) >> 23), 227u), down = min(254u - up, 215u);
    const float scale = scale_log2 * __uint_as_float(up << 23);
#pragma unroll
    for (uint32_t j = 0; j < 2; j++) unit[j] = __uint_as_float(__shfl_sync(0xFFFFFFFFu, down, 8u * (lane & 3u) + 4u * j) << 23);
#pragma unroll
    for (int k = 0; k < KS; k++) {
#pragma unroll
      for (int e = 0; e < 2; e++) ap_split2(q[k][e].x * scale, q[k][e].y * scale, qh[k][e], ql[k][e]);
#pragma unroll
      for (int e = 0; e < 4; e++) o[k][e] = 0.0f;
    }
    m[0] = m[1] = -INFINITY, l[0] = l[1] = 0.0f;
  }
  // N chunks at once, each with `valid` positions
  template <int N>
  __device__ __forceinline__ void chunks(const uint8_t *const (&stage)[N], const uint32_t (&valid)[N], int lane) {
    const uint32_t lm = lane >> 3, lr = lane & 7, hq = lane >> 2;
    float s[N][4], al[2];  // s[.][j]: position lane / 4, s[.][2 + j]: + 8, of head 2 (lane % 4) + j
    float sl[N][4] = {}, s0[N][4] = {}, s1[N][4] = {};
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
      for (int n = 0; n < N; n++) {
        uint32_t a[4];  // (positions lo, dims lo), (positions hi, dims lo), (positions lo, dims hi), (positions hi, dims hi)
        ap_ldsm4(a, smem_u32(stage[n]) + Gm::at((lm & 1) * 8 + lr, 2 * k + (lm >> 1)));
        ap_mma(sl[n], a, ql[k][0], ql[k][1]);
        if (k & 1) ap_mma(s1[n], a, qh[k][0], qh[k][1]);
        else ap_mma(s0[n], a, qh[k][0], qh[k][1]);
      }
#pragma unroll
    for (int n = 0; n < N; n++) {
#pragma unroll
      for (int e = 0; e < 4; e++) s[n][e] = (s0[n][e] + s1[n][e]) + sl[n][e];
      if (valid[n] < 16u) {
        if (hq >= valid[n]) s[n][0] = s[n][1] = -INFINITY;
        if (hq + 8u >= valid[n]) s[n][2] = s[n][3] = -INFINITY;
      }
    }
#pragma unroll
    for (int j = 0; j < 2; j++) {
      float mx = fmaxf(s[0][j], s[0][2 + j]);
#pragma unroll
      for (int n = 1; n < N; n++) mx = fmaxf(mx, fmaxf(s[n][j], s[n][2 + j]));
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 4));
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 8));
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 16));
      const float m_new = fmaxf(m[j], mx * unit[j]), base = m_new == -INFINITY ? 0.0f : m_new;
      al[j] = ex2(m[j] - base);
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < N; n++) {  // from here on the weights
        s[n][j] = ex2(fmaf(s[n][j], unit[j], -base)), s[n][2 + j] = ex2(fmaf(s[n][2 + j], unit[j], -base));
        sum += s[n][j] + s[n][2 + j];
      }
      l[j] = fmaf(l[j], al[j], sum);  // (of this lane's positions: the lanes meet in finish())
      m[j] = m_new;
    }
    uint32_t ph[N][2], pl[N][2];  // each 8 x 8 block [positions x heads] transposed into the B fragment [positions x heads]
#pragma unroll
    for (int n = 0; n < N; n++) {
      ap_split2(s[n][0] * 0x1p15f, s[n][1] * 0x1p15f, ph[n][0], pl[n][0]);
      ap_split2(s[n][2] * 0x1p15f, s[n][3] * 0x1p15f, ph[n][1], pl[n][1]);
#pragma unroll
      for (int e = 0; e < 2; e++) ph[n][e] = ap_movm_t(ph[n][e]), pl[n][e] = ap_movm_t(pl[n][e]);
    }
#pragma unroll
    for (int u = 0; u < KS; u++) {
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < N; n++) {
        uint32_t a[4];  // transposed on load: (dims lo, positions lo), (dims hi, positions lo), (dims lo, positions hi), (dims hi, positions hi)
        ap_ldsm4t(a, smem_u32(stage[n]) + Gm::CH * Gm::ROWB + Gm::at((lm >> 1) * 8 + lr, 2 * u + (lm & 1)));
        ap_mma(c, a, pl[n][0], pl[n][1]);
        ap_mma(c, a, ph[n][0], ph[n][1]);
      }
#pragma unroll
      for (int e = 0; e < 4; e++) o[u][e] = fmaf(o[u][e], al[e & 1], c[e]);
    }
  }
  __device__ __forceinline__ void chunk(const uint8_t *stage, uint32_t valid, int lane) {
    const uint8_t *const st[1] = {stage};
    const uint32_t v[1] = {valid};
    chunks<1>(st, v, lane);
  }
  // this warp's record: red [heads][HD] outputs (2^15 times; red_at), ml [heads][2]
  __device__ __forceinline__ void finish(float *red, float *ml, int lane) {
    const uint32_t hq = lane >> 2, tq = lane & 3;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      float sum = l[j];
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 4);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 8);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 16);
      const uint32_t h = 2 * tq + j;
#pragma unroll
      for (int u = 0; u < KS; u++) red[Gm::red_at(h, 16 * u + hq)] = o[u][j], red[Gm::red_at(h, 16 * u + hq + 8)] = o[u][2 + j];
      if (hq == 0) ml[2 * h] = m[j], ml[2 * h + 1] = sum * 0x1p15f;
    }
  }
};

template <int HD, int W>
struct ApWarp<float, HD, W> {
  using Gm = ApGeom<float, HD, 4>;
  static constexpr int DPL = HD / 32;  // output dims of a lane
  float o[AP_HEADS][DPL], m[2], l[2];  // m, l: of heads lane % 4 and that + 4
  static constexpr int QPT = AP_HEADS * HD / (32 * W);
  float q[QPT];  // this thread's part of the next unit's q, on its way
  const float *qs;
  bool few;

  __device__ __forceinline__ void load(const float *src, uint32_t heads, uint32_t tid) {
#pragma unroll
    for (int i = 0; i < QPT; i++) q[i] = tid + 32u * W * i < heads * HD ? src[tid + 32u * W * i] : 0.0f;
  }
  // (All threads call it, behind a barrier after which nobody reads what is at q_smem.)
  __device__ __forceinline__ void start(uint32_t heads, float *q_smem, float scale_log2, uint32_t tid) {
#pragma unroll
    for (int i = 0; i < QPT; i++) q_smem[tid + 32u * W * i] = q[i] * scale_log2;
    __syncthreads();
    clear(heads, q_smem);
  }
  // The same for one warp, q from where it is.
  __device__ __forceinline__ void start_alone(const float *src, uint32_t heads, float *q_smem, float scale_log2, uint32_t lane) {
#pragma unroll 8
    for (uint32_t i = 4u * lane; i < heads * HD; i += 128u) {
      const float2 a = *reinterpret_cast<const float2 *>(src + i), b = *reinterpret_cast<const float2 *>(src + i + 2);
      *reinterpret_cast<float4 *>(q_smem + i) = make_float4(a.x * scale_log2, a.y * scale_log2, b.x * scale_log2, b.y * scale_log2);
    }
    for (uint32_t i = heads * HD + lane; i < AP_HEADS * HD; i += 32u) q_smem[i] = 0.0f;
    __syncwarp();
    clear(heads, q_smem);
  }
  __device__ __forceinline__ void clear(uint32_t heads, const float *q_smem) {
    few = heads <= 4u, qs = q_smem;
#pragma unroll
    for (int h = 0; h < AP_HEADS; h++)
#pragma unroll
      for (int d = 0; d < DPL; d++) o[h][d] = 0.0f;
    m[0] = m[1] = -INFINITY, l[0] = l[1] = 0.0f;
  }
  // H: heads worked on, 4 or 8 (half the arithmetic where the unit has no more than four)
  template <int H>
  __device__ __forceinline__ void chunk_of(uint8_t *stage, uint32_t valid, int lane) {
    const uint32_t pos = lane >> 2, part = lane & 3;  // lane: a quarter of the dims of one position
    float s[H];
#pragma unroll
    for (int h = 0; h < H; h++) s[h] = 0.0f;
#pragma unroll 4
    for (int i = 0; i < HD / 16; i++) {
      const uint32_t piece = 4 * i + part;
      const float4 k = *reinterpret_cast<const float4 *>(stage + Gm::at(pos, piece));
#pragma unroll
      for (int h = 0; h < H; h++) {
        const float4 x = *reinterpret_cast<const float4 *>(qs + h * HD + 4 * piece);
        s[h] = fmaf(x.x, k.x, s[h]), s[h] = fmaf(x.y, k.y, s[h]), s[h] = fmaf(x.z, k.z, s[h]), s[h] = fmaf(x.w, k.w, s[h]);
      }
    }
    // The four lanes' parts meet, and the heads part: lane `part` is left with the scores of head `part` and, of eight, of part + 4 (with all heads in
    // every lane, 253 x 868 of heads of 64 took 164 us for 141).
    const bool odd = part & 1u, upper = part & 2u;
    float t[H / 2];
#pragma unroll
    for (int i = 0; i < H / 2; i++) t[i] = (odd ? s[2 * i + 1] : s[2 * i]) + __shfl_xor_sync(0xFFFFFFFFu, odd ? s[2 * i] : s[2 * i + 1], 1);
    float w_own[H / 4], al_own[H / 4];
#pragma unroll
    for (int i = 0; i < H / 4; i++) {
      float x = (upper ? t[2 * i + 1] : t[2 * i]) + __shfl_xor_sync(0xFFFFFFFFu, upper ? t[2 * i] : t[2 * i + 1], 2);
      if (pos >= valid) x = -INFINITY;
      float mx = x;
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 4));
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 8));
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 16));
      const float m_new = fmaxf(m[i], mx), base = m_new == -INFINITY ? 0.0f : m_new;
      al_own[i] = ex2(m[i] - base);
      w_own[i] = ex2(x - base);
      l[i] = fmaf(l[i], al_own[i], w_own[i]);  // (of this lane's position: the lanes meet in finish())
      m[i] = m_new;
    }
    // The weights [position][head], and what the outputs so far count for, where the K rows were: every lane has read its part of them.
    float *ws = reinterpret_cast<float *>(stage), *als = ws + Gm::CH * AP_HEADS;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < H / 4; i++) {
      ws[pos * AP_HEADS + 4 * i + part] = w_own[i];
      if (pos == 0) als[4 * i + part] = al_own[i];
    }
    __syncwarp();
#pragma unroll
    for (int h = 0; h < H; h += 4) {
      const float4 x = *reinterpret_cast<const float4 *>(als + h);
#pragma unroll
      for (int d = 0; d < DPL; d++) o[h][d] *= x.x, o[h + 1][d] *= x.y, o[h + 2][d] *= x.z, o[h + 3][d] *= x.w;
    }
    const uint8_t *vs = stage + Gm::CH * Gm::ROWB;
#pragma unroll
    for (int j = 0; j < Gm::CH; j++) {
      float v[DPL], w[H];
      const uint8_t *at = vs + Gm::at(j, (lane * DPL) / 4) + ((lane * DPL) & 3) * 4;
      if (DPL == 4) {
        const float4 x = *reinterpret_cast<const float4 *>(at);
        v[0] = x.x, v[1 % DPL] = x.y, v[2 % DPL] = x.z, v[3 % DPL] = x.w;
      } else if (DPL == 2) {
        const float2 x = *reinterpret_cast<const float2 *>(at);
        v[0] = x.x, v[1 % DPL] = x.y;
      } else {
        v[0] = *reinterpret_cast<const float *>(at);
      }
#pragma unroll
      for (int h = 0; h < H; h += 4) {
        const float4 x = *reinterpret_cast<const float4 *>(stage + j * 32u + 4 * h);
        w[h] = x.x, w[h + 1] = x.y, w[h + 2] = x.z, w[h + 3] = x.w;
      }
#pragma unroll
      for (int h = 0; h < H; h++)
#pragma unroll
        for (int d = 0; d < DPL; d++) o[h][d] = fmaf(w[h], v[d], o[h][d]);
    }
  }
  __device__ __forceinline__ void chunk(uint8_t *stage, uint32_t valid, int lane) {
    if (few) chunk_of<4>(stage, valid, lane);
    else chunk_of<8>(stage, valid, lane);
  }
  __device__ __forceinline__ void finish(float *red, float *ml, int lane) {
#pragma unroll
    for (int h = 0; h < AP_HEADS; h++)
#pragma unroll
      for (int d = 0; d < DPL; d++) red[Gm::red_at(h, lane * DPL + d)] = o[h][d];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      float sum = l[i];
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 4);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 8);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 16);
      if (lane < 4) ml[2 * (4 * i + lane)] = m[i], ml[2 * (4 * i + lane) + 1] = sum;
    }
  }
};

// Where a CTA's share stands: chunks [j, j1) of unit `unit` of row r (this share's part of it), and what is left behind them.
struct ApCursor {
  uint32_t r, seq, len, unit, j0, j1;
  uint32_t left, first;  // chunk numbers left behind j1; number of the unit's first chunk
};

// Positions and sequence of row r: 0 positions where the row pads the batch.
__device__ __forceinline__ uint32_t ap_row(const PagedAttnArgs &a, uint32_t r, uint32_t &seq) {
  seq = a.seq ? __ldg(a.seq + r) : r + a.seq0;
  return seq < a.kv.n_seq ? min(__ldg(a.len + r), table_positions(a.kv)) : 0u;
}

// MANY: more units than CTAs.
template <typename KV, int HD, int W, bool MANY>
__global__ void __launch_bounds__(32 * W, ApGeom<KV, HD, W>::CTAS) attn_paged_kernel(const PagedAttnArgs a) {
  using Gm = ApGeom<KV, HD, W>;
  constexpr int WARPS = W, THREADS = 32 * W, STAGES = Gm::STAGES;
  constexpr uint32_t CH = Gm::CH;
  extern __shared__ __align__(128) uint8_t smem_ap[];
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t *ring = smem_ap + Gm::RING_OFF + warp * STAGES * Gm::STAGE;
  float *red = reinterpret_cast<float *>(smem_ap + Gm::RED_OFF), *ml = reinterpret_cast<float *>(smem_ap + Gm::ML_OFF);
  uint32_t *valid_of = reinterpret_cast<uint32_t *>(smem_ap + Gm::VALID_OFF) + warp * STAGES, *misc = reinterpret_cast<uint32_t *>(smem_ap + Gm::MISC_OFF);
  pdl_prologue();
  const uint32_t units = a.kv.n_kv * a.groups;

  // ---- the share: chunks [x0, x1) of all, and the row it starts in. Where there are few units, each is numbered as if it had whole
  // shares, if that makes them little longer: a CTA then has a part of one unit only.
  const uint32_t per = (a.R + THREADS - 1u) / THREADS, r_lo = min(a.R, tid * per), r_hi = min(a.R, r_lo + per);
  auto chunks = [&](uint32_t r) {
    uint32_t seq;
    return (ap_row(a, r, seq) + CH - 1u) / CH;
  };
  auto block_sum = [&](uint32_t mine, uint32_t &before) {  // of all threads, and of those ahead
    uint32_t incl = mine, all = 0u;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if ((int)lane >= o) incl += v;
    }
    __syncthreads();
    if (lane == 31) misc[warp] = incl;
    __syncthreads();
    before = incl - mine;
#pragma unroll
    for (uint32_t w = 0; w < WARPS; w++) {
      const uint32_t v = misc[w];
      if (w < warp) before += v;
      all += v;
    }
    return all;
  };
  // Behind the chunks of a unit come some numbers without any, for what its end costs (about as long as a chunk of each warp).
  constexpr uint32_t END = WARPS;
  uint32_t longest = 0u, before = 0u, mine = 0u;  // (chunk numbers fit in 32 bits: the launcher sees to it)
  for (uint32_t r = r_lo; r < r_hi; r++) {
    const uint32_t lc = chunks(r);
    mine += lc ? lc + END : 0u, longest = max(longest, lc);
  }
  uint32_t all = block_sum(mine, before) * units, share = (all + gridDim.x - 1u) / gridDim.x;
  // More units than CTAs, and short: a warp has a unit to itself, and no two of them ever meet (235 rows of one position, 40 x 8 heads, 20 -> 9.6 us;
  // 32 x 8: 256 of 50 21 -> 17, 256 of 1 to 200 39 -> 30; with longer ones, or fewer, a unit is too long a chain for one warp: 1200 units of 250 40 against 35,
  // 300 of 60 8.3 against 6.2; float cache, 235 x 1 22 -> 13, 300 x 70 of 8 x 4 heads of 32 13.9 -> 11.7, 256 of 1 to 100, 32 x 8 of 64, 28 against 26).
  bool each_alone = false;
  if constexpr (MANY) {
    constexpr uint32_t MEAN = 9u, LONGEST = Gm::F16 ? 18u : 9u;  // chunks
    each_alone = all <= (uint64_t)(MEAN + END) * units * a.R && !__syncthreads_or(longest > LONGEST);
    if (each_alone) all = 0u;
  }
  if (share < a.min_share) share = a.min_share;
  uint32_t whole_shares = 1u;  // more: unit lengths are rounded up to a multiple of this
  if (!MANY && a.R <= gridDim.x && a.R * units <= gridDim.x) {  // a warp tries a length
    const uint32_t s = share + 2u * warp;
    uint32_t parts = 0u;
    for (uint32_t r = lane; r < a.R; r += 32u) parts += (chunks(r) + s - 1u) / s;
    parts = __reduce_add_sync(0xFFFFFFFFu, parts);
    if (lane == 0) misc[20 + warp] = parts * units <= gridDim.x ? s : 0xFFFFFFFFu;
    __syncthreads();
    uint32_t best = 0xFFFFFFFFu;
    for (uint32_t w = 0; w < WARPS; w++) best = min(best, misc[20 + w]);
    if (best != 0xFFFFFFFFu) {
      mine = 0u;
      for (uint32_t r = r_lo; r < r_hi; r++) mine += (chunks(r) + best - 1u) / best;
      share = whole_shares = best, all = block_sum(mine, before) * units * best, before *= best, mine *= best;
    }
  }
  before *= units, mine *= units;
  auto numbered = [&](uint32_t lc) { return whole_shares > 1u ? (lc + whole_shares - 1u) / whole_shares * whole_shares : lc ? lc + END : 0u; };  // of a unit of lc chunks
  const uint32_t x0 = min(all, share * blockIdx.x), x1 = min(all, x0 + share);
  if (x0 < x1 && before <= x0 && x0 < before + mine) {  // one thread
    uint32_t r = r_lo;
    for (;; r++) {
      const uint32_t row = numbered(chunks(r)) * units;
      if (x0 < before + row) break;
      before += row;
    }
    misc[16] = r, misc[17] = x0 - before;  // row, chunk of the row
  }
  __syncthreads();

  auto work = [&](auto by_warp) {
    constexpr bool alone = decltype(by_warp)::value;
    const uint32_t total_warps = gridDim.x * WARPS, own_unit = blockIdx.x * WARPS + warp;  // (alone) the first unit of this warp
    if (alone ? own_unit >= a.R * units : x0 >= x1) return;
    ApCursor c;  // what is worked on
    auto stand = [&](ApCursor &k) {  // (alone) at unit k.first of all; k.left: units left to this warp
      k.r = k.first / units, k.unit = k.first - k.r * units;
      k.len = ap_row(a, k.r, k.seq);
      k.j0 = 0u, k.j1 = (k.len + CH - 1u) / CH;
    };
    if constexpr (alone) {
      c.first = own_unit, c.left = (a.R * units - 1u - own_unit) / total_warps;
      stand(c);
    } else {
      c.r = misc[16];
      c.len = ap_row(a, c.r, c.seq);
      const uint32_t lc = (c.len + CH - 1u) / CH, num = numbered(lc);
      const uint32_t at = misc[17];
      c.unit = at / num, c.j0 = at - c.unit * num;
      c.first = x0 - c.j0;
      const uint32_t end = min(c.first + num, x1);  // of the share's numbers in this unit
      c.left = x1 - end, c.j1 = min(lc, end - c.first);
    }
    auto advance = [&](ApCursor &k) {  // to the next unit (k.left > 0: there is one)
      if constexpr (alone) {
        k.first += total_warps, k.left--, stand(k);
        return;
      }
      k.first = x1 - k.left;
      if (++k.unit == units) {
        k.unit = 0u;
        do k.len = ap_row(a, ++k.r, k.seq);
        while (k.len == 0u);
      }
      const uint32_t lc = (k.len + CH - 1u) / CH;
      const uint32_t end = min(k.first + numbered(lc), x1);
      k.left = x1 - end, k.j0 = 0u, k.j1 = min(lc, end - k.first);
    };
    bool any = true;
    if (!alone && c.j0 >= c.j1) {  // the share starts behind the chunks of a unit
      any = c.left != 0u;
      if (any) advance(c);
    }

    // ---- the ring: this warp's chunks, in the order in which they are worked on, STAGES - 1 ahead
    ApCursor f = c;  // what is fetched: chunk fj, in page column f_col of the sequence's row of the table f_row, chunk f_off of the page
    const uint32_t lane_of = alone ? 0u : warp, step = alone ? 1u : (uint32_t)WARPS;  // of this warp's chunks in a unit: the first, and from one to the next
    uint32_t fj = f.j0 + lane_of, f_num = 0u, f_stage = 0u, f_col = fj / a.cpp, f_off = fj - f_col * a.cpp;
    const uint32_t *f_row = nullptr;
    size_t f_head = 0u;  // byte offset of the KV head in a page
    auto enter = [&] { f_row = a.kv.table + (size_t)f.seq * a.kv.table_stride, f_head = (size_t)(f.unit / a.groups) * a.kv.page * Gm::ROWB; };
    bool more = any;
    auto find = [&] {  // the next chunk of this warp and its page number (needed only one chunk later: nobody waits for it)
      while (fj >= f.j1) {
        if (f.left == 0u) {
          more = false;
          return;
        }
        advance(f);
        enter();
        fj = lane_of, f_col = lane_of / a.cpp, f_off = lane_of - f_col * a.cpp;
      }
      f_num = f_row[f_col];
    };
    const uint32_t to0 = Gm::at(lane / Gm::PIECES, lane % Gm::PIECES);
    auto fetch = [&] {
      if (more) {
        const bool there = f_num < a.kv.n_pages;
        const uint32_t valid = there ? min(CH, f.len - fj * CH) : 0u;
        if (!there && a.err && lane == 0) atomicExch(a.err, ERR_PAGES);
        const size_t from = (there ? (size_t)f_num * a.kv.page_stride + f_head + f_off * (uint32_t)(CH * Gm::ROWB) : 0u) + lane * 16u;
        const char *ks = static_cast<const char *>(a.kv.kp) + from, *vs = static_cast<const char *>(a.kv.vp) + from;
        uint8_t *st = ring + f_stage * Gm::STAGE;
        if (valid == CH) {
#pragma unroll
          for (int i = 0; i < Gm::PER_LANE; i++) {
            const uint32_t to = Gm::step(to0, i);
            __pipeline_memcpy_async(st + to, ks + 512 * i, 16);
            __pipeline_memcpy_async(st + CH * Gm::ROWB + to, vs + 512 * i, 16);
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < Gm::PER_LANE; i++) {
            const uint32_t row = (lane + 32u * i) / Gm::PIECES, to = Gm::at(row, lane % Gm::PIECES);
            const bool in = row < valid;  // (a row that is not is zeros; no address behind the last page)
            const size_t src = in ? 512u * i : 0u;
            __pipeline_memcpy_async(st + to, ks + src, 16, in ? 0 : 16);
            __pipeline_memcpy_async(st + CH * Gm::ROWB + to, vs + src, 16, in ? 0 : 16);
          }
        }
        if (lane == 0) valid_of[f_stage] = valid;
        fj += step, f_col += alone ? a.cpp == 1u : a.step_col, f_off += alone ? a.cpp != 1u : a.step_off;
        if (f_off >= a.cpp) f_off -= a.cpp, f_col++;
        find();
      }
      __pipeline_commit();
      f_stage = f_stage + 1u == STAGES ? 0u : f_stage + 1u;
    };
    if (any) enter(), find();
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) fetch();

    ApWarp<KV, HD, W> w;
    auto heads_of = [&](const ApCursor &k, uint32_t &h0) {  // the first head of the cursor's unit, and how many
      const uint32_t kvh = k.unit / a.groups, grp = k.unit - kvh * a.groups;
      h0 = kvh * a.G + grp * a.gw;
      return min(a.gw, a.G - grp * a.gw);
    };
    auto q_of = [&](const ApCursor &k, uint32_t h0) { return reinterpret_cast<const float *>(reinterpret_cast<const char *>(a.q) + a.q_stride * k.r) + (size_t)h0 * HD; };
    auto load_q = [&](const ApCursor &k) {
      uint32_t h0;
      const uint32_t heads = heads_of(k, h0);
      if (Gm::F16 || !alone) w.load(q_of(k, h0), heads, tid);
    };
    if (any) load_q(c);
    uint32_t stage = 0u;
    while (any) {
      uint32_t h0;
      const uint32_t heads = heads_of(c, h0);
      if constexpr (Gm::F16) {
        w.start(a.scale_log2, lane);
      } else {
        if (alone) w.start_alone(q_of(c, h0), heads, red + warp * AP_HEADS * HD, a.scale_log2, lane);  // (where its record goes)
        else w.start(heads, reinterpret_cast<float *>(smem_ap + Gm::Q_OFF), a.scale_log2, tid);
      }
      uint32_t j = c.j0 + lane_of;
      if constexpr (Gm::PAIRS) {
        for (; j + step < c.j1; j += 2u * step) {
          __pipeline_wait_prior(STAGES - 3);
          __syncwarp();
          const uint32_t second = stage + 1u == STAGES ? 0u : stage + 1u;
          const uint8_t *const st[2] = {ring + stage * Gm::STAGE, ring + second * Gm::STAGE};
          const uint32_t valid[2] = {valid_of[stage], valid_of[second]};
          fetch();
          w.template chunks<2>(st, valid, lane);
          __syncwarp();
          fetch();
          stage = second + 1u == STAGES ? 0u : second + 1u;
        }
      }
      for (; j < c.j1; j += step) {
        __pipeline_wait_prior(STAGES - 2);
        __syncwarp();
        const uint32_t valid = valid_of[stage];
        fetch();
        w.chunk(ring + stage * Gm::STAGE, valid, lane);
        stage = stage + 1u == STAGES ? 0u : stage + 1u;
      }
      // ---- the warps' records meet; the next unit's q sets out meanwhile
      ApCursor next = c;
      const bool go_on = c.left != 0u;
      if (go_on) advance(next), load_q(next);
      if constexpr (alone) {
        __syncwarp();
        w.finish(red + warp * AP_HEADS * HD, ml + warp * AP_HEADS * 2, lane);
        __syncwarp();
        if (c.j1) {
#pragma unroll 2
          for (uint32_t i0 = 0; i0 < heads * (HD / 4u); i0 += 32u) {
            const uint32_t i = i0 + lane, h = min(i / (HD / 4u), AP_HEADS - 1u), d = i % (HD / 4u) * 4u;
            const float L = ml[warp * AP_HEADS * 2 + 2 * h + 1], inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;  // (a NaN stays one)
            const float4 v = *reinterpret_cast<const float4 *>(red + warp * AP_HEADS * HD + Gm::red_at(h, d));
            store_row4<HD>(a.out, a.out_stride, a.oq, a.oq_stride, a.wide, a.n_head * HD / 32u, c.r, h0 + h, d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv),
                           i < heads * (HD / 4u));
          }
        }
        if (!go_on) break;
        c = next;
        __syncwarp();
        continue;
      }
      if (!Gm::F16) __syncthreads();  // (q lies where the records go)
      w.finish(red + warp * AP_HEADS * HD, ml + warp * AP_HEADS * 2, lane);
      __syncthreads();
      const uint32_t lc = (c.len + CH - 1u) / CH;
      const bool whole = c.j0 == 0u && c.j1 == lc;
      constexpr uint32_t QUADS = HD / 4, REC = AP_HEADS * Gm::REC_ROW;
      for (uint32_t i0 = warp * 32u; i0 < heads * QUADS; i0 += THREADS) {
        const uint32_t i = i0 + lane, h = min(i / QUADS, AP_HEADS - 1u), d = i % QUADS * 4u;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int k = 0; k < WARPS; k++) M = fmaxf(M, ml[k * AP_HEADS * 2 + 2 * h]);
        const float base = M == -INFINITY ? 0.0f : M;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < WARPS; k++) {
          const float f = ex2(ml[k * AP_HEADS * 2 + 2 * h] - base);
          const float4 v = *reinterpret_cast<const float4 *>(red + k * AP_HEADS * HD + Gm::red_at(h, d));
          L = fmaf(f, ml[k * AP_HEADS * 2 + 2 * h + 1], L);
          acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
        }
        const bool in = i < heads * QUADS;
        if (whole) {
          const float inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;  // (a NaN stays one)
          acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
          store_row4<HD>(a.out, a.out_stride, a.oq, a.oq_stride, a.wide, a.n_head * HD / 32u, c.r, h0 + h, d, acc, in);
        } else if (in) {
          float *to = a.rec + ((size_t)blockIdx.x * 2u + (c.j0 == 0u ? 1u : 0u)) * REC + h * Gm::REC_ROW;
          *reinterpret_cast<float4 *>(to + d) = acc;
          if (d == 0u) to[HD] = M, to[HD + 1] = L;
        }
      }
      if (!whole) {
        // The parts of the unit, in the order of its positions: the second record of the CTA it starts in, then the first ones of the
        // CTAs behind. Whoever is the last to have written adds them up.
        const uint32_t c0 = c.first / share, parts = (c.first + lc - 1u) / share - c0 + 1u;
        __threadfence();
        __syncthreads();
        if (tid == 0) {
          const bool last = atomicAdd(&a.count[c0], 1u) == parts - 1u;
          if (last) a.count[c0] = 0u;  // left zero for the next launch
          misc[30] = last;
        }
        __syncthreads();
        if (misc[30]) {
          __threadfence();
          // A warp per head, or per several heads of fewer than 128 dims: the lanes share out the parts' (max, sum) and their weights, then
          // FLIGHT parts at a time are on their way.
          constexpr uint32_t PER_WARP = 32u / QUADS, FLIGHT = HD == 128 ? 16u : 8u;  // heads; parts (as the registers allow)
          for (uint32_t g = warp; g * PER_WARP < heads; g += WARPS) {
            const uint32_t h = g * PER_WARP + lane / QUADS, hh = min(h, heads - 1u), d = lane % QUADS * 4u;
            const float *rec = a.rec + (size_t)c0 * 2u * REC + hh * Gm::REC_ROW;
            auto part = [&](uint32_t k) { return rec + (size_t)(2u * k + (k == 0u ? 1u : 0u)) * REC; };
            float M = -INFINITY, L = 0.0f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (uint32_t k0 = 0; k0 < parts; k0 += QUADS) {  // the lanes of a head: a part each
              const uint32_t mine_k = k0 + lane % QUADS, n = min(QUADS, parts - k0);
              const float2 e = mine_k < parts ? __ldcg(reinterpret_cast<const float2 *>(part(mine_k) + HD)) : make_float2(-INFINITY, 0.0f);
              float old = 1.0f, f = 0.0f;
              for (uint32_t q0 = 0; q0 < n; q0 += FLIGHT) {
                float4 v[FLIGHT];
#pragma unroll
                for (uint32_t q = 0; q < FLIGHT; q++)
                  v[q] = q0 + q < n ? __ldcg(reinterpret_cast<const float4 *>(part(k0 + q0 + q) + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
                if (q0 == 0u) {  // (the first outputs are on their way by now)
                  float m = e.x;
#pragma unroll
                  for (uint32_t o = 1; o < QUADS; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
                  const float M_new = fmaxf(M, m), base = M_new == -INFINITY ? 0.0f : M_new;
                  old = ex2(M - base), f = ex2(e.x - base);
                  float l = f * e.y;
#pragma unroll
                  for (uint32_t o = 1; o < QUADS; o <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
                  L = fmaf(L, old, l), M = M_new;
                  acc.x *= old, acc.y *= old, acc.z *= old, acc.w *= old;
                }
#pragma unroll
                for (uint32_t q = 0; q < FLIGHT; q++) {
                  const float w = __shfl_sync(0xFFFFFFFFu, f, lane / QUADS * QUADS + ((q0 + q) & (QUADS - 1u)));
                  if (q0 + q < n) acc.x = fmaf(w, v[q].x, acc.x), acc.y = fmaf(w, v[q].y, acc.y), acc.z = fmaf(w, v[q].z, acc.z), acc.w = fmaf(w, v[q].w, acc.w);
                }
              }
            }
            const float inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;
            acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
            store_row4<HD>(a.out, a.out_stride, a.oq, a.oq_stride, a.wide, a.n_head * HD / 32u, c.r, h0 + hh, d, acc, h < heads);
          }
        }
      }
      if (!go_on) break;
      c = next;
      __syncthreads();  // everybody has read the records (and misc): the next unit's may be written
    }
    __pipeline_wait_prior(0);
  };
  if constexpr (MANY) {
    if (each_alone) work(std::true_type());
    else work(std::false_type());
  } else {
    work(std::false_type());
  }

  // ---- rows that see nothing, and the padding of new outputs: zeros (a lane looks at a row, its warp writes it)
  const uint32_t warps = gridDim.x * WARPS;
  for (uint32_t r0 = blockIdx.x * WARPS + warp; r0 < a.R; r0 += 32u * warps) {
    const uint32_t r = r0 + lane * warps;
    uint32_t seq = 0xFFFFFFFFu, len = 1u;
    if (r < a.R) len = ap_row(a, r, seq);
    const bool real = r < a.R && seq < a.kv.n_seq;
    if (real && a.err && __ldg(a.len + r) > len) atomicExch(a.err, ERR_PAGES);
    const uint32_t reals = __ballot_sync(0xFFFFFFFFu, real);
    for (uint32_t empty = __ballot_sync(0xFFFFFFFFu, r < a.R && len == 0u && (real || a.fill)); empty; empty &= empty - 1u) {
      const uint32_t k = __ffs(empty) - 1u, e = r0 + k * warps, which = reals >> k & 1u ? 3u : a.fill;
      float *out = reinterpret_cast<float *>(reinterpret_cast<char *>(a.out) + a.out_stride * e);
      if (which & 1u)
        for (uint32_t i = lane; i < a.n_head * HD; i += 32u) out[i] = 0.0f;
      if (a.oq && (which & 2u))
        for (uint32_t i = lane; i < a.n_head * HD / 32u * 10u; i += 32u) reinterpret_cast<uint32_t *>(a.oq + a.oq_stride * e)[i] = 0u;
    }
  }
}

constexpr size_t AP_COUNT_BYTES = AP_MAX_CTAS * 4u;
static size_t ap_record_bytes(uint32_t hd) { return (size_t)AP_HEADS * (hd + 4u) * sizeof(float); }

template <typename KV, int HD, int W>
static int launch_ap(PagedAttnArgs &a, cudaStream_t st) {
  using Gm = ApGeom<KV, HD, W>;
  const uint32_t sms = (uint32_t)sm_count(), ctas = sms * Gm::CTAS < AP_MAX_CTAS ? sms * Gm::CTAS : AP_MAX_CTAS;
  a.cpp = a.kv.page / Gm::CH, a.step_col = W / a.cpp, a.step_off = W % a.cpp;
  a.min_share = 128u / Gm::CH;  // 128 positions: 1 x 100 of 8 KV heads in 5.5 us (64: 7.5, 256: 5.5), 1 x 500 in 8.1 (8.0, 9.3)
  for (uint32_t R = a.R; R;) {
    a.R = R < a.most ? R : a.most;
    const uint64_t units = (uint64_t)a.R * a.kv.n_kv * a.groups;
    constexpr bool CAN = Gm::F16 || W == 4;  // (eight warps with the float cache: few units)
    const auto k = units > ctas && units < 1ull << 31 ? attn_paged_kernel<KV, HD, W, CAN> : attn_paged_kernel<KV, HD, W, false>;
    if (int r = ensure_dynamic_smem(reinterpret_cast<const void *>(k), Gm::TOTAL)) return r;
    IEB_LAUNCH_PDL("attn_paged_kernel", k, dim3(ctas), dim3(32 * W), Gm::TOTAL, st, a);
    R -= a.R;
    a.q = reinterpret_cast<const float *>(reinterpret_cast<const char *>(a.q) + a.q_stride * a.R), a.out = reinterpret_cast<float *>(reinterpret_cast<char *>(a.out) + a.out_stride * a.R);
    a.oq = a.oq ? a.oq + a.oq_stride * a.R : nullptr, a.len += a.R, a.seq = a.seq ? a.seq + a.R : nullptr, a.seq0 += a.R;
  }
  return IE_B200_OK;
}
// Eight warps to a CTA, or four and twice the CTAs: eight where there are few units, whose parts are then longer and fewer to merge (1 x
// 32768 positions of 8 KV heads 28.8 against 30.4 us, 1 x 4000 11.6 / 12.4; at 64 units, 8 x 8192 at most, 33.7 / 32.3), and with the half
// cache where units have many heads and may be long (28 x 4 heads: 64 x 8192 at most 90.1 / 91.6, 32 x 4096 29.7 / 31.8; with 32 x 8
// 172 / 168, 128 x 2500 at most 108 / 101). Four else: a unit's end waits for fewer warps (256 x 200 57 / 45; float cache, 64 x 3001 at most, 137 / 132).
// What the host knows of the lengths is how wide the table is; short rows of a wide one (8192 positions) get eight all the same: 256 x 200 of 28 x 4 heads 37
// against 31 us, of 40 x 8 61 / 49, but 16 x 500 10.6 / 11.3 and 12.0 / 15.6.
template <typename KV, int HD>
static int launch_ap(PagedAttnArgs &a, cudaStream_t st) {
  const bool few = 4u * (uint64_t)a.R * a.kv.n_kv * a.groups <= (uint32_t)sm_count(), maybe_long = sizeof(KV) == 2 && a.gw > 4u && table_positions(a.kv) >= 2048u;
  return few || maybe_long ? launch_ap<KV, HD, 8>(a, st) : launch_ap<KV, HD, 4>(a, st);
}

}  // namespace ieb

using namespace ieb;

extern "C" size_t ie_b200_attn_decode_paged_scratch_bytes(uint32_t n_head, uint32_t n_kv, uint32_t hd) {
  (void)n_head, (void)n_kv;
  return AP_COUNT_BYTES + (size_t)AP_MAX_CTAS * 2u * ap_record_bytes(hd);
}

extern "C" int ie_b200_attn_decode_paged(const float *d_q, const ie_b200_kv_pages *pages, float *d_out, void *d_oq, const uint32_t *d_len, const uint32_t *d_seq,
                                         uint32_t n_head, uint32_t R, size_t q_stride, size_t out_stride, size_t oq_stride, void *d_scratch, uint32_t *d_err,
                                         void *stream) {
  return ie_b200_attn_decode_paged_fill(d_q, pages, d_out, d_oq, d_len, d_seq, n_head, R, q_stride, out_stride, oq_stride, d_scratch, d_err, 0u, stream);
}

extern "C" int ie_b200_attn_decode_paged_fill(const float *d_q, const ie_b200_kv_pages *pages, float *d_out, void *d_oq, const uint32_t *d_len, const uint32_t *d_seq,
                                              uint32_t n_head, uint32_t R, size_t q_stride, size_t out_stride, size_t oq_stride, void *d_scratch, uint32_t *d_err,
                                              uint32_t fill, void *stream) {
  if (R == 0) return IE_B200_OK;  // (an empty tensor may have no address)
  if (int r = check_pages("ie_b200_attn_decode_paged", pages, 16u)) return r;
  if (!d_q || !d_out || !d_len || !d_scratch) return fail(IE_B200_E_ARG, "ie_b200_attn_decode_paged: NULL pointer");
  if ((((uintptr_t)d_q | q_stride) & 7u) || (((uintptr_t)d_out | out_stride | (uintptr_t)d_oq | oq_stride | (uintptr_t)d_len | (uintptr_t)d_seq) & 3u) || !aligned16(d_scratch))
    return fail(IE_B200_E_ARG, "ie_b200_attn_decode_paged: alignment (q 8 bytes, outputs 4, scratch 16)");
  if (fill > 3u) return fail(IE_B200_E_ARG, "ie_b200_attn_decode_paged_fill: fill %u (0 to 3)", fill);
  const uint32_t hd = pages->hd, n_kv = pages->n_kv;
  if (n_head == 0 || n_head % n_kv || n_head > 65535u) return fail(IE_B200_E_SIZE, "ie_b200_attn_decode_paged: %u heads over %u KV heads", n_head, n_kv);
  if (hd != 32 && hd != 64 && hd != 128) return fail(IE_B200_E_SIZE, "ie_b200_attn_decode_paged: head dim %u unsupported (32, 64, 128)", hd);
  const size_t row = (size_t)n_head * hd;
  if (R > (1u << 20) || (R > 1u && (q_stride < row * 4u || out_stride < row * 4u || (d_oq && oq_stride < row / 32u * 40u))))
    return fail(IE_B200_E_SIZE, "ie_b200_attn_decode_paged: %u rows (at most 2^20) with strides of %zu, %zu and %zu bytes", R, q_stride, out_stride, oq_stride);
  // Chunk numbers of a launch stay below 2^31: a batch whose tables could hold more goes in several.
  const uint32_t groups = (n_head / n_kv + AP_HEADS - 1u) / AP_HEADS;
  const uint64_t numbers = ((uint64_t)table_positions(*pages) / (pages->kv_f32 ? 8u : 16u) + 9u) * n_kv * groups;
  if (numbers >= (1ull << 31)) return fail(IE_B200_E_SIZE, "ie_b200_attn_decode_paged: tables of %u positions for %u KV heads", table_positions(*pages), n_kv);
  PagedAttnArgs a = {};
  a.most = (uint32_t)(((1ull << 31) - 1u) / numbers);
  a.q = d_q, a.out = d_out, a.oq = static_cast<uint8_t *>(d_oq), a.len = d_len, a.seq = d_seq, a.err = d_err, a.kv = *pages;
  a.count = static_cast<uint32_t *>(d_scratch), a.rec = reinterpret_cast<float *>(static_cast<char *>(d_scratch) + AP_COUNT_BYTES);
  a.n_head = n_head, a.G = n_head / n_kv, a.groups = groups, a.gw = (a.G + a.groups - 1u) / a.groups, a.R = R, a.fill = fill;
  a.wide = (((uintptr_t)d_out | out_stride) & 15u) == 0u;
  a.q_stride = q_stride, a.out_stride = out_stride, a.oq_stride = oq_stride;
  a.scale_log2 = 1.44269504088896340736f / sqrtf((float)hd);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (pages->kv_f32) return hd == 32 ? launch_ap<float, 32>(a, st) : hd == 64 ? launch_ap<float, 64>(a, st) : launch_ap<float, 128>(a, st);
  return hd == 32 ? launch_ap<__half, 32>(a, st) : hd == 64 ? launch_ap<__half, 64>(a, st) : launch_ap<__half, 128>(a, st);
}
