// rope_paged.cu -- RoPE of a batch of new tokens and the store of their K / V rows into a paged cache, one pass: q rotated to its
// own buffer, k rotated and v as it is into row (position % page) of the page that the table names.
//
// y_a = x_a c - x_b s, y_b = x_a s + x_b c for each pair (a, b) of dimensions and the table row of the token's position, every
// product and sum rounded on its own (the bits of rope_kv_kernel in glue.cu and of the CPU path).
// Bound: HBM for many tokens (8192 of 32 x 8 heads of 128, half pools: 58.5 us, 6.3 TB/s, 97 % of the measured copy rate), latency for few
// (1: 2.0 us; 64: 2.3). A CTA per token keeps its table row and page number in registers for all its heads.
#include "paged.cuh"

namespace ieb {

int check_pages(const char *who, const ie_b200_kv_pages *p, uint32_t page_multiple) {
  if (!p || !p->kp || !p->vp || !p->table) return fail(IE_B200_E_ARG, "%s: NULL pages, pool or table", who);
  if (!aligned16(p->kp) || !aligned16(p->vp) || (p->page_stride & 15u) || ((uintptr_t)p->table & 3u))
    return fail(IE_B200_E_ARG, "%s: pools and page stride must be 16-byte aligned, the table 4-byte", who);
  if (p->kv_f32 != 0 && p->kv_f32 != 1) return fail(IE_B200_E_ARG, "%s: kv_f32 %d is neither 0 nor 1", who, p->kv_f32);
  if (!p->n_pages || !p->page || p->page % page_multiple || p->page > (1u << 20) || !p->n_kv || p->n_kv > 65535u || !p->table_cols || !p->n_seq ||
      (uint64_t)p->table_cols * p->page > 0x7FFFFFFFull)
    return fail(IE_B200_E_SIZE, "%s: %u pages of %u positions (a multiple of %u), %u KV heads, a table of %u x %u (at most 2^31 - 1 positions)", who, p->n_pages, p->page, page_multiple, p->n_kv,
                p->n_seq, p->table_cols);
  if (p->hd == 0 || p->hd > 512u || p->hd % 8u) return fail(IE_B200_E_SIZE, "%s: head dim %u (a multiple of 8, at most 512)", who, p->hd);
  if (p->page_stride < (size_t)p->n_kv * p->page * p->hd * (p->kv_f32 ? 4u : 2u) || p->table_stride < p->table_cols)
    return fail(IE_B200_E_SIZE, "%s: a page stride of %zu bytes or a table stride of %u columns is less than a page or a row has", who, p->page_stride, p->table_stride);
  return IE_B200_OK;
}

struct RopePagedArgs {
  const float *q, *k, *v, *cs, *sn;
  float *q_out;
  const uint32_t *pos, *seq;
  uint32_t *err;
  ie_b200_kv_pages kv;
  uint32_t nq, n_rope, fill;
  size_t stride, q_out_stride;
};

template <int W>
struct Floats {
  float v[W];
};
template <int W>
__device__ __forceinline__ Floats<W> ld_floats(const float *p) {
  Floats<W> r;
  if (W == 4) {
    const float4 x = *reinterpret_cast<const float4 *>(p);
    r.v[0] = x.x, r.v[1 % W] = x.y, r.v[2 % W] = x.z, r.v[3 % W] = x.w;
  } else {
    r.v[0] = *p;
  }
  return r;
}
template <int W>
__device__ __forceinline__ void st_row(float *p, const Floats<W> &x) {
  if (W == 4) *reinterpret_cast<float4 *>(p) = make_float4(x.v[0], x.v[1 % W], x.v[2 % W], x.v[3 % W]);
  else *p = x.v[0];
}
template <int W>
__device__ __forceinline__ void st_row(__half *p, const Floats<W> &x) {
  if (W == 4) {
    const __half2 a = __floats2half2_rn(x.v[0], x.v[1 % W]), b = __floats2half2_rn(x.v[2 % W], x.v[3 % W]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
  } else {
    *p = __float2half_rn(x.v[0]);
  }
}

// blockIdx.x: token; threadIdx.x: 2 W dimensions of a head (W pairs, or two runs of W values of v); the heads q | k | v of a token are
// dealt to threadIdx.y and blockIdx.y. W 4: rows and strides are 16-byte aligned; W 1: any alignment.
template <typename KV, int W>
__global__ void __launch_bounds__(256) rope_kv_paged_kernel(const RopePagedArgs a, const int neox) {
  pdl_prologue();
  const uint32_t t = blockIdx.x, hd = a.kv.hd, h2 = hd / 2u, nkv = a.kv.n_kv;
  const uint32_t pos = a.pos[t], seq = a.seq ? a.seq[t] : t;
  const bool real = seq < a.kv.n_seq;  // (else a row that pads the batch)
  const uint32_t col = pos / a.kv.page, i = threadIdx.x * W, at0 = neox ? i : 2u * i, at1 = at0 + (neox ? h2 : W);  // i: first pair; at0, at1: first dimension of the two runs
  float *qo = reinterpret_cast<float *>(reinterpret_cast<char *>(a.q_out) + a.q_out_stride * t);
  const uint32_t number = real && pos < table_positions(a.kv) && pos < a.n_rope ? page_number(a.kv, seq, col) : 0xFFFFFFFFu;
  if (number >= a.kv.n_pages) {
    if (real && a.err && threadIdx.x == 0 && threadIdx.y == 0) atomicExch(a.err, ERR_PAGES);
    const Floats<W> zero = {};
    for (uint32_t h = blockIdx.y * blockDim.y + threadIdx.y; a.fill && h < a.nq; h += gridDim.y * blockDim.y)
      st_row<W>(qo + (size_t)h * hd + at0, zero), st_row<W>(qo + (size_t)h * hd + at1, zero);
    return;
  }
  const Floats<W> c = ld_floats<W>(a.cs + (size_t)pos * h2 + i), s = ld_floats<W>(a.sn + (size_t)pos * h2 + i);
  const size_t row0 = page_row(a.kv, number, 0u, pos - col * a.kv.page, hd * (uint32_t)sizeof(KV)), head_step = (size_t)a.kv.page * hd * sizeof(KV);
  const float *q = reinterpret_cast<const float *>(reinterpret_cast<const char *>(a.q) + a.stride * t), *k = reinterpret_cast<const float *>(reinterpret_cast<const char *>(a.k) + a.stride * t),
              *v = reinterpret_cast<const float *>(reinterpret_cast<const char *>(a.v) + a.stride * t);
  for (uint32_t h = blockIdx.y * blockDim.y + threadIdx.y; h < a.nq + 2u * nkv; h += gridDim.y * blockDim.y) {
    const bool is_q = h < a.nq, is_v = h >= a.nq + nkv;
    const uint32_t g = is_q ? h : is_v ? h - a.nq - nkv : h - a.nq;
    const float *x = (is_q ? q : is_v ? v : k) + (size_t)g * hd;
    const Floats<W> x0 = ld_floats<W>(x + at0), x1 = ld_floats<W>(x + at1);
    Floats<W> y0 = x0, y1 = x1;
    if (!is_v) {
      if (neox || W == 1) {
#pragma unroll
        for (int e = 0; e < W; e++) {
          y0.v[e] = __fsub_rn(__fmul_rn(x0.v[e], c.v[e]), __fmul_rn(x1.v[e], s.v[e]));
          y1.v[e] = __fadd_rn(__fmul_rn(x0.v[e], s.v[e]), __fmul_rn(x1.v[e], c.v[e]));
        }
      } else {  // the W pairs lie side by side: two in each of the two runs
#pragma unroll
        for (int e = 0; e < W; e += 2) {
          const int p = e / 2, r = (p + W / 2) % W;
          const float a0 = x0.v[e], b0 = x0.v[(e + 1) % W], a1 = x1.v[e], b1 = x1.v[(e + 1) % W];
          y0.v[e] = __fsub_rn(__fmul_rn(a0, c.v[p]), __fmul_rn(b0, s.v[p])), y0.v[(e + 1) % W] = __fadd_rn(__fmul_rn(a0, s.v[p]), __fmul_rn(b0, c.v[p]));
          y1.v[e] = __fsub_rn(__fmul_rn(a1, c.v[r]), __fmul_rn(b1, s.v[r])), y1.v[(e + 1) % W] = __fadd_rn(__fmul_rn(a1, s.v[r]), __fmul_rn(b1, c.v[r]));
        }
      }
    }
    if (is_q) {
      st_row<W>(qo + (size_t)g * hd + at0, y0), st_row<W>(qo + (size_t)g * hd + at1, y1);
    } else {
      KV *dst = reinterpret_cast<KV *>(static_cast<char *>(is_v ? a.kv.vp : a.kv.kp) + row0 + g * head_step);
      st_row<W>(dst + at0, y0), st_row<W>(dst + at1, y1);
    }
  }
}

template <typename KV, int W>
static int launch_rope_paged(const RopePagedArgs &a, int neox, uint32_t T, cudaStream_t st) {
  const uint32_t x = a.kv.hd / (2u * W), y = 256u / x, heads = a.nq + 2u * a.kv.n_kv;
  const uint32_t parts = (heads + y - 1u) / y;
  // Few tokens: a CTA for every 256 / x heads, so that no thread has more than one to do.
  const uint32_t gy = (uint64_t)T * parts <= 4u * (uint32_t)sm_count() ? parts : 1u;
  IEB_LAUNCH_PDL("rope_kv_paged_kernel", (rope_kv_paged_kernel<KV, W>), dim3(T, gy), dim3(x, y), 0, st, a, neox);
  return IE_B200_OK;
}

}  // namespace ieb

using namespace ieb;

extern "C" int ie_b200_rope_kv_paged(const float *d_q, const float *d_k, const float *d_v, float *d_q_out, const ie_b200_kv_pages *pages, const float *d_cos,
                                     const float *d_sin, uint32_t n_rope, const uint32_t *d_pos, const uint32_t *d_seq, uint32_t nq, int neox, uint32_t T,
                                     size_t qkv_stride, size_t q_out_stride, uint32_t *d_err, void *stream) {
  return ie_b200_rope_kv_paged_fill(d_q, d_k, d_v, d_q_out, pages, d_cos, d_sin, n_rope, d_pos, d_seq, nq, neox, T, qkv_stride, q_out_stride, d_err, 0u, stream);
}

extern "C" int ie_b200_rope_kv_paged_fill(const float *d_q, const float *d_k, const float *d_v, float *d_q_out, const ie_b200_kv_pages *pages, const float *d_cos,
                                          const float *d_sin, uint32_t n_rope, const uint32_t *d_pos, const uint32_t *d_seq, uint32_t nq, int neox, uint32_t T,
                                          size_t qkv_stride, size_t q_out_stride, uint32_t *d_err, uint32_t fill, void *stream) {
  if (T == 0) return IE_B200_OK;  // (an empty tensor may have no address)
  if (int r = check_pages("ie_b200_rope_kv_paged", pages, 1u)) return r;
  if ((nq && (!d_q || !d_q_out)) || !d_k || !d_v || !d_cos || !d_sin || !d_pos) return fail(IE_B200_E_ARG, "ie_b200_rope_kv_paged: NULL pointer");
  if (((uintptr_t)d_q | (uintptr_t)d_k | (uintptr_t)d_v | (uintptr_t)d_q_out | (uintptr_t)d_cos | (uintptr_t)d_sin | (uintptr_t)d_pos | (uintptr_t)d_seq | qkv_stride | q_out_stride) & 3u)
    return fail(IE_B200_E_ARG, "ie_b200_rope_kv_paged: pointers and strides must be 4-byte aligned");
  if (fill > 1u) return fail(IE_B200_E_ARG, "ie_b200_rope_kv_paged_fill: fill %u is neither 0 nor 1", fill);
  if (nq > 65535u) return fail(IE_B200_E_SIZE, "ie_b200_rope_kv_paged: %u query heads", nq);
  if (T > 0x7FFFFFFFu || (T > 1u && (qkv_stride < (size_t)pages->n_kv * pages->hd * 4u || (nq && q_out_stride < (size_t)nq * pages->hd * 4u))))
    return fail(IE_B200_E_SIZE, "ie_b200_rope_kv_paged: %u tokens with rows %zu and %zu bytes apart", T, qkv_stride, q_out_stride);
  RopePagedArgs a = {d_q, d_k, d_v, d_cos, d_sin, d_q_out, d_pos, d_seq, d_err, *pages, nq, n_rope, fill, qkv_stride, q_out_stride};
  const bool wide = (((uintptr_t)d_q | (uintptr_t)d_k | (uintptr_t)d_v | (uintptr_t)d_q_out | (uintptr_t)d_cos | (uintptr_t)d_sin | qkv_stride | q_out_stride) & 15u) == 0u;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (pages->kv_f32) return wide ? launch_rope_paged<float, 4>(a, neox, T, st) : launch_rope_paged<float, 1>(a, neox, T, st);
  return wide ? launch_rope_paged<__half, 4>(a, neox, T, st) : launch_rope_paged<__half, 1>(a, neox, T, st);
}
