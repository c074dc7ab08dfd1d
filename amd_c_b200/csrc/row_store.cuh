// row_store.cuh -- what the attention kernels' epilogues share: 2^x, and the store of a head's outputs with their Q8 copy.
#pragma once

#include "common.cuh"

namespace ieb {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four neighbouring outputs of a (token, head) row per lane, eight lanes per block of 32: the row's floats and its Q8 copy.
template <int HD>
__device__ __forceinline__ void store_row4(float *out, size_t out_stride, uint8_t *oq, size_t oq_stride, uint32_t wide, uint32_t nbq, uint32_t tok, uint32_t head,
                                           uint32_t col, const float4 &o, bool in) {
  float *dst = reinterpret_cast<float *>(reinterpret_cast<char *>(out) + out_stride * tok) + (size_t)head * HD + col;
  if (in) {
    if (wide) *reinterpret_cast<float4 *>(dst) = o;
    else dst[0] = o.x, dst[1] = o.y, dst[2] = o.z, dst[3] = o.w;
  }
  if (!oq) return;
  float amax = fmaxf(fmaxf(fabsf(o.x), fabsf(o.y)), fmaxf(fabsf(o.z), fabsf(o.w)));
#pragma unroll
  for (int s = 1; s < 8; s <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, s));
  const float d = __fdiv_rn(amax, 127.0f), v[4] = {o.x, o.y, o.z, o.w};
  const Q8Div qd = q8_div(d);
  int sum = 0;
  uint32_t w = 0u;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const int q = q8_round(v[e], qd);
    sum += q, w |= (uint32_t)(q & 255) << (8 * e);
  }
#pragma unroll
  for (int s = 1; s < 8; s <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, s);
  if (!in) return;
  uint8_t *qrow = oq + oq_stride * tok;
  const uint32_t at = head * HD + col;
  *reinterpret_cast<uint32_t *>(qrow + at) = w;
  if ((at & 31u) == 0u) reinterpret_cast<float *>(qrow + 32u * (size_t)nbq)[at / 32u] = d, reinterpret_cast<int *>(qrow + 36u * (size_t)nbq)[at / 32u] = sum;
}

}  // namespace ieb
