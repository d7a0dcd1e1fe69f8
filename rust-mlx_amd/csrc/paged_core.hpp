// What the paged-cache kernels share: the cache's description, its e4m3 form,
// operand types and the softmax's units.
//
// A page holds K as [kv_head][position][head_dim] and V transposed, as
// [kv_head][head_dim][position].  Both products contract along what is
// contiguous then (scores over head_dim, outputs over positions), so a lane
// reads its matrix-core operand of either as 16 bytes straight from the page:
// no transposition in LDS for the reader, once per position for the writer.
#pragma once

#include "common.hpp"
#include "kernels.hpp"

namespace mx {
namespace pg {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4_t __attribute__((ext_vector_type(4)));
typedef float floatx16_t __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxGroup = 16;  // q heads per kv head

__device__ __forceinline__ float neg_inf() { return u2f(0xff800000u); }

// Four e4m3 values (a dword) as bf16: every e4m3 value is a bf16 value.
__device__ __forceinline__ uint2 widen4(uint32_t v) {
  const bf16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(int(v), 1.0f, false);
  const bf16x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(int(v), 1.0f, true);
  return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}
__device__ __forceinline__ uint4 widen8(uint32_t a, uint32_t b) {
  const uint2 x = widen4(a), y = widen4(b);
  return make_uint4(x.x, x.y, y.x, y.y);
}
// The nearest e4m3 value (ties to even), the largest finite one beyond it; NaN stays NaN.
__device__ __forceinline__ uint8_t narrow(float v) {
  const float c = v > 448.0f ? 448.0f : (v < -448.0f ? -448.0f : v);
  return uint8_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, c, 0, false) & 0xff);
}

// Two fp32 as bf16 in a word, each to the nearest (ties to even).
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  bf16x2_t r;
  r[0] = __bf16(a);
  r[1] = __bf16(b);
  return __builtin_bit_cast(uint32_t, r);
}

// 1 / (1 + e^-x) by the hardware exponential.
__device__ __forceinline__ float gate_of(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-x * kLog2e));
}

// Sixteen bytes a lane from memory to LDS: lane l's land at lds + 16 l (lds: the same for the wave).
__device__ __forceinline__ void copy_to_lds(const char* src, char* lds) {
  __builtin_amdgcn_global_load_lds(
      src, reinterpret_cast<__attribute__((address_space(3))) void*>(reinterpret_cast<uintptr_t>(lds)),
      16, 0, 0);
}

// The page id of table entry `index` of `seq`, or -1 where it names no page of the cache.
__device__ __forceinline__ int page_at(const int32_t* __restrict__ table, const PageDims& d, int seq,
                                       int index) {
  const int p = table[int64_t(seq) * d.table_width + index];
  return unsigned(p) < unsigned(d.pages) ? p : -1;
}

}  // namespace pg
}  // namespace mx
