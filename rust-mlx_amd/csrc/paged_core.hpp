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

// Sixteen bytes a lane from memory to LDS: lane l's land at lds + 16 l (lds: the same for the
// wave), once the wave has waited for its vector memory (copies_done).  Written out because
// the compiler takes every later LDS read for one of these bytes and waits for the copy at
// once; here a tile's copy runs under the work on the tile before.
__device__ __forceinline__ void copy_to_lds(const char* src, uint32_t lds) {
  uint32_t m0;  // an output, so that the compiler knows that it is written
  asm volatile("s_mov_b32 %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               : "=&{m0}"(m0)
               : "v"(src), "s"(lds)
               : "memory");
}
// The same from src + off, src the same for the wave.  src may come from a vector instruction (a read
// of one lane), which has to lie five wait states before a memory instruction that uses it: the
// compiler does not look into the block, so the block has them all.
__device__ __forceinline__ void copy_to_lds(const char* src, uint32_t off, uint32_t lds) {
  const uint64_t at = reinterpret_cast<uint64_t>(src);
  const uint64_t lo = uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(at))));
  const uint64_t hi = uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(at >> 32))));
  uint32_t m0;
  asm volatile("s_mov_b32 %0, %3\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2"
               : "=&{m0}"(m0)
               : "v"(off), "s"(hi << 32 | lo), "s"(lds)
               : "memory");
}
// Waits until at most `N` of the wave's vector memory operations, the latest, are under way.
template <int N>
__device__ __forceinline__ void copies_done() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// Sums over groups of N neighbouring lanes (8, 16 or 32), in every lane of the group.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return u2f(uint32_t(__builtin_amdgcn_mov_dpp(int(f2u(v)), CTRL, 0xf, 0xf, true)));
}
template <int N>
__device__ __forceinline__ float group_sum(float v) {
  v += dpp<0xb1>(v);                     // quad_perm 1 0 3 2
  v += dpp<0x4e>(v);                     // quad_perm 2 3 0 1
  v += dpp<0x141>(v);                    // row_half_mirror: the other four of eight
  if (N >= 16) v += dpp<0x140>(v);       // row_mirror: the other eight of sixteen
  if (N >= 32) v += __shfl_xor(v, 16, 64);
  return v;
}

// The larger of this lane's value and that of the lane 32 away.
__device__ __forceinline__ float max_across_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return fmaxf(u2f(r[0]), u2f(r[1]));
}

// Sums over the lanes up to each one (all 64 lanes active), in registers.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);   // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);   // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);   // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row 0's and 2's last to 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // lane 31's to rows 2 and 3
  return v;
}

// The page id of table entry `index` of `seq`, or -1 where it names no page of the cache.
__device__ __forceinline__ int page_at(const int32_t* __restrict__ table, const PageDims& d, int seq,
                                       int index) {
  const int p = table[int64_t(seq) * d.table_width + index];
  return unsigned(p) < unsigned(d.pages) ? p : -1;
}

}  // namespace pg
}  // namespace mx
