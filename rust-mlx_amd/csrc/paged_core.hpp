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

template <class T>
__device__ __forceinline__ T lds_read(uint32_t at) {
  return *reinterpret_cast<__attribute__((address_space(3))) const T*>(at);
}
// Of sixteen lanes, four rows of sixteen 16-bit values (lane j: four values of row j / 4 at `at`), lane j
// gets the four rows' value j.
__device__ __forceinline__ uint2 lds_read_tr16(uint32_t at) {
  typedef short vec __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       reinterpret_cast<__attribute__((address_space(3))) vec*>(at)));
}
// The same of bytes: eight rows of sixteen (lane j: eight of row j / 2).
__device__ __forceinline__ uint2 lds_read_tr8(uint32_t at) {
  typedef int vec __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                                       reinterpret_cast<__attribute__((address_space(3))) vec*>(at)));
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
template <class Dims>
__device__ __forceinline__ int page_at(const int32_t* __restrict__ table, const Dims& d, int seq,
                                       int index) {
  const int p = table[int64_t(seq) * d.table_width + index];
  return unsigned(p) < unsigned(d.pages) ? p : -1;
}

// sin and cos of 2 pi t
__device__ __forceinline__ void sincos_turn(double t, float* sn, float* cs) {
  const double f = __builtin_amdgcn_fract(t);           // [0, 1)
  const double quarter = __builtin_rint(f * 4.0);       // 0 .. 4
  const float r = float((f - quarter * 0.25) * 6.283185307179586477);  // |r| <= pi / 4
  const float z = r * r;
  float s = fmaf_(z, 2.7557319e-6f, -1.9841270e-4f);    // 1/9!, 1/7!
  s = fmaf_(z, s, 8.3333333e-3f);                       // 1/5!
  s = fmaf_(z, s, -1.6666667e-1f);                      // 1/3!
  s = fmaf_(r * z, s, r);
  float c = fmaf_(z, -2.7557319e-7f, 2.4801587e-5f);    // 1/10!, 1/8!
  c = fmaf_(z, c, -1.3888889e-3f);                      // 1/6!
  c = fmaf_(z, c, 4.1666667e-2f);                       // 1/4!
  c = fmaf_(z, c, -0.5f);
  c = fmaf_(z, c, 1.0f);
  const int n = int(quarter) & 3;
  const float a = n & 1 ? c : s, b = n & 1 ? s : c;
  *sn = n & 2 ? -a : a;
  *cs = (n == 1 || n == 2) ? -b : b;
}

// ---- attention of one token a row: how the keys are shared out, and the join ----

// The length of a row's context, or -1 for a padding row.
template <class Dims>
__device__ __forceinline__ int row_len(const int32_t* __restrict__ seqs,
                                       const int32_t* __restrict__ lens, const Dims& d, int r,
                                       int rows) {
  if (r >= rows) return -1;
  const int seq = seqs ? seqs[r] : r;
  const int len = lens[r];
  if (unsigned(seq) >= unsigned(d.sequences)) return -1;
  const int most = int(min(int64_t(d.table_width) << d.page_log2, int64_t(0x7fffffff)));
  return len < 0 ? 0 : min(len, most);
}

__device__ __forceinline__ int units_of(int len, int unit) {
  return len > 0 ? (len + unit - 1) / unit : 0;
}

// The plan, formed by every wave: the most units of a chunk (a row's chunks are even), the
// fewest that give at most `target` chunks (or two rounds of them, where they are long) where
// some number up to twice the even share does; `len0`: the lengths of the first 64 rows, a lane each.
struct KeyPlan {
  int chunk_units, len0;
};
__device__ __forceinline__ KeyPlan key_plan(const int32_t* seqs, const int32_t* lens,
                                            const PageDims& d, int rows, int unit, int target) {
  const int lane = threadIdx.x & 63;
  KeyPlan p;
  p.len0 = row_len(seqs, lens, d, lane, rows);
  auto sum = [&](auto&& of) {
    int64_t total = __builtin_amdgcn_readlane(wave_scan(of(units_of(p.len0, unit))), 63);
    for (int r = 64; r < rows; r += 64)
      total += __builtin_amdgcn_readlane(
          wave_scan(of(units_of(row_len(seqs, lens, d, r + lane, rows), unit))), 63);
    return total * d.kv_heads;
  };
  const int64_t total = sum([](int u) { return u; });
  if (total >= 16 * int64_t(target)) target *= 2;  // long chunks: a second round evens out the units' speeds
  const int64_t share = (total + target - 1) / target;
  const int c0 = share < 1 ? 1 : int(share), step = (c0 + 7) / 8;
  int c = c0;
  while (c < 2 * c0 && sum([&](int u) { return (u + c - 1) / c; }) > target) c += step;
  p.chunk_units = c;
  return p;
}

// Chunk `want` in the order of rows; row -1: there are fewer.  before: the chunks of the rows before.
struct Chunk {
  int row, index, chunks, before, len;
};
__device__ __forceinline__ Chunk find_chunk(const KeyPlan& plan, const int32_t* seqs,
                                            const int32_t* lens, const PageDims& d, int rows, int unit,
                                            int want) {
  const int lane = threadIdx.x & 63, cu = plan.chunk_units;
  Chunk ch = {-1, 0, 0, 0, 0};
  for (int r = 0; r < rows; r += 64) {
    const int l = r == 0 ? plan.len0 : row_len(seqs, lens, d, r + lane, rows);
    const int n = (units_of(l, unit) + cu - 1) / cu;
    const int sum = wave_scan(n);
    const uint64_t past = __ballot(ch.before + sum > want);
    if (past) {
      const int f = __builtin_ctzll(past);
      ch.row = r + f;
      ch.len = __builtin_amdgcn_readlane(l, f);
      ch.chunks = __builtin_amdgcn_readlane(n, f);
      ch.before += __builtin_amdgcn_readlane(sum, f) - ch.chunks;
      ch.index = want - ch.before;
      break;
    }
    ch.before += __builtin_amdgcn_readlane(sum, 63);
  }
  return ch;
}

constexpr int kDecodeMaxChunks = 2048 + 1;  // of one row: twice decode_target and the rounding
// Joins the chunks of DW dims of one (row, head) in a fixed order; rows without
// keys become 0, rows of one chunk are done already.  Each wave takes every NW-th
// chunk, eight at a time, whose sums are on their way while the weights form.
template <int HD, int DW, int NW>
__global__ __launch_bounds__(64 * NW) void decode_join_kernel(
    const uint16_t* __restrict__ qkv, int64_t qkv_stride, int rows,
    const int32_t* __restrict__ seqs, const int32_t* __restrict__ lens,
    const float* __restrict__ v_scale, PageDims d, const int2* __restrict__ row_chunks,
    const float* __restrict__ o_part, const float* __restrict__ ml_part,
    uint16_t* __restrict__ out) {
  constexpr int DB = HD / DW, DPL = DW / 64;
  typedef float vec __attribute__((ext_vector_type(DPL)));
  __shared__ float ws[kDecodeMaxChunks];
  __shared__ float red[2][NW];
  __shared__ vec os[NW][64];
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int dim = DW * (blockIdx.x % DB) + DPL * lane;
  const int head = blockIdx.x / DB % d.heads, row = blockIdx.x / DB / d.heads;
  const int group = d.heads / d.kv_heads, kvh = head / group;
  const int len = row_len(seqs, lens, d, row, rows);
  const int2 rc = row_chunks[row];  // meaningful where there are keys
  if (len < 0) return;
  uint16_t* dst = out + (int64_t(row) * d.heads + head) * HD + dim;
  if (len == 0) {
    if (wave == 0)
      for (int i = 0; i < DPL; ++i) dst[i] = 0;
    return;
  }
  const int n = rc.y;  // 2 .. kDecodeMaxChunks
  if (n <= 1) return;
  const int64_t part0 = int64_t(rc.x) * d.heads + head;  // chunk c's partial: c heads further on
  auto part_of = [&](int c) {
    return *reinterpret_cast<const vec*>(o_part + (part0 + int64_t(c) * d.heads) * HD + dim);
  };
  vec v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = part_of(min(wave + NW * i, n - 1));
  float M = neg_inf();
  for (int c = t; c < n; c += 64 * NW) M = fmaxf(M, ml_part[(part0 + int64_t(c) * d.heads) * 2]);
  for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  if (lane == 0) red[0][wave] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) M = fmaxf(M, red[0][w]);
  const float ref = M == neg_inf() ? 0.0f : M;
  float L = 0.0f;
  for (int c = t; c < n; c += 64 * NW) {
    const float2 ml = *reinterpret_cast<const float2*>(ml_part + (part0 + int64_t(c) * d.heads) * 2);
    const float e = __builtin_amdgcn_exp2f(ml.x - ref);
    ws[c] = e;
    L = fmaf_(ml.y, e, L);
  }
  for (int o = 32; o > 0; o >>= 1) L += __shfl_xor(L, o, 64);
  if (lane == 0) red[1][wave] = L;
  __syncthreads();
  vec O = 0.0f;
  for (int c0 = wave; c0 < n; c0 += 8 * NW) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + NW * i < n) {  // uniform
        const float e = ws[c0 + NW * i];
        // (an infinite sum stays one, however small its chunk's weight)
        for (int k = 0; k < DPL; ++k) O[k] = fmaf_(v[i][k], __builtin_isinf(v[i][k]) ? 1.0f : e, O[k]);
      }
    if (c0 + 8 * NW < n) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = part_of(min(c0 + NW * (8 + i), n - 1));
    }
  }
  os[wave][lane] = O;
  __syncthreads();
  if (wave != 0) return;
  L = red[1][0];
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    L += red[1][w];
    O += os[w][lane];
  }
  const float inv = (L == 0.0f ? 0.0f : 1.0f / L) * (v_scale ? v_scale[kvh] : 1.0f);
  const uint16_t* gp = qkv + int64_t(row) * qkv_stride + int64_t(head) * 2 * HD + HD + dim;
#pragma unroll
  for (int k = 0; k < DPL; ++k) {
    float y = L == 0.0f ? 0.0f : O[k] * inv;
    if (d.gated) y *= gate_of(bf16_to_f32(gp[k]));
    dst[k] = f32_to_bf16(y);
  }
}

}  // namespace pg
}  // namespace mx
