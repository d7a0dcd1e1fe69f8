// Causal attention of the last rows of packed sequences over their pages.
//
// Sequence s has rows starts[s] .. starts[s + 1] - 1; they are its last
// positions, lens[s] in all, and row i sees the positions up to its own.
//
// A workgroup of four waves takes 128 (row, q head) pairs of one sequence and
// kv head - rows in order, each row's heads of the group side by side, so any
// group size fills its tiles - and walks that sequence's keys in tiles.  Each
// wave owns 32 pairs as matrix-core columns for the whole walk:
//   S^T = K Q^T       A: K rows from LDS, B: the pairs' q in registers
//   O^T = V^T P^T     A: V^T rows from LDS, B: P as it stands
// Lane (pair c = l % 32, half h = l / 32) receives the scores of K rows
// 8 a + 4 h + b (a, b in 0..3) of a 32-row operand and supplies the k-slots
// 8 h + i of each 16 keys for the second product.  K's rows enter with bits 2
// and 3 of the row exchanged, and then the two are the same keys: P never
// leaves its lane, and the pair's maximum, sum and rescaling are one value a
// lane.  The cache holds V transposed, so both operands are 16-byte reads.
//
// P is rounded to bf16 for the product: its relative error of 2^-9 is at most
// that of the output's own rounding, and the sum that divides takes P before it.
//
// Tiles are copied to LDS one ahead (e4m3 through registers, where it is
// widened once for all waves).  16-byte pieces of a row are exchanged by the
// row's number, so that operand reads of 16 rows meet no bank twice.
//
// With few workgroups the keys are split over several, and a second launch
// joins their partials.
#include "paged_core.hpp"

namespace mx {

namespace {

using namespace pg;

constexpr int kPairs = 128;  // pairs of a workgroup: 32 a wave

// Keys of a tile: two stages of K and V fit twice into a compute unit's LDS.
template <int HD>
constexpr int tile_keys() {
  return HD == 256 ? 32 : 64;
}
template <int HD>
constexpr int stage_bytes() {
  return 2 * tile_keys<HD>() * HD * 2;  // K and V
}

// The sequence and block of query block `want`; a sequence's blocks in reverse
// order, those with the most keys first.
struct Block {
  int seq, first, count, pair0, len;  // pair0: the block's first pair within the sequence
};
__device__ __forceinline__ bool find_block(const int32_t* __restrict__ starts,
                                           const int32_t* __restrict__ lens, const PageDims& d,
                                           int rows, int group, int want, Block* out) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < d.sequences; s0 += 64) {
    const int s = s0 + lane;
    int first = 0, count = 0;
    if (s < d.sequences) {
      first = min(max(starts[s], 0), rows);
      count = max(min(starts[s + 1], rows) - first, 0);
    }
    const int n = int((int64_t(count) * group + kPairs - 1) / kPairs);
    const int sum = wave_scan(n);
    const uint64_t past = __ballot(before + sum > want);
    if (past) {
      const int f = __builtin_ctzll(past);
      // uniform values, into scalar registers
      out->seq = __builtin_amdgcn_readfirstlane(s0 + f);
      out->first = __builtin_amdgcn_readlane(first, f);
      out->count = __builtin_amdgcn_readlane(count, f);
      out->pair0 = (before + __builtin_amdgcn_readlane(sum, f) - 1 - want) * kPairs;
      const int64_t most = int64_t(d.table_width) << d.page_log2;
      const int len = lens[out->seq];
      out->len = len < 0 ? 0 : (len > most ? int(most) : len);
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

template <int HD>
__device__ __forceinline__ int k_swizzle(int row) {
  return HD >= 128 ? (row & 15) : (row & 7);
}
template <int HD>
__device__ __forceinline__ int v_swizzle(int dim) {
  return tile_keys<HD>() == 64 ? (dim & 7) : ((dim >> 2) & 3);
}

template <int HD, bool F8>
__global__ __launch_bounds__(256, 2) void prefill_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ qkv, int64_t qkv_stride, int rows,
    const int32_t* __restrict__ starts, const int32_t* __restrict__ lens,
    const int32_t* __restrict__ table, const void* __restrict__ k_cache,
    const void* __restrict__ v_cache, const float* __restrict__ k_scale,
    const float* __restrict__ v_scale, PageDims d, float scale, int splits,
    float* __restrict__ o_part, float* __restrict__ ml_part, uint16_t* __restrict__ out) {
  constexpr int KT = tile_keys<HD>();
  constexpr int KS = HD / 16;          // steps of S^T
  constexpr int KB = KT / 32;          // 32-key operands of a tile
  constexpr int ND = HD / 32;          // 32-dim operands of the output
  constexpr int KP = HD / 8;           // 16-byte pieces of a K row in LDS
  constexpr int VP = KT / 8;           // 16-byte pieces of a V^T row
  constexpr int NK = KT * KP / 256;    // K pieces a thread copies: 16 keys a wave's quarter
  constexpr int NVV = HD * VP / 256;   // V pieces a thread copies
  constexpr int RPW = KT / 4;          // K rows a wave copies (8 or 16: one page)
  extern __shared__ __align__(16) char lds[];  // two stages of [K | V^T]
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int col = lane & 31, h = lane >> 5;
  const int group = d.heads / d.kv_heads;
  const int item = blockIdx.x;
  const int kvh = item % d.kv_heads, rest = item / d.kv_heads;
  const int split = rest % splits;
  Block b;
  if (!find_block(starts, lens, d, rows, group, rest / splits, &b)) return;  // uniform
  const int prior = b.len - b.count;  // the first row's position (negative: rows without one)
  const int pairs = b.count * group;
  const int last_pair = min(b.pair0 + kPairs, pairs) - 1;
  const int kall = max(prior + last_pair / group + 1, 0);  // keys that the block sees
  const int tiles = (kall + KT - 1) / KT;
  const int per = (tiles + splits - 1) / splits;
  const int tile0 = split * per, tile1 = min(tiles, tile0 + per);
  const bool whole = tile0 == 0 && tile1 == tiles;  // also a block without keys
  if (tile0 >= tile1 && !(split == 0 && tiles == 0)) return;

  // this lane's pair
  const int pair = b.pair0 + 32 * wave + col;
  const bool alive = pair < pairs;
  const int token = pair / group, head = kvh * group + pair - token * group;
  const int64_t qrow = b.first + token;
  const int limit = alive ? prior + token : -1;  // the last key that the pair sees
  uint4 qb[KS];
  {
    const uint16_t* src = q + (qrow * d.heads + head) * HD + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qb[s] = alive ? *reinterpret_cast<const uint4*>(src + 16 * s) : make_uint4(0, 0, 0, 0);
  }
  // the wave's pairs see at least the keys up to low, at most those up to high
  int low = alive ? limit : 0x7fffffff, high = limit;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    low = min(low, __shfl_xor(low, o, 64));
    high = max(high, __shfl_xor(high, o, 64));
  }
  low = __builtin_amdgcn_readfirstlane(low);
  high = __builtin_amdgcn_readfirstlane(high);

  const char* kc = static_cast<const char*>(k_cache);
  const char* vc = static_cast<const char*>(v_cache);
  constexpr int E = F8 ? 1 : 2;
  const int page = 1 << d.page_log2, last_page = max(b.len - 1, 0) >> d.page_log2;
  const float sl2 = scale * kLog2e * (F8 && k_scale ? k_scale[kvh] : 1.0f);
  const int64_t head_at = (int64_t(kvh) << d.page_log2) * HD;

  // Page ids of a tile: of the wave's K rows, of this lane's V pieces, and, on lanes
  // 0 .. KT/16 - 1, of its 16-key parts.  They are read two tiles ahead, the copy one.
  struct Ids {
    int k, v, part;
  };
  constexpr int VL = F8 ? VP / 2 : VP;  // lanes that copy one V^T row
  const int vdim = wave * (HD / 4) + lane / VL;
  // the lane's keys of the rows that it copies: the same piece of every row
  const int vkey = F8 ? 16 * (lane % VL) : 8 * ((lane % VL) ^ v_swizzle<HD>(vdim));
  auto id_at = [&](int key) { return page_at(table, d, b.seq, min(key >> d.page_log2, last_page)); };
  auto ids_of = [&](int tile) {
    return Ids{id_at(tile + RPW * wave), id_at(tile + vkey),
               id_at(tile + 16 * (lane & (KT / 16 - 1)))};
  };
  constexpr uint32_t kAllParts = (1u << (KT / 16)) - 1u;

  // One tile's copy.  Slot i of a stage's K part is piece i % KP of row i / KP
  // and holds that row's piece (i % KP) ^ swizzle(row); V^T alike.
  constexpr int kStage = stage_bytes<HD>();
  constexpr int kVAt = KT * HD * 2;
  const uint32_t lds_at = uint32_t(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) char*)lds));
  uint4 kreg[F8 ? NK / 2 : 1], vreg[F8 ? NVV / 2 : 1];
  auto copy = [&](int tile, int stage, const Ids& id) {
    const int kid = __builtin_amdgcn_readfirstlane(max(id.k, 0));
    const int vid = max(id.v, 0);
    const char* kbase =
        kc + (kid * d.page_stride + head_at + int64_t((tile + RPW * wave) & (page - 1)) * HD) * E;
    const char* vbase = vc + (vid * d.page_stride + head_at + (int64_t(vdim) << d.page_log2) +
                              ((tile + vkey) & (page - 1))) * E;
    if constexpr (!F8) {
      const uint32_t ks = lds_at + stage * kStage + RPW * wave * KP * 16;
      const uint32_t vs = lds_at + stage * kStage + kVAt + wave * (HD / 4) * VP * 16;
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const int slot = 64 * i + lane, r = slot / KP, p = slot % KP;
        copy_to_lds(kbase + (r * HD + 8 * (p ^ k_swizzle<HD>(RPW * wave + r))) * E, ks + 1024 * i);
      }
#pragma unroll
      for (int i = 0; i < NVV; ++i)
        copy_to_lds(vbase + (int64_t(64 / VP * i) << d.page_log2) * E, vs + 1024 * i);
    } else {
      // 16 e4m3 values at a time: two neighbouring pieces
#pragma unroll
      for (int i = 0; i < NK / 2; ++i) {
        const int slot = 64 * i + lane, r = slot / (KP / 2), p = slot % (KP / 2);
        kreg[i] = *reinterpret_cast<const uint4*>(kbase + r * HD + 16 * p);
      }
#pragma unroll
      for (int i = 0; i < NVV / 2; ++i)
        vreg[i] = *reinterpret_cast<const uint4*>(vbase + (int64_t(64 / VL * i) << d.page_log2));
    }
  };
  auto store = [&](int stage) {
    if constexpr (F8) {
      char* ks = lds + stage * kStage;
      char* vs = ks + kVAt;
#pragma unroll
      for (int i = 0; i < NK / 2; ++i) {
        const int slot = 64 * i + lane, r = slot / (KP / 2), p = slot % (KP / 2);
        const int row = RPW * wave + r, sw = k_swizzle<HD>(row);
        *reinterpret_cast<uint4*>(ks + (row * KP + ((2 * p) ^ sw)) * 16) = widen8(kreg[i].x, kreg[i].y);
        *reinterpret_cast<uint4*>(ks + (row * KP + ((2 * p + 1) ^ sw)) * 16) = widen8(kreg[i].z, kreg[i].w);
      }
#pragma unroll
      for (int i = 0; i < NVV / 2; ++i) {
        const int dim = vdim + 64 / VL * i, p = lane % VL;
        const int sw = v_swizzle<HD>(dim);
        *reinterpret_cast<uint4*>(vs + (dim * VP + ((2 * p) ^ sw)) * 16) = widen8(vreg[i].x, vreg[i].y);
        *reinterpret_cast<uint4*>(vs + (dim * VP + ((2 * p + 1) ^ sw)) * 16) = widen8(vreg[i].z, vreg[i].w);
      }
    }
  };

  float m_run = neg_inf(), l_run = 0.0f;
  floatx16_t o[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[n][r] = 0.0f;

  Ids now = ids_of(tile0 * KT), next = ids_of((tile0 + 1) * KT);
  if (tile0 < tile1) {
    copy(tile0 * KT, 0, now);
    store(0);
  }
  const int krow = (col & 0x13) | ((col & 4) << 1) | ((col & 8) >> 1);  // bits 2 and 3 exchanged
  for (int ti = tile0; ti < tile1; ++ti) {
    const int tile = ti * KT, stage = (ti - tile0) & 1;
    copies_done();    // this wave's part of the tile is in LDS, and `next` is here
    __syncthreads();  // everyone's is; the other stage is consumed
    const uint32_t parts = uint32_t(__ballot(now.part >= 0)) & kAllParts;
    const bool ragged = tile + KT > kall || parts != kAllParts;
    char* ks = lds + stage * kStage;
    char* vs = ks + kVAt;
    if (ragged) {  // uniform: V of positions that are no keys may be anything, and becomes 0
      for (int i = t; i < HD * VP; i += 256) {
        const int dim = i / VP, key0 = 8 * ((i % VP) ^ v_swizzle<HD>(dim));
        const int n = (parts >> (key0 >> 4)) & 1 ? min(max(kall - tile - key0, 0), 8) : 0;
        if (n == 8) continue;
        uint16_t* p = reinterpret_cast<uint16_t*>(vs + i * 16);
        for (int j = n; j < 8; ++j) p[j] = 0;
      }
      __syncthreads();
    }
    now = next;
    if (ti + 1 < tile1) {
      copy((ti + 1) * KT, stage ^ 1, now);
      next = ids_of((ti + 2) * KT);
    }
    if (tile <= high) {
      floatx16_t sc[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[kb][r] = 0.0f;
      const char* krp = ks + krow * KP * 16;
      int swap = h ^ k_swizzle<HD>(krow);  // of krow + 32 alike
      asm("" : "+v"(swap));                // formed anew for every tile: held, the addresses spill
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const uint4 a =
              *reinterpret_cast<const uint4*>(krp + ((2 * s) ^ swap) * 16 + kb * (32 * KP * 16));
          sc[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                           __builtin_bit_cast(bf16x8_t, qb[s]),
                                                           sc[kb], 0, 0, 0);
        }
      if (tile + KT - 1 > low || parts != kAllParts) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = 32 * kb + 16 * (r >> 3) + 8 * h + (r & 7);
            const bool in = tile + key <= limit && (parts >> (2 * kb + (r >> 3)) & 1);
            sc[kb][r] = in ? sc[kb][r] : neg_inf();
          }
      }
      float mt = sc[0][0];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, sc[kb][r]);
      mt = fmaxf(mt, __shfl_xor(mt, 32, 64)) * sl2;
      // The reference follows the maximum in steps of at least 8 (a factor of 256, far from any
      // limit of fp32 or bf16), so that most tiles rescale nothing.
      if (__any(mt > m_run + 8.0f || m_run == neg_inf())) {
        const float mn = fmaxf(m_run, mt);
        const float alpha = __builtin_amdgcn_exp2f(m_run - (mn == neg_inf() ? 0.0f : mn));
        l_run *= alpha;
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[n][r] *= alpha;
        m_run = mn;
      }
      const float ref = m_run == neg_inf() ? 0.0f : m_run;  // no key yet: every weight is 0
      uint32_t pb[KB * 8];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const float x = __builtin_amdgcn_exp2f(fmaf_(sc[kb][r], sl2, -ref));
          const float y = __builtin_amdgcn_exp2f(fmaf_(sc[kb][r + 1], sl2, -ref));
          l_run += x + y;
          pb[8 * kb + r / 2] = pack2(x, y);
        }
      const int vswap = h ^ v_swizzle<HD>(col);  // of col + 32 n alike
#pragma unroll
      for (int s = 0; s < 2 * KB; ++s) {
        const bf16x8_t p = __builtin_bit_cast(
            bf16x8_t, make_uint4(pb[4 * s], pb[4 * s + 1], pb[4 * s + 2], pb[4 * s + 3]));
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          const uint4 a = *reinterpret_cast<const uint4*>(
              vs + (col * VP + ((2 * s) ^ vswap)) * 16 + n * (32 * VP * 16));
          o[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), p, o[n],
                                                         0, 0, 0);
        }
      }
    }
    if (ti + 1 < tile1) store(stage ^ 1);
  }
  if (!alive) return;
  l_run += __shfl_xor(l_run, 32, 64);
  if (whole) {
    const float inv = (l_run == 0.0f ? 0.0f : 1.0f / l_run) * (F8 && v_scale ? v_scale[kvh] : 1.0f);
    uint16_t* dst = out + (qrow * d.heads + head) * HD;
    const uint16_t* gp = qkv + qrow * qkv_stride + int64_t(head) * 2 * HD + HD;
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const int dim = 32 * n + 8 * a + 4 * h;
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = l_run == 0.0f ? 0.0f : o[n][4 * a + r] * inv;
        if (d.gated) {
          const uint2 gv = *reinterpret_cast<const uint2*>(gp + dim);
          y[0] *= gate_of(u2f(gv.x << 16));
          y[1] *= gate_of(u2f(gv.x & 0xffff0000u));
          y[2] *= gate_of(u2f(gv.y << 16));
          y[3] *= gate_of(u2f(gv.y & 0xffff0000u));
        }
        *reinterpret_cast<uint2*>(dst + dim) = make_uint2(pack2(y[0], y[1]), pack2(y[2], y[3]));
      }
    return;
  }
  const int64_t part = (qrow * d.heads + head) * splits + split;
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      *reinterpret_cast<float4*>(o_part + part * HD + 32 * n + 8 * a + 4 * h) = make_float4(
          o[n][4 * a], o[n][4 * a + 1], o[n][4 * a + 2], o[n][4 * a + 3]);
  if (h == 0) {
    ml_part[part * 2] = m_run;
    ml_part[part * 2 + 1] = l_run;
  }
}

// Joins the splits of 128 pairs of a query block in order, a wave a pair at a time.
template <int HD>
__global__ __launch_bounds__(256) void prefill_join_kernel(
    const uint16_t* __restrict__ qkv, int64_t qkv_stride, int rows,
    const int32_t* __restrict__ starts, const int32_t* __restrict__ lens,
    const float* __restrict__ v_scale, PageDims d, int splits, const float* __restrict__ o_part,
    const float* __restrict__ ml_part, uint16_t* __restrict__ out) {
  constexpr int KT = tile_keys<HD>(), DPL = HD / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int group = d.heads / d.kv_heads;
  const int kvh = blockIdx.x % d.kv_heads;
  Block b;
  if (!find_block(starts, lens, d, rows, group, int(blockIdx.x / d.kv_heads / 8), &b)) return;
  const int prior = b.len - b.count, pairs = b.count * group;
  const int last_pair = min(b.pair0 + kPairs, pairs) - 1;
  const int kall = max(prior + last_pair / group + 1, 0);
  const int tiles = (kall + KT - 1) / KT, per = (tiles + splits - 1) / splits;
  if (per >= tiles) return;  // one split (or none) wrote the result
  const int n = (tiles + per - 1) / per;
  const int first = int(blockIdx.x / d.kv_heads) % 8 * (kPairs / 8);  // an eighth of the block
  for (int i = first + wave; i < first + kPairs / 8; i += 4) {
    const int pair = b.pair0 + i;
    if (pair > last_pair) return;
    const int token = pair / group, head = kvh * group + pair - token * group;
    const int64_t row = b.first + token, part = (row * d.heads + head) * splits;
    float M = neg_inf();
    for (int c = 0; c < n; ++c) M = fmaxf(M, ml_part[(part + c) * 2]);
    const float ref = M == neg_inf() ? 0.0f : M;
    float L = 0.0f, O[DPL];
#pragma unroll
    for (int k = 0; k < DPL; ++k) O[k] = 0.0f;
#pragma unroll 4
    for (int c = 0; c < n; ++c) {
      const float e = __builtin_amdgcn_exp2f(ml_part[(part + c) * 2] - ref);
      L = fmaf_(ml_part[(part + c) * 2 + 1], e, L);
#pragma unroll
      for (int k = 0; k < DPL; ++k) O[k] = fmaf_(o_part[(part + c) * HD + DPL * lane + k], e, O[k]);
    }
    const float inv = (L == 0.0f ? 0.0f : 1.0f / L) * (v_scale ? v_scale[kvh] : 1.0f);
#pragma unroll
    for (int k = 0; k < DPL; ++k) {
      float y = L == 0.0f ? 0.0f : O[k] * inv;
      if (d.gated)
        y *= gate_of(bf16_to_f32(qkv[row * qkv_stride + int64_t(head) * 2 * HD + HD + DPL * lane + k]));
      out[(row * d.heads + head) * HD + DPL * lane + k] = f32_to_bf16(y);
    }
  }
}

// The most query blocks (times kv heads) that any starts give.
int64_t prefill_blocks(int rows, const PageDims& d) {
  const int group = d.heads / d.kv_heads;
  const int64_t n = int64_t(rows) * group / kPairs + (d.sequences < rows ? d.sequences : rows);
  return n * d.kv_heads;
}

// Workgroups that share a block's keys: as many as bring the launch to two a
// compute unit, each with at least four tiles of the longest possible context.
int prefill_splits(int rows, const PageDims& d) {
  const int64_t blocks = prefill_blocks(rows, d);
  const int64_t want = 512 / (blocks < 1 ? 1 : blocks);
  const int64_t room = (int64_t(d.table_width) << d.page_log2) / 256;
  int64_t s = want < room ? want : room;
  s = s > 64 ? 64 : s;
  return s < 1 ? 1 : int(s);
}

}  // namespace

size_t paged_prefill_workspace(int rows, const PageDims& d) {
  const int s = prefill_splits(rows, d);
  return s == 1 ? 0 : size_t(rows) * d.heads * s * (d.head_dim + 2) * 4;
}

int paged_prefill(const uint16_t* q, const uint16_t* qkv, int64_t qkv_stride, int rows,
                  const int32_t* starts, const int32_t* lens, const int32_t* table,
                  const void* k_cache, const void* v_cache, const float* k_scale,
                  const float* v_scale, const PageDims& d, float scale, void* workspace,
                  uint16_t* out, hipStream_t s) {
  const int splits = prefill_splits(rows, d);
  const int64_t blocks = prefill_blocks(rows, d);
  if (blocks * splits > 0x7fffffff || blocks * 8 > 0x7fffffff) return MX_EUNSUPPORTED;
  float* o_part = static_cast<float*>(workspace);
  float* ml_part = o_part + size_t(rows) * d.heads * splits * d.head_dim;
#define MX_PREFILL(HH, FF)                                                                        \
  if (d.head_dim == HH && d.f8 == FF) {                                                           \
    const auto fn = prefill_kernel<HH, FF>;                                                       \
    constexpr int lb = 2 * stage_bytes<HH>();                                                     \
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(fn),                                    \
                            hipFuncAttributeMaxDynamicSharedMemorySize, lb) != hipSuccess)        \
      return MX_EHIP;                                                                             \
    hipLaunchKernelGGL(fn, dim3(unsigned(blocks* splits)), dim3(256), lb, s, q, qkv, qkv_stride,  \
                       rows, starts, lens, table, k_cache, v_cache, k_scale, v_scale, d, scale,   \
                       splits, o_part, ml_part, out);                                             \
    if (hipGetLastError() != hipSuccess) return MX_EHIP;                                          \
    if (splits == 1) return MX_OK;                                                                \
    hipLaunchKernelGGL((prefill_join_kernel<HH>), dim3(unsigned(blocks * 8)), dim3(256), 0, s,    \
                       qkv, qkv_stride, rows, starts, lens, FF ? v_scale : nullptr, d, splits,    \
                       o_part, ml_part, out);                                                     \
    return hipGetLastError() == hipSuccess ? MX_OK : MX_EHIP;                                     \
  }
  MX_PREFILL(64, false) MX_PREFILL(128, false) MX_PREFILL(256, false)
  MX_PREFILL(64, true) MX_PREFILL(128, true) MX_PREFILL(256, true)
#undef MX_PREFILL
  return MX_EUNSUPPORTED;
}

}  // namespace mx
