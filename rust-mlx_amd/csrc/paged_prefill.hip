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
// P is rounded to bf16 for the product, each p by at most 2^-8 of itself, as the
// output is; the sum that divides takes P before it.  A second part of P, as
// attention of one token has it, would make the second product's work twice as
// much where the matrix units are the bound.
//
// Tiles are copied to LDS one ahead (e4m3 through registers, where it is
// widened once for all waves).  16-byte pieces of a row are exchanged by the
// row's number, so that operand reads of 8 rows meet no bank twice (of 16 rows
// at 128 dims too: 562 us against 555 for 8192 tokens, the bits cost more).
//
// With few workgroups the keys are split over several, and a second launch
// joins their partials.
//
// The matrix cores and the vector ALUs bound it together, under a falling clock:
// 8192 tokens of 32 q / 8 kv heads of 128 take 560 to 592 us from card to card (930 to
// 980 TFLOP/s).  512 rows of 16 / 2 heads of 256 on 12001 keys take 123 to 130 us, 17
// of them to join eight splits; there the registers bound it, see R and kHalves.
#include <type_traits>
#include <utility>

#include "paged_core.hpp"

namespace mx {

namespace {

using namespace pg;

constexpr int NW = 4;            // waves of a workgroup
constexpr int D = 2;             // stages of a tile in LDS
constexpr int kPairs = 32 * NW;  // its pairs

// Keys of a tile: two stages of K and V fit twice into a compute unit's LDS.
template <int HD>
constexpr int tile_keys() {
  return HD == 256 ? 32 : 64;
}
template <int HD>
constexpr int stage_bytes() {
  return 2 * tile_keys<HD>() * HD * 2;  // K and V
}

// Lambdas that hold registers by reference: a call would put them into memory.
#define MX_LAMBDA __attribute__((always_inline))

// f(integral_constant<int, 0>) .. f(integral_constant<int, N - 1>)
template <class F, int... I>
__device__ __forceinline__ void each_(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
  each_(static_cast<F&&>(f), std::make_integer_sequence<int, N>{});
}

// Rows of a sequence, which are the packed ones from `first` on, and its length, cut to the table's.
struct Rows {
  int first, count, len;
};
__device__ __forceinline__ Rows rows_of(const int32_t* __restrict__ starts,
                                        const int32_t* __restrict__ lens, const PageDims& d,
                                        int rows, int s) {
  Rows r = {0, 0, 0};
  if (s < d.sequences) {
    r.first = min(max(starts[s], 0), rows);
    r.count = max(min(starts[s + 1], rows) - r.first, 0);
    const int64_t most = int64_t(d.table_width) << d.page_log2;
    const int len = lens[s];
    r.len = len < 0 ? 0 : (len > most ? int(most) : len);
  }
  return r;
}
__device__ __forceinline__ int blocks_of(const Rows& r, int group) {
  return int((int64_t(r.count) * group + kPairs - 1) / kPairs);
}

// How many workgroups share the keys of a query block, with `blocks` of them: as many as bring the
// launch to two workgroups a compute unit, each with at least four tiles of the longest possible
// context; in eights with the kv heads where that is possible, for whole XCDs (512 rows on 12001
// keys, two kv heads: 8 splits 126 us, 7 splits 138).  At most 64, never more with more blocks.
__host__ __device__ __forceinline__ int splits_of(int64_t blocks, const PageDims& d) {
  const int64_t all = blocks * d.kv_heads, room = (int64_t(d.table_width) << d.page_log2) / 256;
  int s = all > 256 ? 1 : 512 / int(all < 1 ? 1 : all);
  s = s > room ? int(room) : s;
  s = s > 64 ? 64 : s < 1 ? 1 : s;
  const int low = d.kv_heads & -d.kv_heads, step = low >= 8 ? 1 : 8 / low;  // powers of two
  const int e = (s + step - 1) & -step;
  return s > 1 && e < 2 * s && e <= room ? e : s;
}
// The fewest blocks that a call of so many rows is laid out for.
__host__ __device__ __forceinline__ int64_t least_blocks(int rows, const PageDims& d) {
  return (int64_t(rows) * (d.heads / d.kv_heads) + kPairs - 1) / kPairs;
}

// What follows from all sequences' rows, formed by every wave: the number of query blocks (sequences
// without rows have none, however many the table has) and the splits; `r0`: the rows of the first 64
// sequences, a lane each.
struct Plan {
  Rows r0;
  int blocks, splits;
};
__device__ __forceinline__ Plan make_plan(const int32_t* __restrict__ starts,
                                          const int32_t* __restrict__ lens, const PageDims& d,
                                          int rows, int group) {
  const int lane = threadIdx.x & 63;
  Plan p;
  p.r0 = rows_of(starts, lens, d, rows, lane);
  int n = blocks_of(p.r0, group);
  constexpr int AHEAD = 8;  // loads on their way; past the last sequence there are no rows
  const int all = min(starts[d.sequences], rows);
  int done = __builtin_amdgcn_readlane(p.r0.first + p.r0.count, 63);  // rows of the sequences so far
  for (int s0 = 64; s0 < d.sequences && done < all; s0 += 64 * AHEAD) {
    int at[AHEAD], to[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      at[i] = starts[min(s0 + 64 * i + lane, d.sequences)];
      to[i] = starts[min(s0 + 64 * i + lane + 1, d.sequences)];
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int first = min(max(at[i], 0), rows);
      n += blocks_of({first, max(min(to[i], rows) - first, 0), 0}, group);
    }
    done = __builtin_amdgcn_readlane(to[AHEAD - 1], 63);
  }
  p.blocks = max(__builtin_amdgcn_readlane(wave_scan(n), 63), int(least_blocks(rows, d)));
  p.splits = splits_of(p.blocks, d);
  return p;
}

// The sequence and block of query block `want`; a sequence's blocks in reverse
// order, those with the most keys first.
struct Block {
  int seq, first, count, pair0, len;  // pair0: the block's first pair within the sequence
};
__device__ __forceinline__ bool find_block(const Plan& p, const int32_t* __restrict__ starts,
                                           const int32_t* __restrict__ lens, const PageDims& d,
                                           int rows, int group, int want, Block* out) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < d.sequences; s0 += 64) {
    const Rows r = s0 == 0 ? p.r0 : rows_of(starts, lens, d, rows, s0 + lane);
    const int sum = wave_scan(blocks_of(r, group));
    const uint64_t past = __ballot(before + sum > want);
    if (past) {
      const int f = __builtin_ctzll(past);
      // uniform values, into scalar registers
      out->seq = __builtin_amdgcn_readfirstlane(s0 + f);
      out->first = __builtin_amdgcn_readlane(r.first, f);
      out->count = __builtin_amdgcn_readlane(r.count, f);
      out->pair0 = (before + __builtin_amdgcn_readlane(sum, f) - 1 - want) * kPairs;
      out->len = __builtin_amdgcn_readlane(r.len, f);
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// The query block, kv head and split of a workgroup.  Workgroups go to the eight XCDs in turn
// (id mod 8).  Those of one kv head and split read the same keys, whatever their block, so with
// eight such pairs or more each XCD takes whole pairs, and its L2 what they read.
struct Item {
  int block, kvh, split;
};
__host__ __device__ __forceinline__ bool by_xcd(int kv_heads, int splits) {
  return kv_heads * splits >= 8;
}
// Workgroups of a block: its pairs of kv head and split, in whole XCDs or, without enough of them,
// every workgroup in turn.
__host__ __device__ __forceinline__ int items_of(int kv_heads, int splits) {
  const int pairs = kv_heads * splits;
  return by_xcd(kv_heads, splits) ? 8 * ((pairs + 7) / 8) : pairs;
}
// Where all workgroups run at once, the second 256 beside the first on the same compute units,
// those take the blocks from the last one on: a sequence's blocks have fewer and fewer keys, and
// so a long one shares its unit with a short one (four prompts of up to 2047 rows on up to 3001,
// e4m3: 144 us against 152).
__device__ __forceinline__ Item item_of(int id, const Plan& p, int kv_heads) {
  const int pairs = kv_heads * p.splits, a_block = items_of(kv_heads, p.splits);
  const bool xcd = by_xcd(kv_heads, p.splits);
  const int each = a_block / 8;  // pairs of an XCD
  const int j = id >> 3, pair = xcd ? (id & 7) + 8 * (j % each) : id % pairs;
  int block = xcd ? j / each : id / pairs;
  if (block >= p.blocks) return Item{block, 0, p.splits};  // past the last block: none
  const int64_t all = int64_t(p.blocks) * a_block;
  if (all > 256 && all <= 512) {
    const int first = 256 / a_block;
    if (block >= first) block = p.blocks - 1 - (block - first);
  }
  return Item{block, pair % kv_heads, pair / kv_heads};  // split >= splits: none
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
__global__ __launch_bounds__(64 * NW, 2) void prefill_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ qkv, int64_t qkv_stride, int rows,
    const int32_t* __restrict__ starts, const int32_t* __restrict__ lens,
    const int32_t* __restrict__ table, const void* __restrict__ k_cache,
    const void* __restrict__ v_cache, const float* __restrict__ k_scale,
    const float* __restrict__ v_scale, PageDims d, float scale, float* __restrict__ o_part,
    float* __restrict__ ml_part, uint16_t* __restrict__ out) {
  constexpr int KT = tile_keys<HD>();
  constexpr int KS = HD / 16;          // steps of S^T
  constexpr int KB = KT / 32;          // 32-key operands of a tile
  constexpr int ND = HD / 32;          // 32-dim operands of the output
  constexpr int KP = HD / 8;           // 16-byte pieces of a K row in LDS
  constexpr int VP = KT / 8;           // 16-byte pieces of a V^T row
  constexpr int NK = KT * KP / (64 * NW);   // K pieces a thread copies
  static_assert(!F8 || NK % 2 == 0, "two pieces of e4m3 at a time");
  constexpr int NVV = HD * VP / (64 * NW);  // V pieces a thread copies
  constexpr int RPW = KT / NW;              // K rows a wave copies (at most 16: one page)
  extern __shared__ __align__(16) char lds[];  // [D] of K, then [D] of V^T
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int col = lane & 31, h = lane >> 5;
  const int group = d.heads / d.kv_heads;
  const Plan plan = make_plan(starts, lens, d, rows, group);
  const int splits = plan.splits;
  const Item it = item_of(blockIdx.x, plan, d.kv_heads);
  if (it.split >= splits) return;
  const int kvh = it.kvh, split = it.split;
  Block b;
  if (!find_block(plan, starts, lens, d, rows, group, it.block, &b)) return;  // uniform
  const int prior = b.len - b.count;  // the first row's position (negative: rows without one)
  const int pairs = b.count * group;
  const int last_pair = min(b.pair0 + kPairs, pairs) - 1;
  const int kall = max(prior + last_pair / group + 1, 0);  // keys that the block sees
  const int tiles = (kall + KT - 1) / KT;
  const int per = (tiles + splits - 1) / splits;
  const int tile0 = split * per, tile1 = min(tiles, tile0 + per);
  const bool whole = tile0 == 0 && tile1 == tiles;  // also a block without keys
  if (tile0 >= tile1 && !(split == 0 && tiles == 0)) return;

  // this lane's pair; lanes past the last pair take that, see nothing and write nothing
  const bool alive = b.pair0 + 32 * wave + col < pairs;
  const int pair = min(b.pair0 + 32 * wave + col, pairs - 1);
  const int token = pair / group, head = kvh * group + pair - token * group;
  const int64_t qrow = b.first + token;
  const int limit = alive ? prior + token : -1;  // the last key that the pair sees
  uint4 qb[KS];
  {
    const uint16_t* src = q + (qrow * d.heads + head) * HD + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s) qb[s] = *reinterpret_cast<const uint4*>(src + 16 * s);
  }
  // the wave's pairs see at least the keys up to low
  int low = alive ? limit : 0x7fffffff;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) low = min(low, __shfl_xor(low, o, 64));
  low = __builtin_amdgcn_readfirstlane(low);

  const int sees_all = prior + b.pair0 / group;  // the last key that every pair of the block sees

  const char* kc = static_cast<const char*>(k_cache);
  const char* vc = static_cast<const char*>(v_cache);
  constexpr int E = F8 ? 1 : 2;
  const int page = 1 << d.page_log2, last_page = max(b.len - 1, 0) >> d.page_log2;
  float sl2 = scale * kLog2e * (F8 && k_scale ? k_scale[kvh] : 1.0f);
  // A tile's maximum is taken before the product with sl2, and masked scores of -inf stay below
  // everything only under a positive one: the sign of a kv head's scale, or its zero, goes to q.
  if constexpr (F8) {
    const uint32_t flip = sl2 < 0.0f ? 0x80008000u : 0u, keep = sl2 == 0.0f ? 0u : 0xffffffffu;
    sl2 = sl2 < 0.0f ? -sl2 : sl2 == 0.0f ? 1.0f : sl2;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qb[s] = make_uint4((qb[s].x & keep) ^ flip, (qb[s].y & keep) ^ flip, (qb[s].z & keep) ^ flip,
                         (qb[s].w & keep) ^ flip);
  }
  const int64_t head_at = (int64_t(kvh) << d.page_log2) * HD;

  // Page ids of a tile's 16-key parts, through scalar loads (they have a counter of their
  // own, so waiting for one waits for no copy), read one tile ahead of the copy.
  constexpr int PT = KT / 16;
  struct Ids {
    int part[PT];
  };
  constexpr int VL = F8 ? VP / 2 : VP;  // lanes that copy one V^T row
  const int vdim = wave * (HD / NW) + lane / VL;
  // the lane's keys of the rows that it copies: the same piece of every row
  const int vkey = F8 ? 16 * (lane % VL) : 8 * ((lane % VL) ^ v_swizzle<HD>(vdim));
  auto ids_of = [&](int tile) MX_LAMBDA {
    Ids id;
#pragma unroll
    for (int i = 0; i < PT; ++i)
      id.part[i] = page_at(table, d, b.seq, min((tile + 16 * i) >> d.page_log2, last_page));
    return id;
  };
  constexpr uint32_t kAllParts = (1u << PT) - 1u;
  auto bits_of = [&](const Ids& id) MX_LAMBDA {  // bit i: keys 16 i .. 16 i + 15 lie in a page
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < PT; ++i) m |= (id.part[i] >= 0 ? 1u : 0u) << i;
    return m;
  };

  // One tile's copies.  Slot i of a K stage is piece i % KP of row i / KP and
  // holds that row's piece (i % KP) ^ swizzle(row); V^T alike.
  constexpr int kPart = KT * HD * 2;  // bytes of a K (or V^T) stage
  const uint32_t lds_at = uint32_t(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) char*)lds));
  uint4 kreg[F8 ? NK / 2 : 1], vreg[F8 ? NVV / 2 : 1];
  // from where this lane copies a tile's K and V
  auto k_from = [&](int tile, const Ids& id) MX_LAMBDA {
    int kid = id.part[0];
#pragma unroll
    for (int i = 1; i < PT; ++i) kid = (RPW * wave) >> 4 == i ? id.part[i] : kid;
    return kc + (max(kid, 0) * d.page_stride + head_at +
                 int64_t((tile + RPW * wave) & (page - 1)) * HD) * E;
  };
  auto v_from = [&](int tile, const Ids& id) MX_LAMBDA {
    int vid = id.part[0];
#pragma unroll
    for (int i = 1; i < PT; ++i) vid = vkey >> 4 == i ? id.part[i] : vid;
    return vc + (max(vid, 0) * d.page_stride + head_at + (int64_t(vdim) << d.page_log2) +
                 ((tile + vkey) & (page - 1))) * E;
  };
  // piece i of a wave's copies, to LDS, or of e4m3 (16 values: two pieces of LDS) to registers
  constexpr int CK = F8 ? NK / 2 : NK, CV = F8 ? NVV / 2 : NVV;
  // K piece `lane` of the wave's rows, in bytes from the first; piece 64 i + lane differs in the
  // bits of its 1 KB and of the rows' part in the exchange
  const uint32_t koff = lane / KP * (HD * 2) + 16 * ((lane % KP) ^ k_swizzle<HD>(RPW * wave + lane / KP));
  auto copy_k = [&](const char* from, int stage, int i) MX_LAMBDA {
    if constexpr (!F8) {
      copy_to_lds(from, koff ^ (1024 * i | 16 * k_swizzle<HD>(64 / KP * i)),
                  lds_at + stage * kPart + RPW * wave * KP * 16 + 1024 * i);
    } else {
      const int slot = 64 * i + lane, r = slot / (KP / 2), p = slot % (KP / 2);
      kreg[i] = *reinterpret_cast<const uint4*>(from + r * HD + 16 * p);
    }
  };
  auto copy_v = [&](const char* from, int stage, int i) MX_LAMBDA {
    const char* src = from + (int64_t(64 / VL * i) << d.page_log2) * E;
    if constexpr (!F8)
      copy_to_lds(src, lds_at + (D + stage) * kPart + wave * (HD / NW) * VP * 16 + 1024 * i);
    else
      vreg[i] = *reinterpret_cast<const uint4*>(src);
  };
  auto store_k = [&](int stage) MX_LAMBDA {
    if constexpr (F8) {
      char* ks = lds + stage * kPart;
#pragma unroll
      for (int i = 0; i < NK / 2; ++i) {
        const int slot = 64 * i + lane, r = slot / (KP / 2), p = slot % (KP / 2);
        const int row = RPW * wave + r, sw = k_swizzle<HD>(row);
        *reinterpret_cast<uint4*>(ks + (row * KP + ((2 * p) ^ sw)) * 16) = widen8(kreg[i].x, kreg[i].y);
        *reinterpret_cast<uint4*>(ks + (row * KP + ((2 * p + 1) ^ sw)) * 16) = widen8(kreg[i].z, kreg[i].w);
      }
    }
  };
  auto store_v = [&](int stage) MX_LAMBDA {
    if constexpr (F8) {
      char* vs = lds + (D + stage) * kPart;
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

  // Tile ti's K and V lie in stages ti % D.  Two workgroups share each matrix unit: while a wave of
  // one forms its exponentials, one of the other has the products.  Forming a tile's exponentials
  // under the next tile's products within one wave was no faster (HD 128, 8192 tokens: 608 us
  // against 565), the two workgroups do that already.
  // With 256 dims of e4m3 the registers hold a tile's K or V on their way, not both: K is widened
  // after the scores, V after P V (512 rows on 12001 keys: 152 us, both after P V 181; with 128
  // dims both together are faster, four prompts of up to 2047 on up to 3001: 147 us against 151).
  constexpr bool kHalves = F8 && HD == 256;
  constexpr int kCopies = F8 ? 0 : CK + CV;  // of a step, by a wave
  constexpr int R = HD == 256 ? 2 : 4;       // operands read ahead of their products
  // The order as it is written: left alone, the compiler reads each operand just before its
  // product.  With 256 dims it has no registers for that, and its own order is faster (124 us
  // against 125 for 512 rows on 12001 keys; operands four ahead 132), and so it is with e4m3 (151
  // against 157 for four prompts of up to 2047 on up to 3001, before their blocks' order).
  auto keep_order = [] {
    if constexpr (HD < 256 && !F8) __builtin_amdgcn_sched_barrier(0);
  };
  const int krow = (col & 0x13) | ((col & 4) << 1) | ((col & 8) >> 1);  // bits 2 and 3 exchanged
  const int kswap = h ^ k_swizzle<HD>(krow);  // of krow + 32 alike
  const int vswap = h ^ v_swizzle<HD>(col);   // of col + 32 n alike
  // operands of product i of the scores, and of P V
  auto k_operand = [&](int stage, int i) MX_LAMBDA {
    return *reinterpret_cast<const uint4*>(lds + stage * kPart + krow * (KP * 16) +
                                           ((2 * (i / KB)) ^ kswap) * 16 +
                                           (i % KB) * (32 * KP * 16));
  };
  auto v_operand = [&](int stage, int i) MX_LAMBDA {
    return *reinterpret_cast<const uint4*>(lds + (D + stage) * kPart + col * (VP * 16) +
                                           ((2 * (i / ND)) ^ vswap) * 16 +
                                           (i % ND) * (32 * VP * 16));
  };
  auto score = [&](int i, const uint4& a, floatx16_t (&sc)[KB]) MX_LAMBDA {
    sc[i % KB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                         __builtin_bit_cast(bf16x8_t, qb[i / KB]),
                                                         sc[i % KB], 0, 0, 0);
  };
  // all scores of the tile in K stage `stage`, with between(i) after product i
  auto scores = [&](int stage, floatx16_t (&sc)[KB], auto&& between) MX_LAMBDA {
    uint4 a[R];
    each<R>([&](auto i) MX_LAMBDA { a[i] = k_operand(stage, i); });
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[kb][r] = 0.0f;
    each<KS * KB>([&](auto i) MX_LAMBDA {
      keep_order();
      score(i, a[i % R], sc);
      if constexpr (i + R < KS * KB) a[i % R] = k_operand(stage, i + R);
      between(i);
    });
    keep_order();
  };
  // Tiles past the last one are copied like it, into stages that nobody reads: every step
  // has the same copies, so waiting for all but the latest is waiting for their number.
  const int last = (tile1 - 1) * KT;
  uint32_t queue = 0;  // parts of the tiles from the present one on, PT bits each
  Ids id;
  if (tile0 < tile1) {
    id = ids_of(tile0 * KT);
#pragma unroll
    for (int i = 0; i < D - 1; ++i) {
      const int at = min((tile0 + i) * KT, last);
      queue |= bits_of(id) << (PT * i);
      const char* kf = k_from(at, id);
      const char* vf = v_from(at, id);
      each<CK>([&](auto j) MX_LAMBDA { copy_k(kf, i, j); });
      each<CV>([&](auto j) MX_LAMBDA { copy_v(vf, i, j); });
      store_k(i);
      store_v(i);
      id = ids_of(min((tile0 + i + 1) * KT, last));
    }
  }
  int stage = 0;
  for (int ti = tile0; ti < tile1; ++ti) {
    const int tile = ti * KT;
    // this wave's part of the tile is in LDS ...
    copies_done<(D - 2) * kCopies>();
    __syncthreads();  // ... and everyone's; the stage of the tile before is free
    const uint32_t parts = queue & kAllParts;
    queue >>= PT;
    const bool ragged = tile + KT > kall || parts != kAllParts;
    char* vs = lds + (D + stage) * kPart;
    if (ragged) {  // uniform: V of positions that are no keys may be anything, and becomes 0
      for (int i = t; i < HD * VP; i += 64 * NW) {
        const int dim = i / VP, key0 = 8 * ((i % VP) ^ v_swizzle<HD>(dim));
        const int n = (parts >> (key0 >> 4)) & 1 ? min(max(kall - tile - key0, 0), 8) : 0;
        if (n == 8) continue;
        uint16_t* p = reinterpret_cast<uint16_t*>(vs + i * 16);
        for (int j = n; j < 8; ++j) p[j] = 0;
      }
      __syncthreads();
    }
    const int ahead = stage == 0 ? D - 1 : stage - 1;  // of tile ti + D - 1
    queue |= bits_of(id) << (PT * (D - 2));
    const int at = min((ti + D - 1) * KT, last);
    const char* kf = k_from(at, id);
    const char* vf = v_from(at, id);
    // Issued together the copies hold up every wave of the workgroup at once, for as long as the
    // memory path takes for all of them, so they are spread over the scores' products (512 rows
    // on 12001 keys, 256 dims: 124 us against 133).
    auto copy = [&](auto i) MX_LAMBDA {
      if constexpr (i < CK)
        copy_k(kf, ahead, i);
      else
        copy_v(vf, ahead, i - CK);
    };
    floatx16_t sc[KB];
    scores(stage, sc, [&](auto i) MX_LAMBDA {
      constexpr int nc = kHalves ? CK : CK + CV;
      constexpr int n = KS * KB, first = i * nc / n, end = (i + 1) * nc / n;
      each<end - first>([&](auto j) MX_LAMBDA { copy(std::integral_constant<int, first + j>{}); });
    });
    if constexpr (kHalves) {
      store_k(ahead);
      each<CV>([&](auto i) MX_LAMBDA { copy_v(vf, ahead, i); });
    }
    uint4 a[R];
    each<R>([&](auto i) MX_LAMBDA { a[i] = v_operand(stage, i); });
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
    for (int i = 1; i < 16 * KB; ++i) mt = fmaxf(mt, sc[i / 16][i % 16]);
    mt = max_across_halves(mt) * sl2;
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
    // Where a pair does not see all of the tile, its p of 0 must not meet an infinite or NaN value:
    // such values go to the sums of the pairs that see them (they stay infinite or NaN whatever
    // their weight) and become 0 for the product.
    if (tile + KT - 1 > sees_all) {  // uniform
      char* vs = lds + (D + stage) * kPart;
      auto odd = [](uint32_t w) MX_LAMBDA {
        return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
      };
      bool some = false;
      for (int i = t; i < HD * VP; i += 64 * NW) {
        const uint4 v = *reinterpret_cast<const uint4*>(vs + i * 16);
        some |= odd(v.x) || odd(v.y) || odd(v.z) || odd(v.w);
      }
      if (__syncthreads_or(some)) {
        for (int key = 0; key < KT; ++key) {
          const bool in = tile + key <= limit && (parts >> (key >> 4) & 1);
          int half = h;  // addresses formed for each key: kept over the keys they would take
          asm volatile("" : "+v"(half));  // a register for every sum, in the loop over tiles too
#pragma unroll
          for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int dim = 32 * n + 8 * (r >> 2) + 4 * half + (r & 3);
              const uint16_t v = *reinterpret_cast<const uint16_t*>(
                  vs + (dim * VP + ((key >> 3) ^ v_swizzle<HD>(dim))) * 16 + (key & 7) * 2);
              if (in && (v & 0x7f80u) == 0x7f80u) o[n][r] += bf16_to_f32(v);
            }
        }
        __syncthreads();
        for (int i = t; i < HD * VP * 8; i += 64 * NW) {
          uint16_t* v = reinterpret_cast<uint16_t*>(vs) + i;
          if ((*v & 0x7f80u) == 0x7f80u) *v = 0;
        }
        __syncthreads();
        each<R>([&](auto i) MX_LAMBDA { a[i] = v_operand(stage, i); });
      }
    }
    uint32_t pb[KB * 8];
    auto pair = [&](auto j) MX_LAMBDA {
      constexpr int kb = j / 8, r = 2 * (j % 8);
      const float x = __builtin_amdgcn_exp2f(fmaf_(sc[kb][r], sl2, -ref));
      const float y = __builtin_amdgcn_exp2f(fmaf_(sc[kb][r + 1], sl2, -ref));
      l_run += x + y;
      pb[j] = pack2(x, y);
    };
    // P V of 16 keys takes four pairs; the next four form between its products
    each<4>(pair);
    constexpr int kP = 2 * KB * ND;
    each<kP>([&](auto i) MX_LAMBDA {
      constexpr int s = i / ND, n = i % ND;
      keep_order();
      o[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          __builtin_bit_cast(bf16x8_t, a[i % R]),
          __builtin_bit_cast(bf16x8_t, make_uint4(pb[4 * s], pb[4 * s + 1], pb[4 * s + 2],
                                                  pb[4 * s + 3])),
          o[n], 0, 0, 0);
      if constexpr (i + R < kP) a[i % R] = v_operand(stage, i + R);
      if constexpr (s + 1 < 2 * KB) {
        constexpr int first = 4 * n / ND, end = 4 * (n + 1) / ND;
        each<end - first>([&](auto j) MX_LAMBDA {
          pair(std::integral_constant<int, 4 * (s + 1) + first + j>{});
        });
      }
    });
    keep_order();
    // read here, the ids are there after the barrier; before, they would hold up the first
    // products, whose LDS reads wait on the same counter
    id = ids_of(min((ti + D) * KT, last));
    if constexpr (!kHalves) store_k(ahead);
    store_v(ahead);
    stage = stage == D - 1 ? 0 : stage + 1;
  }
  copies_done<0>();  // none lands in LDS that is no longer this workgroup's
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

// Joins the splits (at most 64) of some pairs of a kv head in order, a wave a pair at a time.
constexpr int kJoinPairs = 8;
template <int HD>
__global__ __launch_bounds__(256) void prefill_join_kernel(
    const uint16_t* __restrict__ qkv, int64_t qkv_stride, int rows,
    const int32_t* __restrict__ starts, const int32_t* __restrict__ lens,
    const float* __restrict__ v_scale, PageDims d, const float* __restrict__ o_part,
    const float* __restrict__ ml_part, uint16_t* __restrict__ out) {
  constexpr int KT = tile_keys<HD>(), DPL = HD / 64;
  typedef float vec __attribute__((ext_vector_type(DPL)));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = d.heads / d.kv_heads;
  const int kvh = blockIdx.x % d.kv_heads;
  const Plan plan = make_plan(starts, lens, d, rows, group);
  const int splits = plan.splits;
  const int all = rows * group, first = int(blockIdx.x / d.kv_heads) * kJoinPairs;  // below 2^31
  for (int i = first + wave; i < min(first + kJoinPairs, all); i += 4) {
    const int row = i / group, head = kvh * group + i - row * group;
    // the row's sequence
    int token = 0, pairs = 0, prior = 0;
    for (int s0 = 0; s0 < d.sequences && pairs == 0; s0 += 64) {
      const Rows r = s0 == 0 ? plan.r0 : rows_of(starts, lens, d, rows, s0 + lane);
      const uint64_t here = __ballot(row >= r.first && row < r.first + r.count);
      if (here) {
        const int f = __builtin_ctzll(here);
        token = row - __builtin_amdgcn_readlane(r.first, f);
        pairs = __builtin_amdgcn_readlane(r.count, f) * group;
        prior = __builtin_amdgcn_readlane(r.len - r.count, f);
      }
    }
    if (pairs == 0) continue;  // a row outside every sequence
    const int pair0 = (token * group + head - kvh * group) / kPairs * kPairs;  // of its block
    const int last_pair = min(pair0 + kPairs, pairs) - 1;
    const int kall = max(prior + last_pair / group + 1, 0);
    const int tiles = (kall + KT - 1) / KT, per = (tiles + splits - 1) / splits;
    if (per >= tiles) continue;  // one split (or none) wrote the result
    const int n = (tiles + per - 1) / per;
    const int64_t at = int64_t(row) * d.heads + head, part = at * splits;
    // eight splits' sums on their way while the weights form, a lane a split
    vec v[8];
#pragma unroll
    for (int c = 0; c < 8; ++c)
      v[c] = *reinterpret_cast<const vec*>(o_part + (part + min(c, n - 1)) * HD + DPL * lane);
    const float2 ml = *reinterpret_cast<const float2*>(ml_part + (part + min(lane, n - 1)) * 2);
    float M = ml.x;
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    const float e = lane < n ? __builtin_amdgcn_exp2f(ml.x - (M == neg_inf() ? 0.0f : M)) : 0.0f;
    float L = ml.y * e;
    for (int o = 32; o > 0; o >>= 1) L += __shfl_xor(L, o, 64);
    vec O = 0.0f;
    for (int c0 = 0; c0 < n; c0 += 8) {
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c0 + c < n) {  // uniform
          const float w = u2f(__builtin_amdgcn_readlane(int(f2u(e)), c0 + c));
          for (int k = 0; k < DPL; ++k) O[k] = fmaf_(v[c][k], w, O[k]);
        }
      if (c0 + 8 < n) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          v[c] = *reinterpret_cast<const vec*>(o_part + (part + min(c0 + 8 + c, n - 1)) * HD +
                                               DPL * lane);
      }
    }
    const float inv = (L == 0.0f ? 0.0f : 1.0f / L) * (v_scale ? v_scale[kvh] : 1.0f);
#pragma unroll
    for (int k = 0; k < DPL; ++k) {
      float y = L == 0.0f ? 0.0f : O[k] * inv;
      if (d.gated)
        y *= gate_of(bf16_to_f32(qkv[int64_t(row) * qkv_stride + int64_t(head) * 2 * HD + HD + DPL * lane + k]));
      out[at * HD + DPL * lane + k] = f32_to_bf16(y);
    }
  }
}

}  // namespace

// For any call of at most `rows` rows.  Fewer rows are split more, so that 300 rows may need more than
// 512, and 2048 none: the most that any number of rows gives, each with the fewest blocks.
size_t paged_prefill_workspace(int rows, const PageDims& d) {
  const int64_t group = d.heads / d.kv_heads;
  int64_t most = 0;  // rows times splits
  for (int64_t b = 1; (b - 1) * kPairs < rows * group; ++b) {
    const int splits = splits_of(b, d);
    if (splits == 1) break;  // and so for more blocks
    const int64_t r = b * kPairs / group < rows ? b * kPairs / group : rows;  // the last row with b blocks
    most = r * splits > most ? r * splits : most;
  }
  return size_t(most) * d.heads * (d.head_dim + 2) * 4;
}

bool paged_prefill_splits(int rows, const PageDims& d) { return splits_of(least_blocks(rows, d), d) > 1; }

int paged_prefill(const uint16_t* q, const uint16_t* qkv, int64_t qkv_stride, int rows,
                  const int32_t* starts, const int32_t* lens, const int32_t* table,
                  const void* k_cache, const void* v_cache, const float* k_scale,
                  const float* v_scale, const PageDims& d, float scale, void* workspace,
                  uint16_t* out, hipStream_t s) {
  // Workgroups for any number of blocks that starts may give: the number itself is the kernel's to
  // find.  Beyond 256 blocks of a kv head nothing is split, and more blocks have more workgroups.
  const int64_t group = d.heads / d.kv_heads, least = least_blocks(rows, d);
  const int64_t most = int64_t(rows) * group / kPairs + (d.sequences < rows ? d.sequences : rows);
  int64_t grid = most * items_of(d.kv_heads, splits_of(most, d));
  for (int64_t b = least; b < most && b * d.kv_heads <= 256; ++b) {
    const int64_t n = b * items_of(d.kv_heads, splits_of(b, d));
    grid = n > grid ? n : grid;
  }
  const int splits = splits_of(least, d);  // at most
  const int64_t joins = (int64_t(rows) * group + kJoinPairs - 1) / kJoinPairs * d.kv_heads;
  if (grid > 0x7fffffff || joins > 0x7fffffff) return MX_EUNSUPPORTED;
  float* o_part = static_cast<float*>(workspace);
  float* ml_part = o_part + size_t(rows) * d.heads * splits * d.head_dim;
  const float* vs = d.f8 ? v_scale : nullptr;
#define MX_PREFILL(HH, FF)                                                                       \
  if (d.head_dim == HH && d.f8 == FF) {                                                          \
    const auto fn = prefill_kernel<HH, FF>;                                                      \
    constexpr int lb = D * stage_bytes<HH>();                                                    \
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(fn),                                   \
                            hipFuncAttributeMaxDynamicSharedMemorySize, lb) != hipSuccess)       \
      return MX_EHIP;                                                                            \
    hipLaunchKernelGGL(fn, dim3(unsigned(grid)), dim3(64 * NW), lb, s, q, qkv, qkv_stride, rows, \
                       starts, lens, table, k_cache, v_cache, k_scale, v_scale, d, scale,        \
                       o_part, ml_part, out);                                                    \
    if (hipGetLastError() != hipSuccess) return MX_EHIP;                                         \
    if (splits == 1) return MX_OK;                                                               \
    hipLaunchKernelGGL((prefill_join_kernel<HH>), dim3(unsigned(joins)), dim3(256), 0, s, qkv,   \
                       qkv_stride, rows, starts, lens, vs, d, o_part, ml_part, out);             \
    return hipGetLastError() == hipSuccess ? MX_OK : MX_EHIP;                                    \
  }
  MX_PREFILL(64, false) MX_PREFILL(128, false) MX_PREFILL(256, false)
  MX_PREFILL(64, true) MX_PREFILL(128, true) MX_PREFILL(256, true)
#undef MX_PREFILL
  return MX_EUNSUPPORTED;
}

}  // namespace mx
