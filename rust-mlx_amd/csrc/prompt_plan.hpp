// Attention of the last rows of packed sequences: how their (row, q head) pairs are shared out over
// workgroups, the keys over splits, and the join of the splits' partials.
#pragma once

#include <utility>

#include "paged_core.hpp"

namespace mx {
namespace pg {

// Of the description Dims: kPairs, the pairs of a workgroup, and kAtOnce, the workgroups that run at once.

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

// The length of sequence s, cut to what the cache's table can hold, and the most that it can be.
__device__ __forceinline__ int context_of(const int32_t* __restrict__ lens, const PageDims& d, int s) {
  const int64_t most = int64_t(d.table_width) << d.page_log2;
  const int len = lens[s];
  return len < 0 ? 0 : (len > most ? int(most) : len);
}
__host__ __device__ __forceinline__ int64_t longest_context(const PageDims& d) {
  return int64_t(d.table_width) << d.page_log2;
}
// Of keys that lie packed like the rows: lens is where each sequence's begin.
__device__ __forceinline__ int context_of(const int32_t* __restrict__ lens, const LatentPromptDims& d,
                                          int s) {
  return max(min(lens[s + 1], d.kv_rows) - max(lens[s], 0), 0);
}
__host__ __device__ __forceinline__ int64_t longest_context(const LatentPromptDims& d) {
  return d.kv_rows;
}

// Rows of a sequence, which are the packed ones from `first` on, and its length.
struct Rows {
  int first, count, len;
};
template <class Dims>
__device__ __forceinline__ Rows rows_of(const int32_t* __restrict__ starts,
                                        const int32_t* __restrict__ lens, const Dims& d, int rows,
                                        int s) {
  Rows r = {0, 0, 0};
  if (s < d.sequences) {
    r.first = min(max(starts[s], 0), rows);
    r.count = max(min(starts[s + 1], rows) - r.first, 0);
    r.len = context_of(lens, d, s);
  }
  return r;
}
template <class Dims>
__device__ __forceinline__ int blocks_of(const Rows& r, int group) {
  return int((int64_t(r.count) * group + Dims::kPairs - 1) / Dims::kPairs);
}

// How many workgroups share the keys of a query block, with `blocks` of them: as many as bring the
// launch to what runs at once, each with at least 256 keys of the longest possible context; in eights with the
// kv heads where that is possible, for whole XCDs (512 rows on 12001 keys, two kv heads: 8 splits 126 us, 7 splits
// 138).  At most 64, never more with more blocks.
template <class Dims>
__host__ __device__ __forceinline__ int splits_of(int64_t blocks, const Dims& d) {
  const int64_t all = blocks * d.kv_heads, room = longest_context(d) / 256;
  int s = all > Dims::kAtOnce / 2 ? 1 : Dims::kAtOnce / int(all < 1 ? 1 : all);
  s = s > room ? int(room) : s;
  s = s > 64 ? 64 : s < 1 ? 1 : s;
  const int low = d.kv_heads & -d.kv_heads, step = low >= 8 ? 1 : 8 / low;  // powers of two
  const int e = (s + step - 1) & -step;
  return s > 1 && e < 2 * s && e <= room ? e : s;
}
// The fewest blocks that a call of so many rows is laid out for.
template <class Dims>
__host__ __device__ __forceinline__ int64_t least_blocks(int rows, const Dims& d) {
  return (int64_t(rows) * (d.heads / d.kv_heads) + Dims::kPairs - 1) / Dims::kPairs;
}

// What follows from all sequences' rows, formed by every wave: the number of query blocks (sequences
// without rows have none, however many the table has) and the splits; `r0`: the rows of the first 64
// sequences, a lane each.
struct PromptPlan {
  Rows r0;
  int blocks, splits;
};
template <class Dims>
__device__ __forceinline__ PromptPlan prompt_plan(const int32_t* __restrict__ starts,
                                          const int32_t* __restrict__ lens, const Dims& d,
                                          int rows, int group) {
  const int lane = threadIdx.x & 63;
  PromptPlan p;
  p.r0 = rows_of(starts, lens, d, rows, lane);
  int n = blocks_of<Dims>(p.r0, group);
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
      n += blocks_of<Dims>({first, max(min(to[i], rows) - first, 0), 0}, group);
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
template <class Dims>
__device__ __forceinline__ bool find_block(const PromptPlan& p, const int32_t* __restrict__ starts,
                                           const int32_t* __restrict__ lens, const Dims& d,
                                           int rows, int group, int want, Block* out) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < d.sequences; s0 += 64) {
    const Rows r = s0 == 0 ? p.r0 : rows_of(starts, lens, d, rows, s0 + lane);
    const int sum = wave_scan(blocks_of<Dims>(r, group));
    const uint64_t past = __ballot(before + sum > want);
    if (past) {
      const int f = __builtin_ctzll(past);
      // uniform values, into scalar registers
      out->seq = __builtin_amdgcn_readfirstlane(s0 + f);
      out->first = __builtin_amdgcn_readlane(r.first, f);
      out->count = __builtin_amdgcn_readlane(r.count, f);
      out->pair0 = (before + __builtin_amdgcn_readlane(sum, f) - 1 - want) * Dims::kPairs;
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
// e4m3: 144 us against 152).  Only where two workgroups share a unit, so never of latent prompts.
template <class Dims>
__device__ __forceinline__ Item item_of(int id, const PromptPlan& p, int kv_heads) {
  const int pairs = kv_heads * p.splits, a_block = items_of(kv_heads, p.splits);
  const bool xcd = by_xcd(kv_heads, p.splits);
  const int each = a_block / 8;  // pairs of an XCD
  const int j = id >> 3, pair = xcd ? (id & 7) + 8 * (j % each) : id % pairs;
  int block = xcd ? j / each : id / pairs;
  if (block >= p.blocks) return Item{block, 0, p.splits};  // past the last block: none
  const int64_t all = int64_t(p.blocks) * a_block;
  if (all > 256 && all <= Dims::kAtOnce) {
    const int first = 256 / a_block;
    if (block >= first) block = p.blocks - 1 - (block - first);
  }
  return Item{block, pair % kv_heads, pair / kv_heads};  // split >= splits: none
}

// Joins the splits (at most 64) of some pairs of a kv head in order, a wave a pair at a time.
constexpr int kJoinPairs = 8;
template <int HD, int KT, class Dims>
__global__ __launch_bounds__(256) void prefill_join_kernel(
    const uint16_t* __restrict__ qkv, int64_t qkv_stride, int rows,
    const int32_t* __restrict__ starts, const int32_t* __restrict__ lens,
    const float* __restrict__ v_scale, Dims d, const float* __restrict__ o_part,
    const float* __restrict__ ml_part, uint16_t* __restrict__ out) {
  constexpr int DPL = HD / 64;
  typedef float vec __attribute__((ext_vector_type(DPL)));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = d.heads / d.kv_heads;
  const int kvh = blockIdx.x % d.kv_heads;
  const PromptPlan plan = prompt_plan(starts, lens, d, rows, group);
  const int splits = plan.splits;
  if (splits == 1) return;  // the rows lie in more blocks than they could have
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
    const int pair0 = (token * group + head - kvh * group) / Dims::kPairs * Dims::kPairs;  // of its block
    const int last_pair = min(pair0 + Dims::kPairs, pairs) - 1;
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

// For any call of at most `rows` rows.  Fewer rows are split more, so that 300 rows may need more than
// 512, and 2048 none: the most that any number of rows gives, each with the fewest blocks.
template <class Dims>
size_t prompt_workspace(int rows, int head_dim, const Dims& d) {
  const int64_t group = d.heads / d.kv_heads;
  int64_t most = 0;  // rows times splits
  for (int64_t b = 1; (b - 1) * Dims::kPairs < rows * group; ++b) {
    const int splits = splits_of(b, d);
    if (splits == 1) break;  // and so for more blocks
    const int64_t r = b * Dims::kPairs / group < rows ? b * Dims::kPairs / group : rows;  // the last row with b blocks
    most = r * splits > most ? r * splits : most;
  }
  return size_t(most) * d.heads * (head_dim + 2) * 4;
}

template <class Dims>
int64_t prompt_grid(int rows, const Dims& d) {
  // Workgroups for any number of blocks that starts may give: the number itself is the kernel's to
  // find.  Beyond kAtOnce / 2 blocks and kv heads nothing is split, and more blocks have more workgroups.
  const int64_t group = d.heads / d.kv_heads, least = least_blocks(rows, d);
  const int64_t most = int64_t(rows) * group / Dims::kPairs + (d.sequences < rows ? d.sequences : rows);
  int64_t grid = most * items_of(d.kv_heads, splits_of(most, d));
  for (int64_t b = least; b < most && b * d.kv_heads <= Dims::kAtOnce / 2; ++b) {
    const int64_t n = b * items_of(d.kv_heads, splits_of(b, d));
    grid = n > grid ? n : grid;
  }
  return grid;
}
template <class Dims>
int64_t prompt_joins(int rows, const Dims& d) {
  return (int64_t(rows) * (d.heads / d.kv_heads) + kJoinPairs - 1) / kJoinPairs * d.kv_heads;
}

}  // namespace pg
}  // namespace mx
