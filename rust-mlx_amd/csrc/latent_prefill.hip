// Causal attention of the last rows of packed sequences, whose keys and values have been formed from the
// latents for every head: expanded, so that a (row, key) pair costs 2 (nope + rope + v) operations a head
// where the latents themselves would cost 2 (2 latent + rope).
//
// Sequence s has the rows starts[s] .. starts[s + 1] - 1 and the keys kv_starts[s] .. kv_starts[s + 1] - 1;
// its rows are its last positions, and each sees the keys up to its own.  A head's key is its nope part
// beside the rotary key that all heads share; kv rows hold [head][nope | v].
//
// The shape is that of the paged cache's prompt attention with one row a pair: eight waves take 256 rows
// of one sequence and head, 32 matrix-core columns a wave, and walk the keys in tiles of 64:
//   S^T = K Q^T       A: key rows from LDS, 16 bytes a lane, B: q in registers
//   O^T = V^T P^T     A: value rows read transposed from LDS, B: P as it stands
// with rows entering in the order that leaves P in the lane that supplies it (bits 2 and 3 exchanged).
//
// P is rounded to bf16 for the product, each p by at most 2^-8 of itself, as the output is; the sum that
// divides takes P before it.
//
// The matrix units bound it: 8192 rows of 32 heads take 622 to 675 us from card to card (1.02 to 1.11
// PFLOP/s), 512 rows of 20 heads on 12001 positions 96 to 105 (six splits, 9 of it the join).  256 rows a
// workgroup read each key half as often as 128; with 128 and tiles of 32 keys these took 746 and 113 us.  A
// tile's copies are all issued at its top: spread over its products they take a quarter longer.
#include <type_traits>

#include "prompt_plan.hpp"

namespace mx {

namespace {

using namespace pg;

constexpr int NW = 8;   // waves of a workgroup
constexpr int kRows = LatentPromptDims::kPairs;
static_assert(kRows == 32 * NW, "32 rows a wave");
constexpr int KT = 64;  // keys of a tile
constexpr int D = 3;    // stages of a tile in LDS
constexpr int DR = 64;  // rope_dim

// A stage holds blocks of 64 values of its keys' rows: a head's keys and values, then the rotary keys.
constexpr int kBlock = KT * 128;
template <int HD>
constexpr int stage_bytes() {
  return (2 * HD + DR) / 64 * kBlock;
}

// 16-byte pieces of a block's row are exchanged by the row's number: sixteen rows' operands meet none of the
// 64 banks twice, nor do four pieces of four rows, as the transposed reads take them.
__device__ __forceinline__ int swizzle(int row) {
  return (row & 2) << 1 | (row >> 1 & 2) | (row >> 3 & 1);
}

template <int HD>  // nope_dim and v_dim
__global__ __launch_bounds__(64 * NW, 2) void prefill_kernel(
    const uint16_t* __restrict__ q, int64_t q_stride, const uint16_t* __restrict__ q_rope, int rows,
    const int32_t* __restrict__ starts, const uint16_t* __restrict__ kv, int64_t kv_stride,
    const uint16_t* __restrict__ k_rope, int64_t rope_stride, const int32_t* __restrict__ kv_starts,
    LatentPromptDims d, float scale, float* __restrict__ o_part, float* __restrict__ ml_part,
    uint16_t* __restrict__ out) {
  constexpr int KN = HD / 16, KS = KN + DR / 16;  // steps of S^T: of the nope part, all
  constexpr int KB = KT / 32;                     // 32-key operands of a tile
  constexpr int ND = HD / 32;                     // 32-dim operands of the output
  constexpr int NB = (2 * HD + DR) / 64;          // blocks of a stage, the rotary one last
  constexpr int G = KT / NW / 8;                  // eights of rows that a wave copies
  constexpr int NC = NB * G;                      // its copies: eight rows of a block
  constexpr int STAGE = stage_bytes<HD>();
  constexpr int R = 4;                            // operands read ahead of their products
  extern __shared__ __align__(128) char lds[];
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int col = lane & 31, h = lane >> 5;
  const PromptPlan plan = prompt_plan(starts, kv_starts, d, rows, 1);
  const int splits = plan.splits;
  const Item it = item_of<LatentPromptDims>(blockIdx.x, plan, d.kv_heads);
  if (it.split >= splits) return;
  const int head = it.kvh, split = it.split;
  Block b;
  if (!find_block(plan, starts, kv_starts, d, rows, 1, it.block, &b)) return;  // uniform
  const int kv_first = max(kv_starts[b.seq], 0);
  const int prior = b.len - b.count;  // the first row's position (negative: rows without one)
  const int last_row = min(b.pair0 + kRows, b.count) - 1;
  const int kall = max(prior + last_row + 1, 0);  // keys that the block sees
  const int tiles = (kall + KT - 1) / KT;
  const int per = (tiles + splits - 1) / splits;
  const int tile0 = split * per, tile1 = min(tiles, tile0 + per);
  const bool whole = tile0 == 0 && tile1 == tiles;  // also a block without keys
  if (tile0 >= tile1 && !(split == 0 && tiles == 0)) return;

  // this lane's row; lanes past the last one take that, see nothing and write nothing
  const bool alive = b.pair0 + 32 * wave + col < b.count;
  const int token = min(b.pair0 + 32 * wave + col, b.count - 1);
  const int64_t qrow = b.first + token;
  const int limit = alive ? prior + token : -1;  // the last key that the row sees
  uint4 qb[KS];
  {
    const uint16_t* src = q + qrow * q_stride + int64_t(head) * (HD + DR) + 8 * h;
    const uint16_t* rot = q_rope + (qrow * d.heads + head) * DR + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qb[s] = *reinterpret_cast<const uint4*>(s < KN ? src + 16 * s : rot + 16 * (s - KN));
  }
  // every live row of the wave sees the keys up to low, none one past high
  const int low = prior + b.pair0 + 32 * wave;
  const int high = b.pair0 + 32 * wave < b.count ? min(low + 31, prior + b.count - 1) : -1;
  const bool full = b.pair0 + 32 * wave + 31 < b.count;  // no lane past the last row
  const int sees_all = prior + b.pair0;  // the last key that every row of the block sees
  const float sl2 = scale * kLog2e;

  // One tile's copies: a wave takes some of its rows, eight a copy of 1 KB of one block.  A lane copies the piece of
  // its row that its place is for.  Keys past the last one are that one: their scores are masked and their
  // values zeroed.
  const uint32_t lds_at =
      uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
  const char* kv_at = reinterpret_cast<const char*>(kv + kv_first * kv_stride + int64_t(head) * 2 * HD);
  const char* rope_at = reinterpret_cast<const char*>(k_rope + kv_first * rope_stride);
  const int64_t kv_bytes = kv_stride * 2, rope_bytes = rope_stride * 2;
  uint32_t kv_off[G], rope_off[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const uint32_t piece = 16 * ((lane & 7) ^ swizzle(8 * (G * wave + g) + (lane >> 3)));
    kv_off[g] = uint32_t(lane >> 3) * uint32_t(kv_bytes) + piece;
    rope_off[g] = uint32_t(lane >> 3) * uint32_t(rope_bytes) + piece;
  }
  auto copy = [&](int tile, int stage, int i) MX_LAMBDA {  // i: 0 .. NC - 1
    const int block = i / G, g = i % G, r = 8 * (G * wave + g);
    const uint32_t to = lds_at + stage * STAGE + block * kBlock + r * 128;
    if (tile + KT <= b.len) {  // uniform
      if (block < NB - 1)
        copy_to_lds(kv_at + (tile + r) * kv_bytes + block * 128, kv_off[g], to);
      else
        copy_to_lds(rope_at + (tile + r) * rope_bytes, rope_off[g], to);
    } else {
      const int key = min(tile + r + (lane >> 3), b.len - 1);
      const uint32_t piece = 16 * ((lane & 7) ^ swizzle(r + (lane >> 3)));
      copy_to_lds((block < NB - 1 ? kv_at + key * kv_bytes + block * 128 : rope_at + key * rope_bytes) + piece, to);
    }
  };

  // Operands of product i of the scores, and of P V.  Steps differ by the exchanged bits within a block's row.
  const int krow = (col & 0x13) | ((col & 4) << 1) | ((col & 8) >> 1);  // bits 2 and 3 exchanged
  const uint32_t k_at = lds_at + krow * 128 + 16 * (h ^ swizzle(krow));
  const int vrow = 8 * h + ((lane & 15) >> 2);  // and four rows on
  const uint32_t v_at = lds_at + HD / 64 * kBlock + vrow * 128 + 8 * (lane & 1) +
                        16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ swizzle(vrow));
  uint32_t kb[4], vb[2][2];
  auto enter = [&](uint32_t stage_at) MX_LAMBDA {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      kb[j] = (k_at ^ (32 * j)) + stage_at;
      vb[j >> 1][j & 1] = (v_at ^ (64 * (j >> 1) | 32 * (j & 1))) + (stage_at + (j & 1) * 512);
    }
  };
  auto k_operand = [&](int i) MX_LAMBDA {
    const int s = i / KB;
    typedef uint32_t vec __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(uint4, lds_read<vec>(kb[s & 3] + ((s < KN ? s >> 2 : NB - 1) * kBlock + i % KB * (32 * 128))));
  };
  auto v_operand = [&](int i) MX_LAMBDA {
    const int n = i % ND, s = i / ND;
    const uint32_t off = (n >> 1) * kBlock + s * (16 * 128);
    const uint2 x = lds_read_tr16(vb[n & 1][0] + off), y = lds_read_tr16(vb[n & 1][1] + off);
    return make_uint4(x.x, x.y, y.x, y.y);
  };

  // A row's weight of 0 must not meet an infinite or NaN value that it does not see.  It would leave NaN in
  // the row's sums, so tiles are taken as they are, and where a sum is not finite all of them are taken once
  // more, with care, in code of its own, so that the first turn's has the registers.  (One prompt of 256 rows
  // takes 17.5 us; 17.9 with one loop for both turns, 19.6 with care at once.)
  float m_run, l_run;
  floatx16_t o[ND];
  auto walk = [&](auto careful) MX_LAMBDA {
    // (below every score, and finite, so that a masked one's -inf has the weight 0)
    m_run = -__FLT_MAX__, l_run = 0.0f;
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[n][r] = 0.0f;

    // Tiles past the last one are copied like it, into stages that nobody reads: every step has
    // the same copies, so waiting for all but the latest is waiting for their number.
    const int last = (tile1 - 1) * KT;
    if (tile0 < tile1)
#pragma unroll
      for (int i = 0; i < D - 1; ++i)
        each<NC>([&](auto j) MX_LAMBDA { copy(min((tile0 + i) * KT, last), i, j); });
    int stage = 0;
    for (int ti = tile0; ti < tile1; ++ti) {
      const int tile = ti * KT;
      copies_done<(D - 2) * NC>();  // this wave's part of the tile is in LDS ...
      __syncthreads();  // ... and everyone's; the stage of the tile before is free
      const uint32_t stage_at = stage * STAGE;
      const int ahead = stage == 0 ? D - 1 : stage - 1;  // of tile ti + D - 1
      const int at = min((ti + D - 1) * KT, last);
      each<NC>([&](auto j) MX_LAMBDA { copy(at, ahead, j); });
      stage = stage == D - 1 ? 0 : stage + 1;
      // uniform: nothing here that a row of this wave sees (the careful turn's barriers are for all waves)
      if (!careful && tile > high) continue;
      enter(stage_at);
      floatx16_t sc[KB];
#pragma unroll
      for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[k][r] = 0.0f;
      uint4 a[R];
      each<R>([&](auto i) MX_LAMBDA { a[i] = k_operand(i); });
      each<KS * KB>([&](auto i) MX_LAMBDA {
        __builtin_amdgcn_sched_barrier(0);
        sc[i % KB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a[i % R]),
                                                             __builtin_bit_cast(bf16x8_t, qb[i / KB]),
                                                             sc[i % KB], 0, 0, 0);
        if constexpr (i + R < KS * KB) a[i % R] = k_operand(i + R);
      });
      __builtin_amdgcn_sched_barrier(0);
      if (!careful) each<R>([&](auto i) MX_LAMBDA { a[i] = v_operand(i); });
      // sc[k][r]: key 32 k + 16 (r / 8) + 8 h + r % 8 of the tile
      if (tile + KT - 1 > low || !full) {
        const int end = limit + 1 - tile - 8 * h;
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[k][r] = 32 * k + 16 * (r >> 3) + (r & 7) < end ? sc[k][r] : neg_inf();
      }
      float mt = sc[0][0];
#pragma unroll
      for (int i = 1; i < 16 * KB; ++i) mt = fmaxf(mt, sc[i / 16][i % 16]);
      mt = max_across_halves(mt) * sl2;
      // The reference follows the maximum in steps of at least 8 (a factor of 256, far from any
      // limit of fp32 or bf16), so that most tiles rescale nothing.
      if (__any(mt > m_run + 8.0f)) {
        const float mn = mt > m_run + 8.0f ? mt : m_run;  // each column by its own scores alone
        const float alpha = __builtin_amdgcn_exp2f(m_run - mn);
        l_run *= alpha;
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[n][r] *= alpha;
        m_run = mn;
      }
      // The careful turn: keys past the last one become 0, in a tile that has any; in one that some rows see
      // and some do not, infinite and NaN values go to the sums of the rows that see them (they stay infinite or
      // NaN whatever their weight, but for that of a score of -inf, which makes NaN of them) and become 0 for the
      // product.
      if (careful && tile + KT - 1 > sees_all) {  // uniform
        auto value_at = [&](int key, int piece) MX_LAMBDA {
          return lds + stage_at + (HD / 64 + (piece >> 3)) * kBlock + key * 128 +
                 16 * ((piece & 7) ^ swizzle(key));
        };
        auto odd = [](uint32_t w) MX_LAMBDA {
          return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
        };
        bool some = false;
        for (int i = t; i < KT * HD / 8; i += 64 * NW) {
          uint4* p = reinterpret_cast<uint4*>(value_at(i / (HD / 8), i % (HD / 8)));
          if (tile + i / (HD / 8) >= kall) {
            *p = make_uint4(0, 0, 0, 0);
          } else {
            const uint4 v = *p;
            some |= odd(v.x) || odd(v.y) || odd(v.z) || odd(v.w);
          }
        }
        if (__syncthreads_or(some)) {
          uint32_t counts[KB];  // the row's scores above -inf, a key a bit
#pragma unroll
          for (int k = 0; k < KB; ++k) {
            counts[k] = 0;
#pragma unroll
            for (int r = 0; r < 16; ++r)
              counts[k] |= uint32_t(sc[k][r] != neg_inf()) << (16 * (r >> 3) + 8 * h + (r & 7));
            counts[k] |= __shfl_xor(counts[k], 32, 64);
          }
          for (int key = 0; key < KT; ++key) {
            const bool in = tile + key <= limit;
            uint32_t mine = counts[0];
#pragma unroll
            for (int k = 1; k < KB; ++k) mine = key >> 5 == k ? counts[k] : mine;
            const float by = mine >> (key & 31) & 1 ? 1.0f : 0.0f;
            int half = h;  // addresses formed for each key: kept over the keys they would take
            asm volatile("" : "+v"(half));  // a register for every sum, in the loop over tiles too
#pragma unroll
            for (int n = 0; n < ND; ++n)
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const int dim = 32 * n + 8 * (r >> 2) + 4 * half + (r & 3);
                const uint16_t v = reinterpret_cast<const uint16_t*>(value_at(key, dim >> 3))[dim & 7];
                if (in && (v & 0x7f80u) == 0x7f80u) o[n][r] += bf16_to_f32(v) * by;
              }
          }
          __syncthreads();
          for (int i = t; i < KT * HD; i += 64 * NW) {
            uint16_t* v = reinterpret_cast<uint16_t*>(value_at(i / HD, i % HD / 8)) + i % 8;
            if ((*v & 0x7f80u) == 0x7f80u) *v = 0;
          }
          __syncthreads();
        }
      }
      if (careful) each<R>([&](auto i) MX_LAMBDA { a[i] = v_operand(i); });  // as they are now
      uint32_t pb[8 * KB];
      auto pair = [&](auto j) MX_LAMBDA {
        constexpr int k = j / 8, r = 2 * (j % 8);
        const float x = __builtin_amdgcn_exp2f(fmaf_(sc[k][r], sl2, -m_run));
        const float y = __builtin_amdgcn_exp2f(fmaf_(sc[k][r + 1], sl2, -m_run));
        l_run += x + y;
        pb[j] = pack2(x, y);
      };
      // P V of 16 keys takes four pairs; the next four form between its products
      each<4>(pair);
      constexpr int kP = 2 * KB * ND;
      each<kP>([&](auto i) MX_LAMBDA {
        constexpr int s = i / ND, n = i % ND;
        __builtin_amdgcn_sched_barrier(0);
        o[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8_t, a[i % R]),
            __builtin_bit_cast(bf16x8_t,
                               make_uint4(pb[4 * s], pb[4 * s + 1], pb[4 * s + 2], pb[4 * s + 3])),
            o[n], 0, 0, 0);
        if constexpr (i + R < kP) a[i % R] = v_operand(i + R);
        if constexpr (s + 1 < 2 * KB) {
          constexpr int first = 4 * n / ND, end = 4 * (n + 1) / ND;
          each<end - first>([&](auto j) MX_LAMBDA { pair(std::integral_constant<int, 4 * (s + 1) + first + j>{}); });
        }
      });
      __builtin_amdgcn_sched_barrier(0);
    }
    copies_done<0>();  // none lands in LDS that is no longer this workgroup's, or the next turn's
  };
  walk(std::false_type{});
  float most = 0.0f;
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) most += o[n][r] * 0.0f;  // NaN of what is not finite
  if (__syncthreads_or(alive && !(most == 0.0f))) walk(std::true_type{});
  if (!alive) return;
  l_run += __shfl_xor(l_run, 32, 64);
  const int64_t at = qrow * d.heads + head;
  if (whole) {
    const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
    uint16_t* dst = out + at * HD + 4 * h;
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = l_run == 0.0f ? 0.0f : o[n][4 * a + r] * inv;
        *reinterpret_cast<uint2*>(dst + 32 * n + 8 * a) = make_uint2(pack2(y[0], y[1]), pack2(y[2], y[3]));
      }
    return;
  }
  const int64_t part = at * splits + split;
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

LatentPromptDims prompt_dims(int kv_rows, const LatentDims& d) {
  return LatentPromptDims{d.heads, d.heads, d.sequences, kv_rows};
}

}  // namespace

size_t latent_prefill_workspace(int rows, int kv_rows, const LatentDims& d) {
  return prompt_workspace(rows, d.v_dim, prompt_dims(kv_rows, d));
}

bool latent_prefill_splits(int rows, int kv_rows, const LatentDims& d) {
  const LatentPromptDims p = prompt_dims(kv_rows, d);
  return splits_of(least_blocks(rows, p), p) > 1;
}

int latent_prefill(const uint16_t* q, int64_t q_stride, const uint16_t* q_rope, int rows,
                   const int32_t* starts, const uint16_t* kv, int64_t kv_stride,
                   const uint16_t* k_rope, int64_t rope_stride, int kv_rows,
                   const int32_t* kv_starts, const LatentDims& dims, float scale, void* workspace,
                   uint16_t* out, hipStream_t s) {
  const LatentPromptDims d = prompt_dims(kv_rows, dims);
  const int64_t grid = prompt_grid(rows, d), joins = prompt_joins(rows, d);
  const int splits = splits_of(least_blocks(rows, d), d);  // at most
  if (grid > 0x7fffffff || joins > 0x7fffffff) return MX_EUNSUPPORTED;
  float* o_part = static_cast<float*>(workspace);
  float* ml_part = o_part + size_t(rows) * d.heads * splits * dims.v_dim;
#define MX_PREFILL(HD)                                                                             \
  if (dims.v_dim == HD) {                                                                          \
    const auto fn = prefill_kernel<HD>;                                                            \
    constexpr int lb = D * stage_bytes<HD>();                                                      \
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(fn),                                     \
                            hipFuncAttributeMaxDynamicSharedMemorySize, lb) != hipSuccess)         \
      return MX_EHIP;                                                                              \
    hipLaunchKernelGGL(fn, dim3(unsigned(grid)), dim3(64 * NW), lb, s, q, q_stride, q_rope, rows,  \
                       starts, kv, kv_stride, k_rope, rope_stride, kv_starts, d, scale, o_part,    \
                       ml_part, out);                                                              \
    if (hipGetLastError() != hipSuccess) return MX_EHIP;                                           \
    if (splits == 1) return MX_OK;                                                                 \
    hipLaunchKernelGGL((prefill_join_kernel<HD, KT, LatentPromptDims>), dim3(unsigned(joins)),     \
                       dim3(256), 0, s, nullptr, 0, rows, starts, kv_starts, nullptr, d, o_part,   \
                       ml_part, out);                                                              \
    return hipGetLastError() == hipSuccess ? MX_OK : MX_EHIP;                                      \
  }
  MX_PREFILL(64) MX_PREFILL(128)
#undef MX_PREFILL
  return MX_EUNSUPPORTED;
}

}  // namespace mx
