// Attention of one new token a row over the latent cache: absorbed, so that a position's row of
// latent and rotary key is the key of every head, and its latent their value:
//
//   s[h, p] = scale (q_latent[h] . c[p] + q_rope[h] . k[p]),  out[h] = sum_p softmax(s[h])[p] c[p]
//
// A workgroup takes one chunk of one row's positions and all heads, and walks it in tiles of 32 positions
// that are copied to LDS ahead.  Heads are matrix-core columns, 32 a wave, and two or four waves share
// them: each forms the scores over its part of a position's row, the parts meet in LDS, and each has its
// part of the output's dims (one wave alone would hold 400 registers of q and sums).
//   S^T = K Q^T       A: positions from LDS, 16 bytes a lane, B: q in registers
//   O^T = C^T P^T     A: the same positions, read transposed from LDS, B: P as it stands
// Lane (head c = l % 32, half h = l / 32) receives the scores of rows 8 a + 4 h + b of the tile and
// supplies the k-slots 8 h + i of each 16 positions for the second product; rows enter with bits 2 and
// 3 exchanged, so the two are the same positions and P never leaves its lane.
//
// P is rounded to bf16 for the product, each p by at most 2^-8 of itself, as the output is; the sum
// that divides takes P before it.
//
// Rows that need several chunks leave partials in fp32, which a second launch joins in order.
#include <type_traits>

#include "prompt_plan.hpp"

namespace mx {

namespace {

using namespace pg;

constexpr int KT = 32;   // positions of a tile
constexpr int DR = 64;   // rope_dim
typedef short shortx4_t __attribute__((ext_vector_type(4)));

// Head waves (32 heads each), and waves that share their heads.
template <int HW>
constexpr int shares() {
  return HW == 4 ? 2 : 4;
}
constexpr int kPartBytes = KT * 32 * 4;  // of a wave's scores
template <bool F8>
constexpr int stages() {
  return F8 ? 2 : 3;
}
template <int DC, int HW, bool F8>
constexpr int lds_bytes() {
  return stages<F8>() * (KT * (DC + DR) * 2 + (F8 ? KT * 4 : 0)) + HW * shares<HW>() * kPartBytes;
}

// 16-byte pieces of a row are exchanged by the row's number within their 128 bytes: eight rows'
// operands meet no bank twice, nor do two pieces of four rows, as the transposed reads take them.
__device__ __forceinline__ int swizzle(int row) {
  return (row & 3) << 1 | ((row >> 2 ^ row >> 3) & 1);
}
__device__ __forceinline__ uint4 lds_read16(uint32_t at) {
  typedef uint32_t vec __attribute__((ext_vector_type(4)));
  const vec v = *reinterpret_cast<__attribute__((address_space(3))) const vec*>(at);
  return make_uint4(v.x, v.y, v.z, v.w);
}
// Of sixteen lanes, four rows of sixteen values (lane j: four values of row j / 4 at `at`), lane j gets
// the four rows' value j.
__device__ __forceinline__ uint2 lds_read_tr(uint32_t at) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       reinterpret_cast<__attribute__((address_space(3))) shortx4_t*>(at)));
}

template <int DC, int HW, bool F8>
__global__ __launch_bounds__(64 * HW * shares<HW>(), 1) void decode_kernel(
    const uint16_t* __restrict__ q_latent, const uint16_t* __restrict__ q_rope, int rows,
    const int32_t* __restrict__ seqs, const int32_t* __restrict__ lens,
    const int32_t* __restrict__ table, const void* __restrict__ cache,
    const float* __restrict__ scales, LatentDims d, float scale, int target,
    float* __restrict__ o_part, float* __restrict__ ml_part, int2* __restrict__ row_chunks,
    uint16_t* __restrict__ out) {
  constexpr int W = DC + DR;             // values of a position
  constexpr int RB = W * 2;              // bytes of its row in LDS
  constexpr int P = W / 8;               // 16-byte pieces of the row
  constexpr int DW = shares<HW>();       // waves that share 32 heads
  constexpr int NT = 64 * HW * DW;       // threads
  constexpr int KS = W / 16 / DW;        // a wave's steps of S^T
  constexpr int ND = DC / 32 / DW;       // 32-dim operands of a wave's outputs
  constexpr int RW = KT / (HW * DW);     // rows that a wave copies (4 or 8: within a page)
  constexpr int NC = (RW * P + 63) / 64; // their pieces, a lane
  constexpr int D = stages<F8>();
  constexpr int STAGE = KT * RB;
  constexpr int R = 3;  // operands read ahead of their products
  constexpr int E = F8 ? 1 : 2;
  static_assert(P % 8 == 0 && RB % 128 == 0 && ND % 2 == 0, "whole operands");
  static_assert(W / 16 % DW == 0, "equal parts of a row");
  // [D][KT] rows, then the waves' scores, then of e4m3 [D][KT] scales
  extern __shared__ __align__(128) char lds[];
  constexpr int PARTS = D * STAGE, SCALES = PARTS + HW * DW * kPartBytes;
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int col = lane & 31, h = lane >> 5;
  const int hw = wave % HW, dw = wave / HW;  // its heads, its part of the dims
  const KeyPlan plan = key_plan(seqs, lens, d, rows, KT, target);
  const Chunk ch = find_chunk(plan, seqs, lens, d, rows, KT, int(blockIdx.x));
  // uniform values, into scalar registers
  const int row = __builtin_amdgcn_readfirstlane(ch.row), chunk = __builtin_amdgcn_readfirstlane(ch.index);
  const int len = __builtin_amdgcn_readfirstlane(ch.len);
  const int chunks = __builtin_amdgcn_readfirstlane(ch.chunks);
  if (row < 0) return;  // past the last chunk
  if (chunk == 0 && t == 0) row_chunks[row] = make_int2(ch.before, chunks);
  const int seq = __builtin_amdgcn_readfirstlane(seqs ? seqs[row] : row);
  // units / chunks each, the first ones one more
  const int units = units_of(len, KT), few = units / chunks, more_units = units % chunks;
  const int tile0 = chunk * few + min(chunk, more_units), tile1 = tile0 + few + (chunk < more_units);
  const int k1 = min(len, tile1 * KT);
  const bool whole = chunks == 1;
  const int page = 1 << d.page_log2, last_page = (len - 1) >> d.page_log2;
  const float sl2 = scale * kLog2e;  // scores in log2 units

  // q of this lane's head (lanes past the last one have q = 0 and write nothing)
  uint4 qb[KS];
  {
    const int head = 32 * hw + col;
    const int64_t q_row = int64_t(row) * d.heads + (head < d.heads ? head : 0);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int at = 16 * (dw * KS + s);
      const uint16_t* src = at < DC ? q_latent + q_row * DC + at : q_rope + q_row * DR + at - DC;
      qb[s] = *reinterpret_cast<const uint4*>(src + 8 * h);
      if (head >= d.heads) qb[s] = make_uint4(0, 0, 0, 0);
    }
  }

  // Page ids of a tile's two 16-position parts, through scalar loads, read one tile ahead of the copy.
  struct Ids {
    int part[2];
  };
  auto ids_of = [&](int tile) MX_LAMBDA {
    Ids id;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      id.part[i] = page_at(table, d, seq, min((tile + 16 * i) >> d.page_log2, last_page));
    return id;
  };
  auto bits_of = [&](const Ids& id) MX_LAMBDA {  // bit i: part i lies in a page
    return uint32_t(id.part[0] >= 0) | uint32_t(id.part[1] >= 0) << 1;
  };

  // One tile's copies: a wave takes RW rows, which lie in a page one after the other.  Slot i of
  // them holds piece i ^ swizzle(its row).
  const uint32_t lds_at =
      uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
  uint32_t offs[(NC + 1) / 2];  // of this lane's pieces, from the first row's start: two in a register
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int slot = 64 * i + lane;
    const uint32_t off = (slot ^ swizzle(RW * wave + slot / P)) * (8 * E);
    offs[i / 2] = i & 1 ? offs[i / 2] | off << 16 : off;
  }
  auto off_of = [&](int i) MX_LAMBDA { return i & 1 ? offs[i / 2] >> 16 : offs[i / 2] & 0xffffu; };
  auto has = [&](int i) MX_LAMBDA { return 64 * (i + 1) <= RW * P || 64 * i + lane < RW * P; };
  uint2 kreg[F8 ? NC : 1];
  float sreg = 0.0f;
  auto copy = [&](int tile, const Ids& id, int stage) MX_LAMBDA {
    const int pid = max(RW * wave < 16 ? id.part[0] : id.part[1], 0);
    const char* from = static_cast<const char*>(cache) +
                       (pid * d.page_stride + int64_t((tile + RW * wave) & (page - 1)) * W) * E;
    if constexpr (F8) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (has(i)) kreg[i] = *reinterpret_cast<const uint2*>(from + off_of(i));
      if (t < KT)
        sreg = scales[(int64_t(max(t < 16 ? id.part[0] : id.part[1], 0)) << d.page_log2) +
                      ((tile + t) & (page - 1))];
    } else {
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (has(i)) copy_to_lds(from, off_of(i), lds_at + stage * STAGE + wave * RW * RB + 1024 * i);
    }
  };
  auto store = [&](int stage) MX_LAMBDA {
    if constexpr (F8) {
      char* to = lds + stage * STAGE + wave * RW * RB;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (has(i)) *reinterpret_cast<uint4*>(to + 16 * (64 * i + lane)) = widen8(kreg[i].x, kreg[i].y);
      if (t < KT) *reinterpret_cast<float*>(lds + SCALES + (stage * KT + t) * 4) = sreg;
    }
  };

  // operands of the scores' step s, and of output dims 32 n and 16 positions s
  const int krow = (col & 0x13) | ((col & 4) << 1) | ((col & 8) >> 1);  // bits 2 and 3 exchanged
  // Of step s, piece 2 s + h: within 128 bytes the steps differ by the exchanged bits alone.  Of dims
  // 32 n + 16 g + 4 x and positions 16 s + 8 h + 4 u + r, piece 4 n + 2 g + x / 2, likewise.  The present
  // stage's addresses are opaque: the compiler would add each operand's constant outside of the loop,
  // to a register of its own, instead of leaving it to the instruction.
  const uint32_t k_at = lds_at + krow * RB + 16 * (h ^ swizzle(krow));
  const int vrow = 8 * h + ((lane & 15) >> 2);
  const uint32_t v_at = lds_at + vrow * RB +
                        16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ swizzle(vrow)) + 8 * (lane & 1);
  uint32_t kb[4], vb[2][2];
  auto enter_k = [&](uint32_t stage_at) MX_LAMBDA {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s = dw * KS + j;
      kb[j] = (k_at ^ (32 * (s & 3))) + (stage_at + (s >> 2) * 128);
      asm volatile("" : "+v"(kb[j]));
    }
  };
  auto enter_v = [&](uint32_t stage_at) MX_LAMBDA {
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        vb[e][u] = (v_at ^ (64 * e | 16 * u)) + (stage_at + dw * (ND / 2) * 128 + u * 4 * RB);
        asm volatile("" : "+v"(vb[e][u]));
      }
  };
  auto k_operand = [&](int s) MX_LAMBDA { return lds_read16(kb[s & 3] + (s >> 2) * 128); };
  auto v_operand = [&](int n, int s) MX_LAMBDA {
    const uint32_t off = (n >> 1) * 128 + s * 16 * RB;
    const uint2 a = lds_read_tr(vb[n & 1][0] + off), b = lds_read_tr(vb[n & 1][1] + off);
    return make_uint4(a.x, a.y, b.x, b.y);
  };

  // (below every score, and finite, so that a masked one's -inf has the weight 0)
  float m_run = -__FLT_MAX__, l_run = 0.0f;
  floatx16_t o[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[n][r] = 0.0f;

  // Tiles past the last one are copied like it, into stages that nobody reads: every step has
  // the same copies, so waiting for all but the latest is waiting for their number.
  const int last = (tile1 - 1) * KT;
  uint32_t queue = 0;  // parts of the tiles from the present one on, two bits each
  Ids id = ids_of(tile0 * KT);
#pragma unroll
  for (int i = 0; i < D - 1; ++i) {
    queue |= bits_of(id) << (2 * i);
    copy(min((tile0 + i) * KT, last), id, i);
    store(i);
    id = ids_of(min((tile0 + i + 1) * KT, last));
  }
  int stage = 0;
  for (int ti = tile0; ti < tile1; ++ti) {
    const int tile = ti * KT;
    copies_done<F8 ? 0 : (D - 2) * NC>();  // this wave's part of the tile is in LDS ...
    __syncthreads();  // ... and everyone's; the stage of the tile before is free
    const uint32_t parts = queue & 3u;
    queue >>= 2;
    const bool ragged = tile + KT > k1 || parts != 3u;
    if (ragged) {  // uniform: rows that are no positions may be anything, and become 0
      int from = t;  // addresses formed here: kept over the tiles they would take registers
      asm volatile("" : "+v"(from));
#pragma unroll 1
      for (int i = from; i < KT * P; i += NT) {
        const int r = i / P;
        if (tile + r >= k1 || !(parts >> (r >> 4) & 1))
          *reinterpret_cast<uint4*>(lds + stage * STAGE + 16 * i) = make_uint4(0, 0, 0, 0);
      }
      if constexpr (F8)
        if (t < KT && (tile + t >= k1 || !(parts >> (t >> 4) & 1)))
          *reinterpret_cast<float*>(lds + SCALES + (stage * KT + t) * 4) = 0.0f;
      __syncthreads();
    }
    const int ahead = stage == 0 ? D - 1 : stage - 1;  // of tile ti + D - 1
    queue |= bits_of(id) << (2 * (D - 2));
    copy(min((ti + D - 1) * KT, last), id, ahead);
    enter_k(stage * STAGE);
    floatx16_t sc;
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[r] = 0.0f;
    {
      uint4 a[R];
      each<R>([&](auto s) MX_LAMBDA { a[s] = k_operand(s); });
      each<KS>([&](auto s) MX_LAMBDA {
        __builtin_amdgcn_sched_barrier(0);
        sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a[s % R]),
                                                     __builtin_bit_cast(bf16x8_t, qb[s]), sc, 0, 0, 0);
        if constexpr (s + R < KS) a[s % R] = k_operand(s + R);
      });
      __builtin_amdgcn_sched_barrier(0);
    }
    {  // the parts' sum, the same bits in each wave: (0 + 1) + (2 + 3)
      auto part = [&](int w) MX_LAMBDA {
        return reinterpret_cast<floatx4_t*>(lds + PARTS + (hw + HW * w) * kPartBytes) + lane;
      };
#pragma unroll
      for (int r = 0; r < 4; ++r)
        part(dw)[64 * r] = floatx4_t{sc[4 * r], sc[4 * r + 1], sc[4 * r + 2], sc[4 * r + 3]};
      __syncthreads();
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const floatx4_t v = part(dw ^ 1)[64 * r];
#pragma unroll
        for (int k = 0; k < 4; ++k) sc[4 * r + k] += v[k];
        if constexpr (DW == 4) {
          const floatx4_t x = part(dw ^ 2)[64 * r], y = part(dw ^ 3)[64 * r];
#pragma unroll
          for (int k = 0; k < 4; ++k) sc[4 * r + k] += x[k] + y[k];
        }
      }
    }
    // sc[r]: position 16 (r / 8) + 8 h + r % 8 of the tile
    const float* by = reinterpret_cast<const float*>(lds + SCALES) + stage * KT + 8 * h;
    if constexpr (F8) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] *= by[16 * (r >> 3) + (r & 7)];
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[r] *= sl2;
    if (ragged) {
      const int end = k1 - tile - 8 * h;
      const int ends[2] = {parts & 1 ? end : 0, parts & 2 ? end - 16 : 0};  // in each part
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = (r & 7) < ends[r >> 3] ? sc[r] : neg_inf();
    }
    float mt = sc[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mt = fmaxf(mt, sc[r]);
    mt = max_across_halves(mt);
    if constexpr (F8) asm volatile("" ::: "memory");
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
    enter_v(stage * STAGE);
    uint32_t pb[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float x = __builtin_amdgcn_exp2f(sc[2 * j] - m_run);
      float y = __builtin_amdgcn_exp2f(sc[2 * j + 1] - m_run);
      l_run += x + y;
      if constexpr (F8) {  // read again: held, they would be sixteen registers more
        x *= by[16 * (j >> 2) + 2 * (j & 3)];
        y *= by[16 * (j >> 2) + 2 * (j & 3) + 1];
      }
      pb[j] = pack2(x, y);
    }
    {
      uint4 a[R];
      each<R>([&](auto i) MX_LAMBDA { a[i] = v_operand(i % ND, i / ND); });
      each<2 * ND>([&](auto i) MX_LAMBDA {
        constexpr int s = i / ND, n = i % ND;
        __builtin_amdgcn_sched_barrier(0);
        o[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8_t, a[i % R]),
            __builtin_bit_cast(bf16x8_t,
                               make_uint4(pb[4 * s], pb[4 * s + 1], pb[4 * s + 2], pb[4 * s + 3])),
            o[n], 0, 0, 0);
        if constexpr (i + R < 2 * ND) a[i % R] = v_operand((i + R) % ND, (i + R) / ND);
      });
      __builtin_amdgcn_sched_barrier(0);
    }
    id = ids_of(min((ti + D) * KT, last));
    store(ahead);
    stage = stage == D - 1 ? 0 : stage + 1;
  }
  copies_done<0>();  // none lands in LDS that is no longer this workgroup's
  int last_t = t;  // what follows is formed here, not held over the tiles
  asm volatile("" : "+v"(last_t));
  const int head = 32 * hw + (last_t & 31), half = last_t >> 5 & 1;
  if (head >= d.heads) return;
  l_run += __shfl_xor(l_run, 32, 64);
  const int dim0 = dw * ND * 32 + 4 * half;
  if (whole) {
    const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
    uint16_t* dst = out + (int64_t(row) * d.heads + head) * DC + dim0;
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
  const int64_t part = int64_t(blockIdx.x) * d.heads + head;
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      *reinterpret_cast<float4*>(o_part + part * DC + dim0 + 32 * n + 8 * a) = make_float4(
          o[n][4 * a], o[n][4 * a + 1], o[n][4 * a + 2], o[n][4 * a + 3]);
  if (half == 0 && dw == 0) {
    ml_part[part * 2] = m_run;
    ml_part[part * 2 + 1] = l_run;
  }
}

// Waves side by side over the heads.
int head_waves(const LatentDims& d) { return d.heads <= 32 ? 1 : d.heads <= 64 ? 2 : 4; }
// Chunks wanted: as many as run at once, one a compute unit.
constexpr int kDecodeTarget = 256;

// The most chunks that any lengths give.
int64_t decode_items(int rows, const LatentDims& d) {
  const int64_t most = ((int64_t(d.table_width) << d.page_log2) + KT - 1) / KT;
  const int64_t target = 2 * kDecodeTarget;
  return rows * most < target + rows ? rows * most : target + rows;
}

}  // namespace

size_t latent_decode_workspace(int rows, const LatentDims& d) {
  return size_t(decode_items(rows, d)) * d.heads * (d.latent_dim + 2) * 4 + size_t(rows) * 8;
}

int latent_decode(const uint16_t* q_latent, const uint16_t* q_rope, int rows, const int32_t* seqs,
                  const int32_t* lens, const int32_t* table, const void* cache, const float* scales,
                  const LatentDims& d, float scale, void* workspace, uint16_t* out, hipStream_t s) {
  const int64_t items = decode_items(rows, d), joins = int64_t(rows) * d.heads;
  if (items > 0x7fffffff || joins * (d.latent_dim / 64) > 0x7fffffff) return MX_EUNSUPPORTED;
  float* o_part = static_cast<float*>(workspace);
  float* ml_part = o_part + items * d.heads * d.latent_dim;
  int2* row_chunks = reinterpret_cast<int2*>(ml_part + items * d.heads * 2);
  const int target = kDecodeTarget, hw = head_waves(d);
#define MX_JOIN(DC, DW, NJ)                                                                      \
  hipLaunchKernelGGL((decode_join_kernel<DC, DW, NJ, LatentDims>),                               \
                     dim3(unsigned(joins * (DC / DW))), dim3(64 * NJ), 0, s, nullptr, 0, rows,   \
                     seqs, lens, nullptr, d, row_chunks, o_part, ml_part, out)
#define MX_DECODE(DC, HW, FF)                                                                    \
  if (d.latent_dim == DC && hw == HW && d.f8 == FF) {                                            \
    const auto fn = decode_kernel<DC, HW, FF>;                                                   \
    constexpr int lb = lds_bytes<DC, HW, FF>();                                                  \
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(fn),                                   \
                            hipFuncAttributeMaxDynamicSharedMemorySize, lb) != hipSuccess)       \
      return MX_EHIP;                                                                            \
    hipLaunchKernelGGL(fn, dim3(unsigned(items)), dim3(64 * HW * shares<HW>()), lb, s, q_latent, q_rope, rows,  \
                       seqs, lens, table, cache, scales, d, scale, target, o_part, ml_part,      \
                       row_chunks, out);                                                         \
    if (hipGetLastError() != hipSuccess) return MX_EHIP;                                         \
    /* few rows have many chunks each */                                                         \
    if (joins <= 64)                                                                             \
      MX_JOIN(DC, 64, 16);                                                                       \
    else                                                                                         \
      MX_JOIN(DC, DC, 4);                                                                        \
    return hipGetLastError() == hipSuccess ? MX_OK : MX_EHIP;                                    \
  }
  MX_DECODE(256, 1, false) MX_DECODE(256, 2, false) MX_DECODE(256, 4, false)
  MX_DECODE(512, 1, false) MX_DECODE(512, 2, false) MX_DECODE(512, 4, false)
  MX_DECODE(256, 1, true) MX_DECODE(256, 2, true) MX_DECODE(256, 4, true)
  MX_DECODE(512, 1, true) MX_DECODE(512, 2, true) MX_DECODE(512, 4, true)
#undef MX_DECODE
#undef MX_JOIN
  return MX_EUNSUPPORTED;
}

}  // namespace mx
