// Attention of one new token a row over the latent cache: absorbed, so that a position's row of
// latent and rotary key is the key of every head, and its latent their value:
//
//   s[h, p] = scale (q_latent[h] . c[p] + q_rope[h] . k[p]),  out[h] = sum_p softmax(s[h])[p] c[p]
//
// The tiles of 32 positions of all rows in order are shared out evenly, and a workgroup walks its share, all
// heads of it, with the tiles copied to LDS ahead.  Heads are matrix-core columns, 32 a wave:
//   S^T = K Q^T       A: positions from LDS, B: q in registers
//   O^T = C^T P^T     A: the same positions, read transposed from LDS, B: P as it stands
// Lane (head c = l % 32, half h = l / 32) receives the scores of rows 8 a + 4 h + b of the tile and
// supplies the k-slots 8 h + i of each 16 positions for the second product; rows enter with bits 2 and
// 3 exchanged, so the two are the same positions and P never leaves its lane.
//
// Two or four waves share 32 heads: each forms their scores over its part of a position's row, the parts meet
// in LDS, and each has its part of the output's dims.  (A wave alone would hold 400 registers of q and sums.
// Four that form all scores each need no exchange, but their q takes four times as long to load, and a 40-row
// batch of 20 heads as long in all.)
//
// The sum that divides takes P in fp32.  For the product P is split in two bf16 parts, which keep 16 bits, of
// up to 64 heads; of more, where that would double the work of what bounds it, it is rounded to bf16, each p by
// at most 2^-8 of itself, as the output is.
//
// e4m3 lies in LDS as it is, half the bytes, and is widened where an operand is read; a position's scale goes
// to its scores and to its p.
//
// A row whose tiles meet several workgroups' shares leaves partials in fp32, which a second launch joins in
// order.
//
// 64 rows of 128 heads on up to 8192 positions: 118 to 123 us, of which the tiles (298 MB, memory's bound) take
// about 63, the rows' beginnings and ends in each workgroup 37, and the join 20.  A piece's beginning and end
// move 147 KB of q and 256 KB of sums, but they are a chain too: with a latent of 512 and more than 64 heads a
// wave's q and sums leave too few registers, so 16 are kept in scratch memory (of e4m3 11), whose reloads between
// the first tiles' copies wait for these, and the last six of q's 18 loads follow one after another.  Forms with
// fewer heads or a latent of 256 keep everything in registers.  40 rows of 20 heads on up to 12001 of e4m3: 58 us
// (145 MB; without either product three quarters of that).  One row of 16 heads on 60001: 26 us, 6 of them the
// join.
//
// Heads are taken in whole 32s, and past 64 in whole 128s: 65 heads compute as 128 do.
#include <type_traits>

#include "prompt_plan.hpp"

namespace mx {

namespace {

using namespace pg;

constexpr int KT = 32;   // positions of a tile
constexpr int DR = 64;   // rope_dim

// By the number of head waves (of 32 heads each): waves that share their heads; workgroups that share a
// compute unit; stages of a tile in LDS.
template <int HW>
constexpr int shares() {
  return HW == 4 ? 2 : 4;
}
template <int HW, bool F8>
constexpr int groups_a_unit() {
  return HW == 1 && F8 ? 2 : 1;
}
template <int HW, bool F8>
constexpr int stages() {
  return F8 && HW > 1 ? 4 : 3;
}
constexpr int kPartBytes = KT * 32 * 4;  // of a wave's scores
template <int DC, int HW, bool F8>
constexpr int lds_bytes() {
  return stages<HW, F8>() * KT * (F8 ? DC + DR + 4 : 2 * (DC + DR)) + HW * shares<HW>() * kPartBytes;
}

// A tile lies in LDS as blocks of 64 values of its 32 rows, so that a copy of 1 KB is some rows of a block.
// 16-byte pieces are exchanged by the row's number within a block's row, so that neither sixteen rows' operands
// nor the transposed reads, of four rows of bf16 or eight of e4m3 at once, meet one of the 64 banks twice
// (e4m3 rows' operands of 8 bytes do, which costs them what 16 bytes cost).
template <bool F8>
__device__ __forceinline__ int swizzle(int row) {
  return F8 ? ((row >> 1) & 2) ^ ((row >> 3) & 2) ^ ((row >> 1 ^ row >> 3) & 1)
            : (row & 2) << 1 | (row >> 1 & 2) | (row >> 3 & 1);
}
// Four bytes a lane from memory to LDS, lane l's to lds + 4 l (as copy_to_lds).
__device__ __forceinline__ void copy4_to_lds(const void* src, uint32_t lds) {
  uint32_t m0;
  asm volatile("s_mov_b32 %0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               : "=&{m0}"(m0)
               : "v"(src), "s"(lds)
               : "memory");
}

// How the tiles of all rows are shared out: as many to each workgroup, at least `least`, so that all run
// at once.  To begin a row within a share costs as long as kRowTiles tiles, which its length has in front.
template <int HW, bool F8>
constexpr int groups() {
  return 256 * groups_a_unit<HW, F8>();
}
template <int HW>
constexpr int kRowTiles = HW == 4 ? 8 : 4;
template <int HW>
__device__ __forceinline__ int row_tiles(int len) {
  return len > 0 ? units_of(len, KT) + kRowTiles<HW> : 0;
}
struct Share {
  int all, each, len0;  // len0: the lengths of the first 64 rows, a lane each
};
template <int HW, bool F8>
__device__ __forceinline__ Share share_of(const int32_t* seqs, const int32_t* lens,
                                          const LatentDims& d, int rows, int least) {
  Share s;
  s.len0 = row_len(seqs, lens, d, threadIdx.x & 63, rows);
  s.all = __builtin_amdgcn_readlane(wave_scan(row_tiles<HW>(s.len0)), 63);
  for (int r = 64; r < rows; r += 64)
    s.all += __builtin_amdgcn_readlane(
        wave_scan(row_tiles<HW>(row_len(seqs, lens, d, r + (threadIdx.x & 63), rows))), 63);
  s.each = max((s.all + groups<HW, F8>() - 1) / groups<HW, F8>(), least);
  return s;
}
// The row that `unit` of all falls to (there is one), its length, and its first unit.
struct Piece {
  int row, len, first;
};
template <int HW>
__device__ __forceinline__ Piece piece_at(const Share& s, const int32_t* seqs, const int32_t* lens,
                                          const LatentDims& d, int rows, int unit) {
  int before = 0;
  for (int r = 0;; r += 64) {
    const int l = r == 0 ? s.len0 : row_len(seqs, lens, d, r + (threadIdx.x & 63), rows);
    const int n = row_tiles<HW>(l), sum = wave_scan(n);
    const uint64_t past = __ballot(before + sum > unit);
    if (past || r + 64 >= rows) {
      const int f = past ? __builtin_ctzll(past) : 63;
      // uniform values, into scalar registers
      return Piece{__builtin_amdgcn_readfirstlane(r + f), __builtin_amdgcn_readlane(l, f),
                   __builtin_amdgcn_readfirstlane(before + __builtin_amdgcn_readlane(sum, f) -
                                                  __builtin_amdgcn_readlane(n, f))};
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
}

template <int DC, int HW, bool F8>
__global__ __launch_bounds__(64 * HW * shares<HW>(), HW == 1 && !F8 ? 1 : 2) void decode_kernel(
    const uint16_t* __restrict__ q_latent, const uint16_t* __restrict__ q_rope, int rows,
    const int32_t* __restrict__ seqs, const int32_t* __restrict__ lens,
    const int32_t* __restrict__ table, const void* __restrict__ cache,
    const float* __restrict__ scales, LatentDims d, float scale, int least,
    float* __restrict__ o_part, float* __restrict__ ml_part, int2* __restrict__ row_pieces,
    uint16_t* __restrict__ out) {
  constexpr int W = DC + DR;             // values of a position
  constexpr int CB = W / 64;             // blocks of its row in LDS
  constexpr int DW = shares<HW>();       // waves that share 32 heads
  constexpr bool TWO = HW < 4;           // P in two parts
  constexpr int NW = HW * DW, NT = 64 * NW;
  constexpr int KS = W / 16 / DW;        // a wave's steps of S^T
  constexpr int ND = DC / 32 / DW;       // 32-dim operands of a wave's outputs
  constexpr int E = F8 ? 1 : 2;          // bytes of a value
  constexpr int RB = 64 * E, BLOCK = KT * RB;  // a block's row, a block
  constexpr int RC = 1024 / RB, RG = KT / RC;  // rows of a copy, copies of a block
  constexpr int CW = NW / RG;            // waves that copy the same rows, in turn over their blocks
  constexpr int NC = (CB + CW - 1) / CW; // copies of a wave, at most (one less where they do not go round)
  constexpr int D = stages<HW, F8>();
  constexpr int STAGE = CB * BLOCK;
  constexpr int R = 3;                   // operands read ahead of their products
  static_assert(NW % RG == 0 && ND % 2 == 0 && W / 16 % DW == 0, "whole operands, equal parts");
  // [D] tiles, then of e4m3 [D][KT] scales, then the waves' parts of the scores
  extern __shared__ __align__(128) char lds[];
  constexpr int SCALES = D * STAGE, PARTS = SCALES + (F8 ? D * KT * 4 : 0);
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int col = lane & 31, h = lane >> 5;
  const int hw = wave % HW, dw = wave / HW;  // its heads, its part of the dims
  const Share share = share_of<HW, F8>(seqs, lens, d, rows, least);
  int unit = int(blockIdx.x) * share.each;
  const int unit1 = min(unit + share.each, share.all);
  if (unit >= unit1) return;
  Piece pc = piece_at<HW>(share, seqs, lens, d, rows, unit);
  const float sl2 = scale * kLog2e;  // scores in log2 units
  const int page = 1 << d.page_log2;
  int seq = 0, last_page = 0;  // of the present row

  // Page ids of a tile's two 16-position parts, from a register that has them for 32 tiles, a part a lane: a
  // load a tile, through scalar loads, is waited for with the LDS reads that it counts with (64 rows of
  // 128 heads: 23 us of 136).
  int ids = 0, ids0 = 0;  // from tile ids0 on
  struct Ids {
    int part[2];
  };
  auto load_ids = [&](int ti) MX_LAMBDA {
    ids0 = ti;
    ids = page_at(table, d, seq, min((ti * KT + 16 * lane) >> d.page_log2, last_page));
    asm volatile("" : "+v"(ids));  // waited for here, not at every use
  };
  auto ids_of = [&](int ti) MX_LAMBDA {
    if (ti - ids0 >= 32) load_ids(ti);  // uniform
    Ids id;
#pragma unroll
    for (int i = 0; i < 2; ++i) id.part[i] = __builtin_amdgcn_readlane(ids, 2 * (ti - ids0) + i);
    return id;
  };
  auto bits_of = [&](const Ids& id) MX_LAMBDA {  // bit i: part i lies in a page
    return uint32_t(id.part[0] >= 0) | uint32_t(id.part[1] >= 0) << 1;
  };

  // One tile's copies: a wave takes RC rows, which lie in a page one after the other, and every CW-th
  // block.  A lane copies the piece of its row that its place is for.
  const uint32_t lds_at =
      uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
  const int rows_at = wave % RG * RC, block0 = wave / RG;
  constexpr int LR = 64 / RC;  // lanes of a row
  const uint32_t off = lane / LR * (W * E) + 16 * ((lane % LR) ^ swizzle<F8>(rows_at + lane / LR));
  auto has = [&](int i) MX_LAMBDA { return CW * (i + 1) <= CB || block0 + CW * i < CB; };  // uniform
  auto copy = [&](int tile, const Ids& id, int stage) MX_LAMBDA {
    const int pid = max(rows_at < 16 ? id.part[0] : id.part[1], 0);
    const char* from = static_cast<const char*>(cache) +
                       (pid * d.page_stride + int64_t((tile + rows_at) & (page - 1)) * W) * E + block0 * RB;
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (has(i))
        copy_to_lds(from + CW * i * RB, off,
                    lds_at + stage * STAGE + (block0 + CW * i) * BLOCK + wave % RG * 1024);
    if constexpr (F8)  // every wave the same, so that their copies count alike
      if (lane < KT)
        copy4_to_lds(scales + (int64_t(max(lane < 16 ? id.part[0] : id.part[1], 0)) << d.page_log2) +
                         ((tile + lane) & (page - 1)),
                     lds_at + SCALES + stage * KT * 4);
  };
  auto copied = [&]() MX_LAMBDA {  // this wave's copies of all but the latest tiles are done
    if (has(NC - 1))
      copies_done<(D - 2) * (NC + F8)>();
    else
      copies_done<(D - 2) * (NC - 1 + F8)>();
  };

  // Operands of the scores' step s, and of output dims 32 n and 16 positions s.  Steps differ by the
  // exchanged bits within a block's row.  The present stage's addresses are opaque: the compiler would add
  // each operand's constant outside of the loop, to a register of its own, instead of leaving it to the
  // instruction.
  const int krow = (col & 0x13) | ((col & 4) << 1) | ((col & 8) >> 1);  // bits 2 and 3 exchanged
  const uint32_t k_at = lds_at + krow * RB + (F8 ? 16 * swizzle<F8>(krow) + 8 * h : 16 * (h ^ swizzle<F8>(krow)));
  // bf16: row 8 h + j / 4 (and four on), dims 16 g + 4 (j % 4); e4m3: row 8 h + j / 2, dims 16 g + 8 (j % 2)
  const int vj = lane & 15, vg = (lane >> 4) & 1, vrow = 8 * h + (F8 ? vj >> 1 : vj >> 2);
  const uint32_t v_at =
      lds_at + vrow * RB + 8 * (vj & 1) +
      16 * ((F8 ? vg : 2 * vg + ((vj & 3) >> 1)) ^ swizzle<F8>(vrow));
  uint32_t kb[4], vb[2][2];
  auto enter_k = [&](uint32_t stage_at) MX_LAMBDA {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s = dw * KS + j;
      kb[j] = (k_at ^ ((F8 ? 16 : 32) * (s & 3))) + (stage_at + (s >> 2) * BLOCK);
      asm volatile("" : "+v"(kb[j]));
    }
  };
  auto enter_v = [&](uint32_t stage_at) MX_LAMBDA {
    const uint32_t at = stage_at + dw * (ND / 2) * BLOCK;
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int u = 0; u < (F8 ? 1 : 2); ++u) {
        vb[e][u] = (v_at ^ (F8 ? 32 * e : 64 * e | 32 * u)) + (at + u * 4 * RB);
        asm volatile("" : "+v"(vb[e][u]));
      }
  };
  typedef std::conditional_t<F8, uint2, uint4> Raw;
  auto k_operand = [&](int s) MX_LAMBDA {
    typedef uint32_t vec __attribute__((ext_vector_type(sizeof(Raw) / 4)));
    return __builtin_bit_cast(Raw, lds_read<vec>(kb[s & 3] + (s >> 2) * BLOCK));
  };
  auto v_operand = [&](int n, int s) MX_LAMBDA {
    const uint32_t o = (n >> 1) * BLOCK + s * 16 * RB;
    if constexpr (F8) {
      return lds_read_tr8(vb[(n ^ s) & 1][0] + o);  // sixteen rows on, the second bit is exchanged
    } else {
      const uint2 a = lds_read_tr16(vb[n & 1][0] + o), b = lds_read_tr16(vb[n & 1][1] + o);
      return make_uint4(a.x, a.y, b.x, b.y);
    }
  };
  auto wide = [&](const Raw& v) MX_LAMBDA {
    if constexpr (F8)
      return __builtin_bit_cast(bf16x8_t, widen8(v.x, v.y));
    else
      return __builtin_bit_cast(bf16x8_t, v);
  };

  for (;;) {
    // the present row, and its tiles in this workgroup's share
    const int row = pc.row, len = pc.len, tiles = units_of(len, KT), begin = pc.first + kRowTiles<HW>;
    const int tile0 = max(unit - begin, 0), tile1 = min(unit1 - begin, tiles);
    if (tile0 < tile1) {
      const int k1 = min(len, tile1 * KT);
      const int piece0 = begin / share.each;  // the first workgroup that has any of the row's
      const int pieces = (begin + tiles - 1) / share.each - piece0 + 1;
      if (tile0 == 0 && t == 0) row_pieces[row] = make_int2(piece0 + row, pieces);
      seq = __builtin_amdgcn_readfirstlane(seqs ? seqs[row] : row);
      last_page = (len - 1) >> d.page_log2;

      // Tiles past the last one are copied like it, into stages that nobody reads: every step has
      // the same copies, so waiting for all but the latest is waiting for their number.
      uint32_t queue = 0;  // parts of the tiles from the present one on, two bits each
      load_ids(tile0);
#pragma unroll
      for (int i = 0; i < D - 1; ++i) {
        const int next = min(tile0 + i, tile1 - 1);
        const Ids id = ids_of(next);
        queue |= bits_of(id) << (2 * i);
        copy(next * KT, id, i);
      }
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
      // (below every score, and finite, so that a masked one's -inf has the weight 0)
      float m_run = -__FLT_MAX__, l_run = 0.0f;
      floatx16_t o[ND];
#pragma unroll
      for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[n][r] = 0.0f;

      int stage = 0;
      for (int ti = tile0; ti < tile1; ++ti) {
        const int tile = ti * KT;
        copied();        // this wave's part of the tile is in LDS ...
        __syncthreads();  // ... and everyone's; the stage of the tile before is free
        const uint32_t in = queue & 3u;
        queue >>= 2;
        const bool ragged = tile + KT > k1 || in != 3u;
        if (ragged) {  // uniform: rows that are no positions may be anything, and become 0
#pragma unroll 1
          for (int i = t; i < KT * STAGE / KT / 16; i += NT) {  // piece by piece of 32 rows
            const int r = i & (KT - 1), piece = i / KT;
            if (tile + r >= k1 || !(in >> (r >> 4) & 1))
              *reinterpret_cast<uint4*>(lds + stage * STAGE + piece / LR * BLOCK + r * RB +
                                        16 * (piece % LR)) = make_uint4(0, 0, 0, 0);
          }
          if constexpr (F8)
            if (t < KT && (tile + t >= k1 || !(in >> (t >> 4) & 1)))
              *reinterpret_cast<float*>(lds + SCALES + (stage * KT + t) * 4) = 0.0f;
          __syncthreads();
        }
        const int ahead = stage == 0 ? D - 1 : stage - 1;  // of tile ti + D - 1
        const int next = min(ti + D - 1, tile1 - 1);
        const Ids id = ids_of(next);
        queue |= bits_of(id) << (2 * (D - 2));
        copy(next * KT, id, ahead);
        enter_k(stage * STAGE);
        floatx16_t sc;
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[r] = 0.0f;
        {
          Raw a[R];
          each<R>([&](auto s) MX_LAMBDA { a[s] = k_operand(s); });
          each<KS>([&](auto s) MX_LAMBDA {
            __builtin_amdgcn_sched_barrier(0);
            sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wide(a[s % R]), __builtin_bit_cast(bf16x8_t, qb[s]),
                                                         sc, 0, 0, 0);
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
        if (ragged) {
          const int end = k1 - tile - 8 * h;
          const int ends[2] = {in & 1 ? end : 0, in & 2 ? end - 16 : 0};  // in each part
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[r] = (r & 7) < ends[r >> 3] ? sc[r] : neg_inf();
        }
        float mt = sc[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mt = fmaxf(mt, sc[r]);
        mt = max_across_halves(mt) * sl2;
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
        uint32_t ph[8], pl[TWO ? 8 : 1];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float x = __builtin_amdgcn_exp2f(fmaf_(sc[2 * j], sl2, -m_run));
          float y = __builtin_amdgcn_exp2f(fmaf_(sc[2 * j + 1], sl2, -m_run));
          l_run += x + y;
          if constexpr (F8) {  // read again: held, they would be sixteen registers more
            x *= by[16 * (j >> 2) + 2 * (j & 3)];
            y *= by[16 * (j >> 2) + 2 * (j & 3) + 1];
          }
          ph[j] = pack2(x, y);
          if constexpr (TWO) pl[j] = pack2(x - u2f(ph[j] << 16), y - u2f(ph[j] & 0xffff0000u));
        }
        auto p_operand = [&](const uint32_t* p, int s) MX_LAMBDA {
          return __builtin_bit_cast(bf16x8_t, make_uint4(p[4 * s], p[4 * s + 1], p[4 * s + 2], p[4 * s + 3]));
        };
        {
          Raw a[R];
          each<R>([&](auto i) MX_LAMBDA { a[i] = v_operand(i % ND, i / ND); });
          each<2 * ND>([&](auto i) MX_LAMBDA {
            constexpr int s = i / ND, n = i % ND;
            __builtin_amdgcn_sched_barrier(0);
            const bf16x8_t v = wide(a[i % R]);
            if constexpr (i + R < 2 * ND) a[i % R] = v_operand((i + R) % ND, (i + R) / ND);
            o[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, p_operand(ph, s), o[n], 0, 0, 0);
            if constexpr (TWO)
              o[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, p_operand(pl, s), o[n], 0, 0, 0);
          });
          __builtin_amdgcn_sched_barrier(0);
        }
        stage = stage == D - 1 ? 0 : stage + 1;
      }
      copies_done<0>();  // none lands in LDS that is no longer this workgroup's
      int last_t = t;  // what follows is formed here, not held over the tiles
      asm volatile("" : "+v"(last_t));
      const int head = 32 * hw + (last_t & 31), half = last_t >> 5 & 1;
      l_run += __shfl_xor(l_run, 32, 64);
      if (head >= d.heads) {
        // nothing to write
      } else if (pieces == 1) {
        const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
        uint16_t* dst = out + (int64_t(row) * d.heads + head) * DC + dw * ND * 32 + 4 * half;
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
          for (int a = 0; a < 4; ++a) {
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = l_run == 0.0f ? 0.0f : o[n][4 * a + r] * inv;
            *reinterpret_cast<uint2*>(dst + 32 * n + 8 * a) =
                make_uint2(pack2(y[0], y[1]), pack2(y[2], y[3]));
          }
      } else {
        // [dims / 4][heads][4]: neighbouring lanes write neighbouring heads
        const int64_t slot = int64_t(blockIdx.x) + row;
        float4* dst = reinterpret_cast<float4*>(o_part) +
                      (slot * (DC / 4) + dw * ND * 8 + half) * d.heads + head;
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
          for (int a = 0; a < 4; ++a)
            dst[int64_t(8 * n + 2 * a) * d.heads] =
                make_float4(o[n][4 * a], o[n][4 * a + 1], o[n][4 * a + 2], o[n][4 * a + 3]);
        if (half == 0 && dw == 0)
          *reinterpret_cast<float2*>(ml_part + (slot * d.heads + head) * 2) = make_float2(m_run, l_run);
      }
      __syncthreads();  // every wave is done with LDS
    }
    unit = begin + tiles;
    if (unit >= unit1) return;
    pc = piece_at<HW>(share, seqs, lens, d, rows, unit);
  }
}

// Joins the pieces of a row in order, four dims of a head a thread, EL threads beside each other and G sets of
// them, each of which takes every G-th piece; rows without positions become 0, rows of one piece are done.
template <int DC, int EL, int G>
__global__ __launch_bounds__(EL * G) void join_kernel(const int32_t* __restrict__ seqs,
                                                      const int32_t* __restrict__ lens, int rows,
                                                      LatentDims d, const int2* __restrict__ row_pieces,
                                                      const float* __restrict__ o_part,
                                                      const float* __restrict__ ml_part,
                                                      uint16_t* __restrict__ out, int blocks) {
  __shared__ float red[G > 1 ? G : 1][EL], mx[G > 1 ? G : 1][EL];
  __shared__ floatx4_t os[G > 1 ? G : 1][EL];
  const int row = blockIdx.x / blocks, e = threadIdx.x % EL, g = threadIdx.x / EL;
  const int all = d.heads * (DC / 4);
  const int at = blockIdx.x % blocks * EL + e, i = min(at, all - 1);  // element [dims / 4][heads]
  const int len = row_len(seqs, lens, d, row, rows);
  const int2 rp = row_pieces[row];  // meaningful where there are positions
  if (len < 0) return;  // uniform, as what follows
  const int head = i % d.heads, dim = 4 * (i / d.heads);
  uint16_t* dst = out + (int64_t(row) * d.heads + head) * DC + dim;
  if (len == 0) {
    if (g == 0 && at < all) *reinterpret_cast<uint2*>(dst) = make_uint2(0, 0);
    return;
  }
  const int n = rp.y;
  if (n <= 1) return;
  const floatx4_t* po = reinterpret_cast<const floatx4_t*>(o_part) + int64_t(rp.x) * all + i;
  const float2* pm = reinterpret_cast<const float2*>(ml_part) + int64_t(rp.x) * d.heads + head;
  constexpr int A = G > 4 ? 4 : 8;  // pieces on their way
  // each set by its own running maximum; the sets' sums are brought together below
  float M = -__FLT_MAX__, L = 0.0f;
  floatx4_t O = 0.0f;
  for (int c = g; c < n; c += G * A) {
    floatx4_t v[A];
    float2 ml[A];
#pragma unroll
    for (int k = 0; k < A; ++k) {
      const int64_t p = c + G * k;
      ml[k] = make_float2(-__FLT_MAX__, 0.0f);
      v[k] = 0.0f;
      if (p < n) {
        v[k] = po[p * all];
        ml[k] = pm[p * d.heads];
      }
    }
    float m = M;
#pragma unroll
    for (int k = 0; k < A; ++k) m = fmaxf(m, ml[k].x);
    const float w0 = __builtin_amdgcn_exp2f(M - m);
    L *= w0;
    for (int j = 0; j < 4; ++j) O[j] *= w0;
    M = m;
#pragma unroll
    for (int k = 0; k < A; ++k) {
      const float w = __builtin_amdgcn_exp2f(ml[k].x - M);
      L = fmaf_(ml[k].y, w, L);
      for (int j = 0; j < 4; ++j) O[j] = fmaf_(v[k][j], w, O[j]);
    }
  }
  if constexpr (G > 1) {
    mx[g][e] = M;
    __syncthreads();
    float m = M;
#pragma unroll
    for (int k = 0; k < G; ++k) m = fmaxf(m, mx[k][e]);
    const float w = __builtin_amdgcn_exp2f(M - m);
    L *= w;
    for (int j = 0; j < 4; ++j) O[j] *= w;
  }
  if constexpr (G > 1) {
    red[g][e] = L;
    os[g][e] = O;
    __syncthreads();
    if (g > 0) return;
#pragma unroll
    for (int k = 1; k < G; ++k) {
      L += red[k][e];
      O += os[k][e];
    }
  }
  if (at >= all) return;
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  float y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = L == 0.0f ? 0.0f : O[j] * inv;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(y[0], y[1]), pack2(y[2], y[3]));
}

int head_waves(const LatentDims& d) { return d.heads <= 32 ? 1 : d.heads <= 64 ? 2 : 4; }
// The fewest tiles of a share: below, joining partials (heads times latent_dim of fp32) costs more.  Set where all
// compute units have work; one row of 128 heads on 1000 positions takes 4 of them, on 8192 32.
int least_tiles(const LatentDims& d) { return d.heads > 64 ? 8 : 4; }
// The most pieces of rows: a workgroup's and a row's end each begin one.
int64_t decode_pieces(int rows, const LatentDims& d) {
  return int64_t(head_waves(d) == 1 && d.f8 ? groups<1, true>() : groups<1, false>()) + rows;
}

}  // namespace

size_t latent_decode_workspace(int rows, const LatentDims& d) {
  return size_t(decode_pieces(rows, d)) * d.heads * (d.latent_dim + 2) * 4 + size_t(rows) * 8;
}

int latent_decode(const uint16_t* q_latent, const uint16_t* q_rope, int rows, const int32_t* seqs,
                  const int32_t* lens, const int32_t* table, const void* cache, const float* scales,
                  const LatentDims& d, float scale, void* workspace, uint16_t* out, hipStream_t s) {
  const int64_t pieces = decode_pieces(rows, d);
  // the tiles of all rows are counted in 32 bits
  const int64_t most = ((int64_t(d.table_width) << d.page_log2) + KT - 1) / KT + kRowTiles<4>;
  if (rows * most > (1 << 30)) return MX_EUNSUPPORTED;
  float* o_part = static_cast<float*>(workspace);
  float* ml_part = o_part + pieces * d.heads * d.latent_dim;
  int2* row_pieces = reinterpret_cast<int2*>(ml_part + pieces * d.heads * 2);
  const int least = least_tiles(d), hw = head_waves(d);
#define MX_JOIN(DC, EL, G)                                                                       \
  {                                                                                              \
    const int64_t blocks = (int64_t(d.heads) * (DC / 4) + EL - 1) / EL;                          \
    if (rows * blocks > 0x7fffffff) return MX_EUNSUPPORTED;                                      \
    hipLaunchKernelGGL((join_kernel<DC, EL, G>), dim3(unsigned(rows * blocks)), dim3(EL * G), 0, \
                       s, seqs, lens, rows, d, row_pieces, o_part, ml_part, out, int(blocks));   \
  }
#define MX_DECODE(DC, HW, FF)                                                                    \
  if (d.latent_dim == DC && hw == HW && d.f8 == FF) {                                            \
    const auto fn = decode_kernel<DC, HW, FF>;                                                   \
    constexpr int lb = lds_bytes<DC, HW, FF>();                                                  \
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(fn),                                   \
                            hipFuncAttributeMaxDynamicSharedMemorySize, lb) != hipSuccess)       \
      return MX_EHIP;                                                                            \
    hipLaunchKernelGGL(fn, dim3(groups<HW, FF>()), dim3(64 * HW * shares<HW>()), lb, s, q_latent,    \
                       q_rope, rows, seqs, lens, table, cache, scales, d, scale, least, o_part,  \
                       ml_part, row_pieces, out);                                                \
    if (hipGetLastError() != hipSuccess) return MX_EHIP;                                         \
    /* few rows have many pieces each */                                                         \
    if (rows <= 4)                                                                               \
      MX_JOIN(DC, 16, 64)                                                                        \
    else if (rows <= 16)                                                                         \
      MX_JOIN(DC, 64, 4)                                                                         \
    else                                                                                         \
      MX_JOIN(DC, 256, 1)                                                                        \
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
