// The paged cache: rows appended to it, and attention of one new token a row over it.
#include <type_traits>

#include "paged_core.hpp"

namespace mx {

namespace {

using namespace pg;

// ---------------------------------------------------------------------------
// Append: RMS norm, rotary positions and the cache's writes, in one launch.
//
//   y = x rsqrt(mean x^2 + eps) (w + 1)       (q and k heads; w absent: y = x)
//   pair (i, i + rot/2), a = position[axis(i)] inv_freq[i]:
//     (y1 cos a - y2 sin a, y2 cos a + y1 sin a)
//
// all in fp32 with one rounding, to bf16 or, divided by the kv head's scale, to
// e4m3.  The angle is formed in 64 bits as a fraction of a turn, so positions
// of millions keep their low bits; its sine and cosine are then fp32 series
// around the nearest quarter turn, once per row and wave.
//
// Bytes bound it (4093 rows of 32 q / 8 kv heads of 128, e4m3: 25 us, 3.8 TB/s; 8 rows of 16 / 2
// heads of 256 5 us, the chain of loads).  The first workgroups of the grid take one kv head's V of 32
// rows each: they pass through LDS so that neighbouring lanes store neighbouring
// positions of a page, where V lies transposed.  The waves of the others take q
// and k heads of a row, eight values a lane, several at a time, without meeting.
constexpr int kQkThreads = 256;
constexpr int kVRows = 32;

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

template <int HD, bool F8>
__global__ __launch_bounds__(kQkThreads) void append_kernel(
    const uint16_t* __restrict__ qkv, int64_t qkv_stride, int rows,
    const int32_t* __restrict__ seqs, const int32_t* __restrict__ pos,
    const int32_t* __restrict__ rope_pos, RopeAxes rope, const uint16_t* __restrict__ q_norm,
    const uint16_t* __restrict__ k_norm, float eps, const int32_t* __restrict__ table, PageDims d,
    const float* __restrict__ k_scale, const float* __restrict__ v_scale,
    uint16_t* __restrict__ q_out, void* __restrict__ k_cache, void* __restrict__ v_cache,
    int groups, int each, int v_blocks) {
  constexpr int LPH = HD / 8;           // lanes per head
  constexpr int HPW = 64 / LPH;         // heads of a group, which a wave takes at once
  constexpr int PLD = 12;               // a lane's eight values in LDS, padded
  constexpr int AHEAD = 4;              // groups on their way
  __shared__ float trigs[kQkThreads / 64][2][128];
  constexpr int VLD = HD + 2;
  __shared__ __align__(16) union {
    float pairs[kQkThreads * PLD];
    uint16_t v[kVRows * VLD];
  } buf;
  float* pairs = buf.pairs;
  const int t = threadIdx.x;
  const int page = 1 << d.page_log2;
  const int q_width = d.gated ? 2 * HD : HD;
  if (int(blockIdx.x) >= v_blocks) {
    // a wave takes `each` groups of heads of one row
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
    const int per_row = (groups + each - 1) / each;
    const int64_t b = int64_t(int(blockIdx.x) - v_blocks) * (kQkThreads / 64) + wave;
    if (b >= int64_t(rows) * per_row) return;
    const int row = int(b / per_row), g0 = int(b % per_row) * each, g1 = min(groups, g0 + each);
    float(&trig)[2][128] = trigs[wave];
    const int seq = seqs ? seqs[row] : row;
    const int p = pos[row];
    const int piece = t % LPH, heads = d.heads + d.kv_heads;
    const uint16_t* src = qkv + int64_t(row) * qkv_stride + 8 * piece;
    auto load = [&](int group) {
      const int head = group * HPW + lane / LPH;
      if (group >= g1 || head >= heads) return make_uint4(0, 0, 0, 0);
      const int64_t at = head < d.heads ? int64_t(head) * q_width
                                        : int64_t(d.heads) * q_width + int64_t(head - d.heads) * HD;
      return *reinterpret_cast<const uint4*>(src + at);
    };
    uint4 raws[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) raws[i] = load(g0 + i);
    const int half = rope.rotary_dim / 2;
    uint4 qn = make_uint4(0, 0, 0, 0), kn = qn;  // norm weights: the same piece of every head
    if (q_norm) qn = *reinterpret_cast<const uint4*>(q_norm + 8 * piece);
    if (k_norm) kn = *reinterpret_cast<const uint4*>(k_norm + 8 * piece);
    if (unsigned(seq) >= unsigned(d.sequences)) return;  // a padding row (uniform)
    const int pid = p >= 0 && (p >> d.page_log2) < d.table_width
                        ? page_at(table, d, seq, p >> d.page_log2)
                        : -1;
    for (int i = lane; i < half; i += 64)
      sincos_turn(double(rope_pos[int64_t(rope.pair_axis[i]) * rows + row]) * rope.inv_freq[i] *
                      0.15915494309189533577,
                  &trig[1][i], &trig[0][i]);
    wave_sync();
    // The lane's eight places are the same in every head, and so are their sines (signed for
    // the sum) and their partners' place, half a rotary width away in a lane of this wave.
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = 8 * piece + i;
      cs[i] = c < 2 * half ? trig[0][c < half ? c : c - half] : 1.0f;
      sn[i] = c < half ? -trig[1][c] : c < 2 * half ? trig[1][c - half] : 0.0f;
    }
    const int partner =
        (t - piece + (8 * piece < half ? 8 * piece + half : 8 * piece - half) / 8) * PLD;
    auto widen = [](const uint4& v, float (&y)[8]) {
      const uint32_t w4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[2 * i] = u2f(w4[i] << 16);
        y[2 * i + 1] = u2f(w4[i] & 0xffff0000u);
      }
    };
    auto put = [&](int group, const uint4& raw) {
      const int head = group * HPW + lane / LPH;
      const bool is_q = head < d.heads;
      const int kvh = head - d.heads;
      float y[8];
      widen(raw, y);
      if (is_q ? q_norm != nullptr : k_norm != nullptr) {
        float w[8];
        widen(is_q ? qn : kn, w);
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf_(y[i], y[i], ss);
        ss = group_sum<LPH>(ss);
        const float inv = 1.0f / __builtin_sqrtf(ss * (1.0f / HD) + eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * inv * (w[i] + 1.0f);
      }
      if (half > 0) {
        wave_sync();
        float4* mine = reinterpret_cast<float4*>(pairs + t * PLD);
        mine[0] = make_float4(y[0], y[1], y[2], y[3]);
        mine[1] = make_float4(y[4], y[5], y[6], y[7]);
        wave_sync();
        if (half % 8 == 0) {  // a lane's eight values have another lane's eight for partners
          if (8 * piece < 2 * half) {
            const float4* op = reinterpret_cast<const float4*>(pairs + partner);
            const float4 o0 = op[0], o1 = op[1];
            const float x[8] = {o0.x, o0.y, o0.z, o0.w, o1.x, o1.y, o1.z, o1.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = fmaf_(x[i], sn[i], y[i] * cs[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int c = 8 * piece + i, other = c < half ? c + half : c - half;
            if (c < 2 * half)
              y[i] = fmaf_(pairs[(t - piece + (other >> 3)) * PLD + (other & 7)], sn[i], y[i] * cs[i]);
          }
        }
      }
      if (head >= heads) return;
      if (is_q) {
        *reinterpret_cast<uint4*>(q_out + (int64_t(row) * d.heads + head) * HD + 8 * piece) =
            make_uint4(pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(y[4], y[5]), pack2(y[6], y[7]));
        return;
      }
      if (pid < 0) return;
      const int64_t at =
          pid * d.page_stride + (int64_t(kvh) * page + (p & (page - 1))) * HD + 8 * piece;
      if constexpr (F8) {
        const float s = k_scale ? k_scale[kvh] : 1.0f;
        uint32_t o[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i >> 2] |= uint32_t(narrow(y[i] / s)) << (8 * (i & 3));
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(k_cache) + at) = make_uint2(o[0], o[1]);
      } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(k_cache) + at) =
            make_uint4(pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(y[4], y[5]), pack2(y[6], y[7]));
      }
    };
    for (int g = g0; g < g1; g += AHEAD) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (g + i >= g1) break;
        put(g + i, raws[i]);
        raws[i] = load(g + AHEAD + i);
      }
    }
    return;
  }
  // V of kVRows rows and one kv head
  const int kvh = int(blockIdx.x) % d.kv_heads;
  const int row0 = int(blockIdx.x) / d.kv_heads * kVRows;
  const int64_t col = int64_t(d.heads) * q_width + int64_t(d.kv_heads + kvh) * HD;
  for (int i = t; i < kVRows * LPH; i += kQkThreads) {
    const int r = i / LPH, piece = i % LPH;
    if (row0 + r < rows) {
      const uint4 v =
          *reinterpret_cast<const uint4*>(qkv + int64_t(row0 + r) * qkv_stride + col + 8 * piece);
      uint32_t* dst = reinterpret_cast<uint32_t*>(buf.v + r * VLD + 8 * piece);  // 4-byte aligned
      dst[0] = v.x;
      dst[1] = v.y;
      dst[2] = v.z;
      dst[3] = v.w;
    }
  }
  __syncthreads();
  const int r = t % kVRows, row = row0 + r;
  if (row >= rows) return;
  const int seq = seqs ? seqs[row] : row, p = pos[row];
  if (unsigned(seq) >= unsigned(d.sequences) || p < 0 || (p >> d.page_log2) >= d.table_width) return;
  const int pid = page_at(table, d, seq, p >> d.page_log2);
  if (pid < 0) return;
  const int64_t at = pid * d.page_stride + (int64_t(kvh) * HD << d.page_log2) + (p & (page - 1));
  float s = 1.0f;
  if constexpr (F8) s = v_scale ? v_scale[kvh] : 1.0f;
  for (int c = t / kVRows; c < HD / 2; c += kQkThreads / kVRows) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(buf.v + r * VLD + 2 * c);
    const int64_t o = at + (int64_t(2 * c) << d.page_log2);
    if constexpr (F8) {
      uint8_t* dst = static_cast<uint8_t*>(v_cache);
      dst[o] = narrow(u2f(v << 16) / s);
      dst[o + page] = narrow(u2f(v & 0xffff0000u) / s);
    } else {
      uint16_t* dst = static_cast<uint16_t*>(v_cache);
      dst[o] = uint16_t(v);
      dst[o + page] = uint16_t(v >> 16);
    }
  }
}

// ---------------------------------------------------------------------------
// Decode: softmax(q k^T scale) v of one row over its sequence's positions.
//
// The keys of all rows are cut into chunks of whole units (four waves' tiles)
// whose length follows from all rows' lengths, so that a few chunks a compute
// unit cover any mix of short and long contexts; every wave forms that plan
// from the lengths itself.  A workgroup takes one (row, chunk, kv head) for the
// group's q heads, so each K and V value is read once; its four waves take
// tiles of KT keys in turn with a running maximum, sum and output each, and
// join through LDS.  Rows of one chunk are finished there, the others leave
// partials that the second launch joins in order.
//
// Matrix cores do both products with the q heads as columns (columns past the
// group are zero): S^T = K Q^T gives lane (head, quarter g) the scores of keys
// KT/4 g .. of the tile, because K's rows enter in that order, and these are the
// k-slots that the same lane supplies as P^T for O^T = V^T P^T.  So scores never
// leave their lane, and K and V come from memory straight into operands.  P is
// split in two bf16 parts: the matrix cores have time, and P keeps 16 bits.
//
// The memory bounds it where there are many keys: 64 rows of 32 q / 8 kv heads of 128
// on up to 16384 take 386 us and 6 to join (5.5 TB/s), 40 e4m3 rows of 28 / 4 heads on
// up to 12001 48 and 5.  Of one row of 60001 keys (16 / 2 heads of 256, 30 us and 6), 2.7
// us go to the plan, the first keys are there after 6.4, and 2.5 join the waves; 8 rows of
// up to 4000 (14 and 5) are little else.
constexpr int kDecodeMaxChunks = 2048 + 1;  // of one row: twice decode_target and the rounding
template <bool F8>
struct DecodeTile {
  static constexpr int kKeys = F8 ? 64 : 32;  // a lane's 16 bytes of V: 16 or 8 keys
  static constexpr int kUnit = 4 * kKeys;
};
// Workgroups that a compute unit holds, by registers.
constexpr int decode_occupancy(int head_dim) { return head_dim == 256 ? 2 : head_dim == 128 ? 3 : 4; }
// Chunks wanted: as many as run at once.
int decode_target(const PageDims& d) { return 256 * decode_occupancy(d.head_dim); }

// The length of a row's context, or -1 for a padding row.
__device__ __forceinline__ int row_len(const int32_t* __restrict__ seqs,
                                       const int32_t* __restrict__ lens, const PageDims& d, int r,
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
struct Plan {
  int chunk_units, len0;
};
__device__ __forceinline__ Plan make_plan(const int32_t* seqs, const int32_t* lens,
                                          const PageDims& d, int rows, int unit, int target) {
  const int lane = threadIdx.x & 63;
  Plan p;
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

// The sum of the infinite and NaN values among positions k0 .. k1 - 1 of one dim (at: from a page's
// start to that dim's first position), 0 where there is none.
__device__ __forceinline__ float sum_of_odd(const uint16_t* __restrict__ v_cache,
                                            const int32_t* __restrict__ table, const PageDims& d,
                                            int seq, int k0, int k1, int64_t at) {
  float sum = 0.0f;
  for (int key = k0; key < k1; ++key) {
    const int pid = page_at(table, d, seq, key >> d.page_log2);
    if (pid < 0) continue;
    const uint16_t v = v_cache[pid * d.page_stride + at + (key & ((1 << d.page_log2) - 1))];
    if ((v & 0x7f80u) == 0x7f80u) sum += bf16_to_f32(v);
  }
  return sum;
}

template <int HD, bool F8>
__global__ __launch_bounds__(256, decode_occupancy(HD)) void decode_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ qkv, int64_t qkv_stride, int rows,
    const int32_t* __restrict__ seqs, const int32_t* __restrict__ lens,
    const int32_t* __restrict__ table, const void* __restrict__ k_cache,
    const void* __restrict__ v_cache, const float* __restrict__ k_scale,
    const float* __restrict__ v_scale, PageDims d, float scale, int target,
    float* __restrict__ o_part, float* __restrict__ ml_part, int2* __restrict__ row_chunks,
    uint16_t* __restrict__ out) {
  constexpr int KT = DecodeTile<F8>::kKeys, kUnit = DecodeTile<F8>::kUnit;
  constexpr int T = KT / 16;        // score tiles
  constexpr int KG = KT / 4;        // keys of a lane quarter
  constexpr int NV = HD / 16;       // dim tiles of the output
  constexpr int KL = HD / (F8 ? 64 : 32);  // 16-byte pieces of a K row a lane
  constexpr int QLD = HD + 8;       // padded q row in LDS
  constexpr int OLD = HD + 4;       // padded output row in LDS
  // the next tile's K is requested once this one's scores are done; at 256 dims the
  // registers hold one tile of each, and the other waves cover its latency
  constexpr bool kAhead = HD < 256;
  __shared__ __align__(16) uint16_t qs[16 * QLD];
  __shared__ float mls[2][4][16];
  extern __shared__ __align__(16) float os[];  // [4 waves][group][OLD]
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int col = lane & 15, g = lane >> 4;
  const int group = d.heads / d.kv_heads;
  // this workgroup's (row, chunk, kv head)
  const int item = blockIdx.x, kvh = item % d.kv_heads;
  const int want = item / d.kv_heads;
  const Plan plan = make_plan(seqs, lens, d, rows, kUnit, target);
  const int cu = plan.chunk_units;
  int row = -1, chunk = 0, chunks = 0, before = 0, len = 0;
  for (int r = 0; r < rows; r += 64) {
    const int l = r == 0 ? plan.len0 : row_len(seqs, lens, d, r + lane, rows);
    const int n = (units_of(l, kUnit) + cu - 1) / cu;
    const int sum = wave_scan(n);
    const uint64_t past = __ballot(before + sum > want);
    if (past) {
      const int f = __builtin_ctzll(past);
      row = r + f;
      len = __builtin_amdgcn_readlane(l, f);
      chunks = __builtin_amdgcn_readlane(n, f);
      before += __builtin_amdgcn_readlane(sum, f) - chunks;
      chunk = want - before;
      if (chunk == 0 && kvh == 0 && t == 0)  // for the launch that joins
        row_chunks[row] = make_int2(before, chunks);
      break;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  if (row < 0) return;  // uniform: past the last chunk
  const int seq = seqs ? seqs[row] : row;
  // units / chunks each, the first ones one more
  const int units = units_of(len, kUnit), few = units / chunks, more_units = units % chunks;
  const int k0 = (chunk * few + min(chunk, more_units)) * kUnit;
  const int k1 = min(len, k0 + (few + (chunk < more_units)) * kUnit);  // k0 < k1
  const bool whole = k0 == 0 && k1 == len;
  const int last_page = (len - 1) >> d.page_log2;

  const char* kc = static_cast<const char*>(k_cache);
  const char* vc = static_cast<const char*>(v_cache);
  constexpr int E = F8 ? 1 : 2;
  const int page = 1 << d.page_log2;
  const float sl2 =
      scale * kLog2e * (F8 && k_scale ? k_scale[kvh] : 1.0f);  // scores in log2 units
  // K row of score tile s for this lane's operand row: key KG (col / 4) + 4 s + col % 4
  const int krow = KG * (col >> 2) + (col & 3);
  const int vrow = KG * g;  // first key of this lane's V operands and scores
  float m_run = neg_inf(), l_run = 0.0f;
  floatx4_t o[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) o[n] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};

  uint4 kb[T][KL], vb[NV];
  int pk = 0, pv = 0;
  auto pages_of = [&](int tile) {
    pk = page_at(table, d, seq, min((tile + krow) >> d.page_log2, last_page));
    pv = page_at(table, d, seq, min((tile + vrow) >> d.page_log2, last_page));
  };
  auto load_k = [&](int tile) {
    const int64_t base = (pk < 0 ? 0 : pk) * d.page_stride + (int64_t(kvh) << d.page_log2) * HD;
    const int off = (tile + krow) & (page - 1);
#pragma unroll
    for (int s = 0; s < T; ++s)
#pragma unroll
      for (int i = 0; i < KL; ++i)
        kb[s][i] = *reinterpret_cast<const uint4*>(
            kc + (base + int64_t(off + 4 * s) * HD) * E + 64 * i + 16 * g);
  };
  auto load_v = [&](int tile) {
    const int64_t base = (pv < 0 ? 0 : pv) * d.page_stride + (int64_t(kvh) << d.page_log2) * HD +
                         ((tile + vrow) & (page - 1));
    const char* p = vc + (base + (int64_t(col) << d.page_log2)) * E;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      vb[n] = *reinterpret_cast<const uint4*>(p);
      p += (16 * E) << d.page_log2;
      asm("" : "+v"(p));  // one address that walks: sixteen at once would spill
    }
  };
  int tile = k0 + wave * KT;
  if (tile < k1) {
    pages_of(tile);
    load_k(tile);
    load_v(tile);
  }
  // q heads into LDS (rows past the group zero), under the first tile's way
  for (int i = t; i < 16 * HD / 8; i += 256) {
    const int h = i / (HD / 8), piece = i % (HD / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (h < group)
      v = *reinterpret_cast<const uint4*>(
          q + (int64_t(row) * d.heads + kvh * group + h) * HD + 8 * piece);
    *reinterpret_cast<uint4*>(qs + h * QLD + 8 * piece) = v;
  }
  __syncthreads();
  for (; tile < k1; tile += kUnit) {
    // q is read again for every tile where its registers (up to 32) would spill, held
    if constexpr (HD == 256 || (HD == 128 && F8)) asm volatile("" ::: "memory");
    // valid keys of this lane quarter
    const int nk = pv < 0 ? 0 : min(max(k1 - (tile + vrow), 0), KG);
    floatx4_t sc[T];
#pragma unroll
    for (int s = 0; s < T; ++s) sc[s] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      if constexpr (F8) {
        const uint4 qa = *reinterpret_cast<const uint4*>(qs + col * QLD + 64 * i + 16 * g);
        const uint4 qb = *reinterpret_cast<const uint4*>(qs + col * QLD + 64 * i + 16 * g + 8);
#pragma unroll
        for (int s = 0; s < T; ++s) {
          sc[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8_t, widen8(kb[s][i].x, kb[s][i].y)),
              __builtin_bit_cast(bf16x8_t, qa), sc[s], 0, 0, 0);
          sc[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8_t, widen8(kb[s][i].z, kb[s][i].w)),
              __builtin_bit_cast(bf16x8_t, qb), sc[s], 0, 0, 0);
        }
      } else {
        const uint4 qa = *reinterpret_cast<const uint4*>(qs + col * QLD + 32 * i + 8 * g);
#pragma unroll
        for (int s = 0; s < T; ++s)
          sc[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8_t, kb[s][i]), __builtin_bit_cast(bf16x8_t, qa), sc[s], 0,
              0, 0);
      }
    }
    const int next = tile + kUnit;
    const bool more = next < k1;
    const int nv = nk;
    if (kAhead && more) {
      pages_of(next);
      load_k(next);
    }
    float mt = neg_inf();
#pragma unroll
    for (int s = 0; s < T; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sc[s][r] = 4 * s + r < nk ? sc[s][r] * sl2 : neg_inf();
        mt = fmaxf(mt, sc[s][r]);
      }
    mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
    mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
    const float mn = fmaxf(m_run, mt);
    const float ref = mn == neg_inf() ? 0.0f : mn;  // no key yet: every weight is 0
    if (__any(mn != m_run)) {
      const float alpha = __builtin_amdgcn_exp2f(m_run - ref);
      l_run *= alpha;
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[n][r] *= alpha;
      m_run = mn;
    }
    uint32_t ph[2 * T], pl[2 * T];
#pragma unroll
    for (int s = 0; s < T; ++s)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float a = __builtin_amdgcn_exp2f(sc[s][r] - ref);
        const float b = __builtin_amdgcn_exp2f(sc[s][r + 1] - ref);
        l_run += a + b;
        const uint32_t h = pack2(a, b);
        ph[2 * s + r / 2] = h;
        pl[2 * s + r / 2] = pack2(a - u2f(h << 16), b - u2f(h & 0xffff0000u));
      }
    // keys past the end may hold anything: their values become 0 (the last tile only)
    if (!__all(nv == KG)) {
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        uint32_t w[4] = {vb[n].x, vb[n].y, vb[n].z, vb[n].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          constexpr int P = 4 / E;  // keys a word
          const int left = nv - P * i;
          const int bits = left <= 0 ? 0 : (left >= P ? 32 : left * 8 * E);
          w[i] = bits == 32 ? w[i] : (w[i] & ((1u << bits) - 1u));
        }
        vb[n] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      if constexpr (F8) {
        const bf16x8_t va = __builtin_bit_cast(bf16x8_t, widen8(vb[n].x, vb[n].y));
        const bf16x8_t vd = __builtin_bit_cast(bf16x8_t, widen8(vb[n].z, vb[n].w));
        const uint4 h0 = make_uint4(ph[0], ph[1], ph[2], ph[3]);
        const uint4 h1 = make_uint4(ph[4], ph[5], ph[6], ph[7]);
        const uint4 l0 = make_uint4(pl[0], pl[1], pl[2], pl[3]);
        const uint4 l1 = make_uint4(pl[4], pl[5], pl[6], pl[7]);
        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(bf16x8_t, h0), o[n], 0, 0, 0);
        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(bf16x8_t, l0), o[n], 0, 0, 0);
        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vd, __builtin_bit_cast(bf16x8_t, h1), o[n], 0, 0, 0);
        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vd, __builtin_bit_cast(bf16x8_t, l1), o[n], 0, 0, 0);
      } else {
        const bf16x8_t va = __builtin_bit_cast(bf16x8_t, vb[n]);
        const uint4 h0 = make_uint4(ph[0], ph[1], ph[2], ph[3]);
        const uint4 l0 = make_uint4(pl[0], pl[1], pl[2], pl[3]);
        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(bf16x8_t, h0), o[n], 0, 0, 0);
        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(bf16x8_t, l0), o[n], 0, 0, 0);
      }
    }
    if (!kAhead && more) {
      pages_of(next);
      load_k(next);
    }
    if (more) load_v(next);
  }
  // the four waves' parts
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  if (g == 0) {
    mls[0][wave][col] = m_run;
    mls[1][wave][col] = l_run;
  }
  if (col < group) {
#pragma unroll
    for (int n = 0; n < NV; ++n)
      *reinterpret_cast<floatx4_t*>(os + (wave * group + col) * OLD + 16 * n + 4 * g) = o[n];
  }
  __syncthreads();
  const float vs = F8 && v_scale ? v_scale[kvh] : 1.0f;
  const int64_t part0 = (int64_t(item / d.kv_heads) * d.kv_heads + kvh) * group;
  // output i of the chunk; true where it is NaN under weights that are not.  again: where it was
  auto output = [&](int i, auto again) {
    const int h = i / HD, c = i % HD;
    float M = mls[0][0][h];
#pragma unroll
    for (int w = 1; w < 4; ++w) M = fmaxf(M, mls[0][w][h]);
    const float ref = M == neg_inf() ? 0.0f : M;
    float L = 0.0f, O = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float e = __builtin_amdgcn_exp2f(mls[0][w][h] - ref);
      L = fmaf_(mls[1][w][h], e, L);
      O = fmaf_(os[(w * group + h) * OLD + c], e, O);
    }
    const bool odd = O != O && L == L;
    if constexpr (again) {
      if (!odd) return false;
      const float sum = sum_of_odd(static_cast<const uint16_t*>(v_cache), table, d, seq, k0, k1,
                                   (int64_t(kvh) * HD + c) << d.page_log2);
      if (sum != 0.0f) O = sum;
    }
    if (whole) {
      float y = L == 0.0f ? 0.0f : O / L * vs;
      const int head = kvh * group + h;
      if (d.gated)
        y *= gate_of(bf16_to_f32(qkv[int64_t(row) * qkv_stride + int64_t(head) * 2 * HD + HD + c]));
      out[(int64_t(row) * d.heads + head) * HD + c] = f32_to_bf16(y);
    } else {
      o_part[(part0 + h) * HD + c] = O;
      if (c == 0) {
        ml_part[(part0 + h) * 2] = M;
        ml_part[(part0 + h) * 2 + 1] = L;
      }
    }
    return odd;
  };
  bool odd = false;
  for (int i = t; i < group * HD; i += 256) odd |= output(i, std::false_type{});
  // An infinite value times a p whose low part is 0 or negative, or times a weight that has become
  // 0, is NaN, where a positive weight leaves it infinite.  Such outputs are formed once more, from
  // the values that are no numbers alone: nothing before has to look for them.  (e4m3 has no
  // infinity.)
  if constexpr (!F8)
    if (odd)
      for (int i = t; i < group * HD; i += 256) output(i, std::true_type{});
}

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

int decode_unit(const PageDims& d) {
  return d.f8 ? DecodeTile<true>::kUnit : DecodeTile<false>::kUnit;
}

// The most chunks (times kv heads) that any lengths give.
int64_t decode_items(int rows, const PageDims& d) {
  const int64_t unit = decode_unit(d);
  const int64_t most = ((int64_t(d.table_width) << d.page_log2) + unit - 1) / unit;
  const int64_t all = int64_t(rows) * d.kv_heads;
  const int64_t target = 2 * decode_target(d);
  return all * most < target + all ? all * most : target + all;
}

}  // namespace

int paged_append(const uint16_t* qkv, int64_t qkv_stride, int rows, const int32_t* seqs,
                 const int32_t* pos, const int32_t* rope_pos, const RopeAxes& rope,
                 const uint16_t* q_norm, const uint16_t* k_norm, float eps, const int32_t* table,
                 const PageDims& d, const float* k_scale, const float* v_scale, uint16_t* q_out,
                 void* k_cache, void* v_cache, hipStream_t s) {
  const int per = 64 / (d.head_dim / 8);
  const int groups = (d.heads + d.kv_heads + per - 1) / per;
  // as many groups of a row a wave as leave 12 waves a compute unit: the more, the fewer sines
  // are formed twice (4093 rows of 40 heads of 128: 24.6 us, 26.9 with twice the waves)
  const int64_t share = int64_t(rows) * groups / (12 * 256);
  const int each = int(share < 1 ? 1 : share < groups ? share : groups);
  const int64_t vb = int64_t((rows + kVRows - 1) / kVRows) * d.kv_heads;
  const int64_t waves = int64_t(rows) * ((groups + each - 1) / each);
  const int64_t blocks = vb + (waves + kQkThreads / 64 - 1) / (kQkThreads / 64);
  if (blocks > 0x7fffffff) return MX_EUNSUPPORTED;
#define MX_APPEND(HH, FF)                                                                       \
  if (d.head_dim == HH && d.f8 == FF) {                                                         \
    hipLaunchKernelGGL((append_kernel<HH, FF>), dim3(unsigned(blocks)), dim3(kQkThreads), 0, s, \
                       qkv, qkv_stride, rows, seqs, pos, rope_pos, rope, q_norm, k_norm, eps,   \
                       table, d, k_scale, v_scale, q_out, k_cache, v_cache, groups, each,       \
                       int(vb));                                                                \
    return hipGetLastError() == hipSuccess ? MX_OK : MX_EHIP;                                   \
  }
  MX_APPEND(64, false) MX_APPEND(128, false) MX_APPEND(256, false)
  MX_APPEND(64, true) MX_APPEND(128, true) MX_APPEND(256, true)
#undef MX_APPEND
  return MX_EUNSUPPORTED;
}

size_t paged_decode_workspace(int rows, const PageDims& d) {
  return size_t(decode_items(rows, d)) * (d.heads / d.kv_heads) * (d.head_dim + 2) * 4 +
         size_t(rows) * 8;
}

int paged_decode(const uint16_t* q, const uint16_t* qkv, int64_t qkv_stride, int rows,
                 const int32_t* seqs, const int32_t* lens, const int32_t* table,
                 const void* k_cache, const void* v_cache, const float* k_scale,
                 const float* v_scale, const PageDims& d, float scale, void* workspace,
                 uint16_t* out, hipStream_t s) {
  const int64_t items = decode_items(rows, d), joins = int64_t(rows) * d.heads;
  if (items > 0x7fffffff || joins > 0x7fffffff) return MX_EUNSUPPORTED;
  const int group = d.heads / d.kv_heads;
  float* o_part = static_cast<float*>(workspace);
  float* ml_part = o_part + items * group * d.head_dim;
  const int lds = 4 * group * (d.head_dim + 4) * 4;
  int2* row_chunks = reinterpret_cast<int2*>(ml_part + items * group * 2);
  const int target = decode_target(d);
#define MX_JOIN(HH, DW, NW)                                                                      \
  hipLaunchKernelGGL((decode_join_kernel<HH, DW, NW>), dim3(unsigned(joins * (HH / DW))),        \
                     dim3(64 * NW), 0, s, qkv, qkv_stride, rows, seqs, lens,                     \
                     d.f8 ? v_scale : nullptr, d, row_chunks, o_part, ml_part, out)
#define MX_DECODE(HH, FF)                                                                        \
  if (d.head_dim == HH && d.f8 == FF) {                                                          \
    const auto fn = decode_kernel<HH, FF>;                                                       \
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(fn),                                   \
                            hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)      \
      return MX_EHIP;                                                                            \
    hipLaunchKernelGGL(fn, dim3(unsigned(items)), dim3(256), lds, s, q, qkv, qkv_stride, rows,   \
                       seqs, lens, table, k_cache, v_cache, k_scale, v_scale, d, scale, target,  \
                       o_part, ml_part, row_chunks, out);                                        \
    if (hipGetLastError() != hipSuccess) return MX_EHIP;                                         \
    /* few rows have many chunks each */                                                         \
    if (joins <= 64)                                                                             \
      MX_JOIN(HH, 64, 16);                                                                       \
    else                                                                                         \
      MX_JOIN(HH, HH, 4);                                                                          \
    return hipGetLastError() == hipSuccess ? MX_OK : MX_EHIP;                                    \
  }
  MX_DECODE(64, false) MX_DECODE(128, false) MX_DECODE(256, false)
  MX_DECODE(64, true) MX_DECODE(128, true) MX_DECODE(256, true)
#undef MX_DECODE
#undef MX_JOIN
  return MX_EUNSUPPORTED;
}

}  // namespace mx
