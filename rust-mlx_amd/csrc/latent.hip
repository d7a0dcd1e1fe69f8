// The latent cache: rows appended to it, and positions read back.
//
// A position is one vector for all heads: a latent of latent_dim values, from which the heads' keys and
// values follow by products, and a rotary key of rope_dim that they share.  A page holds its positions
// row after row, so what both of attention's products read is one contiguous row.  An e4m3 cache keeps
// one fp32 scale a position beside the pages: its largest value over 448, formed as it is written.
#include "paged_core.hpp"

namespace mx {

namespace {

using namespace pg;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int DR = 64;          // rope_dim
constexpr int kQHeads = 16;     // heads that a wave rotates at once, four lanes each

// Where position p of a sequence lies: its first element, or -1 where it has no page.
struct Place {
  int64_t at, scale;
};
__device__ __forceinline__ Place place_of(const int32_t* __restrict__ table, const LatentDims& d,
                                          int seq, int64_t p, int wide) {
  Place r = {-1, -1};
  if (p < 0 || (p >> d.page_log2) >= d.table_width) return r;
  const int pid = page_at(table, d, seq, int(p >> d.page_log2));
  if (pid < 0) return r;
  const int off = int(p) & ((1 << d.page_log2) - 1);
  r.at = pid * d.page_stride + int64_t(off) * wide;
  r.scale = (int64_t(pid) << d.page_log2) + off;
  return r;
}

// ---------------------------------------------------------------------------
// Append: RMS norm of the latent, rotation of its key and of the queries, and the
// cache's writes, in one launch.  The formulas and the angle's 64 bits are those of
// the paged cache's append.  Bytes bound it; the first waves of the grid take one
// row of the cache each, the others `each` groups of 16 query heads of a row, whose
// sines they form once.  4093 rows of 20 heads into e4m3 take 8.2 us (28 MB,
// 3.4 TB/s), a wave's chain of position, page and row included; 8 rows of 128
// heads 3 us.
template <int DC, bool F8>
__global__ __launch_bounds__(kThreads) void append_kernel(
    const uint16_t* __restrict__ x, int64_t x_stride, const uint16_t* __restrict__ q,
    int64_t q_stride, int rows, const int32_t* __restrict__ seqs, const int32_t* __restrict__ pos,
    const int32_t* __restrict__ rope_pos, RopeAxes rope, const uint16_t* __restrict__ norm, float eps,
    const int32_t* __restrict__ table, LatentDims d, uint16_t* __restrict__ q_rope,
    void* __restrict__ cache, float* __restrict__ scales, int groups, int each, int kv_blocks) {
  constexpr int VPL = DC / 64;  // latent values a lane
  typedef uint32_t vec __attribute__((ext_vector_type(VPL / 2)));
  __shared__ __align__(16) float trigs[kWaves][2][DR / 2];
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  auto turn = [&](int row, int i, float* sn, float* cs) {
    sincos_turn(double(rope_pos[int64_t(rope.pair_axis[i]) * rows + row]) * rope.inv_freq[i] *
                    0.15915494309189533577,
                sn, cs);
  };
  if (int(blockIdx.x) < kv_blocks) {
    const int row = int(blockIdx.x) * kWaves + wave;
    if (row >= rows) return;
    const uint16_t* src = x + int64_t(row) * x_stride;
    const vec raw = *reinterpret_cast<const vec*>(src + VPL * lane);
    const int i = lane & 31;  // the lane's pair of the rotary key, in both halves of the wave
    const float a = bf16_to_f32(src[DC + i]), b = bf16_to_f32(src[DC + DR / 2 + i]);
    vec w = 0;
    if (norm) w = *reinterpret_cast<const vec*>(norm + VPL * lane);
    const int seq = seqs ? seqs[row] : row;
    if (unsigned(seq) >= unsigned(d.sequences)) return;  // a padding row (uniform)
    const Place to = place_of(table, d, seq, pos[row], DC + DR);
    if (to.at < 0) return;
    float sn, cs;
    turn(row, i, &sn, &cs);
    float y[VPL];
#pragma unroll
    for (int k = 0; k < VPL / 2; ++k) {
      y[2 * k] = u2f(raw[k] << 16);
      y[2 * k + 1] = u2f(raw[k] & 0xffff0000u);
    }
    if (norm) {
      float ss = 0.0f;
#pragma unroll
      for (int k = 0; k < VPL; ++k) ss = fmaf_(y[k], y[k], ss);
      ss = group_sum<32>(ss);
      ss += __shfl_xor(ss, 32, 64);
      const float inv = 1.0f / __builtin_sqrtf(ss * (1.0f / DC) + eps);
#pragma unroll
      for (int k = 0; k < VPL / 2; ++k) {
        y[2 * k] = y[2 * k] * inv * (u2f(w[k] << 16) + 1.0f);
        y[2 * k + 1] = y[2 * k + 1] * inv * (u2f(w[k] & 0xffff0000u) + 1.0f);
      }
    }
    // the lower half of the wave stores the pair's first value, the upper one its second
    const float r = lane < 32 ? fmaf_(b, -sn, a * cs) : fmaf_(a, sn, b * cs);
    if constexpr (F8) {
      float most = __builtin_fabsf(r);
#pragma unroll
      for (int k = 0; k < VPL; ++k) most = fmaxf(most, __builtin_fabsf(y[k]));
      for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
      const float scale = fmaxf(most, 7.888609052210118e-31f) / 448.0f;  // 2^-100
      uint8_t* dst = static_cast<uint8_t*>(cache) + to.at;
      uint32_t o[VPL / 4];
#pragma unroll
      for (int k = 0; k < VPL / 4; ++k) {
        o[k] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[k] |= uint32_t(narrow(y[4 * k + j] / scale)) << (8 * j);
      }
      if constexpr (VPL == 8)
        *reinterpret_cast<uint2*>(dst + 8 * lane) = make_uint2(o[0], o[1]);
      else
        *reinterpret_cast<uint32_t*>(dst + 4 * lane) = o[0];
      dst[DC + lane] = narrow(r / scale);
      if (lane == 0) scales[to.scale] = scale;
    } else {
      uint16_t* dst = static_cast<uint16_t*>(cache) + to.at;
      vec o;
#pragma unroll
      for (int k = 0; k < VPL / 2; ++k) o[k] = pack2(y[2 * k], y[2 * k + 1]);
      *reinterpret_cast<vec*>(dst + VPL * lane) = o;
      dst[DC + lane] = f32_to_bf16(r);
    }
    return;
  }
  const int per_row = (groups + each - 1) / each;
  const int64_t b = int64_t(int(blockIdx.x) - kv_blocks) * kWaves + wave;
  if (b >= int64_t(rows) * per_row) return;
  const int row = int(b / per_row), g0 = int(b % per_row) * each, g1 = min(groups, g0 + each);
  const int seq = seqs ? seqs[row] : row;
  const int piece = lane & 3;
  const int q_dim = d.nope_dim + DR;
  const uint16_t* src = q + int64_t(row) * q_stride + d.nope_dim + 8 * piece;
  uint4 lo, hi;
  auto load = [&](int g) {
    const int head = min(g * kQHeads + lane / 4, d.heads - 1);
    lo = *reinterpret_cast<const uint4*>(src + int64_t(head) * q_dim);
    hi = *reinterpret_cast<const uint4*>(src + int64_t(head) * q_dim + DR / 2);
  };
  load(g0);
  if (unsigned(seq) >= unsigned(d.sequences)) return;  // a padding row (uniform)
  if (lane < DR / 2) turn(row, lane, &trigs[wave][1][lane], &trigs[wave][0][lane]);
  wave_sync();
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cs[i] = trigs[wave][0][8 * piece + i];
    sn[i] = trigs[wave][1][8 * piece + i];
  }
  for (int g = g0; g < g1; ++g) {
    const uint32_t a[4] = {lo.x, lo.y, lo.z, lo.w}, c[4] = {hi.x, hi.y, hi.z, hi.w};
    const int head = g * kQHeads + lane / 4;
    if (g + 1 < g1) load(g + 1);
    uint32_t first[4], second[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a0 = u2f(a[k] << 16), a1 = u2f(a[k] & 0xffff0000u);
      const float c0 = u2f(c[k] << 16), c1 = u2f(c[k] & 0xffff0000u);
      first[k] = pack2(fmaf_(c0, -sn[2 * k], a0 * cs[2 * k]), fmaf_(c1, -sn[2 * k + 1], a1 * cs[2 * k + 1]));
      second[k] = pack2(fmaf_(a0, sn[2 * k], c0 * cs[2 * k]), fmaf_(a1, sn[2 * k + 1], c1 * cs[2 * k + 1]));
    }
    if (head >= d.heads) continue;
    uint16_t* dst = q_rope + (int64_t(row) * d.heads + head) * DR + 8 * piece;
    *reinterpret_cast<uint4*>(dst) = make_uint4(first[0], first[1], first[2], first[3]);
    *reinterpret_cast<uint4*>(dst + DR / 2) = make_uint4(second[0], second[1], second[2], second[3]);
  }
}

// ---------------------------------------------------------------------------
// Read: a copy of scattered rows to packed ones (times the position's scale), bound by bytes.  A
// workgroup takes kReadRows rows, finds where they lie, and then has all of its pieces on their way.
// 60001 positions of e4m3 take 24.7 us (104 MB, 4.2 TB/s), 3300 of bf16 4.6.
constexpr int kReadRows = 32;

template <int DC, bool F8>
__global__ __launch_bounds__(kThreads) void read_kernel(
    const void* __restrict__ cache, const float* __restrict__ scales, int rows,
    const int32_t* __restrict__ starts, const int32_t* __restrict__ first,
    const int32_t* __restrict__ table, LatentDims d, uint16_t* __restrict__ latent,
    int64_t latent_stride, uint16_t* __restrict__ rope, int64_t rope_stride) {
  constexpr int P = (DC + DR) / 8, N = kReadRows * P / kThreads;  // pieces of eight values: of a row, a thread
  constexpr int E = F8 ? 1 : 2;
  __shared__ int64_t from[kReadRows];
  __shared__ float by[kReadRows];
  const int t = threadIdx.x, row0 = blockIdx.x * kReadRows;
  if (t < kReadRows) {
    const int row = row0 + t;
    int64_t at = -2;  // outside every sequence
    float s = 1.0f;
    if (row < rows) {
      int lo = 0, hi = d.sequences;  // the first sequence that ends past the row
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (starts[mid + 1] > row)
          hi = mid;
        else
          lo = mid + 1;
      }
      if (lo < d.sequences && starts[lo] <= row) {
        const Place p = place_of(table, d, lo, int64_t(first ? first[lo] : 0) + row - starts[lo], DC + DR);
        at = p.at;
        if (F8 && at >= 0) s = scales[p.scale];
      }
    }
    from[t] = at;
    by[t] = s;
  }
  __syncthreads();
  uint4 raw[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int slot = t + kThreads * i, r = slot / P, piece = slot % P;
    const int64_t at = from[r];
    raw[i] = make_uint4(0, 0, 0, 0);
    if (at < 0) continue;
    const char* src = static_cast<const char*>(cache) + (at + 8 * piece) * E;
    if constexpr (F8) {
      const uint2 v = *reinterpret_cast<const uint2*>(src);
      raw[i].x = v.x;
      raw[i].y = v.y;
    } else {
      raw[i] = *reinterpret_cast<const uint4*>(src);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int slot = t + kThreads * i, r = slot / P, piece = slot % P;
    if (from[r] == -2) continue;
    uint4 v = raw[i];
    if constexpr (F8) {
      const uint4 w = widen8(v.x, v.y);
      const float s = by[r];
      auto times = [&](uint32_t p) { return pack2(u2f(p << 16) * s, u2f(p & 0xffff0000u) * s); };
      v = make_uint4(times(w.x), times(w.y), times(w.z), times(w.w));
    }
    const int64_t row = row0 + r;
    uint16_t* dst = piece < DC / 8 ? latent + row * latent_stride + 8 * piece
                                   : rope + row * rope_stride + 8 * (piece - DC / 8);
    *reinterpret_cast<uint4*>(dst) = v;
  }
}

}  // namespace

int latent_append(const uint16_t* x, int64_t x_stride, const uint16_t* q, int64_t q_stride, int rows,
                  const int32_t* seqs, const int32_t* pos, const int32_t* rope_pos,
                  const RopeAxes& rope, const uint16_t* norm, float eps, const int32_t* table,
                  const LatentDims& d, uint16_t* q_rope, void* cache, float* scales, hipStream_t s) {
  const int groups = (d.heads + kQHeads - 1) / kQHeads;
  // as many groups of a row a wave as leave 12 waves a compute unit: the sines are formed once for them
  const int64_t share = int64_t(rows) * groups / (12 * 256);
  const int each = int(share < 1 ? 1 : share < groups ? share : groups);
  const int64_t kv_blocks = (int64_t(rows) + kWaves - 1) / kWaves;
  const int64_t waves = int64_t(rows) * ((groups + each - 1) / each);
  const int64_t blocks = kv_blocks + (waves + kWaves - 1) / kWaves;
  if (blocks > 0x7fffffff) return MX_EUNSUPPORTED;
#define MX_APPEND(DC, FF)                                                                           \
  if (d.latent_dim == DC && d.f8 == FF) {                                                           \
    hipLaunchKernelGGL((append_kernel<DC, FF>), dim3(unsigned(blocks)), dim3(kThreads), 0, s, x,    \
                       x_stride, q, q_stride, rows, seqs, pos, rope_pos, rope, norm, eps, table, d, \
                       q_rope, cache, scales, groups, each, int(kv_blocks));                        \
    return hipGetLastError() == hipSuccess ? MX_OK : MX_EHIP;                                       \
  }
  MX_APPEND(256, false) MX_APPEND(512, false) MX_APPEND(256, true) MX_APPEND(512, true)
#undef MX_APPEND
  return MX_EUNSUPPORTED;
}

int latent_read(const void* cache, const float* scales, int rows, const int32_t* starts,
                const int32_t* first, const int32_t* table, const LatentDims& d, uint16_t* latent,
                int64_t latent_stride, uint16_t* rope, int64_t rope_stride, hipStream_t s) {
  const int64_t blocks = (int64_t(rows) + kReadRows - 1) / kReadRows;
#define MX_READ(DC, FF)                                                                            \
  if (d.latent_dim == DC && d.f8 == FF) {                                                          \
    hipLaunchKernelGGL((read_kernel<DC, FF>), dim3(unsigned(blocks)), dim3(kThreads), 0, s, cache, \
                       scales, rows, starts, first, table, d, latent, latent_stride, rope,         \
                       rope_stride);                                                               \
    return hipGetLastError() == hipSuccess ? MX_OK : MX_EHIP;                                      \
  }
  MX_READ(256, false) MX_READ(512, false) MX_READ(256, true) MX_READ(512, true)
#undef MX_READ
  return MX_EUNSUPPORTED;
}

}  // namespace mx
