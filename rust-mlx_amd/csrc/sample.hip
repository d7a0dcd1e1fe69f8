// Sampling from bf16 logits with temperature, top-k, top-p and min-p.
//
// Tokens are ordered by logit, largest first, lowest id first among equals; with
// w_j = exp((l_j - l_0) / T) every filter keeps a prefix of that order:
//   top-k  the first k
//   top-p  the shortest prefix with a mass of at least p times the first k's
//   min-p  those with w_j >= min_p
// n is the shortest of them (at least one token), and the sampled token is the
// first whose prefix mass exceeds u times the mass of n (the n-th from u = 1 on).
//
// bf16 has 65536 values, so a row is known by how often each occurs, and needs an
// exponential per occurring value instead of one per token, without any sort.
// Counts are exact and masses are sums of few products in 64 bits, so neither the
// order of the atomics nor the launch shape can change a token: a u within the
// sums' rounding of a border falls on one side of it, always the same.
//
// Launch 1 counts: a workgroup takes a part of a row (at most 65024 tokens, so
// 16-bit counters suffice: 128 KB of LDS for all values) and writes the segments
// of 64 neighbouring values that occur, with a bit each.
// Launch 2 chooses, a workgroup a row: it adds the parts' segments, weighs them,
// forms prefixes over the 1024 segments, and one wave answers each question
// (which value holds rank k, which holds mass x) by a search over the prefixes
// and then over one segment's 64 values, a lane each.  The rank within the
// value's tokens picks the part by the parts' own counts, and only that part is
// read again for the id.
//
// The latency of few dependent steps bounds it: one row of 151936 takes 6 us to count
// and 14 to choose, 64 rows 10 and 16 (their logits alone would take 4).  One workgroup
// a row that counts, chooses and reads the row three times takes 76 us for 1 to 256
// rows: each read is 19 dependent trips of one compute unit.
#include "common.hpp"
#include "kernels.hpp"

namespace mx {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kSegments = 1024;
constexpr int kPiece = 512;        // tokens of one wave's step: eight a lane
constexpr int kPartPieces = 127;   // pieces of a part at most: 65024 tokens
constexpr int kWavePieces = 8;     // of them a wave's, held in registers
constexpr int kBatchParts = 512;   // parts in flight: two rounds of the device
constexpr int kMaxParts = 32;
constexpr int kSlots = 480;        // segments whose sums launch 2 keeps in LDS
constexpr int kHistBytes = 65536 * 2;
static_assert(kWavePieces * kWaves >= kPartPieces, "a part fits its waves");
static_assert((kSampleMaxVocab / kPiece + 2) / kPartPieces + 1 <= kMaxParts, "parts of the longest row");

// The workspace: counters of every part, then their segment bits, then their first places.
struct Parts {
  uint16_t* counts;  // [part][65536], segments without a bit are not written
  uint32_t* bits;    // [part][32]
  uint32_t* top;     // [part]: the first place that occurs
};

// The place of a bf16 value among all, largest first: +inf at 0x7f, -inf at 0xff80, 0 and -0 at
// 0x7fff; NaN lands before or behind them.
constexpr uint32_t kInfPlace = 0x7fu, kNegInfPlace = 0xff80u;
__device__ __forceinline__ uint32_t place_of(uint32_t b) {
  const uint32_t d = b ^ (b & 0x8000u ? 0u : 0x7fffu);
  return d == 0x8000u ? 0x7fffu : d;
}
__device__ __forceinline__ float value_at(uint32_t place) {
  return bf16_to_f32(uint16_t(place & 0x8000u ? place : place ^ 0x7fffu));
}

// e^x for x <= 0 in 64 bits: x = n ln 2 + r, the series of e^r to r^13 / 13!
// (|r| <= ln 2 / 2: 2e-17 of it is left out), scaled by 2^n.  0 below the
// smallest double, and for NaN; exactly 1 at 0.
__device__ __forceinline__ double weight_of(double x) {
  const double n = __builtin_rint(x * 1.4426950408889634074);
  double r = __builtin_fma(-n, 0x1.62e42ff000000p-1, x);  // ln 2 to 32 bits: n times it is exact
  r = __builtin_fma(-n, -0x1.718432a1b0e26p-35, r);         // and the rest
  double p = 1.6059043836821613e-10;  // 1 / 13!
  p = __builtin_fma(p, r, 2.0876756987868099e-09);
  p = __builtin_fma(p, r, 2.5052108385441720e-08);
  p = __builtin_fma(p, r, 2.7557319223985893e-07);
  p = __builtin_fma(p, r, 2.7557319223985888e-06);
  p = __builtin_fma(p, r, 2.4801587301587302e-05);
  p = __builtin_fma(p, r, 1.9841269841269841e-04);
  p = __builtin_fma(p, r, 1.3888888888888889e-03);
  p = __builtin_fma(p, r, 8.3333333333333332e-03);
  p = __builtin_fma(p, r, 4.1666666666666664e-02);
  p = __builtin_fma(p, r, 1.6666666666666666e-01);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return x > -746.0 ? __builtin_ldexp(p, int(n)) : 0.0;
}

// Sums over the lanes up to each one (all 64 lanes active), in registers.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t shifted(uint32_t v) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROWS, 0xf, true));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double shifted(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = shifted<CTRL, ROWS>(uint32_t(u)), hi = shifted<CTRL, ROWS>(uint32_t(u >> 32));
  return __builtin_bit_cast(double, lo | hi << 32);
}
template <class T>
__device__ __forceinline__ T scan(T v) {
  v += shifted<0x111, 0xf>(v);  // from 1, 2, 4, 8 lanes below in the row of 16
  v += shifted<0x112, 0xf>(v);
  v += shifted<0x114, 0xf>(v);
  v += shifted<0x118, 0xf>(v);
  v += shifted<0x142, 0xa>(v);  // rows 0 and 2 to rows 1 and 3
  v += shifted<0x143, 0xc>(v);  // the first two rows to the others
  return v;
}
// The largest of the lanes up to each one (none negative).
__device__ __forceinline__ double scan_max(double v) {
  v = fmax(v, shifted<0x111, 0xf>(v));
  v = fmax(v, shifted<0x112, 0xf>(v));
  v = fmax(v, shifted<0x114, 0xf>(v));
  v = fmax(v, shifted<0x118, 0xf>(v));
  v = fmax(v, shifted<0x142, 0xa>(v));
  v = fmax(v, shifted<0x143, 0xc>(v));
  return v;
}
__device__ __forceinline__ uint32_t at_lane(uint32_t v, int l) {
  return uint32_t(__builtin_amdgcn_readlane(int(v), l));
}
__device__ __forceinline__ double at_lane(double v, int l) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, uint64_t(at_lane(uint32_t(u), l)) |
                                        uint64_t(at_lane(uint32_t(u >> 32), l)) << 32);
}

// A row in blocks of eight at 16-byte borders: block b holds tokens 8 b - lead .. + 7.
struct Row {
  const uint16_t* x;
  int n, lead;
  __device__ Row(const uint16_t* p, int n_)
      : x(p), n(n_), lead(int((reinterpret_cast<uintptr_t>(p) & 15) >> 1)) {}
  __device__ __forceinline__ int pieces() const { return (n + lead + kPiece - 1) / kPiece; }
  __device__ __forceinline__ int first(int piece, int lane) const {
    return piece * kPiece + 8 * lane - lead;
  }
  // the lane's eight tokens of a piece; those outside the row are -inf
  __device__ __forceinline__ uint4 load(int piece, int lane) const {
    const int at = first(piece, lane);
    if (at >= 0 && at + 8 <= n) return *reinterpret_cast<const uint4*>(x + at);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = at + 2 * j;
      const uint32_t lo = i >= 0 && i < n ? x[i] : 0xff80u;
      const uint32_t hi = i + 1 >= 0 && i + 1 < n ? x[i + 1] : 0xff80u;
      w[j] = lo | hi << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
__device__ __forceinline__ uint32_t token_of(const uint4& v, int j) {
  const uint32_t w = j < 2 ? v.x : j < 4 ? v.y : j < 6 ? v.z : v.w;
  return j & 1 ? w >> 16 : w & 0xffffu;
}

// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kThreads) void count_kernel(const uint16_t* __restrict__ logits,
                                                         int64_t stride, int n, int parts,
                                                         Parts ws) {
  extern __shared__ __align__(16) uint32_t hist[];  // 32768 words, two counters each
  __shared__ uint32_t bits[32], top;
  const int row = blockIdx.x / parts, part = blockIdx.x % parts;
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const Row r(logits + int64_t(row) * stride, n);
  const int each = (r.pieces() + parts - 1) / parts;
  const int p0 = part * each, p1 = min(r.pieces(), p0 + each);
  uint4 v[kWavePieces];
#pragma unroll
  for (int i = 0; i < kWavePieces; ++i)
    if (p0 + wave + kWaves * i < p1) v[i] = r.load(p0 + wave + kWaves * i, lane);
  for (int i = t; i < 32768 / 4; i += kThreads)
    reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
  if (t < 32) bits[t] = 0;
  if (t == 32) top = 0xffffu;
  __syncthreads();
  uint32_t least = 0xffffu;
#pragma unroll
  for (int i = 0; i < kWavePieces; ++i)
    if (p0 + wave + kWaves * i < p1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t d = place_of(token_of(v[i], j));
        const bool counts = d - kInfPlace < kNegInfPlace - kInfPlace;  // not NaN, not -inf
        least = min(least, counts ? d : 0xffffu);
        if (counts) atomicAdd(&hist[d >> 1], d & 1 ? 0x10000u : 1u);
      }
    }
  for (int o = 32; o > 0; o >>= 1) least = min(least, uint32_t(__shfl_xor(int(least), o, 64)));
  if (lane == 0) atomicMin(&top, least);
  __syncthreads();
  // eight counters a lane, eight lanes a segment
  uint16_t* counts = ws.counts + int64_t(blockIdx.x) * 65536;
#pragma unroll
  for (int i = 0; i < kSegments / 8 / kWaves; ++i) {
    const int at = (kWaves * i + wave) * 64 + lane;  // in sixteen bytes
    const uint4 c = reinterpret_cast<const uint4*>(hist)[at];
    const uint64_t some = __ballot((c.x | c.y | c.z | c.w) != 0);
    if (some >> (lane & 56) & 255) {
      reinterpret_cast<uint4*>(counts)[at] = c;
      if ((lane & 7) == 0) atomicOr(&bits[at >> 8], 1u << (at >> 3 & 31));
    }
  }
  __syncthreads();
  if (t < 32) ws.bits[int64_t(blockIdx.x) * 32 + t] = bits[t];
  if (t == 32) ws.top[blockIdx.x] = top;
}

// ---------------------------------------------------------------------------
constexpr int kNone = 0xffff;
struct Shared {
  double mass[kSegments];  // of the segment, then of all up to and with it
  uint32_t count[kSegments];
  uint16_t slot[kSegments];  // its place among the occurring segments, kNone where it does not occur
  uint16_t list[kSegments];  // the occurring segments
  uint32_t bits[kMaxParts * 32];
  double wmass[kWaves];
  uint32_t wcount[kWaves];
  uint32_t pieces[kPartPieces + 1];
  uint32_t top, above;
  uint32_t chosen, rank, part;
};

__global__ __launch_bounds__(kThreads) void choose_kernel(
    const uint16_t* __restrict__ logits, int64_t stride, int n, int parts, Parts ws,
    const float* __restrict__ temperature, const int32_t* __restrict__ top_k,
    const float* __restrict__ top_p, const float* __restrict__ min_p,
    const float* __restrict__ uniform, uint32_t* __restrict__ tokens, float* __restrict__ logprob,
    int32_t* __restrict__ kept) {
  extern __shared__ __align__(16) uint32_t sums[];  // [kSlots][64]
  __shared__ Shared sh;
  const int row = blockIdx.x, t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const uint16_t* counts = ws.counts + int64_t(row) * parts * 65536;
  for (int i = t; i < parts * 32; i += kThreads) sh.bits[i] = ws.bits[int64_t(row) * parts * 32 + i];
  if (wave == kWaves - 1) {
    uint32_t first = lane < parts ? ws.top[int64_t(row) * parts + lane] : 0xffffu;
    for (int o = 32; o > 0; o >>= 1) first = min(first, uint32_t(__shfl_xor(int(first), o, 64)));
    if (lane == 0) {
      sh.top = first;
      sh.above = 0;
    }
  }
  // the row's settings, on their way during the first steps
  const float temp = temperature ? temperature[row] : 1.0f;
  const int32_t k = top_k ? top_k[row] : 0;
  const float p = top_p ? top_p[row] : 1.0f, mp = min_p ? min_p[row] : 0.0f;
  const float u = uniform[row];
  __syncthreads();
  const uint32_t top = sh.top;
  if (top >= kNegInfPlace) {  // uniform: nothing exceeds -inf
    if (t == 0) {
      tokens[row] = 0;
      if (kept) kept[row] = 0;
      if (logprob) logprob[row] = u2f(0xff800000u);
    }
    return;
  }
  const bool greedy = !(temp > 0.0f);
  const double lmax = double(value_at(top)), per_t = greedy ? 1.0 : 1.0 / double(temp);
  auto weight = [&](uint32_t place) {
    if (place == top) return 1.0;
    return weight_of((double(value_at(place)) - lmax) * per_t);  // 0 also where both are infinite
  };
  // lane's counter of a segment over all parts (of one that found no room in LDS)
  auto gather = [&](int seg) {
    uint32_t c = 0;
    for (int i = 0; i < parts; ++i)
      if (sh.bits[i * 32 + (seg >> 5)] >> (seg & 31) & 1)
        c += counts[int64_t(i) * 65536 + seg * 64 + lane];
    return c;
  };

  if (!greedy) {
    {  // the list of occurring segments, in order
      uint32_t a = 0;
      for (int i = 0; i < parts; ++i) a |= sh.bits[i * 32 + (t >> 5)];
      const bool here = a >> (t & 31) & 1;
      const uint64_t m = __ballot(here);
      if (lane == 0) sh.wcount[wave] = uint32_t(__builtin_popcountll(m));
      sh.mass[t] = 0.0;
      sh.count[t] = 0;
      __syncthreads();
      uint32_t at = uint32_t(__builtin_popcountll(m & ((1ull << lane) - 1)));
      for (int w = 0; w < wave; ++w) at += sh.wcount[w];
      sh.slot[t] = here ? uint16_t(at) : uint16_t(kNone);
      if (here) sh.list[at] = uint16_t(t);
      if (t == kThreads - 1) sh.pieces[0] = at + here;
      __syncthreads();
    }
    const int occurring = int(sh.pieces[0]);
    const double floor_w = mp > 0.0f ? double(mp) : 0.0;
    uint32_t above = 0;
    // four segments a wave, a row of 16 lanes each, four counters a lane; the next four's
    // counters of the first eight parts are requested before this four's are weighed
    const int four = 4 * (lane & 15);
    auto request = [&](int at, int first, uint2* v) {
      const int seg = at < occurring ? sh.list[at] : -1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = make_uint2(0, 0);
        if (seg >= 0 && first + i < parts &&
            (sh.bits[(first + i) * 32 + (seg >> 5)] >> (seg & 31) & 1))
          v[i] = *reinterpret_cast<const uint2*>(counts + int64_t(first + i) * 65536 + seg * 64 + four);
      }
    };
    uint2 v[8];
    request(4 * wave + (lane >> 4), 0, v);
    for (int s0 = 4 * wave; s0 < occurring; s0 += 4 * kWaves) {
      const int at = s0 + (lane >> 4);
      uint32_t c[4] = {0, 0, 0, 0};
      auto add = [&]() {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          c[0] += v[i].x & 0xffffu;
          c[1] += v[i].x >> 16;
          c[2] += v[i].y & 0xffffu;
          c[3] += v[i].y >> 16;
        }
      };
      add();
      for (int first = 8; first < parts; first += 8) {
        request(at, first, v);
        add();
      }
      request(at + 4 * kWaves, 0, v);
      const bool here = at < occurring;
      const int seg = here ? sh.list[at] : 0;
      if (here && at < kSlots)
        *reinterpret_cast<uint4*>(sums + at * 64 + four) = make_uint4(c[0], c[1], c[2], c[3]);
      double m = 0.0;
      uint32_t n_in = 0, a = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c[i]) {
          const double w = weight(uint32_t(seg) * 64 + four + i);
          m += double(c[i]) * w;
          n_in += w > 0.0 ? c[i] : 0;
          a += w > 0.0 && w >= floor_w ? c[i] : 0;
        }
      for (int o = 8; o > 0; o >>= 1) {
        m += __shfl_xor(m, o, 64);
        n_in += __shfl_xor(n_in, o, 64);
        a += __shfl_xor(a, o, 64);
      }
      if (here && (lane & 15) == 0) {
        sh.mass[seg] = m;
        sh.count[seg] = n_in;
        above += a;
      }
    }
    if ((lane & 15) == 0 && above) atomicAdd(&sh.above, above);
    __syncthreads();
    // Prefixes over the segments.  Rounding depends on the order of a sum, which differs from lane to
    // lane in the scan: only the prefixes of occurring segments count, each raised to the largest
    // before it, and the waves' totals add up one after another.  So the prefixes never fall and an
    // empty segment has exactly its predecessor's: the first to pass a bound is one with tokens.
    const uint32_t c_own = sh.count[t];
    double m_in = scan(sh.mass[t]);
    m_in = scan_max(c_own ? m_in : 0.0);
    uint32_t c_in = scan(c_own);
    if (lane == 63) {
      sh.wmass[wave] = m_in;
      sh.wcount[wave] = c_in;
    }
    __syncthreads();
    const double m_w = lane < kWaves ? sh.wmass[lane] : 0.0;
    const uint32_t c_w = scan(lane < kWaves ? sh.wcount[lane] : 0u);
    double m_before = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves - 1; ++w) m_before += w < wave ? at_lane(m_w, w) : 0.0;
    m_in += m_before;
    if (wave > 0) c_in += at_lane(c_w, wave - 1);
    sh.mass[t] = m_in;
    sh.count[t] = c_in;
    __syncthreads();
    if (wave == 0) {
      const double m_all = sh.mass[kSegments - 1];
      const uint32_t c_all = sh.count[kSegments - 1];
      // the first segment whose prefix passes (the last with tokens where none does): over every
      // 16th segment, then within sixteen
      auto find = [&](auto&& passes) {
        uint64_t b = __ballot(passes(16 * lane + 15));
        if (!b) b = __ballot(sh.count[16 * lane + 15] >= c_all);
        const int base = 16 * __builtin_ctzll(b);
        b = __ballot(lane < 16 && passes(base + (lane & 15)));
        if (!b) b = __ballot(lane < 16 && sh.count[base + (lane & 15)] >= c_all);
        return base + (b ? __builtin_ctzll(b) : 15);
      };
      uint32_t c = 0, ci = 0;  // of the open segment: the lane's counter, and up to it
      double w = 0.0, mi = 0.0;
      auto open = [&](int seg) {
        const int s = sh.slot[seg];
        c = s == kNone ? 0 : s < kSlots ? sums[s * 64 + lane] : gather(seg);
        w = c ? weight(uint32_t(seg) * 64 + lane) : 0.0;
        c = w > 0.0 ? c : 0;
        ci = scan(c);
        mi = scan(double(c) * w);
        mi += seg ? sh.mass[seg - 1] : 0.0;
        ci += seg ? sh.count[seg - 1] : 0;
      };
      // the lane of the open segment that holds rank `want` (from 1), or the last with tokens
      auto lane_of = [&](uint64_t past) {
        if (!past) past = 1ull << (63 - __builtin_clzll(__ballot(c != 0) | 1ull));
        return __builtin_amdgcn_readfirstlane(__builtin_ctzll(past));
      };
      // the mass of the first `want` tokens (1 <= want <= c_all)
      auto mass_of = [&](uint32_t want) {
        if (want >= c_all) return m_all;
        open(find([&](int s) { return sh.count[s] >= want; }));
        const int f = lane_of(__ballot(ci >= want));
        const uint32_t over = at_lane(ci, f) - want;  // tokens of the value past the rank
        return at_lane(mi, f) - double(over) * at_lane(w, f);
      };
      uint32_t keep = c_all;
      if (k > 0 && uint32_t(k) < keep) keep = uint32_t(k);
      double mass = mass_of(keep);
      const uint32_t first = keep;
      if (p <= 0.0f) {
        keep = 1;
      } else if (p < 1.0f) {
        const double target = double(p) * mass;
        open(find([&](int s) { return sh.mass[s] >= target; }));
        const int f = lane_of(__ballot(mi >= target && c != 0));
        const uint32_t cf = at_lane(c, f);
        const double wf = at_lane(w, f);
        const double before = at_lane(mi, f) - double(cf) * wf;
        double q = __builtin_ceil((target - before) / wf);
        q = q < 1.0 ? 1.0 : (q > double(cf) ? double(cf) : q);
        keep = min(keep, at_lane(ci, f) - cf + uint32_t(q));
      }
      if (floor_w > 0.0) keep = min(keep, sh.above);
      keep = max(keep, 1u);
      if (keep != first) mass = mass_of(keep);
      const double at = (u > 0.0f ? (u < 1.0f ? double(u) : 1.0) : 0.0) * mass;
      int seg = find([&](int s) { return sh.mass[s] > at; });
      open(seg);
      int f = lane_of(__ballot(mi > at && c != 0));
      uint32_t cf = at_lane(c, f);
      double wf = at_lane(w, f);
      const double before = at_lane(mi, f) - double(cf) * wf;
      double q = __builtin_floor((at - before) / wf);
      q = q < 0.0 ? 0.0 : (q > double(cf - 1) ? double(cf - 1) : q);
      uint32_t rank = uint32_t(q);  // among the value's tokens
      // all of the mass, or a rounding past the last kept token: that token
      if (u >= 1.0f || at_lane(ci, f) - cf + rank >= keep) {
        seg = find([&](int s) { return sh.count[s] >= keep; });
        open(seg);
        f = lane_of(__ballot(ci >= keep));
        cf = at_lane(c, f);
        wf = at_lane(w, f);
        rank = keep - 1 - (at_lane(ci, f) - cf);
      }
      if (lane == 0) {
        sh.chosen = uint32_t(seg) * 64 + f;
        sh.rank = rank;
        if (kept) kept[row] = int32_t(keep);
        if (logprob) logprob[row] = float(log(wf / mass));
      }
    }
  } else if (t == 0) {
    sh.chosen = top;
    sh.rank = 0;
    if (kept) kept[row] = 1;
    if (logprob) logprob[row] = 0.0f;
  }
  // the part that holds the rank-th of the value's tokens (ids in order)
  if (wave == 0) {
    wave_sync();
    const uint32_t d = sh.chosen, seg = d >> 6, rank = sh.rank;
    uint32_t c = 0;
    if (lane < parts && (sh.bits[lane * 32 + (seg >> 5)] >> (seg & 31) & 1))
      c = counts[int64_t(lane) * 65536 + d];
    const uint32_t sum = scan(c);
    const int f = __builtin_ctzll(__ballot(sum > rank) | (1ull << 63));
    const uint32_t before = at_lane(sum, f) - at_lane(c, f);
    if (lane == 0) {
      sh.part = min(uint32_t(f), uint32_t(parts - 1));
      sh.rank = rank - before;
    }
  }
  __syncthreads();
  const uint32_t place = sh.chosen, rank = sh.rank;
  const Row r(logits + int64_t(row) * stride, n);
  const int each = (r.pieces() + parts - 1) / parts;
  const int p0 = int(sh.part) * each, np = min(r.pieces(), p0 + each) - p0;
  // matches of every piece, which its wave keeps
  uint4 v[kWavePieces];
#pragma unroll
  for (int i = 0; i < kWavePieces; ++i)
    if (wave + kWaves * i < np) v[i] = r.load(p0 + wave + kWaves * i, lane);
#pragma unroll
  for (int i = 0; i < kWavePieces; ++i) {
    if (wave + kWaves * i >= np) continue;
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) c += place_of(token_of(v[i], j)) == place;
    c = at_lane(scan(c), 63);
    if (lane == 0) sh.pieces[wave + kWaves * i] = c;
  }
  __syncthreads();
  // the piece that holds it: two a lane
  const uint32_t a = 2 * lane < np ? sh.pieces[2 * lane] : 0;
  const uint32_t b = 2 * lane + 1 < np ? sh.pieces[2 * lane + 1] : 0;
  const uint32_t sum = scan(a + b);
  const uint64_t past = __ballot(sum > rank);
  if (!past) return;  // unreachable: the part's counters say that it is there
  const int f = __builtin_ctzll(past);
  uint32_t before = at_lane(sum, f) - at_lane(a + b, f);
  const uint32_t af = at_lane(a, f);
  const int piece = before + af > rank ? 2 * f : 2 * f + 1;
  if (piece & 1) before += af;
#pragma unroll
  for (int i = 0; i < kWavePieces; ++i) {
    if (piece != wave + kWaves * i) continue;  // uniform: one wave's one piece
    uint32_t own = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) own += place_of(token_of(v[i], j)) == place;
    const uint32_t upto = scan(own);
    uint32_t at = before + upto - own;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (place_of(token_of(v[i], j)) == place) {
        if (at == rank) tokens[row] = uint32_t(r.first(p0 + piece, lane) + j);
        ++at;
      }
  }
}

// Parts of a row: enough workgroups for few rows, but no more than eight (launch 2
// adds them up: at 151936 tokens it would then take as long as launch 1 saves), and
// few enough tokens for 16-bit counters.
int sample_parts(int rows, int n) {
  const int pieces = (n + 7 + kPiece - 1) / kPiece;
  const int least = (pieces + kPartPieces - 1) / kPartPieces;
  int p = rows < 32 ? 8 : 256 / rows;
  p = p < pieces / 4 ? p : pieces / 4;
  p = p < 1 ? 1 : p;
  return p > least ? p : least;
}
int sample_batch(int rows, int parts) {
  const int b = kBatchParts / parts;
  return rows < b ? rows : b;
}

}  // namespace

// For any call of at most `rows` rows of at most n tokens.  Fewer rows are cut into more parts, so
// that 32 rows may need more than 33: the most that any number of rows gives (parts of a longer row
// are never fewer).
size_t sample_workspace(int rows, int n) {
  int64_t most = 0;  // parts of a batch
  for (int r = 1; r <= rows && r <= kBatchParts; ++r) {
    const int64_t all = int64_t(r) * sample_parts(r, n);
    most = all > most ? all : most;
  }
  return size_t(most < kBatchParts ? most : kBatchParts) * (kHistBytes + 32 * 4 + 4);
}

int sample_bf16(const uint16_t* logits, int64_t stride, int rows, int n, const float* temperature,
                const int32_t* top_k, const float* top_p, const float* min_p,
                const float* uniform, uint32_t* tokens, float* logprob, int32_t* kept,
                void* workspace, hipStream_t s) {
  const int parts = sample_parts(rows, n), batch = sample_batch(rows, parts);
  Parts ws;
  ws.counts = static_cast<uint16_t*>(workspace);
  ws.bits = reinterpret_cast<uint32_t*>(ws.counts + size_t(batch) * parts * 65536);
  ws.top = ws.bits + size_t(batch) * parts * 32;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(count_kernel),
                          hipFuncAttributeMaxDynamicSharedMemorySize, kHistBytes) != hipSuccess ||
      hipFuncSetAttribute(reinterpret_cast<const void*>(choose_kernel),
                          hipFuncAttributeMaxDynamicSharedMemorySize,
                          kSlots * 256) != hipSuccess)
    return MX_EHIP;
  // batches one after another on the stream share the workspace
  for (int r = 0; r < rows; r += batch) {
    const int m = rows - r < batch ? rows - r : batch;
    const uint16_t* x = logits + int64_t(r) * stride;
    hipLaunchKernelGGL(count_kernel, dim3(m * parts), dim3(kThreads), kHistBytes, s, x, stride, n,
                       parts, ws);
    if (hipGetLastError() != hipSuccess) return MX_EHIP;
    hipLaunchKernelGGL(choose_kernel, dim3(m), dim3(kThreads), kSlots * 256, s, x, stride, n,
                       parts, ws, temperature ? temperature + r : nullptr,
                       top_k ? top_k + r : nullptr, top_p ? top_p + r : nullptr,
                       min_p ? min_p + r : nullptr, uniform + r, tokens + r,
                       logprob ? logprob + r : nullptr, kept ? kept + r : nullptr);
    if (hipGetLastError() != hipSuccess) return MX_EHIP;
  }
  return MX_OK;
}

}  // namespace mx
