// Sampling from bf16 logits with temperature, top-k, top-p and min-p.
//
// Tokens are ordered by logit, largest first, lowest id first among equals; with
// w_j = exp((l_j - l_0) / T) every filter keeps a prefix of that order:
//   top-k  the first k
//   top-p  the shortest prefix with a mass of at least p times the first k's
//   min-p  those with w_j >= min_p
// n is the shortest of them (at least one token), and the sampled token is the
// first whose prefix mass exceeds u times the mass of n.
//
// bf16 has 65536 values, so a row is known by how often each occurs: one
// workgroup counts them in LDS (16-bit counters, 128 KB) and needs an
// exponential per occurring value instead of one per token.  Counts are exact
// and masses are sums of few products in 64 bits, so neither the order of the
// atomics nor the launch shape can change a token, and a u next to a border
// falls on the side that the definition says.
//
// Counters are cut into 1024 segments of 64 neighbouring values.  Each gets its
// count and mass, one scan over the workgroup's threads gives the prefixes, and
// every question (which value holds rank k, which holds mass x) is a search over
// segments and then over one segment's 64 values by a wave.  The rank within the
// value's tokens then picks the id, by counts of matches per 512 tokens.
//
// A row of one value that occurs over 65535 times does not fit 16-bit counters;
// the sum of all counters shows it (a carry or a wrap only ever loses), and such a
// row is counted again with 32-bit counters, half the values at a time.
#include "common.hpp"
#include "kernels.hpp"

namespace mx {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kSegments = 1024;
constexpr int kPiece = 512;  // tokens of one wave's step: eight a lane
constexpr int kHistBytes = 65536 * 2;

struct Shared {
  double mass[kSegments];     // of the segment, then of all before it
  uint32_t count[kSegments];
  double wmass[kWaves];
  uint32_t wcount[kWaves];
  uint32_t seg32[64];         // one segment's counters (32-bit rows)
  uint32_t pieces[kSampleMaxVocab / kPiece];
  int red[kWaves];
  int answer;
  uint32_t total, counted, above;
};

// bf16 bits as a 16-bit key that orders like the values; NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t key_of(uint32_t b) {
  b = (b & 0x7fffu) > 0x7f80u ? 0xff80u : b;
  b = b == 0x8000u ? 0u : b;
  return b & 0x8000u ? b ^ 0xffffu : b | 0x8000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return bf16_to_f32(uint16_t(key & 0x8000u ? key ^ 0x8000u : key ^ 0xffffu));
}
constexpr uint32_t kNegInfKey = 0x007fu;

// One row; a workgroup.
__global__ __launch_bounds__(kThreads) void sample_kernel(
    const uint16_t* __restrict__ logits, int64_t stride, int n,
    const float* __restrict__ temperature, const int32_t* __restrict__ top_k,
    const float* __restrict__ top_p, const float* __restrict__ min_p,
    const float* __restrict__ uniform, uint32_t* __restrict__ tokens, float* __restrict__ logprob,
    int32_t* __restrict__ kept) {
  extern __shared__ __align__(16) uint32_t hist[];  // 32768 words
  __shared__ Shared sh;
  const int row = blockIdx.x, t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const uint16_t* x = logits + int64_t(row) * stride;
  const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const int pieces = (n + kPiece - 1) / kPiece;

  // calls f(key, id) for every token of piece i, eight neighbouring ones a lane
  auto each_of = [&](int i, auto&& f) {
    const int at = i * kPiece + 8 * lane;
    if (aligned && at + 8 <= n) {
      const uint4 v = *reinterpret_cast<const uint4*>(x + at);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) f(key_of(j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu), at + j);
    } else {
      for (int j = 0; j < 8 && at + j < n; ++j) f(key_of(x[at + j]), at + j);
    }
  };

  // the largest key
  int best = 0;
  for (int i = wave; i < pieces; i += kWaves)
    each_of(i, [&](uint32_t k, int) { best = max(best, int(k)); });
  for (int o = 32; o > 0; o >>= 1) best = max(best, __shfl_xor(best, o, 64));
  if (lane == 0) sh.red[wave] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) best = max(best, sh.red[w]);
  const uint32_t top = uint32_t(best);
  if (top <= kNegInfKey) {  // uniform: nothing exceeds -inf
    if (t == 0) {
      tokens[row] = 0;
      if (kept) kept[row] = 0;
      if (logprob) logprob[row] = u2f(0xff800000u);
    }
    return;
  }
  const float temp = temperature ? temperature[row] : 1.0f;
  const bool greedy = !(temp > 0.0f);
  const double lmax = double(value_of(top)), td = greedy ? 1.0 : double(temp);
  // the weight of a key; keys without weight are no tokens
  auto weight = [&](uint32_t key) {
    if (key == top) return 1.0;
    if (key <= kNegInfKey) return 0.0;
    const double w = exp((double(value_of(key)) - lmax) / td);
    return w > 0.0 ? w : 0.0;  // also where both are infinite
  };

  uint32_t chosen = top, rank = 0;  // the value and the rank among its tokens
  if (!greedy) {
    // values that far below the largest weigh 0 even in 64 bits: not counted
    const double cut = lmax - 750.0 * td;
    uint32_t floor_key = kNegInfKey + 1;
    {
      float c = float(cut);
      c = c < -3.3e38f ? -3.4e38f : c;
      const uint32_t b = f2u(c) >> 16;  // towards 0 for negative c: above the cut or equal
      const uint32_t k = key_of(b & 0xffffu);
      if (c > -3.3e38f && k > kNegInfKey + 2) floor_key = k - 1;
    }
    const uint32_t span = min(top - floor_key + 1, 65536u);  // values counted

    auto clear = [&](int words) {
      for (int i = t; i < words / 4; i += kThreads)
        reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
    };
    // a segment's count and mass, from its counters by one wave
    auto reduce = [&](int seg, uint32_t c, double floor_w, uint32_t* above) {
      double m = 0.0;
      if (__ballot(c != 0)) {
        const uint32_t d = uint32_t(seg) * 64 + lane;
        const double w = c ? weight(top - d) : 0.0;
        c = w > 0.0 ? c : 0;
        m = double(c) * w;
        uint32_t a = w >= floor_w ? c : 0;
        for (int o = 32; o > 0; o >>= 1) {
          m += __shfl_xor(m, o, 64);
          c += __shfl_xor(c, o, 64);
          a += __shfl_xor(a, o, 64);
        }
        *above += a;
      }
      if (lane == 0) {
        sh.mass[seg] = m;
        sh.count[seg] = c;
      }
    };
    const float mp = min_p ? min_p[row] : 0.0f;
    const double floor_w = mp > 0.0f ? double(mp) : 0.0;

    // all values in 16-bit counters
    clear(32768);
    if (t == 0) sh.counted = sh.total = sh.above = 0;
    __syncthreads();
    uint32_t mine = 0;
    for (int i = wave; i < pieces; i += kWaves)
      each_of(i, [&](uint32_t k, int) {
        if (k >= floor_key) {
          const uint32_t d = top - k;
          atomicAdd(&hist[d >> 1], d & 1 ? 0x10000u : 1u);
          ++mine;
        }
      });
    for (int o = 32; o > 0; o >>= 1) mine += __shfl_xor(mine, o, 64);
    if (lane == 0) atomicAdd(&sh.counted, mine);
    __syncthreads();
    uint32_t above = 0, sum = 0;
    for (int seg = wave; seg < kSegments; seg += kWaves) {
      const uint32_t c =
          seg * 64 < int(span) ? reinterpret_cast<const uint16_t*>(hist)[seg * 64 + lane] : 0;
      sum += c;
      reduce(seg, c, floor_w, &above);
    }
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) {
      atomicAdd(&sh.total, sum);
      atomicAdd(&sh.above, above);
    }
    __syncthreads();
    const bool wide = sh.total != sh.counted;  // uniform
    if (wide) {
      __syncthreads();
      if (t == 0) sh.above = 0;
      above = 0;
      for (int half = 0; half < 2; ++half) {
        __syncthreads();
        clear(32768);
        __syncthreads();
        for (int i = wave; i < pieces; i += kWaves)
          each_of(i, [&](uint32_t k, int) {
            const uint32_t d = top - k;
            if (k >= floor_key && int(d >> 15) == half) atomicAdd(&hist[d & 32767], 1u);
          });
        __syncthreads();
        for (int seg = wave; seg < kSegments / 2; seg += kWaves)
          reduce(512 * half + seg, hist[seg * 64 + lane], floor_w, &above);
      }
      if (lane == 0) atomicAdd(&sh.above, above);
      __syncthreads();
    }
    // prefixes over the segments
    double m_in = sh.mass[t];
    uint32_t c_in = sh.count[t];
    const uint32_t c_own = c_in;
    for (int o = 1; o < 64; o <<= 1) {
      const double m = __shfl_up(m_in, o, 64);
      const uint32_t c = __shfl_up(c_in, o, 64);
      if (lane >= o) {
        m_in += m;
        c_in += c;
      }
    }
    if (lane == 63) {
      sh.wmass[wave] = m_in;
      sh.wcount[wave] = c_in;
    }
    __syncthreads();
    double m_all = 0.0;
    uint32_t c_all = 0;
    for (int w = 0; w < kWaves; ++w) {
      if (w == wave) {
        m_in += m_all;
        c_in += c_all;
      }
      m_all += sh.wmass[w];
      c_all += sh.wcount[w];
    }
    // A segment starts where the one before it ends, in the same bits.
    sh.mass[t] = m_in;
    sh.count[t] = c_in;
    __syncthreads();
    const double m_before = t ? sh.mass[t - 1] : 0.0;
    const uint32_t c_before = t ? sh.count[t - 1] : 0;

    // the segment whose thread says so (the last with tokens, where none does)
    auto find = [&](bool here) {
      __syncthreads();
      if (t == 0) sh.answer = -1;
      __syncthreads();
      if (here) atomicMax(&sh.answer, t);
      __syncthreads();
      int a = sh.answer;
      if (a < 0) {
        __syncthreads();
        if (c_own) atomicMax(&sh.answer, t);
        __syncthreads();
        a = sh.answer;
      }
      return a;
    };
    // lane's counter and weight of segment seg
    auto open = [&](int seg, uint32_t* c, double* w) {
      if (!wide) {
        *c = seg * 64 < int(span) ? reinterpret_cast<const uint16_t*>(hist)[seg * 64 + lane] : 0;
      } else {
        __syncthreads();
        if (t < 64) sh.seg32[t] = 0;
        __syncthreads();
        for (int i = wave; i < pieces; i += kWaves)
          each_of(i, [&](uint32_t k, int) {
            const uint32_t d = top - k;
            if (k >= floor_key && int(d >> 6) == seg) atomicAdd(&sh.seg32[d & 63], 1u);
          });
        __syncthreads();
        *c = sh.seg32[lane];
      }
      *w = *c ? weight(top - (uint32_t(seg) * 64 + lane)) : 0.0;
      *c = *w > 0.0 ? *c : 0;
    };
    // counts and masses of the segment's values up to and with the lane's own
    auto prefix = [&](int seg, uint32_t c, double w, uint32_t* ci, double* mi) {
      *ci = c;
      *mi = double(c) * w;
      for (int o = 1; o < 64; o <<= 1) {
        const double m = __shfl_up(*mi, o, 64);
        const uint32_t k = __shfl_up(*ci, o, 64);
        if (lane >= o) {
          *mi += m;
          *ci += k;
        }
      }
      *mi += seg ? sh.mass[seg - 1] : 0.0;
      *ci += seg ? sh.count[seg - 1] : 0;
    };
    // the mass of the first `want` tokens (1 <= want <= c_all)
    auto mass_of = [&](uint32_t want) {
      if (want >= c_all) return m_all;
      const int seg = find(c_before < want && want <= c_in);
      uint32_t c, ci;
      double w, mi;
      open(seg, &c, &w);
      prefix(seg, c, w, &ci, &mi);
      const int f = __builtin_ctzll(__ballot(ci >= want) | (1ull << 63));
      const uint32_t left = want - (__shfl(ci, f, 64) - __shfl(c, f, 64));
      return __shfl(mi, f, 64) - double(__shfl(c, f, 64) - left) * __shfl(w, f, 64);
    };
    uint32_t keep = c_all;
    const int32_t k = top_k ? top_k[row] : 0;
    if (k > 0 && uint32_t(k) < keep) keep = uint32_t(k);
    double mass = mass_of(keep);
    const float p = top_p ? top_p[row] : 1.0f;
    bool changed = false;
    if (p <= 0.0f) {
      keep = 1;
      changed = true;
    } else if (p < 1.0f) {
      const double target = double(p) * mass;
      const int seg = find(m_before < target && target <= m_in);
      uint32_t c, ci;
      double w, mi;
      open(seg, &c, &w);
      prefix(seg, c, w, &ci, &mi);
      uint64_t past = __ballot(mi >= target && c != 0);
      if (!past) past = 1ull << (63 - __builtin_clzll(__ballot(c != 0) | 1ull));
      const int f = __builtin_ctzll(past);
      const uint32_t cf = __shfl(c, f, 64);
      const double wf = __shfl(w, f, 64);
      const double before = __shfl(mi, f, 64) - double(cf) * wf;
      double q = __builtin_ceil((target - before) / wf);
      q = q < 1.0 ? 1.0 : (q > double(cf) ? double(cf) : q);
      const uint32_t np = __shfl(ci, f, 64) - cf + uint32_t(q);
      if (np < keep) {
        keep = np;
        changed = true;
      }
    }
    const uint32_t least = sh.above;
    if (floor_w > 0.0 && least < keep) {
      keep = least;
      changed = true;
    }
    if (keep < 1) {
      keep = 1;
      changed = true;
    }
    if (changed) mass = mass_of(keep);
    const float u = uniform[row];
    const double at = (u > 0.0f ? (u < 1.0f ? double(u) : 1.0) : 0.0) * mass;
    const int seg = find(m_before <= at && at < m_in);
    uint32_t c, ci;
    double w, mi;
    open(seg, &c, &w);
    prefix(seg, c, w, &ci, &mi);
    uint64_t past = __ballot(mi > at && c != 0);
    if (!past) past = 1ull << (63 - __builtin_clzll(__ballot(c != 0) | 1ull));
    int f = __builtin_ctzll(past);
    const uint32_t cf = __shfl(c, f, 64);
    const double wf = __shfl(w, f, 64);
    const double before = __shfl(mi, f, 64) - double(cf) * wf;
    double q = __builtin_floor((at - before) / wf);
    q = q < 0.0 ? 0.0 : (q > double(cf - 1) ? double(cf - 1) : q);
    uint32_t place = __shfl(ci, f, 64) - cf + uint32_t(q);  // among all tokens
    double wt = wf;
    uint32_t value = top - (uint32_t(seg) * 64 + f);
    rank = uint32_t(q);
    if (place >= keep) {  // a rounding past the last kept token
      const int s2 = find(c_before < keep && keep <= c_in);
      open(s2, &c, &w);
      prefix(s2, c, w, &ci, &mi);
      f = __builtin_ctzll(__ballot(ci >= keep) | (1ull << 63));
      rank = keep - 1 - (__shfl(ci, f, 64) - __shfl(c, f, 64));
      wt = __shfl(w, f, 64);
      value = top - (uint32_t(s2) * 64 + f);
    }
    chosen = value;
    if (t == 0) {
      if (kept) kept[row] = int32_t(keep);
      if (logprob) logprob[row] = float(log(wt / mass));
    }
  } else if (t == 0) {
    if (kept) kept[row] = 1;
    if (logprob) logprob[row] = 0.0f;
  }

  // the id of the chosen value's rank-th token: matches per piece, then within one
  __syncthreads();
  for (int i = wave; i < pieces; i += kWaves) {
    int c = 0;
    each_of(i, [&](uint32_t k, int) { c += k == chosen; });
    for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
    if (lane == 0) sh.pieces[i] = uint32_t(c);
  }
  __syncthreads();
  if (wave != 0) return;
  uint32_t before = 0;
  for (int i0 = 0; i0 < pieces; i0 += 64) {
    const uint32_t c = i0 + lane < pieces ? sh.pieces[i0 + lane] : 0;
    uint32_t sum = c;
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t v = __shfl_up(sum, o, 64);
      sum += lane >= o ? v : 0;
    }
    const uint64_t past = __ballot(before + sum > rank);
    if (!past) {
      before += __shfl(sum, 63, 64);
      continue;
    }
    const int f = __builtin_ctzll(past);
    before += __shfl(sum, f, 64) - __shfl(c, f, 64);
    uint32_t own = 0;
    each_of(i0 + f, [&](uint32_t k, int) { own += k == chosen; });
    uint32_t mine = own;
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t v = __shfl_up(mine, o, 64);
      mine += lane >= o ? v : 0;
    }
    uint32_t at = before + mine - own;
    each_of(i0 + f, [&](uint32_t k, int id) {
      if (k == chosen) {
        if (at == rank) tokens[row] = uint32_t(id);
        ++at;
      }
    });
    return;
  }
}

}  // namespace

size_t sample_workspace(int, int) { return 0; }

int sample_bf16(const uint16_t* logits, int64_t stride, int rows, int n, const float* temperature,
                const int32_t* top_k, const float* top_p, const float* min_p,
                const float* uniform, uint32_t* tokens, float* logprob, int32_t* kept, void*,
                hipStream_t s) {
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(sample_kernel),
                          hipFuncAttributeMaxDynamicSharedMemorySize, kHistBytes) != hipSuccess)
    return MX_EHIP;
  hipLaunchKernelGGL(sample_kernel, dim3(rows), dim3(kThreads), kHistBytes, s, logits, stride, n,
                     temperature, top_k, top_p, min_p, uniform, tokens, logprob, kept);
  return hipGetLastError() == hipSuccess ? MX_OK : MX_EHIP;
}

}  // namespace mx
