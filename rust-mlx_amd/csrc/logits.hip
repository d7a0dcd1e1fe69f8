// Controls on logits before a token is chosen: penalties for tokens that a sequence holds already,
// biases, and masks.
//
// Of a row's token j, c the times that it occurs in the sequence's own output:
//   x = l_j;  where j occurs in prompt or output: x = x < 0 ? x repetition : x / repetition
//   x -= frequency c;  x -= presence where c > 0;  x += the row's bias of j
//   x = -inf where the row's mask does not allow j
// in fp32, rounded once to bf16.
//
// A workgroup takes kSeg tokens of one row.  It runs over the whole history and counts what falls into
// its tokens in LDS (whole numbers: the order of the counting does not show), the prompt's occurrences as
// the top bit, so no table of the vocabulary is kept between steps; then it changes its logits in one
// pass, eight a thread.  64 rows of 151936 with histories of up to 8192, 300 biases and every second row
// masked take 17.7 us (2.3 TB/s): chains of dependent reads, counts and barriers, two and a half rounds of
// workgroups of them, rather than bytes; so the first reads of the history and of the biases do not wait for
// their numbers (0.8 us).  Two eights of logits a thread, with half the threads, take 23.
// A token that the biases name twice takes the last entry: the largest index wins, whatever the
// order.
#include "kernels.hpp"
#include "paged_core.hpp"

namespace mx {

namespace {

using namespace pg;

constexpr uint32_t kInPrompt = 0x80000000u;

// Rows start at any element, histories at any word.
typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
typedef int32_t tokens4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ bool finite(float x) { return __builtin_fabsf(x) < u2f(0x7f800000u); }

// Where token j of a segment is counted: the first four of eight tokens in one half, the others in the
// other, so that the lanes' reads of 16 bytes lie side by side.
template <int kSeg>
__device__ __forceinline__ unsigned place_of(unsigned j) {
  return (j >> 3) * 4 + (j & 3) + (j & 4) * (kSeg / 8);
}

template <int kSeg>
__global__ __launch_bounds__(kSeg / 8) void control_kernel(const uint16_t* logits, int64_t stride,
                                                           int n, LogitsControls c, uint16_t* out,
                                                           int64_t out_stride, int segs) {
  constexpr int kThreads = kSeg / 8;    // eight logits each
  extern __shared__ uint32_t counts[];  // [kSeg], then with biases [kSeg] of 1 + an entry's index
  uint32_t* entry = counts + kSeg;
  const int t = threadIdx.x;
  const int row = blockIdx.x / segs, first = blockIdx.x % segs * kSeg;
  const int seq = c.tokens && c.seqs ? c.seqs[row] : row;
  const int count = min(kSeg, n - first);
  const uint16_t* src = logits + int64_t(row) * stride + first;
  uint16_t* dst = out + int64_t(row) * out_stride + first;
  const bool in_place = src == dst;  // then only what changes is touched
  // What follows from the row alone is on its way before the history is looked at.
  const int at = 8 * t;
  words4 raw = {0, 0, 0, 0};
  auto load = [&]() {
    if (at + 8 <= count) {
      raw = *reinterpret_cast<const words4*>(src + at);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i < count) raw[i / 2] |= uint32_t(src[at + i]) << (16 * (i & 1));
    }
  };
  if (!in_place) load();
  for (int i = 4 * t; i < kSeg; i += 4 * kThreads) {
    *reinterpret_cast<uint4*>(counts + i) = make_uint4(0, 0, 0, 0);
    if (c.bias_starts) *reinterpret_cast<uint4*>(entry + i) = make_uint4(0, 0, 0, 0);
  }
  const int state = c.masks ? (c.mask_rows ? c.mask_rows[row] : row) : -1;
  const uint8_t* allowed = unsigned(state) < unsigned(c.mask_states)
                               ? reinterpret_cast<const uint8_t*>(c.masks + state * c.mask_stride) + first / 8
                               : nullptr;
  const uint32_t open = allowed && at < count ? allowed[at / 8] : 0xffu;
  int b0 = 0, b1 = 0;
  if (c.bias_starts) {
    b0 = min(max(c.bias_starts[row], 0), c.bias_count);
    b1 = min(max(c.bias_starts[row + 1], b0), c.bias_count);
  }
  float rep = c.repetition ? c.repetition[row] : 0.0f;
  if (!(rep > 0.0f && finite(rep))) rep = 1.0f;  // off: x 1 and x / 1 are x
  float freq = c.frequency ? c.frequency[row] : 0.0f, pres = c.presence ? c.presence[row] : 0.0f;
  if (!finite(freq)) freq = 0.0f;
  if (!finite(pres)) pres = 0.0f;
  if (c.tokens && unsigned(seq) >= unsigned(c.sequences)) return;  // a padding row (uniform)
  const int64_t room = c.tokens_stride;
  const int32_t* tokens = c.tokens + int64_t(seq) * room;
  // The first of the history and of the biases are asked for before their numbers are known.
  constexpr int A = 2;  // reads of a thread on their way
  constexpr unsigned kStep = 4 * kThreads;
  tokens4 ahead[A];
  auto fetch = [&](unsigned base, int64_t end) {
#pragma unroll
    for (int e = 0; e < A; ++e) {
      const unsigned i = base + 4 * t + kStep * e;
      ahead[e] = tokens4{-1, -1, -1, -1};
      if (i + 4 <= end) ahead[e] = *reinterpret_cast<const tokens4*>(tokens + i);
    }
  };
  if (c.tokens) fetch(0, room);
  const int b_first = t < b1 - b0 ? c.bias_tokens[b0 + t] : -1;
  const int len = c.tokens ? int(min(int64_t(max(c.lens[seq], 0)), room)) : 0;
  const unsigned prompt = c.tokens && c.prompt_lens ? min(max(c.prompt_lens[seq], 0), len) : 0;
  __syncthreads();
  auto see = [&](int token, unsigned i) {
    const unsigned j = unsigned(token) - unsigned(first);
    if (j < unsigned(count)) {
      if (i < prompt)
        atomicOr(counts + place_of<kSeg>(j), kInPrompt);
      else
        atomicAdd(counts + place_of<kSeg>(j), 1u);
    }
  };
  // (unsigned: a step past 2^31 tokens does not turn negative)
  const unsigned whole = len & ~3;
  for (unsigned base = 0; base < whole;) {  // uniform
#pragma unroll
    for (int e = 0; e < A; ++e) {
      const unsigned i = base + 4 * t + kStep * e;
      if (i < whole) {
#pragma unroll
        for (int j = 0; j < 4; ++j) see(ahead[e][j], i + j);
      }
    }
    base += kStep * A;
    if (base < whole) fetch(base, whole);
  }
  if (unsigned(t) < len - whole) see(tokens[whole + t], whole + t);
  auto see_bias = [&](int token, unsigned i) {
    const unsigned j = unsigned(token) - unsigned(first);
    if (j < unsigned(count)) atomicMax(entry + place_of<kSeg>(j), i + 1);
  };
  if (t < b1 - b0) see_bias(b_first, t);
  for (unsigned i = b0 + t + kThreads; i < unsigned(b1); i += kThreads) see_bias(c.bias_tokens[i], i - b0);
  __syncthreads();
  if (at >= count) return;
  uint32_t cs[8], es[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    const uint4 k = *reinterpret_cast<const uint4*>(counts + place_of<kSeg>(at + i));
    cs[i] = k.x, cs[i + 1] = k.y, cs[i + 2] = k.z, cs[i + 3] = k.w;
    if (b1 > b0) {
      const uint4 e = *reinterpret_cast<const uint4*>(entry + place_of<kSeg>(at + i));
      es[i] = e.x, es[i + 1] = e.y, es[i + 2] = e.z, es[i + 3] = e.w;
    }
  }
  uint32_t some = open ^ 0xffu;
#pragma unroll
  for (int i = 0; i < 8; ++i) some |= cs[i] | es[i];
  if (in_place) {
    if (some == 0) return;
    load();
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (cs[i] | es[i]) {  // few are
      float x = bf16_to_f32(uint16_t(raw[i / 2] >> (16 * (i & 1))));
      if (cs[i] != 0) {
        x = x < 0.0f ? x * rep : x / rep;
        const uint32_t said = cs[i] & ~kInPrompt;
        x -= freq * float(said);
        if (said != 0) x -= pres;
      }
      if (es[i] != 0) x += c.bias_values[b0 + int(es[i]) - 1];
      const uint32_t y = f32_to_bf16(x);
      raw[i / 2] = i & 1 ? (raw[i / 2] & 0xffffu) | y << 16 : (raw[i / 2] & 0xffff0000u) | y;
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t keep = (open >> (2 * i) & 1 ? 0xffffu : 0u) | (open >> (2 * i) & 2 ? 0xffff0000u : 0u);
    raw[i] = (raw[i] & keep) | (0xff80ff80u & ~keep);
  }
  if (at + 8 <= count) {
    *reinterpret_cast<words4*>(dst + at) = raw;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + i < count) dst[at + i] = uint16_t(raw[i / 2] >> (16 * (i & 1)));
  }
}

}  // namespace

int logits_control(const uint16_t* logits, int64_t stride, int rows, int n, const LogitsControls& c,
                   uint16_t* out, int64_t out_stride, hipStream_t s) {
  // Few rows take short segments, for more workgroups; many take long ones, whose histories are read less
  // often (64 rows of 151936 one after another: 18.2 us, 20.0 with 2048 tokens each, 18.7 with 8192).
#define MX_CONTROL(SEG)                                                                             \
  {                                                                                                 \
    const int64_t segs = (int64_t(n) + SEG - 1) / SEG, blocks = rows * segs;                        \
    if (blocks > 0x7fffffff) return MX_EUNSUPPORTED;                                                \
    hipLaunchKernelGGL((control_kernel<SEG>), dim3(unsigned(blocks)), dim3(SEG / 8),                \
                       SEG * (c.bias_starts ? 8 : 4), s, logits, stride, n, c, out, out_stride,     \
                       int(segs));                                                                  \
  }
  if (int64_t(rows) * n <= 256 * 4096) MX_CONTROL(2048) else MX_CONTROL(4096)
#undef MX_CONTROL
  return hipGetLastError() == hipSuccess ? MX_OK : MX_EHIP;
}

}  // namespace mx
