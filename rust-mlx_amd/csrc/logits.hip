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
// pass.  A token that the biases name twice takes the last entry: the largest index wins, whatever the
// order.
#include "kernels.hpp"
#include "paged_core.hpp"

namespace mx {

namespace {

using namespace pg;

constexpr int kThreads = 256;
constexpr uint32_t kInPrompt = 0x80000000u;

// Rows start at any element, histories at any word.
typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
typedef int32_t tokens4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ bool finite(float x) { return __builtin_fabsf(x) < u2f(0x7f800000u); }

template <int kSeg>
__global__ __launch_bounds__(kThreads) void control_kernel(const uint16_t* logits, int64_t stride,
                                                           int n, LogitsControls c, uint16_t* out,
                                                           int64_t out_stride, int segs) {
  constexpr int NV = kSeg / kThreads / 8;  // vectors of eight logits a thread
  extern __shared__ uint32_t counts[];     // [kSeg], then with biases [kSeg] of 1 + an entry's index
  uint32_t* entry = counts + kSeg;
  const int t = threadIdx.x;
  const int row = blockIdx.x / segs, first = blockIdx.x % segs * kSeg;
  const int seq = c.tokens && c.seqs ? c.seqs[row] : row;
  if (c.tokens && unsigned(seq) >= unsigned(c.sequences)) return;  // a padding row (uniform)
  const int count = min(kSeg, n - first);
  const uint16_t* src = logits + int64_t(row) * stride + first;
  uint16_t* dst = out + int64_t(row) * out_stride + first;
  const bool in_place = src == dst;  // then only what changes is touched
  words4 raw[NV];
  auto load = [&](int v) {
    const int at = 8 * (t + kThreads * v);
    if (at + 8 <= count) {
      raw[v] = *reinterpret_cast<const words4*>(src + at);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i < count) {
          const uint32_t x = src[at + i];
          raw[v][i / 2] = i & 1 ? (raw[v][i / 2] & 0xffffu) | x << 16 : x;
        }
    }
  };
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    raw[v] = words4{0, 0, 0, 0};
    if (!in_place) load(v);
  }
  int b0 = 0, b1 = 0;
  if (c.bias_starts) {
    b0 = min(max(c.bias_starts[row], 0), c.bias_count);
    b1 = min(max(c.bias_starts[row + 1], b0), c.bias_count);
  }
  const int state = c.masks ? (c.mask_rows ? c.mask_rows[row] : row) : -1;
  const uint8_t* allowed = unsigned(state) < unsigned(c.mask_states)
                               ? reinterpret_cast<const uint8_t*>(c.masks + state * c.mask_stride) + first / 8
                               : nullptr;
  for (int i = 4 * t; i < kSeg; i += 4 * kThreads) {
    *reinterpret_cast<uint4*>(counts + i) = make_uint4(0, 0, 0, 0);
    if (b1 > b0) *reinterpret_cast<uint4*>(entry + i) = make_uint4(0, 0, 0, 0);
  }
  const int64_t room = c.tokens_stride;
  const int len = c.tokens ? int(min(int64_t(max(c.lens[seq], 0)), room)) : 0;
  const int prompt = c.tokens && c.prompt_lens ? min(max(c.prompt_lens[seq], 0), len) : 0;
  const int32_t* tokens = c.tokens + int64_t(seq) * room;
  __syncthreads();
  auto see = [&](int token, int i) {
    const unsigned j = unsigned(token) - unsigned(first);
    if (j < unsigned(count)) {
      if (i < prompt)
        atomicOr(counts + j, kInPrompt);
      else
        atomicAdd(counts + j, 1u);
    }
  };
  const int whole = len & ~3;
#pragma unroll 4
  for (int i = 4 * t; i < whole; i += 4 * kThreads) {
    const tokens4 k = *reinterpret_cast<const tokens4*>(tokens + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) see(k[e], i + e);
  }
  if (t < len - whole) see(tokens[whole + t], whole + t);
  for (int i = b0 + t; i < b1; i += kThreads) {
    const unsigned j = unsigned(c.bias_tokens[i]) - unsigned(first);
    if (j < unsigned(count)) atomicMax(entry + j, uint32_t(i - b0) + 1u);
  }
  float rep = c.repetition ? c.repetition[row] : 0.0f;
  if (!(rep > 0.0f && finite(rep))) rep = 1.0f;  // off: x 1 and x / 1 are x
  float freq = c.frequency ? c.frequency[row] : 0.0f, pres = c.presence ? c.presence[row] : 0.0f;
  if (!finite(freq)) freq = 0.0f;
  if (!finite(pres)) pres = 0.0f;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int at = 8 * (t + kThreads * v);
    if (at >= count) break;
    const uint32_t open = allowed ? allowed[at / 8] : 0xffu;
    const uint4 c0 = *reinterpret_cast<const uint4*>(counts + at);
    const uint4 c1 = *reinterpret_cast<const uint4*>(counts + at + 4);
    const uint32_t cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    uint32_t es[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (b1 > b0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) es[i] = entry[at + i];
    }
    uint32_t some = open ^ 0xffu;
#pragma unroll
    for (int i = 0; i < 8; ++i) some |= cs[i] | es[i];
    if (in_place && some == 0) continue;
    if (in_place) load(v);
    if (some != 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float x = bf16_to_f32(uint16_t(raw[v][i / 2] >> (16 * (i & 1))));
        if (cs[i] != 0) {
          x = x < 0.0f ? x * rep : x / rep;
          const uint32_t said = cs[i] & ~kInPrompt;
          x -= freq * float(said);
          if (said != 0) x -= pres;
        }
        if (es[i] != 0) x += c.bias_values[b0 + int(es[i]) - 1];
        if (!(open >> i & 1)) x = neg_inf();
        const uint32_t y = f32_to_bf16(x);
        raw[v][i / 2] = i & 1 ? (raw[v][i / 2] & 0xffffu) | y << 16 : (raw[v][i / 2] & 0xffff0000u) | y;
      }
    }
    if (at + 8 <= count) {
      *reinterpret_cast<words4*>(dst + at) = raw[v];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i < count) dst[at + i] = uint16_t(raw[v][i / 2] >> (16 * (i & 1)));
    }
  }
}

}  // namespace

int logits_control(const uint16_t* logits, int64_t stride, int rows, int n, const LogitsControls& c,
                   uint16_t* out, int64_t out_stride, hipStream_t s) {
  // few rows take short segments, for more workgroups
#define MX_CONTROL(SEG)                                                                             \
  {                                                                                                 \
    const int64_t segs = (n + SEG - 1) / SEG, blocks = rows * segs;                                 \
    if (blocks > 0x7fffffff) return MX_EUNSUPPORTED;                                                \
    hipLaunchKernelGGL((control_kernel<SEG>), dim3(unsigned(blocks)), dim3(kThreads),               \
                       SEG * (c.bias_starts ? 8 : 4), s, logits, stride, n, c, out, out_stride,     \
                       int(segs));                                                                  \
  }
  if (int64_t(rows) * n <= 256 * 4096) MX_CONTROL(2048) else MX_CONTROL(4096)
#undef MX_CONTROL
  return hipGetLastError() == hipSuccess ? MX_OK : MX_EHIP;
}

}  // namespace mx
