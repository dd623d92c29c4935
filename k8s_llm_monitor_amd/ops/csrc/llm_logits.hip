// Rules on logits and the greedy choice of a token. For a row x of logits, its history of prompt and output tokens and
//   seen(v) = v is in the history, c(v) = how often v is in its output part
//     x1 = seen(v) ? (x > 0 ? x / r : x * r) : x         repetition penalty r
//     x2 = x1 - f * c(v)                                 frequency penalty f
//     x3 = c(v) > 0 ? x2 - p : x2                        presence penalty p
//     x4 = x3 + bias(v)                                  a token listed twice: the later entry counts
//     y  = allowed(v) ? x4 : -inf                        a grammar's mask, one bit a token
//   choice = the allowed token of the largest y, the lowest id among equals, a NaN above everything; -1 if none is allowed.
// Every step is one fp32 operation, rounded by itself (no fused multiply-add), so any other implementation in fp32 that
// follows the formulas gives the same bits.
//
// The history is a list, the vocabulary is long: a block counts the tokens that fall into its slice of the vocabulary in LDS
// (whole numbers: the order of the atomic additions does not matter), then passes over the slice's logits once.
//
// No reference counterpart (vLLM is a README bullet in the reference, README.md:73).
#include "llm_common.h"

using namespace klm_llm;

namespace {

struct LogitArgs {
  const void* logits;             // [B][V], rows `stride` elements apart
  const int* history;             // [R][hist_len] token ids
  const int *prompt_lens, *lens;  // [R]
  const float *repetition, *frequency, *presence;   // [R]
  const int* bias_ids;            // [R][n_bias], entries outside the vocabulary are ignored
  const float* bias_values;
  const uint32_t* mask;           // [n_masks][mask_words], bit v % 32 of word v / 32: v is allowed
  const int* mask_rows;           // [R] mask of the row (outside 0 .. n_masks - 1: none), null: mask r for row r
  const int* rows;                // [B] rules of the row (outside 0 .. R - 1: none), null: row b
  float* out;                     // [B][V] or null
  uint64_t* part;                 // [B][slices]
  int64_t* ids;                   // [B]
  float* best;                    // [B]
  int64_t stride;
  int B, V, R, hist_len, n_bias, n_masks, mask_words, first;
};

constexpr int SLICE = 4096;

// larger number = larger value; -0 and +0 are equal, a NaN is above everything; 0 is left for "no token"
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  if (o == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint64_t wave_max(uint64_t k) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t other = __shfl_xor((unsigned long long)k, o);
    k = other > k ? other : k;
  }
  return k;
}
__device__ __forceinline__ void write_choice(const LogitArgs& a, int b, uint64_t key) {
  const bool none = key == 0;
  a.ids[b] = none ? -1 : (int64_t)a.first + (int64_t)(0xffffffffu - (uint32_t)key);
  a.best[b] = none ? -INFINITY : value_of((uint32_t)(key >> 32));
}

__device__ __forceinline__ float apply_rules(float x, uint32_t cnt, float r, float f, float p) {
#pragma clang fp contract(off)
  const float c = (float)(cnt & 0x7fffffffu);
  if (cnt != 0) {
    x = x > 0.f ? x / r : x * r;
    const float fc = f * c;
    x = x - fc;
    if ((cnt & 0x7fffffffu) != 0) x = x - p;
  }
  return x;
}

template <bool F32>
__global__ __launch_bounds__(256) void logits_kernel(LogitArgs a, int slices) {
  __shared__ uint32_t cnt[SLICE];      // bit 31: in the prompt; below: times in the output
  __shared__ uint32_t last[SLICE];     // 1 + the last bias entry of the token
  __shared__ uint64_t red[4];
  const int tid = threadIdx.x, b = blockIdx.y, v0 = blockIdx.x * SLICE;
  const int n = a.V - v0 < SLICE ? a.V - v0 : SLICE;
  const int row = a.rows ? a.rows[b] : b;
  const bool rules = row >= 0 && row < a.R;
  float r = 1.f, f = 0.f, p = 0.f;
  const uint32_t* mask = nullptr;
  const float* bias = nullptr;
  if (rules) {
    const uint32_t lo = (uint32_t)a.first + v0;
    for (int i = tid; i < n; i += 256) { cnt[i] = 0; last[i] = 0; }
    __syncthreads();
    r = a.repetition[row];
    f = a.frequency[row];
    p = a.presence[row];
    int len = a.lens[row];
    len = len < a.hist_len ? len : a.hist_len;
    const int plen = a.prompt_lens[row];
    const int* hist = a.history + (size_t)row * a.hist_len;
    for (int i = tid; i < len; i += 256) {
      const uint32_t t = (uint32_t)hist[i] - lo;
      if (hist[i] >= 0 && t < (uint32_t)n) {
        if (i >= plen) atomicAdd(&cnt[t], 1u);
        else atomicOr(&cnt[t], 0x80000000u);
      }
    }
    if (a.n_bias > 0) {
      bias = a.bias_values + (size_t)row * a.n_bias;
      const int* ids = a.bias_ids + (size_t)row * a.n_bias;
      for (int i = tid; i < a.n_bias; i += 256) {
        const uint32_t t = (uint32_t)ids[i] - lo;
        if (ids[i] >= 0 && t < (uint32_t)n) atomicMax(&last[t], (uint32_t)i + 1);
      }
    }
    if (a.mask) {
      const int m = a.mask_rows ? a.mask_rows[row] : row;
      if (m >= 0 && m < a.n_masks) mask = a.mask + (size_t)m * a.mask_words;
    }
    __syncthreads();
  }
  uint64_t best = 0;
  for (int i = tid; i < n; i += 256) {
    float x = F32 ? ((const float*)a.logits)[b * a.stride + v0 + i] : bf2f(((const uint16_t*)a.logits)[b * a.stride + v0 + i]);
    if (rules) {
      x = apply_rules(x, cnt[i], r, f, p);
      if (bias && last[i]) x = x + bias[last[i] - 1];
    }
    bool allowed = true;
    if (mask) {
      const uint32_t t = (uint32_t)a.first + v0 + i;
      allowed = (mask[t >> 5] >> (t & 31)) & 1;
    }
    if (a.out) a.out[(size_t)b * a.V + v0 + i] = allowed ? x : -INFINITY;
    if (allowed) {
      const uint64_t key = ((uint64_t)order_of(x) << 32) | (0xffffffffu - (uint32_t)(v0 + i));
      best = key > best ? key : best;
    }
  }
  best = wave_max(best);
  if ((tid & 63) == 0) red[tid >> 6] = best;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < 4; ++i) best = red[i] > best ? red[i] : best;
    if (slices == 1) write_choice(a, b, best);
    else a.part[(size_t)b * slices + blockIdx.x] = best;
  }
}

__global__ __launch_bounds__(64) void choose_kernel(LogitArgs a, int slices) {
  const int b = blockIdx.x;
  uint64_t best = 0;
  for (int i = threadIdx.x; i < slices; i += 64) {
    const uint64_t k = a.part[(size_t)b * slices + i];
    best = k > best ? k : best;
  }
  best = wave_max(best);
  if (threadIdx.x == 0) write_choice(a, b, best);
}

}  // namespace

extern "C" {

int klm_logits_slices(int V) { return (V + SLICE - 1) / SLICE; }

int klm_choose_tokens(const void* logits, int fp32, int64_t stride, int B, int V, int first, const int32_t* rows, int R,
                      const int32_t* history, int hist_len, const int32_t* prompt_lens, const int32_t* lens,
                      const float* repetition, const float* frequency, const float* presence, const int32_t* bias_ids,
                      const float* bias_values, int n_bias, const void* mask, int n_masks, int mask_words,
                      const int32_t* mask_rows, float* out, void* part, int64_t* ids, float* best, void* stream) {
  if (B <= 0 || B > 65535 || V <= 0 || stride < V || first < 0 || (int64_t)first + V > INT32_MAX || R < 0 || hist_len < 0 || n_bias < 0 ||
      n_masks < 0)
    return KLM_ERR_SHAPE;
  if (!logits || !ids || !best || !part) return KLM_ERR_ARG;
  if (R > 0 && (!prompt_lens || !lens || !repetition || !frequency || !presence || (hist_len > 0 && !history) ||
                (n_bias > 0 && (!bias_ids || !bias_values)) || (n_masks > 0 && (!mask || (int64_t)mask_words * 32 < (int64_t)first + V))))
    return KLM_ERR_ARG;
  LogitArgs a{logits, history, prompt_lens, lens, repetition, frequency, presence, bias_ids, bias_values,
              n_masks > 0 ? (const uint32_t*)mask : nullptr, mask_rows, rows, out, (uint64_t*)part, ids, best, stride,
              B, V, R, hist_len, n_bias, n_masks, mask_words, first};
  const int slices = klm_logits_slices(V);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (fp32) hipLaunchKernelGGL(logits_kernel<true>, dim3(slices, B), dim3(256), 0, s, a, slices);
  else hipLaunchKernelGGL(logits_kernel<false>, dim3(slices, B), dim3(256), 0, s, a, slices);
  if (hipGetLastError() != hipSuccess) return KLM_ERR_HIP;
  if (slices > 1) hipLaunchKernelGGL(choose_kernel, dim3(B), dim3(64), 0, s, a, slices);
  return launch_status();
}

}  // extern "C"
