// Rules on logits and the greedy choice of a token. For a row x of logits, its history of prompt and output tokens and
//   seen(v) = v is in the history, c(v) = how often v is in its output part
//     x1 = seen(v) ? (x > 0 ? x / r : x * r) : x         repetition penalty r
//     x2 = c(v) > 0 ? x1 - f * c(v) : x1                 frequency penalty f
//     x3 = c(v) > 0 ? x2 - p : x2                        presence penalty p
//     x4 = x3 + bias(v)                                  a token listed twice: the later entry counts
//     y  = allowed(v) ? x4 : -inf                        a grammar's mask, one bit a token
//   choice = the allowed token of the largest y, the lowest id among equals, a NaN above everything; -1 if none is allowed.
// Every step is one fp32 operation, rounded by itself (no fused multiply-add), so any other implementation in fp32 that
// follows the formulas gives the same bits.
//
// The history is a list, the vocabulary is long: a block counts the tokens that fall into its slice of the vocabulary in LDS
// (whole numbers: the order of the atomic additions does not matter), then passes over the slice's logits once.
// MI355X: 96 rows of 128256 bf16 logits with 4096 tokens of history, 50 biases and masks 17.8 us, of which the rows alone take 6,
// the history 6 (every block of a row counts all of it, once a slice), biases and masks 3; 256 rows of 64128 fp32 with the processed
// logits written 25.6 us, 5.1 TB/s; one row 5.1 us. Taking the rules only to the few tokens that have one, a token at a time, made chains of
// dependent loads: 29.9 us where this takes 17.8.
//
// No reference counterpart (vLLM is a README bullet in the reference, README.md:73).
#include "klm_launch.h"
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
  uint64_t* part;                 // [B][klm_logits_parts]
  int64_t* ids;                   // [B]
  float* best;                    // [B]
  int64_t stride;
  int B, V, R, hist_len, n_bias, n_masks, mask_words, first;
};

// A block takes SLICE columns, a chunk of 8 a thread. Columns are counted from the 16-byte boundary at or before the
// row's start, so that every chunk but a row's first and last is whole aligned loads whatever the row stride is.
constexpr int THREADS = 512, SLICE = THREADS * 8;
// Blocks on the chip at once: 3 per CU, 6 waves a SIMD of up to 80 registers (the four kernels take 70 to 76; LDS would hold 5).
constexpr int RESIDENT = 3 * 256;

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
    if ((cnt & 0x7fffffffu) != 0) {
      const float fc = f * c;
      x = x - fc;
      x = x - p;
    }
  }
  return x;
}

// One slice's 8 places of a thread as the bits that came from memory; 0 in places outside the row.
template <bool F32>
struct Raw {
  uint32_t w[F32 ? 8 : 4];
};
template <bool F32>
__device__ __forceinline__ void load_raw(const char* base, int v, int V, Raw<F32>& r) {
  constexpr int ES = F32 ? 4 : 2;
  if (v >= 0 && v + 8 <= V) {
#pragma unroll
    for (int k = 0; k < (F32 ? 2 : 1); ++k) {
      const uint4 w = *reinterpret_cast<const uint4*>(base + (ptrdiff_t)v * ES + k * 16);
      r.w[k * 4] = w.x; r.w[k * 4 + 1] = w.y; r.w[k * 4 + 2] = w.z; r.w[k * 4 + 3] = w.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < (F32 ? 8 : 4); ++k) r.w[k] = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (v + e >= 0 && v + e < V) {
        if (F32) r.w[e] = reinterpret_cast<const uint32_t*>(base)[v + e];
        else r.w[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(base)[v + e] << (16 * (e & 1));
      }
  }
}

// the words that hold the mask's bits of tokens t .. t + 7; t may lie before the vocabulary (places before a row's column 0) or end
// behind it
__device__ __forceinline__ void load_bits(const uint32_t* mask, int words, int64_t t, uint32_t& m0, uint32_t& m1) {
  const int64_t w = t >> 5;
  m0 = w >= 0 && w < words ? mask[w] : 0u;
  m1 = (t & 31) > 24 && w + 1 >= 0 && w + 1 < words ? mask[w + 1] : 0u;
}

template <bool F32, bool BIAS>
__global__ __launch_bounds__(THREADS, 6) void logits_kernel(LogitArgs a, int slices, int per, int wide_out) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  uint32_t* cnt = lds;                 // [SLICE] bit 31: in the prompt; below: times in the output
  uint32_t* last = lds + SLICE;        // [SLICE] 1 + the last bias entry of the token
  __shared__ uint64_t red[THREADS / 64];
  constexpr int ES = F32 ? 4 : 2;
  const int tid = threadIdx.x, b = blockIdx.y, u = tid * 8;
  const char* base = (const char*)a.logits + (size_t)b * a.stride * ES;
  const int pad = (int)((reinterpret_cast<uintptr_t>(base) & 15) / ES);
  const int s0 = blockIdx.x * per, s1 = s0 + per < slices ? s0 + per : slices;
  Raw<F32> raw;
  load_raw<F32>(base, s0 * SLICE - pad + u, a.V, raw);
  const int row = a.rows ? a.rows[b] : b;
  const bool rules = row >= 0 && row < a.R;

  float r = 1.f, f = 0.f, p = 0.f;
  const uint32_t* mask = nullptr;
  const int *hist = nullptr, *ids = nullptr;
  int len = 0, plen = 0;
  if (rules) {
    r = a.repetition[row];
    f = a.frequency[row];
    p = a.presence[row];
    len = a.lens[row];
    len = len < a.hist_len ? len : a.hist_len;
    plen = a.prompt_lens[row];
    if (a.mask) {
      const int m = a.mask_rows ? a.mask_rows[row] : row;
      if (m >= 0 && m < a.n_masks) mask = a.mask + (size_t)m * a.mask_words;
    }
    hist = a.history + (size_t)row * a.hist_len;
    if (BIAS) ids = a.bias_ids + (size_t)row * a.n_bias;
  }
  // the history's first HELD tokens a thread stay in registers for all slices; a longer one is read again from the caches
  constexpr int HELD = 8;
  int held[HELD];
#pragma unroll
  for (int k = 0; k < HELD; ++k) held[k] = tid + k * THREADS < len ? hist[tid + k * THREADS] : -1;
  uint32_t m0 = 0, m1 = 0;             // the words of the mask that hold the 8 places' bits
  if (mask) load_bits(mask, a.mask_words, (int64_t)a.first + s0 * SLICE - pad + u, m0, m1);
  float top = 0.f, kept[8];            // the thread's largest value so far (valid where `kept_bits` is not 0), and the 8 values among which it is
  uint32_t kept_bits = 0;
  int kept_v = 0;
  bool nan_kept = false;
  for (int s = s0; s < s1; ++s) {
    const int v0 = s * SLICE - pad;                                // column of the slice's first place; below 0 in a row's first slice
    const int v = v0 + u;                                          // column of this thread's first place
    const bool whole = v >= 0 && v + 8 <= a.V;
    const int sh = (int)(((int64_t)a.first + v) & 31);
    if (rules) {
#pragma unroll
      for (int j = 0; j < SLICE / THREADS / 4; ++j) {
        reinterpret_cast<uint4*>(cnt)[tid + j * THREADS] = uint4{0, 0, 0, 0};
        if (BIAS) reinterpret_cast<uint4*>(last)[tid + j * THREADS] = uint4{0, 0, 0, 0};
      }
      __syncthreads();
      const uint32_t lo = (uint32_t)(a.first + v0);                // ids at or above `first` only: the difference does not wrap into the slice
      const auto count = [&](int t, int i) {
        const uint32_t at = (uint32_t)t - lo;
        if (t >= a.first && at < (uint32_t)SLICE) {
          if (i >= plen) atomicAdd(&cnt[at], 1u);
          else atomicOr(&cnt[at], 0x80000000u);
        }
      };
#pragma unroll
      for (int k = 0; k < HELD; ++k) count(held[k], tid + k * THREADS);
      for (int i = tid + HELD * THREADS; i < len; i += THREADS) count(hist[i], i);
      if (BIAS) {
        for (int i = tid; i < a.n_bias; i += THREADS) {
          const uint32_t at = (uint32_t)ids[i] - lo;
          if (ids[i] >= a.first && at < (uint32_t)SLICE) atomicMax(&last[at], (uint32_t)i + 1);
        }
      }
      __syncthreads();
    }

    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = F32 ? __uint_as_float(raw.w[e]) : __uint_as_float((e & 1) ? (raw.w[e >> 1] & 0xffff0000u) : (raw.w[e >> 1] << 16));
    uint32_t bits = mask ? (uint32_t)((((uint64_t)m1 << 32) | m0) >> sh) & 0xffu : 0xffu;      // bit e: place e is allowed, and of the row
    if (s + 1 < s1) {                                              // the next slice's logits and mask travel under this one's work
      load_raw<F32>(base, v + SLICE, a.V, raw);
      if (mask) load_bits(mask, a.mask_words, (int64_t)a.first + v + SLICE, m0, m1);
    }
    if (rules) {
      uint32_t c[8];
      *reinterpret_cast<uint4*>(c) = *reinterpret_cast<const uint4*>(cnt + u);
      *reinterpret_cast<uint4*>(c + 4) = *reinterpret_cast<const uint4*>(cnt + u + 4);
      if ((c[0] | c[1] | c[2] | c[3] | c[4] | c[5] | c[6] | c[7]) != 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = apply_rules(x[e], c[e], r, f, p);
      }
      if (BIAS) {
        const float* bias = a.bias_values + (size_t)row * a.n_bias;
        *reinterpret_cast<uint4*>(c) = *reinterpret_cast<const uint4*>(last + u);
        *reinterpret_cast<uint4*>(c + 4) = *reinterpret_cast<const uint4*>(last + u + 4);
        if ((c[0] | c[1] | c[2] | c[3] | c[4] | c[5] | c[6] | c[7]) != 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c[e]) x[e] = x[e] + bias[c[e] - 1];
        }
      }
      if (s + 1 < s1) __syncthreads();                             // the counts are cleared for the next slice
    }
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 8; ++e) bits &= v + e >= 0 && v + e < a.V ? 0xffu : ~(1u << e);
    }
    if (mask || !whole) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (bits >> e) & 1 ? x[e] : -INFINITY;
    }
    if (a.out) {
      float* dst = a.out + (size_t)b * a.V + v;
      if (wide_out && whole) {
        *reinterpret_cast<f32x4*>(dst) = f32x4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4*>(dst + 4) = f32x4{x[4], x[5], x[6], x[7]};
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (v + e >= 0 && v + e < a.V) dst[e] = x[e];
      }
    }
    // the largest value by a plain maximum; its column is looked for at the end, by the threads that hold the block's largest
    float m = x[0];
    bool nan = __builtin_isunordered(x[0], x[1]);
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      m = fmaxf(m, x[e]);
      if (e & 1) nan = nan || __builtin_isunordered(x[e], x[e - 1]);
    }
    // an equal value of a later slice has a higher column; the first slice with a NaN is kept for good
    if (bits && !nan_kept && (nan || !kept_bits || m > top)) {
      top = m;
      kept_bits = bits;
      kept_v = v;
      nan_kept = nan;
#pragma unroll
      for (int e = 0; e < 8; ++e) kept[e] = x[e];
    }
  }
  const uint32_t mine = nan_kept ? 0xffffffffu : kept_bits ? order_of(top) : 0u;
  uint32_t most = mine;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t other = __shfl_xor(most, o);
    most = other > most ? other : most;
  }
  uint32_t at = 0xffffffffu;
  if (mine == most && most != 0) {
#pragma unroll
    for (int e = 7; e >= 0; --e) at = (kept_bits >> e) & 1 && order_of(kept[e]) == most ? (uint32_t)(kept_v + e) : at;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t other = __shfl_xor(at, o);
    at = other < at ? other : at;
  }
  if ((tid & 63) == 0) red[tid >> 6] = most ? ((uint64_t)most << 32) | (0xffffffffu - at) : 0;
  __syncthreads();
  if (tid == 0) {
    uint64_t best = red[0];
    for (int i = 1; i < THREADS / 64; ++i) best = red[i] > best ? red[i] : best;
    if (gridDim.x == 1) write_choice(a, b, best);
    else a.part[(size_t)b * gridDim.x + blockIdx.x] = best;
  }
}

__global__ __launch_bounds__(64) void choose_kernel(LogitArgs a, int parts) {
  const int b = blockIdx.x;
  uint64_t best = 0;
  for (int i = threadIdx.x; i < parts; i += 64) {
    const uint64_t k = a.part[(size_t)b * parts + i];
    best = k > best ? k : best;
  }
  best = wave_max(best);
  if (threadIdx.x == 0) write_choice(a, b, best);
}

int slices_of(int V) { return (int)(((int64_t)V + 7 + SLICE - 1) / SLICE); }     // a row may start up to 7 places into its first slice
// Slices that one block walks: as few as let all blocks be on the chip at once, 8 at most. A block's chain of dependent loads (the
// row's lengths, its history, the mask) is longer than the work of a slice, and a second round runs it again: 256 x 64128 fp32, 8
// biases, processed logits written, 28.2 us with 6 slices a block (768 blocks), 31.6 with 4 (1024) and 37.9 with 1 (4096); 128 x
// 128256, 2000 tokens of history, 22.5 with 6 (768), 25.7 with 4 (1024), 32.1 with 1 (4096). More slices than it takes leave CUs
// idle: 96 x 128256 20.7 with 4 (768), 25.8 with 6 (576).
int slices_per_block(int B, int V) {
  const int slices = slices_of(V);
  int per = 1;
  while (per < 8 && (int64_t)((slices + per - 1) / per) * B > RESIDENT) ++per;
  return per;
}

}  // namespace

extern "C" {

int klm_logits_parts(int B, int V) {
  const int per = slices_per_block(B, V);
  return (slices_of(V) + per - 1) / per;
}

int klm_choose_tokens(const klm_logits_args* c) {
  if (!c) return KLM_ERR_ARG;
  const int B = c->B, V = c->V, fp32 = c->fp32;
  if (B <= 0 || B > 65535 || V <= 0 || c->stride < V || c->first < 0 || (int64_t)c->first + V > INT32_MAX || c->R < 0 || c->hist_len < 0 ||
      c->n_bias < 0 || c->n_masks < 0)
    return KLM_ERR_SHAPE;
  if (!c->logits || !c->ids || !c->best || !c->part) return KLM_ERR_ARG;
  if (c->R > 0 && (!c->prompt_lens || !c->lens || !c->repetition || !c->frequency || !c->presence || (c->hist_len > 0 && !c->history) ||
                   (c->n_bias > 0 && (!c->bias_ids || !c->bias_values)) ||
                   (c->n_masks > 0 && (!c->mask || (int64_t)c->mask_words * 32 < (int64_t)c->first + V))))
    return KLM_ERR_ARG;
  const LogitArgs a{c->logits, c->history, c->prompt_lens, c->lens, c->repetition, c->frequency, c->presence, c->bias_ids, c->bias_values,
                    c->n_masks > 0 ? (const uint32_t*)c->mask : nullptr, c->mask_rows, c->rows, c->out, (uint64_t*)c->part, c->ids, c->best,
                    c->stride, B, V, c->R, c->hist_len, c->n_bias, c->n_masks, c->mask_words, c->first};
  const int slices = slices_of(V), per = slices_per_block(B, V), parts = klm_logits_parts(B, V);
  hipStream_t s = static_cast<hipStream_t>(c->stream);
  // 16-byte stores where every chunk starts on such a boundary of `out`: columns there and in `logits` are off alike
  const int pad = (int)((reinterpret_cast<uintptr_t>(c->logits) & 15) / (fp32 ? 4 : 2));
  const int wide_out = a.out && pad % 4 == 0 && (B == 1 || (V % 4 == 0 && a.stride % (fp32 ? 4 : 8) == 0)) && aligned16(a.out);
  const dim3 grid(parts, B);
  const size_t one = SLICE * 4;
  if (a.n_bias > 0 && a.R > 0) {
    if ((fp32 ? klm_ensure_dyn_lds<logits_kernel<true, true>>(2 * one) : klm_ensure_dyn_lds<logits_kernel<false, true>>(2 * one)) != KLM_OK)
      return KLM_ERR_HIP;
    if (fp32) hipLaunchKernelGGL((logits_kernel<true, true>), grid, dim3(THREADS), 2 * one, s, a, slices, per, wide_out);
    else hipLaunchKernelGGL((logits_kernel<false, true>), grid, dim3(THREADS), 2 * one, s, a, slices, per, wide_out);
  } else {
    if (fp32) hipLaunchKernelGGL((logits_kernel<true, false>), grid, dim3(THREADS), one, s, a, slices, per, wide_out);
    else hipLaunchKernelGGL((logits_kernel<false, false>), grid, dim3(THREADS), one, s, a, slices, per, wide_out);
  }
  if (hipGetLastError() != hipSuccess) return KLM_ERR_HIP;
  if (parts > 1) hipLaunchKernelGGL(choose_kernel, dim3(B), dim3(64), 0, s, a, parts);
  return launch_status();
}

}  // extern "C"
