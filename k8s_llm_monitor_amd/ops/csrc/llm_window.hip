// Attention with a sliding window and sinks over the paged KV cache (layouts: llm_attention.hip).
//
//   o[t, h] = sum_j p_j v_j,  p = softmax over the keys j that token t sees of  scale * q[t, h] . k_j
//   the token at position p sees key j  <=>  j <= p  and  (j > p - window  or  j < sinks)  and j's page exists
//
// A page id outside the cache is no page: nothing is read through it, its tokens are not seen. Pages that lie between the
// sinks and the window are never looked at, so the engine gives them back while the sequence runs. A row that sees nothing
// gives 0. A masked key contributes nothing whatever its bytes are (stale slots, NaN, infinities).
//
// Roundings: scores, maxima, sums and the output's sums are fp32. A weight is rounded to bf16 before it meets V, because the matrix
// instruction takes bf16: off by at most 2^-8 of itself. Its sum is taken unrounded, so that the two do not cancel: the result is
// within 2^-8 sum p |v|, and 2^-8 of itself from its own rounding, of the formula. Un-normalised sums bound V: weights are at most 1
// in the decode, at most 256 in the prefill, so that |V| times the keys, times 256 in the prefill, has to stay within fp32 (over a
// million keys V up to 1e30 does).
//
// No reference counterpart (vLLM is a README bullet in the reference, README.md:73).
#include <type_traits>

#include "klm_launch.h"
#include "llm_common.h"

using namespace klm_llm;

namespace {

struct WinArgs {
  const uint16_t* q;
  const void* kc;
  const void* vc;
  const int* tables;     // [n_seqs][width] page ids
  const int* lens;       // decode: context lengths [B]; prefill: seq_info [n_seqs][3] = q_start, q_len, ctx_len
  uint16_t* out;
  float* part_o;         // [rows * n_q][splits][128], fp32, un-normalised
  float* part_ml;        // [rows * n_q][splits][2]: maximum (scaled, log2) and sum
  int n_seqs, rows;      // rows of q and out
  int q_stride, n_q, n_kv, G;
  int width, pages;      // table width, pages in the cache
  int window, sinks;
  int splits;
  int zero_rest;         // prefill: rows of no sequence become 0
  float scale_log2;
};

// The keys a span of queries at positions [pos_a, pos_b] may see, as steps of 32 keys: the sinks' steps, then the window's.
struct Span {
  int lo, n_sink, lo_step, n;
  __device__ __forceinline__ int step(int i) const { return i < n_sink ? i : lo_step + (i - n_sink); }
};

__device__ __forceinline__ Span make_span(int pos_a, int pos_b, int window, int sinks, int width) {
  Span s;
  const int lim = (pos_b + 1) < width * BLK ? pos_b + 1 : width * BLK;
  s.lo = pos_a - window + 1 > 0 ? pos_a - window + 1 : 0;
  s.lo_step = s.lo >> 5;
  int se = sinks < s.lo ? sinks : s.lo;
  se = se < lim ? se : lim;
  const int ns = (se + 31) >> 5;
  s.n_sink = ns < s.lo_step ? ns : s.lo_step;
  const int end = (lim + 31) >> 5;
  s.n = s.n_sink + (end > s.lo_step ? end - s.lo_step : 0);
  return s;
}

// page of 16 tokens `i` of a sequence; -1: none
__device__ __forceinline__ int page_at(const int* table, int i, int width, int pages) {
  const int id = table[i < width ? i : width - 1];
  return (i < width && id >= 0 && id < pages) ? id : -1;
}

// bits 15 and 31: that bf16 half of x is a NaN or an infinity (all ones in its exponent)
__device__ __forceinline__ uint32_t odd_halves(uint32_t x) { return ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }
// x with those halves 0
__device__ __forceinline__ uint32_t without_odd(uint32_t x) { return x & ~((odd_halves(x) >> 15) * 0xffffu); }

// ---------------------------------------------------------------------------------------------------------------------
// One token per sequence: what bounds it is the cache that has to be read once. Block = (16 query heads of a kv head, sequence,
// split); its 4 waves take the 32-key steps of the split in turn, loaded past the caches straight into matrix operands, the next
// step's 16 KiB (e4m3: 8) in flight under this one's work. e4m3 stays raw until its turn: turned into bf16 as it came it would
// be waited for at once. The operand mapping is llm_attention.hip's. Measured, 8 kv heads, window 4096: 128 sequences of up to
// 8192 tokens 252 us, 5.4 TB/s (through the caches 257 us); 96 of e4m3, 118 us, 4.6 TB/s (64-key steps 121 us). The same loads
// without products and softmax take 247 and 111 us. A sequence's splits are as many for a short context as for a long one: 96 of one
// length, with as many keys in sum as those 96, take 93 us, and 89 unsplit (6.1 TB/s); 33 bf16 ones 41 at best, 44 where they differ.
// ---------------------------------------------------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

template <bool KV8>
struct Raw {
  using V = std::conditional_t<KV8, u32x2, u32x4>;      // 8 tokens of a dim
  u32x4 k[KV8 ? 4 : 8];  // bf16: tile i / 4 (tokens + 4), k-step i % 4; e4m3: tile i / 2, 64 dims i % 2
  V v[8];
  int pv;                // the page that this lane's V comes from, -1: none
};

template <bool KV8>
__device__ __forceinline__ void load_raw(const WinArgs& a, int held, int j, int h, int fr, int fq, Raw<KV8>& f) {
  constexpr int ES = KV8 ? 1 : 2;
  const int pk = __shfl(held, j * 2 + (fr >> 3));
  f.pv = __shfl(held, j * 2 + (fq >> 1));
  const char* kp = (const char*)a.kc + ((size_t)(pk < 0 ? 0 : pk) * a.n_kv + h) * (BLK_ELEMS * ES);
  const char* vp = (const char*)a.vc + ((size_t)(f.pv < 0 ? 0 : f.pv) * a.n_kv + h) * (BLK_ELEMS * ES);
  kp += ((((fr >> 2) & 1) << 3) + (fr & 3)) * HD * ES + fq * 16;
  vp += (fr * BLK + (fq & 1) * 8) * ES;
#pragma unroll
  for (int i = 0; i < (KV8 ? 4 : 8); ++i) {
    const int off = KV8 ? (i >> 1) * 4 * HD + (i & 1) * 64 : ((i >> 2) * 4 * HD + (i & 3) * 32) * 2;
    f.k[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp + off));
  }
#pragma unroll
  for (int n = 0; n < 8; ++n) f.v[n] = __builtin_nontemporal_load(reinterpret_cast<const typename Raw<KV8>::V*>(vp + n * 16 * BLK * ES));
}

struct DAcc {
  f32x4 o[8];
  float m, l;
};

// ctx: every row of the block stands at position ctx - 1, so all rows share one mask.
template <bool KV8>
__device__ __forceinline__ void decode_step(Raw<KV8>& f, const bf16x8 (&qf)[4], int key, bool inside, int ctx, int lo, int sinks,
                                             float scale_log2, DAcc& a) {
  f32x4 s0 = f32x4{0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    bf16x8 k0, k1;
    if constexpr (KV8) {
      const u32x4 r0 = f.k[s >> 1], r1 = f.k[2 + (s >> 1)];
      k0 = (s & 1) ? fp8x8_to_bf16(r0[2], r0[3]) : fp8x8_to_bf16(r0[0], r0[1]);
      k1 = (s & 1) ? fp8x8_to_bf16(r1[2], r1[3]) : fp8x8_to_bf16(r1[0], r1[1]);
    } else {
      k0 = __builtin_bit_cast(bf16x8, f.k[s]);
      k1 = __builtin_bit_cast(bf16x8, f.k[4 + s]);
    }
    s0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, qf[s], s0, 0, 0, 0);
    s1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, qf[s], s1, 0, 0, 0);
  }
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[j] = s0[j] * scale_log2;
    x[j + 4] = s1[j] * scale_log2;
  }
  uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
  if (!inside) {                                            // wave-uniform: the window's two ends and the last sink step
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool see = f.pv >= 0 && key + j < ctx && (key + j >= lo || key + j < sinks);
      x[j] = see ? x[j] : -INFINITY;
      if (!see) keep[j >> 1] &= (j & 1) ? 0xffffu : 0xffff0000u;
    }
  }
  float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
  mx = fmaxf(mx, __shfl_xor(mx, 16));
  mx = fmaxf(mx, __shfl_xor(mx, 32));
  const float m_new = fmaxf(a.m, mx);
  const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
  const float alpha = fast_exp2(a.m - m_use);
  bf16x8 p;
  float rs = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float pj = fast_exp2(x[j] - m_use);
    p[j] = (__bf16)pj;
    rs += pj;
  }
  a.l = a.l * alpha + rs;                                   // this lane's 8 of 32 keys; the four parts are joined at the end
  a.m = m_new;
  if (__ballot(alpha != 1.f) != 0) {
#pragma unroll
    for (int n = 0; n < 8; ++n) a.o[n] *= alpha;
  }
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    u32x4 u;
    if constexpr (KV8) u = __builtin_bit_cast(u32x4, fp8x8_to_bf16(f.v[n][0], f.v[n][1]));
    else u = f.v[n];
    if (!inside) u = u32x4{u[0] & keep[0], u[1] & keep[1], u[2] & keep[2], u[3] & keep[3]};      // a weight of 0 times a NaN would reach the sum
    a.o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, u), p, a.o[n], 0, 0, 0);
  }
}

constexpr int OPAD = HD + 4;

template <bool KV8>
__global__ __launch_bounds__(256, 2) void window_decode_kernel(WinArgs a, int head_tiles) {
  constexpr int HELD = 32;
  __shared__ float sm_o[4][16][OPAD];
  __shared__ float sm_m[4][16], sm_l[4][16];
  const int h = blockIdx.x / head_tiles, ht = blockIdx.x % head_tiles, b = blockIdx.y, split = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int ctx = a.lens[b];
  const int* table = a.tables + (size_t)b * a.width;
  Span sp = make_span(ctx - 1, ctx - 1, a.window, a.sinks, a.width);
  if (ctx <= 0) sp.n = 0;
  const int sps = (sp.n + a.splits - 1) / a.splits;
  const int i0 = split * sps + w, i1 = (split + 1) * sps < sp.n ? (split + 1) * sps : sp.n;      // the wave's steps: i0, i0 + 4, ..
  const int row_head = ht * 16 + fr;
  const bool valid = row_head < a.G;
  // a lane holds one page id of the wave's next HELD steps: the loads of a step wait for no table
  int held = -1;
  const auto hold = [&](int i) {
    const int step = i + (lane >> 1) * 4;
    held = step < i1 ? page_at(table, sp.step(step) * 2 + (lane & 1), a.width, a.pages) : -1;
  };
  DAcc acc;
#pragma unroll
  for (int n = 0; n < 8; ++n) acc.o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  acc.m = -INFINITY;
  acc.l = 0.f;
  if (i0 < i1) {
    hold(i0);
    Raw<KV8> cur, nxt;
    load_raw<KV8>(a, held, 0, h, fr, fq, cur);
    const uint16_t* qrow = a.q + (size_t)b * a.q_stride + ((size_t)h * a.G + (valid ? row_head : 0)) * HD;
    bf16x8 qf[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      // e4m3: a 16-byte K load carries 16 dims = two k-steps of the product, q follows that order
      u32x4 u = u32x4{0, 0, 0, 0};
      if (valid) u = *reinterpret_cast<const u32x4*>(qrow + (KV8 ? (s >> 1) * 64 + fq * 16 + (s & 1) * 8 : s * 32 + fq * 8));
      qf[s] = __builtin_bit_cast(bf16x8, u);
    }
    for (int i = i0, j = 0; i < i1; i += 4) {
      if (++j == HELD) {
        hold(i + 4);
        j = 0;
      }
      if (i + 4 < i1) load_raw<KV8>(a, held, j, h, fr, fq, nxt);
      const int k0 = sp.step(i) << 5, k1 = k0 + 31;
      const bool inside = k1 < ctx && (k0 >= sp.lo || k1 < a.sinks) && __ballot(cur.pv < 0) == 0;
      decode_step<KV8>(cur, qf, k0 + fq * 8, inside, ctx, sp.lo, a.sinks, a.scale_log2, acc);
      cur = nxt;
    }
  }
  acc.l += __shfl_xor(acc.l, 16);
  acc.l += __shfl_xor(acc.l, 32);
#pragma unroll
  for (int n = 0; n < 8; ++n) *reinterpret_cast<f32x4*>(&sm_o[w][fr][n * 16 + fq * 4]) = acc.o[n];
  if (fq == 0) {
    sm_m[w][fr] = acc.m;
    sm_l[w][fr] = acc.l;
  }
  __syncthreads();
  const int row = tid >> 4, d0 = (tid & 15) * 8;
  if (ht * 16 + row < a.G) {
    const float mt = fmaxf(fmaxf(sm_m[0][row], sm_m[1][row]), fmaxf(sm_m[2][row], sm_m[3][row]));
    const float mu = (mt == -INFINITY) ? 0.f : mt;
    float L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ww = 0; ww < 4; ++ww) {
      const float wgt = fast_exp2(sm_m[ww][row] - mu);
      L += sm_l[ww][row] * wgt;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] += sm_o[ww][row][d0 + j] * wgt;
    }
    const size_t head = (size_t)b * a.n_q + (size_t)h * a.G + ht * 16 + row;
    if (a.splits == 1) {
      const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] *= inv;
      *reinterpret_cast<uint4*>(a.out + head * HD + d0) = pack8(o);
    } else {
      float* po = a.part_o + (head * a.splits + split) * HD + d0;
      *reinterpret_cast<f32x4*>(po) = f32x4{o[0], o[1], o[2], o[3]};
      *reinterpret_cast<f32x4*>(po + 4) = f32x4{o[4], o[5], o[6], o[7]};
      if ((tid & 15) == 0) {
        a.part_ml[(head * a.splits + split) * 2] = mt;
        a.part_ml[(head * a.splits + split) * 2 + 1] = L;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Prompts and chunks of prompts. Query rows are (token, head of the kv head's group) pairs in a row; a wave takes QT tiles of
// 16 of them, a block of 4 waves walks the 32-key steps they may see, staged through LDS as bf16. The operand mapping is
// decode's (and llm_attention.hip's): lane (fr, fq) has query row fr and, after S^T = K Q^T, the scores of keys fq*8 .. + 7;
// these are the second operand that O^T = V^T P wants from it, no value changes lanes.
// LDS step: K [32 tokens][16 chunks of 16 bytes], chunk c of token t at c ^ key(t): the 16 rows of a fragment read 16 chunk
// columns. V [page][dims/16][half][dims%16] chunks of 8 tokens: half a wave reads 512 bytes in lane order. Two steps of each: while
// one is worked on the next is brought in, a bf16 cache by LDS-DMA (4 KiB a wave, no registers), an e4m3 cache by LDS-DMA as it
// is and turned into bf16 once per block.
// What bounds it: a step of two tiles is 32 matrix instructions (512 clocks) and 80 vector ones, 16 of them exp2 (400); with three
// waves a SIMD the two come to as long as the step: one is hardly under the other, the waves spend a third of their time at waits.
// Two tiles, because they and their state fit 168 registers, three blocks a CU; three tiles at two blocks a CU, with the scores of a
// step computed under the weights of the one before, took 391 us where this takes 384 (8192 tokens, 32 heads over 8, window 4096:
// 1075 TFLOP/s) and 293 where this takes 260 (e4m3, chunks of a long context). One tile for fewer rows: 128 registers, four blocks a
// CU (e4m3: three, for the 48 KiB of LDS that a block takes). A third step in LDS, wave priorities and sums by matrix instructions
// gave nothing.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int HALF = 8192;      // a step's K, or its V, in LDS

__device__ __forceinline__ int k_key(int tok) { return (tok & 3) | (((tok >> 3) & 3) << 2); }

#define KLM_AS3 __attribute__((address_space(3)))

// A wave brings a quarter of a step, half a page: K tokens 8w .. 8w + 7 (the chunk swizzle is the same for both fours of
// them), V dims 64 (w % 2) .. + 63; `at`: number of the page's block of this kv head in the cache, -1: none; `ko`, `vo`: the lane's
// offsets in bytes inside it. The second half of each lies 1 KiB
// behind the first, in memory as in LDS.
// Written in assembly because the compiler takes the builtin for an access that may hit LDS at any time, and then waits for all
// outstanding LDS reads at each of them (and for the DMA before them); what has landed is said by the kernel's own waits. No
// register is written but m0. s_nop 4: a scalar base that a vector instruction wrote may be
// read by a memory instruction five states later; s_nop 0: m0 before its use.
__device__ __forceinline__ void dma_step(const WinArgs& a, int at, uint32_t st, int w, unsigned ko, unsigned vo) {
  const size_t base = (size_t)(at < 0 ? 0 : at) * (BLK_ELEMS * 2);
  const char* k = (const char*)a.kc + base;
  const char* v = (const char*)a.vc + base;
  asm volatile(
      "s_mov_b32 m0, %4\n\t"
      "s_nop 4\n\t"
      "global_load_lds_dwordx4 %0, %2\n\t"
      "global_load_lds_dwordx4 %0, %2 offset:1024\n\t"
      "s_mov_b32 m0, %5\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %3\n\t"
      "global_load_lds_dwordx4 %1, %3 offset:1024"
      :
      : "v"(ko), "v"(vo), "s"(k), "s"(v), "s"(st + w * 2048), "s"(st + 2 * HALF + w * 2048)
      : "memory", "m0");
}

// The same of an e4m3 cache: a wave's 2 KiB of raw bytes go to a corner of its own, `raw`, from where it turns them into the bf16
// step one step later. A lane's 16 bytes: 16 dims of a key, 16 tokens of a dim.
__device__ __forceinline__ void dma_step8(const WinArgs& a, int at, uint32_t raw, int w, unsigned off) {
  const size_t base = (size_t)(at < 0 ? 0 : at) * BLK_ELEMS + (w & 1) * 1024;
  const char* k = (const char*)a.kc + base;
  const char* v = (const char*)a.vc + base;
  asm volatile(
      "s_mov_b32 m0, %3\n\t"
      "s_nop 4\n\t"
      "global_load_lds_dwordx4 %0, %1\n\t"
      "s_mov_b32 m0, %4\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, %2"
      :
      : "v"(off), "s"(k), "s"(v), "s"(raw), "s"(raw + 1024)
      : "memory", "m0");
}
__device__ __forceinline__ void widen_step8(char* st, const char* raw, int w, int lane) {
  const uint4 k = *reinterpret_cast<const uint4*>(raw + lane * 16), v = *reinterpret_cast<const uint4*>(raw + 1024 + lane * 16);
  const int tok = w * 8 + (lane >> 3), c = (lane & 7) * 2, key = k_key(tok);
  char* kp = st + tok * 256;
  *reinterpret_cast<bf16x8*>(kp + ((c ^ key) << 4)) = fp8x8_to_bf16(k.x, k.y);
  *reinterpret_cast<bf16x8*>(kp + (((c + 1) ^ key) << 4)) = fp8x8_to_bf16(k.z, k.w);
  const int dim = (w & 1) * 64 + lane;
  char* vp = st + 2 * HALF + (w >> 1) * 4096 + (dim >> 4) * 512 + (dim & 15) * 16;
  *reinterpret_cast<bf16x8*>(vp) = fp8x8_to_bf16(v.x, v.y);
  *reinterpret_cast<bf16x8*>(vp + 256) = fp8x8_to_bf16(v.z, v.w);
}

// a row of seq_info that counts: queries inside q, and a context that holds them (rows * G fits 31 bits, see the launcher)
__device__ __forceinline__ bool is_sequence(const WinArgs& a, int q_start, int q_len, int ctx) {
  return q_len > 0 && ctx >= q_len && q_start >= 0 && q_len <= a.rows && q_start <= a.rows - q_len;
}

// Tile t of the launch -> its sequence and its number among the sequence's tiles (seq < 0: the launch has more tiles than
// needed), and how many rows the sequences have together.
__device__ __forceinline__ void find_tile(const WinArgs& a, int rows, int t, int lane, int& seq, int& tile, int& in_use) {
  int base = 0;
  seq = -1;
  tile = 0;
  in_use = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
    const int i = s0 + lane;
    int n = 0, m = 0;
    if (i < a.n_seqs) {
      const int qs = a.lens[i * 3], ql = a.lens[i * 3 + 1], cl = a.lens[i * 3 + 2];
      if (is_sequence(a, qs, ql, cl)) {
        n = (int)(((unsigned)(ql * a.G) + rows - 1) / rows);
        m = ql;
      }
    }
    int inc = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(inc, o);
      if (lane >= o) inc += up;
      if (a.zero_rest) m += __shfl_xor(m, o);
    }
    in_use += __builtin_amdgcn_readfirstlane(m);
    const int total = __builtin_amdgcn_readlane(inc, 63);
    if (seq < 0 && t < base + total) {
      const int first = __builtin_ctzll(__ballot(base + inc > t));
      seq = s0 + first;
      tile = __builtin_amdgcn_readlane(n, first) - 1 - (t - base - __builtin_amdgcn_readlane(inc - n, first));     // latest queries first: they see the most keys
      if (!a.zero_rest) return;
    }
    base += total;
  }
}

// Is `row` one of a sequence's? The same row in all lanes, which look at 64 sequences at a time.
__device__ __forceinline__ bool owned(const WinArgs& a, int row, int lane) {
  bool mine = false;
  for (int i = lane; i < a.n_seqs; i += 64) {
    const int qs = a.lens[i * 3], ql = a.lens[i * 3 + 1];
    mine = mine || (is_sequence(a, qs, ql, a.lens[i * 3 + 2]) && row >= qs && row < qs + ql);
  }
  return __ballot(mine) != 0;
}

// Zeroes the rows from `lo` on, up to 64 of them and below `hi`, that no sequence has, for one kv head's query heads: a lane looks
// at one row, all sequences pass by.
__device__ __forceinline__ void zero_rows(const WinArgs& a, int lo, int hi, int h, int lane) {
  const int row = lo + lane;
  bool mine = row >= hi;
  for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
    int qs = 0, ql = 0;
    if (s0 + lane < a.n_seqs) {
      qs = a.lens[(s0 + lane) * 3];
      ql = a.lens[(s0 + lane) * 3 + 1];
      if (!is_sequence(a, qs, ql, a.lens[(s0 + lane) * 3 + 2])) ql = 0;
    }
    const int n = a.n_seqs - s0 < 64 ? a.n_seqs - s0 : 64;
    for (int j = 0; j < n; ++j) mine = mine || (unsigned)(row - __builtin_amdgcn_readlane(qs, j)) < (unsigned)__builtin_amdgcn_readlane(ql, j);
  }
  for (uint64_t rest = __ballot(!mine); rest != 0; rest &= rest - 1) {
    const size_t head = (size_t)(lo + __builtin_ctzll(rest)) * a.n_q + (size_t)h * a.G;
    for (int e = lane * 8; e < a.G * HD; e += 512) *reinterpret_cast<uint4*>(a.out + head * HD + e) = uint4{0, 0, 0, 0};
  }
}

// A wave's state: QT tiles of 16 query rows, lane (fr, fq) has row fr of each.
template <int QT>
struct Rows {
  bf16x8 q[QT][4];
  f32x4 o[QT][8];
  // weights are exp2(scaled score + shift); a sum of them; the largest exponent that is let through: 8, or -inf before the first key
  float shift[QT], l[QT], lim[QT];
  int pos[QT];
};

// Marks a NaN with 4096, +inf with 1, -inf with 64, all else with 0, as two bf16 numbers.
__device__ __forceinline__ uint32_t odd_marks(uint32_t x) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t e = (x >> (16 * i)) & 0xffffu;
    const uint32_t mark = (e & 0x7f80u) != 0x7f80u ? 0u : (e & 0x7fu) ? 0x4580u : (e >> 15) ? 0x4280u : 0x3f80u;
    r |= mark << (16 * i);
  }
  return r;
}

// The weights of a tile's exponents. The sum is taken of the weights as they are, V meets them rounded to bf16 (half a step, 2^-9,
// of each, as often up as down).
template <int QT>
__device__ __forceinline__ void weights(Rows<QT>& r, const float (&x)[QT][8], int t, bf16x8& p) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float e0 = fast_exp2(x[t][j]), e1 = fast_exp2(x[t][j + 1]);
    p[j] = (__bf16)e0;
    p[j + 1] = (__bf16)e1;
    r.l[t] += e0 + e1;
  }
}

// bit j: the row at `pos` sees key + j, j = 0 .. 7
__device__ __forceinline__ uint32_t seen_bits(const WinArgs& a, int pos, int key) {
  const auto below = [](int n) { return (1u << (n < 0 ? 0 : n > 8 ? 8 : n)) - 1; };         // bits 0 .. n - 1
  return below(pos - key + 1) & (~below(pos - key - a.window + 1) | below(a.sinks - key));
}

// Masks the exponents of a step that some row does not see whole; bit i of `pages`: its page i is there.
template <int QT>
__device__ __forceinline__ void mask_step(const WinArgs& a, int step, int pages, int lane, const Rows<QT>& r, float (&x)[QT][8], float (&mx)[QT]) {
  const int fq = lane >> 4, key = step * 32 + fq * 8;                  // the lane's scores: keys key .. + 7, of one page
  const bool page = (pages >> (fq >> 1)) & 1;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const uint32_t see = page ? seen_bits(a, r.pos[t], key) : 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t all = (uint32_t)((int)(see << (31 - j)) >> 31);
      x[t][j] = __uint_as_float((all & __float_as_uint(x[t][j])) | (~all & 0xff800000u));        // -inf where the bit is not set
      mx[t] = j ? fmaxf(mx[t], x[t][j]) : x[t][j];
    }
  }
}

// The maximum that the weights are relative to is moved only when an exponent passes 8 (a weight of 256): the weights' ratio to
// their sum is what counts, and bf16 keeps it at any size. Most steps then need nothing from another lane.
template <int QT>
__device__ __forceinline__ void move_maximum(Rows<QT>& r, float (&x)[QT][8], float (&mx)[QT]) {
  bool moves = false;
#pragma unroll
  for (int t = 0; t < QT; ++t) moves = moves || mx[t] > r.lim[t];
  if (__ballot(moves) == 0) return;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    if (__ballot(mx[t] > r.lim[t]) == 0) continue;                     // a tile's numbers do not hang on the wave's others
    mx[t] = fmaxf(mx[t], __shfl_xor(mx[t], 16));
    mx[t] = fmaxf(mx[t], __shfl_xor(mx[t], 32));
    const bool first = r.lim[t] < 0.f, seen = mx[t] > -INFINITY;
    const float by = first ? (seen ? mx[t] : 0.f) : fmaxf(mx[t], 0.f);
    const float alpha = first ? 1.f : fast_exp2(-by);
    r.lim[t] = seen ? 8.f : r.lim[t];
    r.shift[t] -= by;
    r.l[t] *= alpha;
#pragma unroll
    for (int n = 0; n < 8; ++n) r.o[t][n] *= alpha;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[t][j] -= by;
  }
}

// The finished rows of one 16-row tile: lane (fr, fq) holds dims n * 16 + fq * 4 .. + 3 of row fr; dst < 0: no row.
__device__ __forceinline__ void write_rows(const WinArgs& a, int64_t dst, int split, int fq, const f32x4 (&o)[8], float m, float l) {
  if (dst < 0) return;
  if (a.splits == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      bf16x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = (__bf16)(o[n][j] * inv);
      *reinterpret_cast<bf16x4*>(a.out + dst * HD + n * 16 + fq * 4) = v;
    }
  } else {
    const size_t at = (size_t)dst * a.splits + split;
#pragma unroll
    for (int n = 0; n < 8; ++n) *reinterpret_cast<f32x4*>(a.part_o + at * HD + n * 16 + fq * 4) = o[n];
    if (fq == 0) {
      a.part_ml[at * 2] = m;
      a.part_ml[at * 2 + 1] = l;
    }
  }
}

// 8 values of the cache as bf16
template <bool KV8>
__device__ __forceinline__ bf16x8 load8(const void* cache, size_t at) {
  if (KV8) {
    const uint2 raw = *reinterpret_cast<const uint2*>((const uint8_t*)cache + at);
    return fp8x8_to_bf16(raw.x, raw.y);
  }
  return *reinterpret_cast<const bf16x8*>((const uint16_t*)cache + at);
}

// One 16-row tile again, from the cache and by itself, where V holds NaN or infinities that some rows see and others do not (a
// weight of 0 times them is NaN): they leave the matrix product, and the rows that see them get them back. Rare and slow: one
// step after another, every load waited for. Each number is made as the fast loop makes it, so what a masked place holds does not
// move a single bit.
template <bool KV8, typename Inside>
__device__ __forceinline__ void careful_tile(const WinArgs& a, const int* table, int h, const Span& sp, int i0, int i1, int split, int lane,
                                             const uint16_t* qrow, int pos, int64_t dst, const Inside& is_inside) {
  const int fr = lane & 15, fq = lane >> 4;
  Rows<1> r;
  r.pos[0] = pos;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint4 u = uint4{0, 0, 0, 0};
    if (dst >= 0) u = *reinterpret_cast<const uint4*>(qrow + c * 32 + fq * 8);
    r.q[0][c] = __builtin_bit_cast(bf16x8, u);
  }
#pragma unroll
  for (int n = 0; n < 8; ++n) r.o[0][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  r.lim[0] = -INFINITY;
  r.shift[0] = 0.f;
  r.l[0] = 0.f;
#pragma unroll 1
  for (int i = i0; i < i1; ++i) {
    const int step = sp.step(i), key = step * 32 + fq * 8;
    const int p0 = page_at(table, step * 2, a.width, a.pages), p1 = page_at(table, step * 2 + 1, a.width, a.pages);
    const int pages = (p0 >= 0 ? 1 : 0) | (p1 >= 0 ? 2 : 0);
    const size_t b0 = ((size_t)(p0 < 0 ? 0 : p0) * a.n_kv + h) * BLK_ELEMS, b1 = ((size_t)(p1 < 0 ? 0 : p1) * a.n_kv + h) * BLK_ELEMS;
    const size_t ko = ((fr >> 3) ? b1 : b0) + ((((fr >> 2) & 1) << 3) + (fr & 3)) * HD + fq * 8;
    const size_t vo = ((fq >> 1) ? b1 : b0) + fr * BLK + (fq & 1) * 8;
    f32x4 s0 = f32x4{0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      s0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(load8<KV8>(a.kc, ko + c * 32), r.q[0][c], s0, 0, 0, 0);
      s1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(load8<KV8>(a.kc, ko + 4 * HD + c * 32), r.q[0][c], s1, 0, 0, 0);
    }
    float x[1][8], mx[1];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[0][j] = fmaf(j < 4 ? s0[j & 3] : s1[j & 3], a.scale_log2, r.shift[0]);
    mx[0] = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), fmaxf(fmaxf(x[0][4], x[0][5]), fmaxf(x[0][6], x[0][7])));
    if (!is_inside(i, pages)) mask_step<1>(a, step, pages, lane, r, x, mx);
    move_maximum<1>(r, x, mx);
    const uint32_t see = (pages >> (fq >> 1)) & 1 ? seen_bits(a, pos, key) : 0u;
    bf16x8 p;
    uint32_t ones[4] = {0u, 0u, 0u, 0u};                               // 1 for a key that the row sees, as bf16 pairs
#pragma unroll
    for (int j = 0; j < 8; ++j) ones[j >> 1] |= ((see >> j) & 1) * 0x3f80u << (16 * (j & 1));
    const bf16x8 one = __builtin_bit_cast(bf16x8, uint4{ones[0], ones[1], ones[2], ones[3]});
    weights<1>(r, x, 0, p);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const uint4 u = __builtin_bit_cast(uint4, load8<KV8>(a.vc, vo + n * 16 * BLK));
      const bf16x8 marks = __builtin_bit_cast(bf16x8, uint4{odd_marks(u.x), odd_marks(u.y), odd_marks(u.z), odd_marks(u.w)});
      const bf16x8 v = __builtin_bit_cast(bf16x8, uint4{without_odd(u.x), without_odd(u.y), without_odd(u.z), without_odd(u.w)});
      // how many of them each row sees in each dim: exact in fp32
      const f32x4 c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(marks, one, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
      r.o[0][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p, r.o[0][n], 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int all = (int)c[j], neg = (all >> 6) & 63, inf = all & 63;
        if (all) r.o[0][n][j] += all >= 4096 || (neg && inf) ? NAN : neg ? -INFINITY : INFINITY;
      }
    }
  }
  r.l[0] += __shfl_xor(r.l[0], 16);
  r.l[0] += __shfl_xor(r.l[0], 32);
  write_rows(a, dst, split, fq, r.o[0], r.lim[0] > 0.f ? -r.shift[0] : -INFINITY, r.l[0]);
}

template <int QT, bool KV8>
__global__ __launch_bounds__(256, QT == 1 && !KV8 ? 4 : 3) void window_prefill_kernel(WinArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int h = blockIdx.x, split = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  constexpr int ROWS = 64 * QT;
  int seq, tile, in_use;
  find_tile(a, ROWS, blockIdx.y, lane, seq, tile, in_use);
  if (a.zero_rest && a.splits == 1 && in_use < a.rows) {               // this block's share of the rows that may be nobody's
    const int share = (a.rows + gridDim.y - 1) / gridDim.y, lo = blockIdx.y * share, hi = lo + share < a.rows ? lo + share : a.rows;
    for (int row = lo + w * 64; row < hi; row += 256) zero_rows(a, row, hi, h, lane);
  }
  if (seq < 0) return;
  const int q_start = a.lens[seq * 3], q_len = a.lens[seq * 3 + 1], ctx = a.lens[seq * 3 + 2];
  const int* table = a.tables + (size_t)seq * a.width;
  const int first = ctx - q_len;                                       // position of the sequence's first query
  const unsigned G = a.G, r0 = (unsigned)tile * ROWS;
  // (readfirstlane: these are the same in all lanes, and the branches on them are to stay scalar)
  const int tok_a = __builtin_amdgcn_readfirstlane(r0 / G), tb = __builtin_amdgcn_readfirstlane((r0 + ROWS - 1) / G), tok_b = tb < q_len ? tb : q_len - 1;
  const Span sp = make_span(first + tok_a, first + tok_b, a.window, a.sinks, a.width);
  const int sps = (sp.n + a.splits - 1) / a.splits;
  const int i0 = split * sps, i1 = (i0 + sps) < sp.n ? (i0 + sps) : sp.n;

  Rows<QT> r;
  // row fr of tile t: its token (>= q_len: none) and head of the group
  const auto row_of = [&](int t, int& token, int& g) {
    const unsigned R = r0 + (w * QT + t) * 16 + fr;
    token = R / G;
    g = R - (unsigned)token * G;
  };
  const unsigned ra = r0 + w * QT * 16;                                // the wave's first and last position; of no rows: nothing is inside
  const int ta = __builtin_amdgcn_readfirstlane(ra / G), tz = __builtin_amdgcn_readfirstlane((ra + QT * 16 - 1) / G);
  const int pmin = ta < q_len ? first + ta : -1, pmax = first + (tz < q_len ? tz : q_len - 1);
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    int token, g;
    row_of(t, token, g);
    const bool valid = token < q_len;
    r.pos[t] = valid ? first + token : -1;                             // a row that is none sees nothing
    const uint16_t* qp = a.q + (valid ? (size_t)(q_start + token) * a.q_stride + ((size_t)h * G + g) * HD : 0);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (valid) r.q[t][s] = *reinterpret_cast<const bf16x8*>(qp + s * 32 + fq * 8);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) r.q[t][s][j] = (__bf16)0.f;
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) r.o[t][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    r.lim[t] = -INFINITY;
    r.shift[t] = 0.f;
    r.l[t] = 0.f;
  }

  // Does every row of the wave see all of step i? (Rows that are none see what they like then: they are not written.) Of the sinks'
  // steps the first `in_sinks`, of the window's those from in_a to in_b.
  const int whole = (pmin + 1) >> 5, in_sinks = (a.sinks >> 5) < whole ? (a.sinks >> 5) : whole;
  const int in_a = (pmax < a.window ? 0 : ((pmax - a.window) >> 5) + 1) - sp.lo_step + sp.n_sink, in_b = whole - sp.lo_step + sp.n_sink;
  const auto is_inside = [&](int i, int pages) {
    return pages == 3 && (i < sp.n_sink ? i < in_sinks : i >= in_a && i < in_b);
  };
  const bool nobody = ta >= q_len;                                     // the wave has no rows: it brings its part of the cache and no more
  if (i0 < i1) {
    const int last = i1 - 1;
    const int tok = w * 8 + (lane >> 4);
    const unsigned ko = (tok & 15) * 256 + (((lane & 15) ^ k_key(tok)) << 4);
    const unsigned vo = ((w & 1) * 64 + (lane >> 5) * 16 + (lane & 15)) * 32 + ((lane >> 4) & 1) * 16;
    // The table's entries for 32 steps at a time lie in one register, a lane each: looking them up in the loop through the scalar
    // cache would share the LDS reads' counter and make every wait on them a wait for all of them. They are numbers of this kv
    // head's blocks in the cache, -1: no page. `there`: which of them are pages.
    int held;
    uint64_t there;
    const auto hold = [&](int i) {                                     // steps i .. i + 31; past the last step: that one again, unused
      const int at = i + (lane >> 1), e = sp.step(at < last ? at : last) * 2 + (lane & 1);
      const int id = table[e < a.width ? e : a.width - 1];
      held = e < a.width && (unsigned)id < (unsigned)a.pages ? id * a.n_kv + h : -1;
      there = __ballot(held >= 0);
    };
    const auto mine_at = [&](int at) { return __builtin_amdgcn_readlane(held, (at & 31) * 2 + (w >> 1)); };       // what this wave brings of step i0 + at
    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((KLM_AS3 char*)lds);
    // e4m3: two raw corners a wave behind the bf16 steps; step i + 1 is widened at step i, while i + 2 lands in the other corner
    const uint32_t raw0 = lds0 + 4 * HALF + w * 2048;
    const char* const raws = lds + 4 * HALF + w * 2048;
    hold(i0);
    if (KV8) {
      dma_step8(a, mine_at(0), raw0, w, lane * 16);
      dma_step8(a, mine_at(1), raw0 + HALF, w, lane * 16);
      asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
      widen_step8(lds, raws, w, lane);
    } else {
      dma_step(a, mine_at(0), lds0, w, ko, vo);
    }
    uint64_t pages = there;                                            // the step's two in its lowest bits
    for (int i = i0; i < i1; ++i) {
      const int at = i - i0, cur = (at & 1) * HALF, other = HALF - cur;
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");      // what was brought, and widened, during the last step
      __builtin_amdgcn_s_barrier();                                    // ... by all waves, and all have left the step before
      asm volatile("" ::: "memory");
      const int now = pages & 3;
      pages >>= 2;
      if (KV8) {
        if (((at + 1) & 31) == 0) pages = there;                       // (held one step ago)
        if (((at + 2) & 31) == 0) hold(i + 2);
        dma_step8(a, mine_at(at + 2), raw0 + cur, w, lane * 16);       // the corner was read one step ago
        widen_step8(lds + other, raws + other, w, lane);
      } else {
        if (((at + 1) & 31) == 0) {
          hold(i + 1);
          pages = there;
        }
        dma_step(a, mine_at(at + 1), lds0 + other, w, ko, vo);
      }
      if (nobody) continue;
      const char* kp = lds + cur + ((fr >> 2) * 8 + (fr & 3)) * 256;   // k_key of both tokens below is fr
      const char* vst = lds + 2 * HALF + cur;
      const bool inside = is_inside(i, now);
      float x[QT][8], mx[QT];
      {
        f32x4 s[QT][2];
#pragma unroll
        for (int t = 0; t < QT; ++t) s[t][0] = s[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const bf16x8 k0 = *reinterpret_cast<const bf16x8*>(kp + (((c * 4 + fq) ^ fr) << 4));
          const bf16x8 k1 = *reinterpret_cast<const bf16x8*>(kp + 1024 + (((c * 4 + fq) ^ fr) << 4));
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            s[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, r.q[t][c], s[t][0], 0, 0, 0);
            s[t][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, r.q[t][c], s[t][1], 0, 0, 0);
          }
        }
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            x[t][j] = fmaf(j < 4 ? s[t][0][j & 3] : s[t][1][j & 3], a.scale_log2, r.shift[t]);
            mx[t] = j ? fmaxf(mx[t], x[t][j]) : x[t][j];
          }
      }
      if (!inside) mask_step<QT>(a, sp.step(i), now, lane, r, x, mx);
      move_maximum<QT>(r, x, mx);
      bf16x8 p[QT];
#pragma unroll
      for (int t = 0; t < QT; ++t) weights<QT>(r, x, t, p[t]);
      const char* vp = vst + (fq >> 1) * 4096 + (lane & 31) * 16;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const bf16x8 v = *reinterpret_cast<const bf16x8*>(vp + n * 512);
#pragma unroll
        for (int t = 0; t < QT; ++t) r.o[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[t], r.o[t][n], 0, 0, 0);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                   // the last, unused steps land before the LDS goes away
  }

  // a NaN in a row's sums: was it the row's to see?
  unsigned odd = 0;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    float any = 0.f;
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) any = fmaf(r.o[t][n][j], 0.f, any);
    odd |= __ballot(r.pos[t] >= 0 && any != 0.f) ? 1u << t : 0u;
  }
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    r.l[t] += __shfl_xor(r.l[t], 16);
    r.l[t] += __shfl_xor(r.l[t], 32);
    int token, g;
    row_of(t, token, g);
    const int64_t dst = token < q_len ? (int64_t)((size_t)(q_start + token) * a.n_q + (size_t)h * G + g) : -1;
    if (((odd >> t) & 1) == 0) write_rows(a, dst, split, fq, r.o[t], r.lim[t] > 0.f ? -r.shift[t] : -INFINITY, r.l[t]);
  }
#pragma unroll 1
  for (; odd; odd &= odd - 1) {
    int token, g;
    row_of(__builtin_ctz(odd), token, g);
    const bool valid = token < q_len;
    const size_t row = q_start + (valid ? token : 0), head = (size_t)h * G + g;
    careful_tile<KV8>(a, table, h, sp, i0, i1, split, lane, a.q + row * a.q_stride + head * HD, valid ? first + token : -1,
                      valid ? (int64_t)(row * a.n_q + head) : -1, is_inside);
  }
}

// Joins the splits' parts: one wave per (row, query head), two dims a lane.
template <bool PREFILL>
__global__ __launch_bounds__(256) void window_join_kernel(WinArgs a) {
  const int lane = threadIdx.x & 63, row = blockIdx.y;
  const int h = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (h >= a.n_q) return;
  const size_t head = (size_t)row * a.n_q + h;
  uint32_t* out = reinterpret_cast<uint32_t*>(a.out + head * HD) + lane;
  if (PREFILL && !owned(a, row, lane)) {                               // its parts were not written
    if (a.zero_rest) *out = 0;
    return;
  }
  const float* ml = a.part_ml + head * a.splits * 2;
  float mt = -INFINITY;
  for (int s = lane; s < a.splits; s += 64) mt = fmaxf(mt, ml[s * 2]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor(mt, o));
  const float mu = (mt == -INFINITY) ? 0.f : mt;
  const float2* po = reinterpret_cast<const float2*>(a.part_o + head * a.splits * HD) + lane;
  float L = 0.f, x = 0.f, y = 0.f;
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float wgt = fast_exp2(ml[s * 2] - mu);
    const float2 v = po[s * (HD / 2)];
    L += ml[s * 2 + 1] * wgt;
    x += v.x * wgt;
    y += v.y * wgt;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  *out = (uint32_t)f2bf(x * inv) | ((uint32_t)f2bf(y * inv) << 16);
}

int check_args(const WinArgs& a) {
  if (a.rows <= 0 || a.n_seqs <= 0 || a.n_seqs > 65535 || a.n_q <= 0 || a.n_kv <= 0 || a.n_q % a.n_kv != 0 || a.width <= 0 || a.pages <= 0 ||
      a.q_stride < a.n_q * HD || a.q_stride % 8 != 0 || a.width > INT32_MAX / BLK - 2 ||
      (int64_t)a.pages * a.n_kv > INT32_MAX)
    return KLM_ERR_SHAPE;
  if (a.window < 1 || a.window > (1 << 30) || a.sinks < 0 || a.sinks > (1 << 30) || a.splits < 1 || a.splits > 256 || !(a.scale_log2 > 0.f))
    return KLM_ERR_ARG;
  if (!a.q || !a.kc || !a.vc || !a.tables || !a.lens || !a.out || (a.splits > 1 && (!a.part_o || !a.part_ml))) return KLM_ERR_ARG;
  if (!aligned16(a.q) || !aligned16(a.kc) || !aligned16(a.vc) || !aligned16(a.out) || !aligned16(a.part_o)) return KLM_ERR_ALIGN;
  return KLM_OK;
}

WinArgs device_args(const klm_window_args* c) {
  return WinArgs{(const uint16_t*)c->q, c->k_cache, c->v_cache, c->tables, c->lens, (uint16_t*)c->out, c->part_o, c->part_ml,
                 c->n_seqs, c->rows, c->q_stride, c->n_q, c->n_kv, c->n_kv > 0 ? c->n_q / c->n_kv : 0, c->width, c->pages,
                 c->window, c->sinks, c->splits, c->zero_rest, c->scale * 1.4426950408889634f};
}

template <bool PREFILL>
int launch_join(const WinArgs& a, hipStream_t s) {
  if (hipGetLastError() != hipSuccess) return KLM_ERR_HIP;
  if (a.splits > 1) hipLaunchKernelGGL(window_join_kernel<PREFILL>, dim3((a.n_q + 3) / 4, a.rows), dim3(256), 0, s, a);
  return launch_status();
}

template <int QT, bool KV8>
int launch_prefill(const WinArgs& a, hipStream_t s) {
  constexpr int LDS = (KV8 ? 6 : 4) * HALF;
  const int64_t tiles = ((int64_t)a.rows * a.G + 64 * QT - 1) / (64 * QT) + a.n_seqs;       // every sequence may end in a partial tile
  if (tiles > 65535 || (int64_t)a.rows * a.G > (1 << 30) || (a.splits > 1 && a.rows > 65535)) return KLM_ERR_SHAPE;
  if (klm_ensure_dyn_lds<window_prefill_kernel<QT, KV8>>(LDS) != KLM_OK) return KLM_ERR_HIP;
  hipLaunchKernelGGL((window_prefill_kernel<QT, KV8>), dim3(a.n_kv, (unsigned)tiles, a.splits), dim3(256), LDS, s, a);
  return launch_join<true>(a, s);
}

}  // namespace

extern "C" {

int klm_window_attn_decode(const klm_window_args* c) {
  if (!c) return KLM_ERR_ARG;
  const WinArgs a = device_args(c);
  const int rc = check_args(a);
  if (rc != KLM_OK) return rc;
  if (a.n_seqs != a.rows) return KLM_ERR_SHAPE;
  const int head_tiles = (a.G + 15) / 16;
  hipStream_t s = static_cast<hipStream_t>(c->stream);
  const dim3 grid(a.n_kv * head_tiles, a.rows, a.splits);
  if (c->kv_fp8) hipLaunchKernelGGL(window_decode_kernel<true>, grid, dim3(256), 0, s, a, head_tiles);
  else hipLaunchKernelGGL(window_decode_kernel<false>, grid, dim3(256), 0, s, a, head_tiles);
  return launch_join<false>(a, s);
}

int klm_window_attn_prefill(const klm_window_args* c) {
  if (!c) return KLM_ERR_ARG;
  const WinArgs a = device_args(c);
  const int rc = check_args(a);
  if (rc != KLM_OK) return rc;
  hipStream_t s = static_cast<hipStream_t>(c->stream);
  switch (c->q_tiles) {
    case 1: return c->kv_fp8 ? launch_prefill<1, true>(a, s) : launch_prefill<1, false>(a, s);
    case 2: return c->kv_fp8 ? launch_prefill<2, true>(a, s) : launch_prefill<2, false>(a, s);
    default: return KLM_ERR_VARIANT;
  }
}

}  // extern "C"
