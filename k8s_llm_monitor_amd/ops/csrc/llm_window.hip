// Attention with a sliding window and sinks over the paged KV cache (layouts: llm_attention.hip).
//
//   o[t, h] = sum_j p_j v_j,  p = softmax over the keys j that token t sees of  scale * q[t, h] . k_j
//   the token at position p sees key j  <=>  j <= p  and  (j > p - window  or  j < sinks)  and j's page exists
//
// A page id outside the cache is no page: nothing is read through it, its tokens are not seen. Pages that lie between the
// sinks and the window are never looked at, so the engine gives them back while the sequence runs. A row that sees nothing
// gives 0. A masked key contributes nothing whatever its bytes are (stale slots, NaN, infinities).
//
// No reference counterpart (vLLM is a README bullet in the reference, README.md:73).
#include "klm_launch.h"
#include "llm_common.h"

using namespace klm_llm;

typedef __attribute__((ext_vector_type(16))) float f32x16;

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
  float scale_log2;
};

// The keys a span of queries at positions [pos_a, pos_b] may see, as 32-key steps: the sinks' steps, then the window's.
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
// One token per sequence. Block = (16 query heads of a kv head, sequence, split); its 4 waves take the 32-key steps of the
// split in turn, K and V^T fragments straight from the cache into matrix operands (see llm_attention.hip for the operand
// mapping), the next step's 16 KiB in flight.
// ---------------------------------------------------------------------------------------------------------------------
struct DFrags {
  bf16x8 k[2][4];
  bf16x8 v[8];
  int p0, p1;            // the step's two pages, -1: none
};

template <bool KV8>
__device__ __forceinline__ void load_step(const WinArgs& a, const int* table, int h, int step, int fr, int fq, DFrags& f) {
  f.p0 = page_at(table, step * 2, a.width, a.pages);
  f.p1 = page_at(table, step * 2 + 1, a.width, a.pages);
  const size_t b0 = ((size_t)(f.p0 < 0 ? 0 : f.p0) * a.n_kv + h) * BLK_ELEMS, b1 = ((size_t)(f.p1 < 0 ? 0 : f.p1) * a.n_kv + h) * BLK_ELEMS;
  const size_t ko = ((fr >> 3) ? b1 : b0) + ((((fr >> 2) & 1) << 3) + (fr & 3)) * HD;
  const size_t vo = ((fq >> 1) ? b1 : b0) + fr * BLK + (fq & 1) * 8;
  if (KV8) {
    const uint8_t* kp = (const uint8_t*)a.kc + ko + fq * 16;
    const uint8_t* vp = (const uint8_t*)a.vc + vo;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {
        const uint4 raw = *reinterpret_cast<const uint4*>(kp + t * 4 * HD + h2 * 64);
        f.k[t][2 * h2] = fp8x8_to_bf16(raw.x, raw.y);
        f.k[t][2 * h2 + 1] = fp8x8_to_bf16(raw.z, raw.w);
      }
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const uint2 raw = *reinterpret_cast<const uint2*>(vp + n * 16 * BLK);
      f.v[n] = fp8x8_to_bf16(raw.x, raw.y);
    }
  } else {
    const uint16_t* kp = (const uint16_t*)a.kc + ko + fq * 8;
    const uint16_t* vp = (const uint16_t*)a.vc + vo;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < 4; ++s) f.k[t][s] = *reinterpret_cast<const bf16x8*>(kp + t * 4 * HD + s * 32);
#pragma unroll
    for (int n = 0; n < 8; ++n) f.v[n] = *reinterpret_cast<const bf16x8*>(vp + n * 16 * BLK);
  }
}

struct DAcc {
  f32x4 o[8];
  float m, l;
};

// ctx: every row of the block stands at position ctx - 1, so all rows share one mask
__device__ __forceinline__ void decode_step(DFrags& f, const bf16x8 (&qf)[4], int step, int fq, int ctx, int lo, int sinks,
                                            float scale_log2, DAcc& a) {
  f32x4 s0 = f32x4{0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    s0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.k[0][s], qf[s], s0, 0, 0, 0);
    s1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.k[1][s], qf[s], s1, 0, 0, 0);
  }
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[j] = s0[j];
    x[j + 4] = s1[j];
  }
  const int k0 = step * 32;
  const bool inside = k0 + 31 < ctx && (k0 >= lo || k0 + 31 < sinks) && f.p0 >= 0 && f.p1 >= 0;
  if (!inside) {                                            // wave-uniform: the window's two ends and the last sink step
    const int tk = k0 + fq * 8;
    const bool page = ((fq >> 1) ? f.p1 : f.p0) >= 0;
    uint32_t keep[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool see = page && tk + j < ctx && (tk + j >= lo || tk + j < sinks);
      x[j] = see ? x[j] : -INFINITY;
      keep[j >> 1] |= see ? (0xffffu << (16 * (j & 1))) : 0u;
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) {                           // a weight of 0 times a NaN would reach the sum: masked values go
      uint4 u = __builtin_bit_cast(uint4, f.v[n]);
      u = uint4{u.x & keep[0], u.y & keep[1], u.z & keep[2], u.w & keep[3]};
      f.v[n] = __builtin_bit_cast(bf16x8, u);
    }
  }
  float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
  mx = fmaxf(mx, __shfl_xor(mx, 16));
  mx = fmaxf(mx, __shfl_xor(mx, 32));
  const float m_new = fmaxf(a.m, mx * scale_log2);
  const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
  const float alpha = fast_exp2(a.m - m_use);
  bf16x8 p;
  float rs = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float pj = fast_exp2(fmaf(x[j], scale_log2, -m_use));
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
  for (int n = 0; n < 8; ++n) a.o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.v[n], p, a.o[n], 0, 0, 0);
}

constexpr int OPAD = HD + 4;

template <bool KV8>
__global__ __launch_bounds__(256) void window_decode_kernel(WinArgs a, int head_tiles) {
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
  const int i0 = split * sps, i1 = (i0 + sps) < sp.n ? (i0 + sps) : sp.n;
  const int row_head = ht * 16 + fr;
  const bool valid = row_head < a.G;
  const uint16_t* qrow = a.q + (size_t)b * a.q_stride + ((size_t)h * a.G + (valid ? row_head : 0)) * HD;
  bf16x8 qf[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    // fp8: a 16-byte K load carries 16 dims = two k-steps of the product, q follows that order
    if (valid) qf[s] = *reinterpret_cast<const bf16x8*>(qrow + (KV8 ? (s >> 1) * 64 + fq * 16 + (s & 1) * 8 : s * 32 + fq * 8));
    else
#pragma unroll
      for (int j = 0; j < 8; ++j) qf[s][j] = (__bf16)0.f;
  }
  DAcc acc;
#pragma unroll
  for (int n = 0; n < 8; ++n) acc.o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  acc.m = -INFINITY;
  acc.l = 0.f;
  if (i0 + w < i1) {
    DFrags cur;
    load_step<KV8>(a, table, h, sp.step(i0 + w), fr, fq, cur);
    for (int i = i0 + w; i < i1; i += 4) {
      DFrags nxt;
      load_step<KV8>(a, table, h, sp.step(i + 4 < i1 ? i + 4 : i), fr, fq, nxt);
      decode_step(cur, qf, sp.step(i), fq, ctx, sp.lo, a.sinks, a.scale_log2, acc);
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

// Joins the splits' parts: one wave per (row, query head), two dims a lane.
__global__ __launch_bounds__(256) void window_join_kernel(WinArgs a, size_t n_heads) {
  const int lane = threadIdx.x & 63;
  const size_t head = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (head >= n_heads) return;
  const float* ml = a.part_ml + head * a.splits * 2;
  float mt = -INFINITY;
  for (int s = lane; s < a.splits; s += 64) mt = fmaxf(mt, ml[s * 2]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor(mt, o));
  const float mu = (mt == -INFINITY) ? 0.f : mt;
  const float2* po = reinterpret_cast<const float2*>(a.part_o + head * a.splits * HD) + lane;
  float L = 0.f, x = 0.f, y = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float wgt = fast_exp2(ml[s * 2] - mu);
    const float2 v = po[s * (HD / 2)];
    L += ml[s * 2 + 1] * wgt;
    x += v.x * wgt;
    y += v.y * wgt;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  reinterpret_cast<uint32_t*>(a.out + head * HD)[lane] = (uint32_t)f2bf(x * inv) | ((uint32_t)f2bf(y * inv) << 16);
}

// ---------------------------------------------------------------------------------------------------------------------
// Prompts and chunks of prompts. Query rows are (token, head of the kv head's group) pairs in a row; a block takes 128 * QT
// of them (4 waves of QT 32-row tiles) and walks the 32-key steps they may see, staged through LDS as bf16.
//   S^T = K Q^T with v_mfma_f32_32x32x16_bf16: first operand lane l = row l%32, k = (l/32)*8 ..+8; result lane l = column
//   (query row) l%32, register i = row 8*(i/4) + 4*(l/32) + i%4. Row r of the K operand holds token
//   16*(r/16) + 8*bit2(r) + 4*bit3(r) + r%4, so that lane l ends up with the scores of tokens 8*(l/32) .. +8 of page 0
//   (registers 0..7) and of page 1 (8..15): the second operand that O^T = V^T P wants from it, no value changes lanes.
// LDS step: K [32 tokens][16 chunks of 16 bytes], chunk c of token t at c ^ key(t); V [page][dims/32][half][dims%32] chunks of
// 8 tokens, so that a fragment is 1 KiB in lane order.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int STEP_BYTES = 16384;

__device__ __forceinline__ int k_key(int tok) { return (tok & 3) | (((tok >> 3) & 1) << 2) | (((tok >> 2) & 1) << 3); }

template <bool KV8>
struct Stage {
  uint4 r[KV8 ? 2 : 4];
};

template <bool KV8>
__device__ __forceinline__ void stage_load(const WinArgs& a, const int* table, int h, int step, int tid, Stage<KV8>& s) {
  const int p0 = page_at(table, step * 2, a.width, a.pages), p1 = page_at(table, step * 2 + 1, a.width, a.pages);
  const size_t b0 = ((size_t)(p0 < 0 ? 0 : p0) * a.n_kv + h) * BLK_ELEMS, b1 = ((size_t)(p1 < 0 ? 0 : p1) * a.n_kv + h) * BLK_ELEMS;
  if (KV8) {
    const size_t o = ((tid >> 7) ? b1 : b0) + (tid & 127) * 16;
    s.r[0] = *reinterpret_cast<const uint4*>((const uint8_t*)a.kc + o);
    s.r[1] = *reinterpret_cast<const uint4*>((const uint8_t*)a.vc + o);
  } else {
    const int e = tid * 8;
    s.r[0] = *reinterpret_cast<const uint4*>((const uint16_t*)a.kc + b0 + e);
    s.r[1] = *reinterpret_cast<const uint4*>((const uint16_t*)a.kc + b1 + e);
    s.r[2] = *reinterpret_cast<const uint4*>((const uint16_t*)a.vc + b0 + e);
    s.r[3] = *reinterpret_cast<const uint4*>((const uint16_t*)a.vc + b1 + e);
  }
}

template <bool KV8>
__device__ __forceinline__ void stage_store(char* st, int tid, const Stage<KV8>& s) {
  if (KV8) {
    const int tok = tid >> 3, c = (tid & 7) * 2, key = k_key(tok & 15);
    char* kp = st + tok * 256;
    *reinterpret_cast<bf16x8*>(kp + ((c ^ key) << 4)) = fp8x8_to_bf16(s.r[0].x, s.r[0].y);
    *reinterpret_cast<bf16x8*>(kp + (((c + 1) ^ key) << 4)) = fp8x8_to_bf16(s.r[0].z, s.r[0].w);
    const int page = tid >> 7, dim = tid & 127;
    char* vp = st + 8192 + page * 4096 + (dim >> 5) * 1024 + (dim & 31) * 16;
    *reinterpret_cast<bf16x8*>(vp) = fp8x8_to_bf16(s.r[1].x, s.r[1].y);
    *reinterpret_cast<bf16x8*>(vp + 512) = fp8x8_to_bf16(s.r[1].z, s.r[1].w);
  } else {
    const int tok = tid >> 4, c = tid & 15;
    const int ko = tok * 256 + ((c ^ k_key(tok)) << 4);
    *reinterpret_cast<uint4*>(st + ko) = s.r[0];
    *reinterpret_cast<uint4*>(st + 4096 + ko) = s.r[1];
    const int dim = tid >> 1, half = tid & 1;
    char* vp = st + 8192 + (dim >> 5) * 1024 + half * 512 + (dim & 31) * 16;
    *reinterpret_cast<uint4*>(vp) = s.r[2];
    *reinterpret_cast<uint4*>(vp + 4096) = s.r[3];
  }
}

// tile t of the launch -> its sequence and its number among the sequence's tiles; false: the launch has more tiles than needed
__device__ __forceinline__ bool find_tile(const WinArgs& a, int rows, int t, int lane, int& seq, int& tile) {
  int base = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
    const int i = s0 + lane;
    int n = 0;
    if (i < a.n_seqs) {
      const int ql = a.lens[i * 3 + 1], cl = a.lens[i * 3 + 2];
      if (ql > 0 && cl >= ql) n = (int)(((int64_t)ql * a.G + rows - 1) / rows);
    }
    int inc = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(inc, o);
      if (lane >= o) inc += up;
    }
    const int total = __shfl(inc, 63);
    if (t < base + total) {
      const int first = __builtin_ctzll(__ballot(base + inc > t));
      seq = s0 + first;
      tile = __shfl(n, first) - 1 - (t - base - __shfl(inc - n, first));       // latest queries first: they see the most keys
      seq = __builtin_amdgcn_readfirstlane(seq);
      tile = __builtin_amdgcn_readfirstlane(tile);
      return true;
    }
    base += total;
  }
  return false;
}

template <int QT, bool KV8>
__global__ __launch_bounds__(256) void window_prefill_kernel(WinArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int h = blockIdx.x, split = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, hi = lane >> 5;
  constexpr int ROWS = 128 * QT;
  int seq, tile;
  if (!find_tile(a, ROWS, blockIdx.y, lane, seq, tile)) return;
  const int q_start = a.lens[seq * 3], q_len = a.lens[seq * 3 + 1], ctx = a.lens[seq * 3 + 2];
  const int* table = a.tables + (size_t)seq * a.width;
  const int first = ctx - q_len;                                       // position of the sequence's first query
  const int64_t r0 = (int64_t)tile * ROWS;
  const int tok_a = (int)(r0 / a.G);
  const int64_t tb = (r0 + ROWS - 1) / a.G;
  const int tok_b = tb < q_len ? (int)tb : q_len - 1;
  const Span sp = make_span(first + tok_a, first + tok_b, a.window, a.sinks, a.width);
  const int sps = (sp.n + a.splits - 1) / a.splits;
  const int i0 = split * sps, i1 = (i0 + sps) < sp.n ? (i0 + sps) : sp.n;

  bf16x8 qf[QT][8];
  f32x16 o[QT][4];
  float m[QT], l[QT];
  int pos[QT];
  int64_t dst[QT];
  int pmin[QT], pmax[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int64_t R = r0 + (w * QT + t) * 32;
    const int64_t tq = (R + col) / a.G;
    const int g = (int)((R + col) % a.G);
    const int64_t qrow = q_start + tq;
    const bool valid = tq < q_len && qrow >= 0 && qrow < a.rows;
    pos[t] = valid ? first + (int)tq : -1;
    dst[t] = valid ? (qrow * a.n_q + (int64_t)h * a.G + g) : -1;
    const uint16_t* qp = a.q + (valid ? qrow * a.q_stride + ((int64_t)h * a.G + g) * HD : 0);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      if (valid) qf[t][s] = *reinterpret_cast<const bf16x8*>(qp + s * 16 + hi * 8);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) qf[t][s][j] = (__bf16)0.f;
    }
    const int64_t ta = R / a.G, tz = (R + 31) / a.G;                   // wave-uniform: the tile's first and last position
    pmin[t] = ta < q_len ? first + (int)ta : 0x7fffffff;               // past the queries: sees nothing, skips every step
    pmax[t] = ta < q_len ? first + (int)(tz < q_len ? tz : q_len - 1) : -1;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[t][n][i] = 0.f;
    m[t] = -INFINITY;
    l[t] = 0.f;
  }

  Stage<KV8> sg;
  if (i0 < i1) stage_load<KV8>(a, table, h, sp.step(i0), tid, sg);
  for (int i = i0; i < i1; ++i) {
    char* st = lds + ((i - i0) & 1) * STEP_BYTES;
    stage_store<KV8>(st, tid, sg);
    if (i + 1 < i1) stage_load<KV8>(a, table, h, sp.step(i + 1), tid, sg);
    __syncthreads();
    const int step = sp.step(i), k0 = step * 32;
    const int pg0 = page_at(table, step * 2, a.width, a.pages), pg1 = page_at(table, step * 2 + 1, a.width, a.pages);
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      // does any row of the tile see a key of this step?
      if (k0 > pmax[t] || (k0 + 31 <= pmin[t] - a.window && k0 >= a.sinks)) continue;
      f32x16 s;
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] = 0.f;
      const int tok = (col & 16) + ((col >> 2) & 1) * 8 + ((col >> 3) & 1) * 4 + (col & 3);
      const char* kp = st + tok * 256;
      const int key = k_key(tok & 15);
#pragma unroll
      for (int c = 0; c < 8; ++c)
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(kp + (((c * 2 + hi) ^ key) << 4)), qf[t][c], s, 0, 0, 0);
      const bool inside = k0 + 31 <= pmin[t] && (k0 > pmax[t] - a.window || k0 + 31 < a.sinks) && pg0 >= 0 && pg1 >= 0;
      if (!inside) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int k = k0 + (j >> 3) * 16 + hi * 8 + (j & 7);
          const bool see = k <= pos[t] && (k > pos[t] - a.window || k < a.sinks) && ((j >> 3) ? pg1 : pg0) >= 0;
          s[j] = see ? s[j] : -INFINITY;
        }
      }
      float mx = s[0];
#pragma unroll
      for (int j = 1; j < 16; ++j) mx = fmaxf(mx, s[j]);
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float m_new = fmaxf(m[t], mx * a.scale_log2);
      const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
      const float alpha = fast_exp2(m[t] - m_use);
      bf16x8 p[2];
      float rs = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float pj = fast_exp2(fmaf(s[j], a.scale_log2, -m_use));
        p[j >> 3][j & 7] = (__bf16)pj;
        rs += pj;
      }
      l[t] = l[t] * alpha + rs;
      m[t] = m_new;
      if (__ballot(alpha != 1.f) != 0) {
#pragma unroll
        for (int n = 0; n < 4; ++n) o[t][n] *= alpha;
      }
      // Some row of the tile may not see a key whose V holds a NaN or an infinity: 0 times that would be NaN. Such values
      // are taken out of the matrix product and added for the rows that do see them.
      uint32_t odd = 0;
      bf16x8 vf[4][2];
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int g = 0; g < 2; ++g) vf[n][g] = *reinterpret_cast<const bf16x8*>(st + 8192 + g * 4096 + n * 1024 + lane * 16);
      if (!inside) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const uint4 u = __builtin_bit_cast(uint4, vf[n][g]);
            odd |= odd_halves(u.x) | odd_halves(u.y) | odd_halves(u.z) | odd_halves(u.w);
          }
        if (__ballot(odd != 0) != 0) {
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              uint4 u = __builtin_bit_cast(uint4, vf[n][g]);
              u = uint4{without_odd(u.x), without_odd(u.y), without_odd(u.z), without_odd(u.w)};
              vf[n][g] = __builtin_bit_cast(bf16x8, u);
            }
          for (int kk = 0; kk < 32; ++kk) {                            // (page, half, token): register (page, token) of lane half
            const int pg = kk >> 4, half = (kk >> 3) & 1, e = kk & 7;
            float pk = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) pk = (pg * 8 + e) == j ? (float)p[j >> 3][j & 7] : pk;
            pk = __shfl(pk, col + half * 32);
            const int k = k0 + kk;
            const bool see = k <= pos[t] && (k > pos[t] - a.window || k < a.sinks) && (pg ? pg1 : pg0) >= 0;
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
              for (int i2 = 0; i2 < 16; ++i2) {
                const int d = 8 * (i2 >> 2) + 4 * hi + (i2 & 3);
                const uint16_t e16 = *reinterpret_cast<const uint16_t*>(st + 8192 + pg * 4096 + n * 1024 + half * 512 + d * 16 + e * 2);
                if (see && (e16 & 0x7f80) == 0x7f80) o[t][n][i2] += pk * bf2f(e16);
              }
          }
        }
      }
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int n = 0; n < 4; ++n) o[t][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[n][g], p[g], o[t][n], 0, 0, 0);
    }
  }

#pragma unroll
  for (int t = 0; t < QT; ++t) {
    l[t] += __shfl_xor(l[t], 32);
    if (dst[t] < 0) continue;
    if (a.splits == 1) {
      const float inv = l[t] == 0.f ? 0.f : 1.f / l[t];
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bf16x4 v;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = (__bf16)(o[t][n][i * 4 + j] * inv);
          *reinterpret_cast<bf16x4*>(a.out + dst[t] * HD + n * 32 + i * 8 + hi * 4) = v;
        }
    } else {
      const size_t at = (size_t)dst[t] * a.splits + split;
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4*>(a.part_o + at * HD + n * 32 + i * 8 + hi * 4) =
              f32x4{o[t][n][i * 4], o[t][n][i * 4 + 1], o[t][n][i * 4 + 2], o[t][n][i * 4 + 3]};
      if (hi == 0) {
        a.part_ml[at * 2] = m[t];
        a.part_ml[at * 2 + 1] = l[t];
      }
    }
  }
}

int check_args(const WinArgs& a) {
  if (a.rows <= 0 || a.n_seqs <= 0 || a.n_seqs > 65535 || a.n_q <= 0 || a.n_kv <= 0 || a.n_q % a.n_kv != 0 || a.width <= 0 || a.pages <= 0 ||
      a.q_stride < a.n_q * HD || a.q_stride % 8 != 0 || a.width > INT32_MAX / BLK - 2)
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
                 c->window, c->sinks, c->splits, c->scale * 1.4426950408889634f};
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
  if (hipGetLastError() != hipSuccess) return KLM_ERR_HIP;
  if (a.splits > 1) {
    const size_t heads = (size_t)a.rows * a.n_q;
    hipLaunchKernelGGL(window_join_kernel, dim3((unsigned)((heads + 3) / 4)), dim3(256), 0, s, a, heads);
  }
  return launch_status();
}

int klm_window_attn_prefill(const klm_window_args* c) {
  if (!c) return KLM_ERR_ARG;
  const WinArgs a = device_args(c);
  const int rc = check_args(a);
  if (rc != KLM_OK) return rc;
  const int64_t tiles = ((int64_t)a.rows * a.G + 255) / 256 + a.n_seqs;       // every sequence may end in a partial tile
  if (tiles > 65535) return KLM_ERR_SHAPE;
  hipStream_t s = static_cast<hipStream_t>(c->stream);
  const dim3 grid(a.n_kv, (unsigned)tiles, 1);
  if (c->kv_fp8) hipLaunchKernelGGL((window_prefill_kernel<2, true>), grid, dim3(256), 2 * STEP_BYTES, s, a);
  else hipLaunchKernelGGL((window_prefill_kernel<2, false>), grid, dim3(256), 2 * STEP_BYTES, s, a);
  return launch_status();
}

}  // extern "C"
