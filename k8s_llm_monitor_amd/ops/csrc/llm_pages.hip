// Copies of pages of the paged KV cache: a fork's private copy of its last, partly filled page, compaction of the pool, the
// move into another cache, and clearing. A page is 16 tokens of every layer and kv head: in the cache tensors
// [layers][blocks][n_kv][16 * 128] it is one contiguous slab of n_kv * 2048 elements per layer, in K and in V.
//
// Nothing is computed: the floor is each page read once and written once. The page numbers travel in the launch's own
// arguments, up to PAIRS of them, so a call needs no copy to the device, no buffer that has to outlive it, and can be captured.
//
// No reference counterpart (vLLM is a README bullet in the reference, README.md:73).
#include "llm_common.h"

using namespace klm_llm;

namespace {

constexpr int PAIRS = 256;
struct PagePairs {
  int src[PAIRS], dst[PAIRS];      // src < 0: clear dst
};

struct PageArgs {
  const char *ks, *vs;
  char *kd, *vd;
  size_t slab;                     // bytes of one page of one layer
  size_t src_layer, dst_layer;     // bytes from one layer to the next
};

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

// One 16-byte load and store a thread, both past the caches: a page is not read again soon by whoever copies it. MI355X, read and
// written: 683 pages of 32 layers, 32 KiB each in K and in V, 539 us, 5.3 TB/s (through the caches, with 64 bytes a thread in
// one pass, 571 us); 250 e4m3 pages of 80 layers 209 us, 6.3 TB/s (241 us). A torch copy of one large tensor reaches 6.6 TB/s.
__global__ __launch_bounds__(256) void copy_pages_kernel(PageArgs a, PagePairs p) {
  const int src = p.src[blockIdx.y], dst = p.dst[blockIdx.y], layer = blockIdx.z >> 1;
  const bool v = blockIdx.z & 1;
  const size_t at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 16;
  if (at >= a.slab) return;
  char* d = (v ? a.vd : a.kd) + (size_t)layer * a.dst_layer + (size_t)dst * a.slab + at;
  u32x4 r = u32x4{0, 0, 0, 0};
  if (src >= 0) r = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>((v ? a.vs : a.ks) + (size_t)layer * a.src_layer + (size_t)src * a.slab + at));
  __builtin_nontemporal_store(r, reinterpret_cast<u32x4*>(d));
}

}  // namespace

extern "C" {

int klm_copy_pages(const klm_pages_args* c) {
  if (!c) return KLM_ERR_ARG;
  const int n = c->n;
  const int32_t* pairs = c->pairs;
  if (n < 0 || c->layers <= 0 || c->layers > 65535 || c->src_blocks <= 0 || c->dst_blocks <= 0 || c->n_kv <= 0) return KLM_ERR_SHAPE;
  if ((c->elem_size != 1 && c->elem_size != 2) || (n > 0 && !pairs) || !c->k_src || !c->v_src || !c->k_dst || !c->v_dst) return KLM_ERR_ARG;
  if (!aligned16(c->k_src) || !aligned16(c->v_src) || !aligned16(c->k_dst) || !aligned16(c->v_dst)) return KLM_ERR_ALIGN;
  for (int i = 0; i < n; ++i)
    if (pairs[2 * i] >= c->src_blocks || pairs[2 * i + 1] < 0 || pairs[2 * i + 1] >= c->dst_blocks) return KLM_ERR_ARG;
  PageArgs a;
  a.ks = (const char*)c->k_src;
  a.vs = (const char*)c->v_src;
  a.kd = (char*)c->k_dst;
  a.vd = (char*)c->v_dst;
  a.slab = (size_t)c->n_kv * BLK_ELEMS * c->elem_size;
  a.src_layer = a.slab * c->src_blocks;
  a.dst_layer = a.slab * c->dst_blocks;
  const size_t chunks = (a.slab + 4095) / 4096;
  if (chunks > INT32_MAX || c->layers > 32767) return KLM_ERR_SHAPE;
  for (int at = 0; at < n; at += PAIRS) {
    const int m = n - at < PAIRS ? n - at : PAIRS;
    PagePairs p;
    for (int i = 0; i < PAIRS; ++i) {
      p.src[i] = i < m ? pairs[2 * (at + i)] : -1;
      p.dst[i] = i < m ? pairs[2 * (at + i) + 1] : 0;
    }
    hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)chunks, m, c->layers * 2), dim3(256), 0, static_cast<hipStream_t>(c->stream), a, p);
    if (hipGetLastError() != hipSuccess) return KLM_ERR_HIP;
  }
  return KLM_OK;
}

}  // extern "C"
