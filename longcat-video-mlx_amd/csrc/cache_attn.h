// What the kernels that read queries against the 8-bit cache share: an item's lengths
// and what a query sees, and loads into LDS.
#pragma once

#include "attn_common.h"
#include "cache_common.h"

namespace lcv {
namespace {

// dma16 where the descriptor may have been brought back from spilled lanes right
// before: a vector instruction's scalar result needs five wait states until a buffer
// load reads it, and the compiler does not see the load inside the asm.
__device__ __forceinline__ void dma16_settled(__amdgpu_buffer_rsrc_t rsrc, uint32_t voffset, int32_t soffset,
                                              uint32_t m0v) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
               ::"v"(voffset), "s"(rsrc), "s"(soffset), "{m0}"(m0v)
               : "memory");
}

// One dword a lane, the same way.
__device__ __forceinline__ void dma4_settled(__amdgpu_buffer_rsrc_t rsrc, uint32_t voffset, uint32_t m0v) {
  asm volatile("s_nop 4\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voffset), "s"(rsrc), "{m0}"(m0v) : "memory");
}

struct Lens {
  int len, ql;  // tokens held, real queries
};
__device__ __forceinline__ Lens item_lens(const CacheAttn& a, int b) {
  Lens r;
  r.len = a.lengths[b];
  r.len = r.len < 0 ? 0 : r.len > a.max_len ? a.max_len : r.len;
  r.ql = a.q_lens ? a.q_lens[b] : a.S;
  r.ql = r.ql < 0 ? 0 : r.ql > a.S ? a.S : r.ql;
  return r;
}
// Tokens that query i sees.
__device__ __forceinline__ int visible(const CacheAttn& a, const Lens& n, int i) {
  if (i >= n.ql) return 0;
  if (!a.causal) return n.len;
  const int v = n.len - n.ql + i + 1;
  return v < 0 ? 0 : v;
}

template <bool B>
struct Flag {
  static constexpr bool value = B;
};

// Keeps what follows from being computed before the branch that it stands in.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

}  // namespace
}  // namespace lcv
