// Eviction from the 8-bit cache (cache_common.h): of each head, the newest `recent`
// tokens and the heaviest of the others stay, keep in all, in their order.
//
// Two kernels.  The first ranks: a radix search over the weights' bits (as unsigned
// numbers in the order of the floats, NaN below everything) for the weight of the
// last token to stay, among equals the lowest tokens, then the list of kept tokens in
// order.  The second gathers: one workgroup makes one block of the new cache, whose
// scale is the least one for the rows it gets.
#include "cache_common.h"

namespace lcv {
namespace {

// Floats as unsigned numbers of the same order; -0 as +0, NaN last.
__device__ __forceinline__ uint32_t rank_bits(float w) {
  if (w != w) return 0u;
  const uint32_t u = __builtin_bit_cast(uint32_t, w == 0.0f ? 0.0f : w);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

constexpr int kRankThreads = 1024;

__global__ __launch_bounds__(kRankThreads) void rank_kernel(const int32_t* lengths, const float* weights, int H,
                                                            int64_t capacity, int keep, int recent,
                                                            int64_t new_capacity, int32_t* kept, float* w_out,
                                                            int32_t* new_lengths) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t found[3];
  __shared__ uint32_t wave_ties[16], wave_kept[16];
  const int bh = blockIdx.x, b = bh / H;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  int64_t len = lengths[b];
  len = len < 0 ? 0 : len > capacity ? capacity : len;
  const int64_t tail = recent < len ? recent : len;
  const int64_t old = len - tail;  // tokens that compete
  const int64_t left = len < keep ? len : keep;
  int64_t want = left - tail;  // of them stay
  const float* w = weights + (int64_t)bh * capacity;

  // The search: after each pass `prefix` holds the top bits of the last kept weight
  // and `want` its place among the weights that share them.
  uint32_t prefix = 0, mask = 0;
  const bool all = want >= old;
  if (!all && want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int64_t i = tid; i < old; i += kRankThreads) {
        const uint32_t u = rank_bits(w[i]);
        if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t above = 0;
        int d = 255;
        for (; d > 0 && above + hist[d] < (uint32_t)want; --d) above += hist[d];
        found[0] = (uint32_t)d;
        found[1] = above;
      }
      __syncthreads();
      prefix |= found[0] << shift;
      mask |= 255u << shift;
      want -= found[1];
      __syncthreads();
    }
  }
  // The list, in order: a token stays if it is newest, above the threshold, or one of
  // the first `want` at it.
  uint32_t ties = 0, out = 0;
  for (int64_t i0 = 0; i0 < len; i0 += kRankThreads) {
    const int64_t i = i0 + tid;
    const float wi = i < len ? w[i] : 0.0f;
    const uint32_t u = rank_bits(wi);
    const bool race = i < old && !all && left > tail;
    const bool tie = race && u == prefix;
    const uint64_t tie_mask = __ballot(tie);
    if (lane == 0) wave_ties[wave] = (uint32_t)__popcll(tie_mask);
    __syncthreads();
    uint32_t before = ties, tie_total = 0;
    for (int k = 0; k < 16; ++k) {
      if (k < wave) before += wave_ties[k];
      tie_total += wave_ties[k];
    }
    before += mbcnt64(tie_mask);
    const bool stay = i < len && (i >= old || (i < old && all) || (race && u > prefix) || (tie && before < (uint32_t)want));
    const uint64_t stay_mask = __ballot(stay);
    if (lane == 0) wave_kept[wave] = (uint32_t)__popcll(stay_mask);
    __syncthreads();
    uint32_t at = out, total = 0;
    for (int k = 0; k < 16; ++k) {
      if (k < wave) at += wave_kept[k];
      total += wave_kept[k];
    }
    at += mbcnt64(stay_mask);
    if (stay) {
      kept[(int64_t)bh * keep + at] = (int32_t)i;
      w_out[(int64_t)bh * new_capacity + at] = wi;
    }
    ties += tie_total;
    out += total;
    __syncthreads();
  }
  for (int64_t i = left + tid; i < keep; i += kRankThreads) kept[(int64_t)bh * keep + i] = -1;
  for (int64_t i = left + tid; i < new_capacity; i += kRankThreads) w_out[(int64_t)bh * new_capacity + i] = 0.0f;
  if (tid == 0 && bh % H == 0) new_lengths[b] = (int32_t)left;
}

template <int D>
__global__ __launch_bounds__(256) void gather_kernel(Cache8 src, Cache8 dst, const int32_t* kept, int keep) {
  __shared__ float wave_max[4];
  __shared__ __attribute__((aligned(16))) uint8_t tile[64 * (D + 4)];
  int64_t id = blockIdx.x;
  const int isv = (int)(id & 1);
  id >>= 1;
  const int j = (int)(id % dst.nb);
  const int64_t bh = id / dst.nb;
  const int tid = threadIdx.x, row = tid / 4, quarter = tid % 4;
  const int64_t slot = 64 * (int64_t)j + row;
  const int64_t cap = (int64_t)src.nb * 64;
  int64_t t = slot < keep ? kept[bh * keep + slot] : -1;
  if (t >= cap) t = -1;
  float x[D / 4];
  float amax = 0.0f;
  if (t >= 0) {
    const int64_t block = bh * src.nb + t / 64;
    const float scale = pow2i(exponent_of((isv ? src.v_scale : src.k_scale)[block]));
    if (!isv) {
      const uint8_t* in = src.k8 + block * (64 * D) + (t % 64) * D + quarter * (D / 4);
#pragma unroll
      for (int u = 0; u < D / 16; ++u) unpack_e4m3(reinterpret_cast<const uint32_t*>(in)[u], x + 4 * u);
    } else {
      const uint8_t* in = src.v8 + block * (64 * D) + (t % 64) + quarter * (D / 4) * 64;
#pragma unroll
      for (int u = 0; u < D / 16; ++u) {
        uint32_t word = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) word |= (uint32_t)in[(4 * u + e) * 64] << (8 * e);
        unpack_e4m3(word, x + 4 * u);
      }
    }
#pragma unroll
    for (int i = 0; i < D / 4; ++i) {
      x[i] *= scale;
      const float a = __builtin_fabsf(x[i]);
      amax = a < __builtin_inff() ? fmaxf(amax, a) : amax;
    }
  } else {
#pragma unroll
    for (int i = 0; i < D / 4; ++i) x[i] = 0.0f;
  }
  for (int o = 1; o < 64; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
  if (tid % 64 == 0) wave_max[tid / 64] = amax;
  const bool filled = __syncthreads_or(t >= 0) != 0;
  amax = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
  const int e = filled ? scale_exponent(amax) : 0;
  const float inv = pow2i(-e);
#pragma unroll
  for (int u = 0; u < D / 16; ++u)
    *reinterpret_cast<uint32_t*>(tile + row * (D + 4) + quarter * (D / 4) + 4 * u) =
        pack_e4m3(x[4 * u] * inv, x[4 * u + 1] * inv, x[4 * u + 2] * inv, x[4 * u + 3] * inv);
  __syncthreads();
  const int64_t block = bh * dst.nb + j;
  if (tid == 0) (isv ? dst.v_scale : dst.k_scale)[block] = pow2i(e);
  uint8_t* out = (isv ? dst.v8 : dst.k8) + block * (64 * D);
  for (int i = tid; i < 64 * D / 4; i += 256) {
    uint32_t word;
    if (!isv) {
      word = *reinterpret_cast<const uint32_t*>(tile + i / (D / 4) * (D + 4) + i % (D / 4) * 4);
    } else {
      const int d = i / 16, r = i % 16 * 4;
      word = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) word |= (uint32_t)tile[(r + q) * (D + 4) + d] << (8 * q);
    }
    reinterpret_cast<uint32_t*>(out)[i] = word;
  }
}

}  // namespace

hipError_t launch_cache_evict(const Cache8& src, const int32_t* lengths, const float* weights, int keep, int recent,
                              const Cache8& dst, float* w_out, int32_t* kept, int32_t* new_lengths, int D,
                              hipStream_t stream) {
  hipLaunchKernelGGL(rank_kernel, dim3(src.B * src.H), dim3(kRankThreads), 0, stream, lengths, weights, src.H,
                     (int64_t)src.nb * 64, keep, recent, (int64_t)dst.nb * 64, kept, w_out, new_lengths);
  const uint32_t grid = (uint32_t)((int64_t)src.B * src.H * dst.nb * 2);
  if (D == 64)
    hipLaunchKernelGGL((gather_kernel<64>), dim3(grid), dim3(256), 0, stream, src, dst, kept, keep);
  else
    hipLaunchKernelGGL((gather_kernel<128>), dim3(grid), dim3(256), 0, stream, src, dst, kept, keep);
  return hipGetLastError();
}

}  // namespace lcv
