// Eviction from the 8-bit cache (cache_common.h): of each head, the newest `recent`
// tokens and the heaviest of the others stay, keep in all, in their order.
//
// Two kernels.  The first ranks, one workgroup a head: weights as unsigned numbers in the
// order of the floats (NaN below everything), held in LDS, and a search for the number T
// of the last token to stay (count above T < want <= count from T on).  A round sorts the
// candidates into 4096 bins of the interval [a, z) by a shift, and goes on in the bin where
// the count passes `want`: three rounds at most, whatever the weights.  As soon as 32 are
// left they are compared with one another.  Each wave holds a run of tokens, so one
// exchange of the waves' counts places every kept token; equal weights at T stay from the
// lowest token on.
//
// The second gathers: one workgroup makes one block of the new cache, whose scale is the
// least one for the rows it gets.  Keys move as 32-byte pieces of rows; of the values,
// whose bytes lie token by token, a wave takes one of the D rows at a time, its lanes the
// 64 tokens: kept tokens are in order, so the lanes' bytes are in few lines.
//
// 9360 of 18,720 tokens of 32 heads of 128: ranking 18 us (32 workgroups, bound by the
// passes' latency), gathering 49 us: 192 MB, as of the values every line is read, 3.9 TB/s
// (40 us from the last-level cache).
#include "cache_common.h"

namespace lcv {
namespace {

// Floats as unsigned numbers of the same order, from 1; -0 as +0, NaN first.
__device__ __forceinline__ uint32_t rank_bits(float w) {
  if (w != w) return 1u;
  const uint32_t u = __builtin_bit_cast(uint32_t, w == 0.0f ? 0.0f : w);
  return (u >> 31) ? ~u : u | 0x80000000u;
}
constexpr uint32_t kAlways = ~0u;          // the newest tokens' key; 0: no token
constexpr uint64_t kKeysEnd = 0xff800001;  // past infinity's

constexpr int kRankThreads = 1024, kRankWaves = kRankThreads / 64;
constexpr int kBins = 4096;
// 18,720 tokens of 32 heads (1000 of 8 heads): 67 (12) us; 512 candidates 72 (20), 16 67 (14).
constexpr uint32_t kLast = 32;

// N: keys that LDS holds, or 0 where the weights are read anew at each pass.  (In
// registers the loops over them would be unrolled, and a launch that runs each
// instruction a few times waits for the instructions: 38 us for 18,720 tokens.)
template <int N>
__global__ __launch_bounds__(kRankThreads) void rank_kernel(const int32_t* lengths, const float* __restrict__ weights,
                                                            int H, int64_t capacity, int keep, int recent,
                                                            int32_t* __restrict__ kept, int32_t* new_lengths) {
  __shared__ __attribute__((aligned(16))) uint32_t bins[kBins];  // later: the last candidates
  __shared__ uint32_t waves[2][kRankWaves];
  __shared__ uint32_t found[3];
  __shared__ __attribute__((aligned(16))) uint32_t held[N > 0 ? N : 4];
  const int bh = blockIdx.x, b = bh / H;
  const int tid = threadIdx.x, lane = tid % 64, wave = uniform_i32(tid / 64);
  int64_t n = lengths[b];
  const int len = (int)(n < 0 ? 0 : n > capacity ? capacity : n);
  const int tail = recent < len ? recent : len;
  const int old = len - tail;  // tokens that compete
  const int left = len < keep ? len : keep;
  const int want = left - tail;  // of them stay
  const float* w = weights + (int64_t)bh * capacity;

  // Wave w holds tokens w * run .. + run - 1, its lane l four of each 256.
  const int quads = (len + 4 * kRankThreads - 1) / (4 * kRankThreads), run = quads * 256;
  const int first = wave * run + 4 * lane;
  struct Four {
    float x[4];
  };
  auto load = [&](int r) {  // 16 bytes, on any float's boundary; capacities are whole blocks
    const int i = first + 256 * r;
    Four v;
    __builtin_memcpy(&v, w + (r < quads && i < old ? i : 0), sizeof(v));
    return v;
  };
  auto keys = [&](int r, const Four& v) {
    const int i = first + 256 * r;
    u32x4 k;
#pragma unroll
    for (int q = 0; q < 4; ++q) k[q] = i + q < old ? rank_bits(v.x[q]) : i + q < len ? kAlways : 0u;
    return k;
  };
  if constexpr (N > 0) {
    for (int r = 0; r < quads; r += 8) {  // eight loads under way together
      Four v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = load(r + q);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (r + q < quads)  // read by the same lane alone
          *reinterpret_cast<u32x4*>(&held[first + 256 * (r + q)]) = keys(r + q, v[q]);
    }
  }
  // f(i, the keys of tokens i .. i + 3) for every token of this lane; key 0 behind the last.
  auto each = [&](auto f) {
    for (int r = 0; r < quads; ++r) {
      const int i = first + 256 * r;
      if constexpr (N > 0) f(i, *reinterpret_cast<const u32x4*>(&held[i]));
      else f(i, keys(r, load(r)));
    }
  };

  // T: the largest key that at least `want` competing tokens reach; the first `ties` of
  // those equal to T stay beside all that exceed it.
  uint32_t T = want >= old ? 0u : kAlways - 1, ties = 0;
  if (want < old && want > 0) {
    const uint32_t goal = (uint32_t)want;
    uint64_t a = 1, z = kKeysEnd;
    uint32_t above = 0, have = (uint32_t)old;  // keys from z on; keys in [a, z)
    while (z - a > 1 && have > kLast) {        // workgroup-uniform
      int shift = 0;
      while ((z - a - 1) >> shift >= kBins) ++shift;
      reinterpret_cast<u32x4*>(bins)[tid] = u32x4{0u, 0u, 0u, 0u};
      __syncthreads();
      each([&](int, u32x4 k) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (k[q] >= a && k[q] < z) atomicAdd(&bins[(k[q] - (uint32_t)a) >> shift], 1u);
      });
      __syncthreads();
      // Thread t: bins 4 t .. 4 t + 3, and how many keys lie in the bins behind them.
      const u32x4 c = reinterpret_cast<u32x4*>(bins)[tid];
      const uint32_t mine = c[0] + c[1] + c[2] + c[3];
      uint32_t from = mine;
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_down(from, o);
        from += lane + o < 64 ? x : 0u;
      }
      if (lane == 0) waves[0][wave] = from;
      __syncthreads();
      uint32_t behind = above + from - mine;
      for (int k = wave + 1; k < kRankWaves; ++k) behind += waves[0][k];
#pragma unroll
      for (int q = 3; q >= 0; --q) {
        if (behind < goal && behind + c[q] >= goal) found[0] = 4 * tid + q, found[1] = behind, found[2] = c[q];
        behind += c[q];
      }
      __syncthreads();
      a += (uint64_t)found[0] << shift;
      z = a + ((uint64_t)1 << shift) < z ? a + ((uint64_t)1 << shift) : z;
      above = found[1], have = found[2];
    }
    T = (uint32_t)a, ties = goal - above;
    if (z - a > 1) {  // at most kLast candidates, against one another
      __syncthreads();
      if (tid < (int)kLast) bins[tid] = 0;
      if (tid == 0) found[0] = 0;
      __syncthreads();
      each([&](int, u32x4 k) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (k[q] >= a && k[q] < z) bins[atomicAdd(&found[0], 1u)] = k[q];  // in any order
      });
      __syncthreads();
      if (tid < (int)have) {
        const uint32_t k = bins[tid];
        uint32_t more = above, from = above;
#pragma unroll 4
        for (uint32_t i = 0; i < kLast; i += 4) {  // zeros behind the last: none reaches a key
          const u32x4 x = *reinterpret_cast<const u32x4*>(&bins[i]);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            more += x[q] > k ? 1u : 0u;
            from += x[q] >= k ? 1u : 0u;
          }
        }
        if (more < goal && from >= goal) {  // equal keys write the same
          found[1] = from == goal ? k - 1 : k;
          found[2] = from == goal ? 0u : goal - more;
        }
      }
      __syncthreads();
      T = found[1], ties = found[2];
    }
  }
  // Where this wave's tokens go, and which ties are its own.
  uint32_t n_new = 0, n_tie = 0;
  each([&](int, u32x4 k) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      n_new += k[q] > T ? 1u : 0u;
      n_tie += k[q] == T ? 1u : 0u;  // counted only where there are ties
    }
  });
  for (int o = 1; o < 64; o <<= 1) n_new += __shfl_xor(n_new, o), n_tie += __shfl_xor(n_tie, o);
  __syncthreads();  // waves is read
  if (lane == 0) waves[0][wave] = n_new, waves[1][wave] = n_tie;
  __syncthreads();
  uint32_t at = 0, tie = 0;
  for (int k = 0; k < wave; ++k) {
    const uint32_t room = ties - tie, use = waves[1][k] < room ? waves[1][k] : room;
    at += waves[0][k] + use;
    tie += use;
  }
  int32_t* list = kept + (int64_t)bh * keep;
  each([&](int i, u32x4 k) {
    bool stay[4];
    if (ties == 0) {  // workgroup-uniform
#pragma unroll
      for (int q = 0; q < 4; ++q) stay[q] = k[q] > T;
    } else {
      uint32_t before = tie, all = 0;  // ties of the lanes before, and of this lane so far
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint64_t mask = __ballot(k[q] == T);
        before += mbcnt64(mask);
        all += (uint32_t)__popcll(mask);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        stay[q] = k[q] > T || (k[q] == T && before < ties);
        before += k[q] == T ? 1u : 0u;
      }
      tie = tie + all < ties ? tie + all : ties;
    }
    uint32_t to = at;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint64_t mask = __ballot(stay[q]);
      to += mbcnt64(mask);
      at += (uint32_t)__popcll(mask);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (stay[q]) list[to] = i + q;
      to += stay[q] ? 1u : 0u;
    }
  });
  for (int i = left + tid; i < keep; i += kRankThreads) list[i] = -1;
  if (tid == 0 && bh % H == 0) new_lengths[b] = left;
}

// The scale's exponent for what `word` holds under `scale`, over the workgroup, and the
// words under it.
template <int W>
__device__ __forceinline__ float largest(const uint32_t (&word)[W], float scale) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    float y[4];
    unpack_e4m3(word[i], y);
#pragma unroll
    for (int e = 0; e < 4; ++e) amax = fmaxf(amax, __builtin_fabsf(y[e]));  // fmaxf leaves NaN out
  }
  amax *= scale;
  for (int o = 1; o < 64; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
  return amax;
}
template <int W>
__device__ __forceinline__ void rescale(uint32_t (&word)[W], float by) {
#pragma unroll
  for (int i = 0; i < W; ++i) {
    float y[4];
    unpack_e4m3(word[i], y);
    word[i] = pack_e4m3(y[0] * by, y[1] * by, y[2] * by, y[3] * by);
  }
}

// One workgroup a block of the new cache, its keys and its values: thread (row, quarter of
// D) of the keys, (quarter of D, row) of the values.
template <int D>
__global__ __launch_bounds__(256) void gather_kernel(Cache8 src, Cache8 dst, const int32_t* __restrict__ kept, int keep,
                                                     const float* __restrict__ weights, float* __restrict__ w_out) {
  constexpr int W = D / 16;  // words of a quarter
  __shared__ float maxima[2][4];
  const int j = (int)(blockIdx.x % dst.nb);
  const int64_t bh = blockIdx.x / dst.nb;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const int krow = tid / 4, kd = tid % 4 * (D / 4), vd = wave * (D / 4);
  const int64_t slot0 = 64 * (int64_t)j, old = bh * src.nb, block = bh * dst.nb + j;
  auto token = [&](int row) {
    const int64_t t = slot0 + row < keep ? kept[bh * keep + slot0 + row] : -1;
    return t < (int64_t)src.nb * 64 ? t : -1;
  };
  const int64_t kt = token(krow), vt = token(lane);
  const bool filled = token(0) >= 0;
  uint32_t kw[W], vw[W];
  float ks = 1.0f, vs = 1.0f, weight = 0.0f;
#pragma unroll
  for (int i = 0; i < W; ++i) kw[i] = vw[i] = 0;
  if (kt >= 0) {
    const u32x4* in = reinterpret_cast<const u32x4*>(src.k8 + (old + kt / 64) * (64 * D) + (kt % 64) * D + kd);
#pragma unroll
    for (int i = 0; i < W / 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) kw[4 * i + e] = in[i][e];
    ks = src.k_scale[old + kt / 64];
  }
  if (vt >= 0) {
    const uint8_t* in = src.v8 + (old + vt / 64) * (64 * D) + vd * 64 + vt % 64;
    uint8_t byte[4 * W];
#pragma unroll
    for (int i = 0; i < 4 * W; ++i) byte[i] = in[i * 64];
#pragma unroll
    for (int i = 0; i < W; ++i)
      vw[i] = byte[4 * i] | (uint32_t)byte[4 * i + 1] << 8 | (uint32_t)byte[4 * i + 2] << 16 |
              (uint32_t)byte[4 * i + 3] << 24;
    vs = src.v_scale[old + vt / 64];
    if (wave == 0) weight = weights[old * 64 + vt];
  }
  if (wave == 0) w_out[block * 64 + lane] = weight;
  ks = pow2i(exponent_of(ks));
  vs = pow2i(exponent_of(vs));
  const float kmax = largest(kw, ks), vmax = largest(vw, vs);
  if (lane == 0) maxima[0][wave] = kmax, maxima[1][wave] = vmax;
  __syncthreads();
  int e[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    e[i] = filled ? scale_exponent(fmaxf(fmaxf(maxima[i][0], maxima[i][1]), fmaxf(maxima[i][2], maxima[i][3]))) : 0;
  if (tid == 0) dst.k_scale[block] = pow2i(e[0]), dst.v_scale[block] = pow2i(e[1]);
  rescale(kw, ks * pow2i(-e[0]));  // by 2^(old - new), within 2^-120 .. 2^120
  u32x4* out = reinterpret_cast<u32x4*>(dst.k8 + block * (64 * D) + krow * D + kd);
#pragma unroll
  for (int i = 0; i < W / 4; ++i) out[i] = u32x4{kw[4 * i], kw[4 * i + 1], kw[4 * i + 2], kw[4 * i + 3]};
  rescale(vw, vs * pow2i(-e[1]));
  uint8_t* vout = dst.v8 + block * (64 * D) + vd * 64 + lane;
#pragma unroll
  for (int i = 0; i < 4 * W; ++i) vout[i * 64] = (uint8_t)(vw[i / 4] >> (8 * (i % 4)));
}

template <int N>
void launch_rank(const Cache8& src, const int32_t* lengths, const float* weights, int keep, int recent,
                 int32_t* kept, int32_t* new_lengths, hipStream_t stream) {
  hipLaunchKernelGGL((rank_kernel<N>), dim3(src.B * src.H), dim3(kRankThreads), 0, stream, lengths, weights, src.H,
                     (int64_t)src.nb * 64, keep, recent, kept, new_lengths);
}

}  // namespace

hipError_t launch_cache_evict(const Cache8& src, const int32_t* lengths, const float* weights, int keep, int recent,
                              const Cache8& dst, float* w_out, int32_t* kept, int32_t* new_lengths, int D,
                              hipStream_t stream) {
  const int64_t most = (int64_t)src.nb * 64;  // LDS holds whole rounds of 4096
  // Weights in LDS up to what it holds (32 heads of 18,720 tokens: the call 67 us, read anew
  // 78; 8 heads of 32,000 and 20,000: 41 and 63), and little of it where little is needed, for
  // two workgroups a CU (8 times 64 heads of 4000 tokens: 67 us, with 35,840's room 72).
  const auto rank = most <= 4096 ? launch_rank<4096> : most <= 32768 ? launch_rank<32768> : launch_rank<0>;
  rank(src, lengths, weights, keep, recent, kept, new_lengths, stream);
  const uint32_t grid = (uint32_t)((int64_t)src.B * src.H * dst.nb);
  if (D == 64)
    hipLaunchKernelGGL((gather_kernel<64>), dim3(grid), dim3(256), 0, stream, src, dst, kept, keep, weights, w_out);
  else
    hipLaunchKernelGGL((gather_kernel<128>), dim3(grid), dim3(256), 0, stream, src, dst, kept, keep, weights, w_out);
  return hipGetLastError();
}

}  // namespace lcv
