// Attention weights per cached token: w_out[j] = w_in[j] + sum over the rows that see
// token j of exp(scale q.k_j - lse), the rows' lse as cached_attention gives it.  What
// an eviction ranks tokens by.
//
// One workgroup owns one block of 64 keys and walks the rows, 16 at a time, its four
// waves taking every fourth tile: the keys stay in registers as the B operand of
// S = Q K^T (16 x 16 x 32 MFMAs), whose accumulators hold 4 rows of one key, so that a
// key's sum over rows is a sum over registers.  No atomics: the order of every sum is
// fixed.
#include "attn_common.h"
#include "cache_common.h"

namespace lcv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

template <typename T, int D>
__global__ __launch_bounds__(256) void weights_kernel(CacheAttn a, const float* w_in, float* w_out) {
  typedef typename Mfma<T>::vec8 vec8;
  __shared__ float sums[4][64];
  const int wid = xcd_linear_work_id(blockIdx.x, gridDim.x);
  const int j = wid % a.c.nb, bh = wid / a.c.nb;
  const int b = bh / a.c.H, kvh = bh - b * a.c.H;
  const int lane = threadIdx.x % 64, G = lane / 16, gi = lane % 16;
  const int wave = uniform_i32(threadIdx.x / 64);
  int len = a.lengths[b];
  len = len < 0 ? 0 : len > a.max_len ? a.max_len : len;
  int ql = a.q_lens ? a.q_lens[b] : a.S;
  ql = ql < 0 ? 0 : ql > a.S ? a.S : ql;
  const int rows = a.group * a.S;

  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (64 * j < len) {
    const uint8_t* kb = a.c.k8 + ((int64_t)bh * a.c.nb + j) * (64 * D) + gi * D + G * (D / 4);
    vec8 kf[4][D / 32];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int u = 0; u < D / 64; ++u) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(kb + 16 * t * D + 16 * u);
        kf[t][2 * u] = From8<T>::cvt(w[0], w[1]);
        kf[t][2 * u + 1] = From8<T>::cvt(w[2], w[3]);
      }
    const float c = a.scale_log2 * a.c.k_scale[(int64_t)bh * a.c.nb + j];
    for (int tile = wave; 16 * tile < rows; tile += 4) {
      int r = 16 * tile + gi;
      r = r < rows ? r : rows - 1;
      const int g = r / a.S, i = r - g * a.S;
      const T* q = reinterpret_cast<const T*>(a.q.ptr) + (int64_t)b * a.q.sb + (int64_t)(kvh * a.group + g) * a.q.sh +
                   (int64_t)i * a.q.ss + G * (D / 4);
      vec8 qf[D / 32];
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks)
        qf[ks] = __builtin_bit_cast(vec8, *reinterpret_cast<const u32x4*>(q + 8 * ks));
      int vis[4];
      float lse[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int re = 16 * tile + 4 * G + e;
        const int ge = re / a.S, ie = re - ge * a.S;
        vis[e] = 0;
        lse[e] = 0.0f;
        if (re < rows && ie < ql) {
          vis[e] = a.causal ? len - ql + ie + 1 : len;
          lse[e] = a.lse[((int64_t)b * a.c.H * a.group + kvh * a.group + ge) * a.S + ie] * kLog2e;
        }
        if (lse[e] == -__builtin_inff()) vis[e] = 0;
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 s = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) s = Mfma<T>::mma(qf[ks], kf[t][ks], s);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sum[t] += 64 * j + 16 * t + gi < vis[e] ? fast_exp2(__builtin_fmaf(s[e], c, -lse[e])) : 0.0f;
      }
    }
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    sum[t] = sum_quarters(sum[t]);
    if (G == 0) sums[wave][16 * t + gi] = sum[t];
  }
  __syncthreads();
  const int t = threadIdx.x;
  if (t < 64) {
    const int64_t at = ((int64_t)bh * a.c.nb + j) * 64 + t;
    const float got = (sums[0][t] + sums[1][t]) + (sums[2][t] + sums[3][t]);
    w_out[at] = (w_in ? w_in[at] : 0.0f) + got;
  }
}

template <typename T, int D>
hipError_t launch(const CacheAttn& a, const float* w_in, float* w_out, hipStream_t stream) {
  hipLaunchKernelGGL((weights_kernel<T, D>), dim3(a.c.B * a.c.H * a.c.nb), dim3(256), 0, stream, a, w_in, w_out);
  return hipGetLastError();
}

}  // namespace

size_t cache_weights_workspace(const CacheAttn& a, int D) { return 0; }

hipError_t launch_cache_weights(const CacheAttn& a, int dtype, int D, const float* w_in, float* w_out,
                                hipStream_t stream) {
  if (dtype == LCV_BSA_F16) return D == 64 ? launch<f16, 64>(a, w_in, w_out, stream) : launch<f16, 128>(a, w_in, w_out, stream);
  return D == 64 ? launch<bf16, 64>(a, w_in, w_out, stream) : launch<bf16, 128>(a, w_in, w_out, stream);
}

}  // namespace lcv
