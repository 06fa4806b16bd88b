// New keys and values into the 8-bit cache (cache_common.h).
//
// Item b's rows go to tokens start[b] ..; a block of 64 tokens takes the least
// scale 2^e that brings its new rows within 448, and where the block keeps earlier
// rows no less than its old one, under which those rows are rounded again (exact but
// for the smallest values, as scales are powers of two).  One workgroup writes one
// block of keys or of values, so nothing is shared between workgroups.  Bound by
// the bytes of the rows.
#include "cache_common.h"

namespace lcv {
namespace {

template <typename T, int D>
__global__ __launch_bounds__(256) void append_kernel(Cache8 c, Tensor4 k, Tensor4 v, const int32_t* start,
                                                     const int32_t* counts, int S, int touched) {
  constexpr int kVec = 16 / sizeof(T);   // values of a 16-byte load
  constexpr int kLoads = D / 4 / kVec;   // loads of one thread: a quarter of a row
  __shared__ float wave_max[4];
  __shared__ __attribute__((aligned(16))) uint8_t tile[64 * (D + 4)];

  int64_t id = blockIdx.x;
  const int isv = (int)(id & 1);
  id >>= 1;
  const int j = (int)(id % touched);
  id /= touched;
  const int h = (int)(id % c.H);
  const int b = (int)(id / c.H);
  const int64_t cap = (int64_t)c.nb * 64;
  const int64_t p = start[b];
  int64_t n = counts ? counts[b] : S;
  if (n > S) n = S;
  if (p < 0 || n <= 0 || p >= cap) return;
  const int64_t end = p + n < cap ? p + n : cap;  // rows past the capacity are dropped
  const int64_t first = p / 64 * 64 + 64 * (int64_t)j;
  if (first >= end) return;
  const int lo = first < p ? (int)(p - first) : 0;            // rows [0, lo) are kept
  const int hi = end - first < 64 ? (int)(end - first) : 64;  // rows [lo, hi) are new

  const Tensor4& src = isv ? v : k;
  const int64_t block = ((int64_t)b * c.H + h) * c.nb + first / 64;
  uint8_t* out = (isv ? c.v8 : c.k8) + block * (64 * D);
  float* scale = (isv ? c.v_scale : c.k_scale) + block;

  const int tid = threadIdx.x, row = tid / 4, quarter = tid % 4;
  const bool fresh = row >= lo && row < hi;
  float x[kLoads][kVec];
  float amax = 0.0f;
  if (fresh) {
    const T* in = reinterpret_cast<const T*>(src.ptr) + (int64_t)b * src.sb + (int64_t)h * src.sh +
                  (first + row - p) * src.ss;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(in + kVec * (4 * u + quarter));
      T t[kVec];
      __builtin_memcpy(t, &w, 16);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        x[u][i] = to_f32(t[i]);
        const float a = __builtin_fabsf(x[u][i]);
        amax = a < __builtin_inff() ? fmaxf(amax, a) : amax;  // infinities and NaN do not set the scale
      }
    }
  }
  for (int o = 1; o < 64; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
  if (tid % 64 == 0) wave_max[tid / 64] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
  int e = scale_exponent(amax);
  const int e_old = lo > 0 ? exponent_of(*scale) : e;
  if (e_old > e) e = e_old;
  const float inv = pow2i(-e);
  // The new rows' bytes: a row of the tile is D bytes (padded against bank conflicts).
  if (fresh) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
#pragma unroll
      for (int i = 0; i < kVec; i += 4)
        *reinterpret_cast<uint32_t*>(tile + row * (D + 4) + kVec * (4 * u + quarter) + i) =
            pack_e4m3(x[u][i] * inv, x[u][i + 1] * inv, x[u][i + 2] * inv, x[u][i + 3] * inv);
  }
  __syncthreads();  // also: every thread has read *scale
  if (tid == 0) *scale = pow2i(e);
  const bool again = lo > 0 && e > e_old;  // the kept rows change their scale
  const float step = pow2i(e_old - e);
  if (!isv) {
    for (int i = tid; i < 64 * D / 4; i += 256) {
      const int r = i / (D / 4), col = i % (D / 4) * 4;
      if (r >= lo && r < hi) {
        *reinterpret_cast<uint32_t*>(out + r * D + col) = *reinterpret_cast<const uint32_t*>(tile + r * (D + 4) + col);
      } else if (again && r < lo) {
        uint32_t* w = reinterpret_cast<uint32_t*>(out + r * D + col);
        float y[4];
        unpack_e4m3(*w, y);
        *w = pack_e4m3(y[0] * step, y[1] * step, y[2] * step, y[3] * step);
      }
    }
  } else {
    for (int i = tid; i < 64 * D / 4; i += 256) {
      const int d = i / 16, r = i % 16 * 4;
      if (r + 4 <= lo && !again) continue;
      if (r >= hi) continue;
      uint32_t* w = reinterpret_cast<uint32_t*>(out + d * 64 + r);
      uint32_t word = 0;
      if (r < lo || r + 4 > hi) word = *w;  // rows behind the last new one keep their bytes
      if (again && r < lo) {
        float y[4];
        unpack_e4m3(word, y);
        const uint32_t moved = pack_e4m3(y[0] * step, y[1] * step, y[2] * step, y[3] * step);
        const int kept = lo - r < 4 ? lo - r : 4;
        const uint32_t m = kept == 4 ? ~0u : (1u << (8 * kept)) - 1u;
        word = (word & ~m) | (moved & m);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (r + q >= lo && r + q < hi)
          word = (word & ~(255u << (8 * q))) | ((uint32_t)tile[(r + q) * (D + 4) + d] << (8 * q));
      *w = word;
    }
  }
}

template <typename T>
hipError_t launch(const Cache8& c, const Tensor4& k, const Tensor4& v, int S, int D, const int32_t* start,
                  const int32_t* counts, hipStream_t stream) {
  const int touched = (int)(((int64_t)S + 126) / 64);  // blocks that S rows can reach, whatever their start
  const int64_t grid = (int64_t)c.B * c.H * touched * 2;
  if (D == 64)
    hipLaunchKernelGGL((append_kernel<T, 64>), dim3((uint32_t)grid), dim3(256), 0, stream, c, k, v, start, counts, S,
                       touched);
  else
    hipLaunchKernelGGL((append_kernel<T, 128>), dim3((uint32_t)grid), dim3(256), 0, stream, c, k, v, start, counts, S,
                       touched);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_append(const Cache8& c, const Tensor4& k, const Tensor4& v, int dtype, int S, int D,
                               const int32_t* start, const int32_t* counts, hipStream_t stream) {
  switch (dtype) {
    case LCV_BSA_F16: return launch<f16>(c, k, v, S, D, start, counts, stream);
    case LCV_BSA_BF16: return launch<bf16>(c, k, v, S, D, start, counts, stream);
    default: return launch<float>(c, k, v, S, D, start, counts, stream);
  }
}

}  // namespace lcv
