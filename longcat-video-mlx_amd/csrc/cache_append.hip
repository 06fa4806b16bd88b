// New keys and values into the 8-bit cache (cache_common.h).
//
// Item b's rows go to tokens start[b] ..; a block of 64 tokens takes the least
// scale 2^e that brings its new rows within 448, and where the block keeps earlier
// rows no less than its old one, under which those rows are rounded again (exact but
// for the smallest values, as scales are powers of two).  One workgroup writes the keys
// and the values of one block, so nothing is shared between workgroups.  Bound by the
// bytes of the rows: both tensors' loads are under way together, the bytes go through LDS
// and leave as 16-byte pieces, the values turned 4 x 4 bytes at a time.  12,480 tokens of 32
// heads of 128 in bf16 (307 MB, from memory) take 71 us, 4.3 TB/s, in fp32 (511 MB) 105 us,
// 4.9 TB/s; one token each of 16 requests 8.4 us.
#include "cache_common.h"

namespace lcv {
namespace {

// Four words of four rows, bytes b0 .. b3 of columns d .. d + 3, to four of one column each.
__device__ __forceinline__ void turn4(uint32_t (&w)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602);
  const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602);
  w[0] = __builtin_amdgcn_perm(c, a, 0x05040100), w[1] = __builtin_amdgcn_perm(c, a, 0x07060302);
  w[2] = __builtin_amdgcn_perm(d, b, 0x05040100), w[3] = __builtin_amdgcn_perm(d, b, 0x07060302);
}

template <typename T, int D>
__global__ __launch_bounds__(256) void append_kernel(Cache8 c, Tensor4 k, Tensor4 v, const int32_t* start,
                                                     const int32_t* counts, int S, int touched) {
  constexpr int kVec = 16 / sizeof(T);   // values of a 16-byte load
  constexpr int kLoads = D / 4 / kVec;   // loads of one thread: a quarter of a row
  constexpr int kRow = D + 4;            // of the tiles, against bank conflicts
  __shared__ float wave_max[2][4];
  __shared__ __attribute__((aligned(16))) uint8_t tiles[2][64 * kRow];

  // Heads next to one another: the rows of a projection hold all of them.
  const int h = (int)(blockIdx.x % c.H), j = (int)(blockIdx.x / c.H % touched);
  const int b = (int)(blockIdx.x / c.H / touched);
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
  const int64_t block = ((int64_t)b * c.H + h) * c.nb + first / 64;

  const int tid = threadIdx.x, row = tid / 4, quarter = tid % 4;
  const bool fresh = row >= lo && row < hi;
  u32x4 w[2][kLoads];
  int e_old[2] = {-kMaxScaleExp, -kMaxScaleExp};
  if (fresh) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Tensor4& src = i ? v : k;
      const T* in = reinterpret_cast<const T*>(src.ptr) + (int64_t)b * src.sb + (int64_t)h * src.sh +
                    (first + row - p) * src.ss;
#pragma unroll
      for (int u = 0; u < kLoads; ++u) w[i][u] = *reinterpret_cast<const u32x4*>(in + kVec * (4 * u + quarter));
    }
  }
  if (lo > 0) e_old[0] = exponent_of(c.k_scale[block]), e_old[1] = exponent_of(c.v_scale[block]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float amax = 0.0f;
    if (fresh) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        T t[kVec];
        __builtin_memcpy(t, &w[i][u], 16);
#pragma unroll
        for (int q = 0; q < kVec; ++q) {
          const float a = __builtin_fabsf(to_f32(t[q]));
          amax = a < __builtin_inff() ? fmaxf(amax, a) : amax;  // infinities and NaN do not set the scale
        }
      }
    }
    for (int o = 1; o < 64; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    if (tid % 64 == 0) wave_max[i][tid / 64] = amax;
  }
  __syncthreads();  // also: every thread has read the old scales
  int e[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    e[i] = scale_exponent(fmaxf(fmaxf(wave_max[i][0], wave_max[i][1]), fmaxf(wave_max[i][2], wave_max[i][3])));
    if (lo > 0 && e_old[i] > e[i]) e[i] = e_old[i];
    if (fresh) {
      const float inv = pow2i(-e[i]);
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        T t[kVec];
        __builtin_memcpy(t, &w[i][u], 16);
#pragma unroll
        for (int q = 0; q < kVec; q += 4)
          *reinterpret_cast<uint32_t*>(tiles[i] + row * kRow + kVec * (4 * u + quarter) + q) = pack_e4m3(
              to_f32(t[q]) * inv, to_f32(t[q + 1]) * inv, to_f32(t[q + 2]) * inv, to_f32(t[q + 3]) * inv);
      }
    }
  }
  if (tid == 0) c.k_scale[block] = pow2i(e[0]), c.v_scale[block] = pow2i(e[1]);
  __syncthreads();
  uint8_t* kout = c.k8 + block * (64 * D);
  uint8_t* vout = c.v8 + block * (64 * D);
  if (lo == 0 && hi == 64) {  // a whole block
#pragma unroll
    for (int u = 0; u < 64 * D / 16 / 256; ++u) {
      const int i = tid + 256 * u, r = i / (D / 16), col = i % (D / 16) * 16;
      const uint32_t* in = reinterpret_cast<const uint32_t*>(tiles[0] + r * kRow + col);
      *reinterpret_cast<u32x4*>(kout + 16 * i) = u32x4{in[0], in[1], in[2], in[3]};
    }
    if (tid < D) {  // columns 4 (tid / 4) .. + 3, rows 16 (tid % 4) .. + 15
      const int d = tid / 4 * 4, r0 = tid % 4 * 16;
      uint32_t t[4][4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
#pragma unroll
        for (int q = 0; q < 4; ++q) t[g][q] = *reinterpret_cast<const uint32_t*>(tiles[1] + (r0 + 4 * g + q) * kRow + d);
        turn4(t[g]);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<u32x4*>(vout + (d + q) * 64 + r0) = u32x4{t[0][q], t[1][q], t[2][q], t[3][q]};
    }
    return;
  }
  // A block at the first or the last new row.
  const bool again[2] = {lo > 0 && e[0] > e_old[0], lo > 0 && e[1] > e_old[1]};  // the kept rows change their scale
  const float step[2] = {pow2i(e_old[0] - e[0]), pow2i(e_old[1] - e[1])};
  auto moved = [&](uint32_t word, float by) {
    float y[4];
    unpack_e4m3(word, y);
    return pack_e4m3(y[0] * by, y[1] * by, y[2] * by, y[3] * by);
  };
  for (int i = tid; i < 64 * D / 4; i += 256) {
    const int r = i / (D / 4), col = i % (D / 4) * 4;
    uint32_t* to = reinterpret_cast<uint32_t*>(kout + r * D + col);
    if (r >= lo && r < hi) *to = *reinterpret_cast<const uint32_t*>(tiles[0] + r * kRow + col);
    else if (again[0] && r < lo) *to = moved(*to, step[0]);
  }
  for (int i = tid; i < 64 * D / 4; i += 256) {
    const int d = i / 16, r = i % 16 * 4;
    if (r >= hi || (r + 4 <= lo && !again[1])) continue;
    uint32_t* to = reinterpret_cast<uint32_t*>(vout + d * 64 + r);
    uint32_t word = 0;
    if (r < lo || r + 4 > hi) word = *to;  // rows behind the last new one keep their bytes
    if (again[1] && r < lo) {
      const int kept = lo - r < 4 ? lo - r : 4;
      const uint32_t m = kept == 4 ? ~0u : (1u << (8 * kept)) - 1u;
      word = (word & ~m) | (moved(word, step[1]) & m);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (r + q >= lo && r + q < hi)
        word = (word & ~(255u << (8 * q))) | ((uint32_t)tiles[1][(r + q) * kRow + d] << (8 * q));
    *to = word;
  }
}

template <typename T>
hipError_t launch(const Cache8& c, const Tensor4& k, const Tensor4& v, int S, int D, const int32_t* start,
                  const int32_t* counts, hipStream_t stream) {
  const int touched = (int)(((int64_t)S + 126) / 64);  // blocks that S rows can reach, whatever their start
  const int64_t grid = (int64_t)c.B * c.H * touched;
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
