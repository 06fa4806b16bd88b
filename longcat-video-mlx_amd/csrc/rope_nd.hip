// Rotary positions with several axes (time, height, width, or any other split of
// the head dim) at positions that the caller gives per token, forward and backward:
//
//   angle t of pair i on axis a: position[s][a] * base^(-2 i / dim_a)
//   y[2i] = x[2i] cos t - x[2i+1] sin t,  y[2i+1] = x[2i] sin t + x[2i+1] cos t
//
// and, since a rotation's transpose turns back, the gradient with -t.  Bound by the
// bytes of x and y.  The angle is taken as turns, position * (frequency / 2 pi), in
// 64 bits with the whole turns dropped, so that a far position keeps its angle to
// fp32's last bits; sine and cosine of the rest are fp32.
#include "cache_common.h"

namespace lcv {
namespace {

template <int N>
struct Words {
  u32x4 w[N];
};

// One thread turns 8 values (4 pairs) of a token over a run of heads.
template <typename T, typename P>
__global__ __launch_bounds__(256) void rope_nd_kernel(RopeNd r, int heads_per_part, int parts, int64_t total) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;
  const int chunks = r.pairs / 4;
  const int c = (int)(id % chunks);
  int64_t t = id / chunks;
  const int s = (int)(t % r.S);
  t /= r.S;
  const int part = (int)(t % parts);
  const int b = (int)(t / parts);
  const P* pos = reinterpret_cast<const P*>(r.positions) + (int64_t)b * r.pos_sb + (int64_t)s * r.pos_ss;
  float cs[4], sn[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int pair = 4 * c + i;
    const double turns = (double)pos[r.axis[pair]] * r.turns[pair];
    const float f = (float)(turns - rint(turns));
    sincospif(2.0f * f, &sn[i], &cs[i]);
    sn[i] *= r.sign;
  }
  const T* x = reinterpret_cast<const T*>(r.x.ptr) + (int64_t)b * r.x.sb + (int64_t)s * r.x.ss + 8 * c;
  T* y = reinterpret_cast<T*>(const_cast<void*>(r.y.ptr)) + (int64_t)b * r.y.sb + (int64_t)s * r.y.ss + 8 * c;
  const int h0 = part * heads_per_part;
  const int h1 = h0 + heads_per_part < r.H ? h0 + heads_per_part : r.H;
  constexpr int kWords = sizeof(T) / 2;
  for (int h = h0; h < h1; ++h) {
    const T* xh = x + (int64_t)h * r.x.sh;
    T* yh = y + (int64_t)h * r.y.sh;
    T v[8];
    u32x4 w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const u32x4*>(xh)[i];
    __builtin_memcpy(v, w, sizeof(v));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = to_f32(v[2 * i]), d = to_f32(v[2 * i + 1]);
      v[2 * i] = from_f32<T>(a * cs[i] - d * sn[i]);
      v[2 * i + 1] = from_f32<T>(a * sn[i] + d * cs[i]);
    }
    __builtin_memcpy(w, v, sizeof(v));
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<u32x4*>(yh)[i] = w[i];
  }
}

template <typename T, typename P>
hipError_t launch(const RopeNd& r, hipStream_t stream) {
  const int per = r.H;
  const int parts = (r.H + per - 1) / per;
  const int64_t total = (int64_t)r.B * parts * r.S * (r.pairs / 4);
  hipLaunchKernelGGL((rope_nd_kernel<T, P>), dim3((uint32_t)((total + 255) / 256)), dim3(256), 0, stream, r, per, parts,
                     total);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_pos(const RopeNd& r, int pos_type, hipStream_t stream) {
  switch (pos_type) {
    case kPosI32: return launch<T, int32_t>(r, stream);
    case kPosI64: return launch<T, int64_t>(r, stream);
    default: return launch<T, float>(r, stream);
  }
}

}  // namespace

hipError_t launch_rope_nd(const RopeNd& r, int dtype, int pos_type, hipStream_t stream) {
  switch (dtype) {
    case LCV_BSA_F16: return launch_pos<f16>(r, pos_type, stream);
    case LCV_BSA_BF16: return launch_pos<bf16>(r, pos_type, stream);
    default: return launch_pos<float>(r, pos_type, stream);
  }
}

}  // namespace lcv
