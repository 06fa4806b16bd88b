// Rotary positions with several axes (time, height, width, or any other split of
// the head dim) at positions that the caller gives per token, forward and backward:
//
//   angle t of pair i on axis a: position[s][a] * base^(-2 i / dim_a)
//   y[2i] = x[2i] cos t - x[2i+1] sin t,  y[2i+1] = x[2i] sin t + x[2i+1] cos t
//
// and, since a rotation's transpose turns back, the gradient with -t.  Bound by the
// bytes of x and y.  The angle is taken as turns, position * (frequency / 2 pi), in
// 64 bits with the whole turns dropped, so that a far position keeps its angle to
// fp32's last bits; sine and cosine of the rest are fp32.  57,600 tokens of 32 heads of 128
// in bf16 (944 MB) take 165 us, 5.7 TB/s (a copy of 1 GiB: 5.0); 8 frames of 30 x 52 tokens
// in fp32 (409 MB) 76 us.
//
// A workgroup takes some tokens and heads: its threads form each pair's sine and cosine
// of each token once, in LDS, and then walk the rows 16 bytes a thread, in the order in
// which they lie in memory (tokens of a head next to one another, or heads of a token).
#include "cache_common.h"

namespace lcv {
namespace {

struct Share {
  int32_t tokens, heads;    // of a workgroup
  int32_t token_parts, head_parts;
  int32_t by_token;         // a token's heads lie next to one another
  FastDiv pairs, chunks, inner;  // inner: heads or tokens, whichever lies closer
};
constexpr int kMaxAngles = 2048;  // tokens * pairs of a workgroup

template <typename T, typename P>
__global__ __launch_bounds__(256) void rope_nd_kernel(RopeNd r, Share w) {
  constexpr int kVec = 16 / sizeof(T), kPairs = kVec / 2;
  __shared__ __attribute__((aligned(16))) float cs[2 * kMaxAngles];
  const int tid = threadIdx.x;
  int id = blockIdx.x;
  const int hp = id % w.head_parts;
  id /= w.head_parts;
  const int tp = id % w.token_parts, b = id / w.token_parts;
  const int s0 = tp * w.tokens, h0 = hp * w.heads;
  const int tokens = r.S - s0 < w.tokens ? r.S - s0 : w.tokens, heads = r.H - h0 < w.heads ? r.H - h0 : w.heads;
  const P* pos = reinterpret_cast<const P*>(r.positions) + (int64_t)b * r.pos_sb + (int64_t)s0 * r.pos_ss;
  for (int i = tid; i < tokens * r.pairs; i += 256) {
    const int s = (int)fast_div(i, w.pairs), pair = i - s * r.pairs;
    const double turns = (double)pos[(int64_t)s * r.pos_ss + r.axis[pair]] * r.turns[pair];
    const float f = (float)(turns - rint(turns));
    float sn, c;
    sincospif(2.0f * f, &sn, &c);
    cs[2 * i] = c;
    cs[2 * i + 1] = sn * r.sign;
  }
  __syncthreads();
  const T* x = reinterpret_cast<const T*>(r.x.ptr) + (int64_t)b * r.x.sb + (int64_t)s0 * r.x.ss + (int64_t)h0 * r.x.sh;
  T* y = reinterpret_cast<T*>(const_cast<void*>(r.y.ptr)) + (int64_t)b * r.y.sb + (int64_t)s0 * r.y.ss + (int64_t)h0 * r.y.sh;
  const int chunks = 2 * r.pairs / kVec;
  // The inner count is a full part's, so that one divisor serves; what it adds is skipped.
  const int inner = w.by_token ? w.heads : w.tokens, outer = w.by_token ? tokens : heads;
  const int all = outer * inner * chunks;
  constexpr int kUnroll = 2;
  for (int i0 = tid; i0 < all; i0 += 256 * kUnroll) {
    u32x4 v[kUnroll];
    int64_t to[kUnroll];
    int at[kUnroll];
#pragma unroll
    for (int q = 0; q < kUnroll; ++q) {
      const int i = i0 + 256 * q;
      const int row = (int)fast_div(i < all ? i : 0, w.chunks), c = (i < all ? i : 0) - row * chunks;
      const int a = (int)fast_div(row, w.inner), e = row - a * inner;
      const int s = w.by_token ? a : e, h = w.by_token ? e : a;
      const bool there = i < all && s < tokens && h < heads;
      at[q] = there ? s * r.pairs + c * kPairs : -1;
      to[q] = (int64_t)s * r.y.ss + (int64_t)h * r.y.sh + kVec * c;
      if (there) v[q] = *reinterpret_cast<const u32x4*>(x + (int64_t)s * r.x.ss + (int64_t)h * r.x.sh + kVec * c);
    }
#pragma unroll
    for (int q = 0; q < kUnroll; ++q) {
      if (at[q] < 0) continue;
      T t[kVec];
      __builtin_memcpy(t, &v[q], 16);
#pragma unroll
      for (int p = 0; p < kPairs; ++p) {
        const float c = cs[2 * (at[q] + p)], sn = cs[2 * (at[q] + p) + 1];
        const float a = to_f32(t[2 * p]), d = to_f32(t[2 * p + 1]);
        t[2 * p] = from_f32<T>(a * c - d * sn);
        t[2 * p + 1] = from_f32<T>(a * sn + d * c);
      }
      __builtin_memcpy(&v[q], t, 16);
      *reinterpret_cast<u32x4*>(y + to[q]) = v[q];
    }
  }
}

template <typename T, typename P>
hipError_t launch(const RopeNd& r, hipStream_t stream) {
  constexpr int kVec = 16 / sizeof(T);
  Share w{};
  // Up to 16 tokens and 16 KB: smaller shares even out.  57,600 tokens of 32 heads of 128 in
  // bf16 (8 KB a token) 166 us, in shares of 128 KB 192, of 8 KB 164; 24 heads of 64 in fp16
  // (3 KB a token) 124 us, of 32 KB 132, of 8 KB 141.  Then the heads are split where that
  // leaves CUs idle (their angles are formed anew): 16 tokens of 64 heads 2.8 us, unsplit 3.7.
  const int chunks = 2 * r.pairs / kVec;
  w.tokens = kMaxAngles / r.pairs < 16 ? kMaxAngles / r.pairs : 16;
  while (w.tokens > 1 && (int64_t)w.tokens * r.H * chunks > 1024) w.tokens /= 2;
  w.heads = r.H;
  while (w.heads > 1 && (int64_t)r.B * ((r.S + w.tokens - 1) / w.tokens) * ((r.H + w.heads - 1) / w.heads) < 512 &&
         w.tokens * w.heads * chunks > 256)
    w.heads = (w.heads + 1) / 2;
  w.token_parts = (r.S + w.tokens - 1) / w.tokens;
  w.head_parts = (r.H + w.heads - 1) / w.heads;
  w.by_token = r.x.sh <= r.x.ss;
  w.pairs = make_fastdiv((uint32_t)r.pairs);
  w.chunks = make_fastdiv((uint32_t)chunks);
  w.inner = make_fastdiv((uint32_t)(w.by_token ? w.heads : w.tokens));
  hipLaunchKernelGGL((rope_nd_kernel<T, P>), dim3((uint32_t)((int64_t)r.B * w.token_parts * w.head_parts)), dim3(256), 0,
                     stream, r, w);
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
