// The 8-bit KV cache: layout, e4m3 conversions and the host-side launchers.
//
// A cache holds, per batch item and head, blocks of 64 tokens.  Keys lie row by
// row, k8 [capacity][D]; values block by block with the tokens innermost,
// v8 [capacity / 64][D][64], which is how the product P V reads them as a matrix
// operand.  Each block has one scale for its keys and one for its values, a power
// of two 2^e with e in [-60, 60]: a stored byte x (e4m3: 4 exponent bits, 3
// mantissa bits, largest value 448, one NaN, no infinity) stands for x 2^e, so a
// change of scale moves exponents and rounds nothing but the smallest values.
#pragma once

#include "bsa_common.h"

namespace lcv {

constexpr int kCacheBlock = 64;    // tokens under one scale
constexpr int kMaxScaleExp = 60;   // scales are 2^-60 .. 2^60

struct Cache8 {
  uint8_t* k8;
  uint8_t* v8;
  float* k_scale;
  float* v_scale;
  int32_t B, H, nb;  // nb: blocks of a head
};

// Queries over a cache: q and out [B, H, S, D] with H = group * c.H.
struct CacheAttn {
  Cache8 c;
  Tensor4 q, out;
  float* lse;              // [B, H, S], or null
  const int32_t* lengths;  // [B] tokens held
  const int32_t* q_lens;   // [B] real queries, or null (all S)
  int32_t group, S, max_len, causal;
  float scale_log2;        // sm_scale * log2(e)
  void* workspace;         // the parts of a split walk, or null
};

hipError_t launch_cache_append(const Cache8& c, const Tensor4& k, const Tensor4& v, int dtype, int S, int D,
                               const int32_t* start, const int32_t* counts, hipStream_t stream);

size_t cache_attn_workspace(const CacheAttn& a, int D);
hipError_t launch_cache_attn(const CacheAttn& a, int dtype, int D, hipStream_t stream);

// a.lse is read; w_in [B, c.H, 64 c.nb] or null, w_out the same shape.
size_t cache_weights_workspace(const CacheAttn& a, int D);
hipError_t launch_cache_weights(const CacheAttn& a, int dtype, int D, const float* w_in, float* w_out,
                                hipStream_t stream);

// src with weights [B, H, 64 src.nb] -> dst (its own nb), w_out [B, H, 64 dst.nb],
// kept [B, H, keep], new_lengths [B].
hipError_t launch_cache_evict(const Cache8& src, const int32_t* lengths, const float* weights, int keep, int recent,
                              const Cache8& dst, float* w_out, int32_t* kept, int32_t* new_lengths, int D,
                              hipStream_t stream);

constexpr int kRopeMaxPairs = 128;
struct RopeNd {
  Tensor4 x, y;
  const void* positions;  // [B or 1, S, axes]
  int64_t pos_sb, pos_ss;
  int32_t B, H, S, pairs;
  float sign;
  uint8_t axis[kRopeMaxPairs];   // of each pair
  double turns[kRopeMaxPairs];   // turns a position step makes
};
enum { kPosI32 = 0, kPosI64 = 1, kPosF32 = 2 };
hipError_t launch_rope_nd(const RopeNd& r, int dtype, int pos_type, hipStream_t stream);

#ifdef __HIPCC__
// The least e in [-60, 60] with amax <= 448 2^e = 0.875 * 2^(e + 9).
__device__ __forceinline__ int scale_exponent(float amax) {
  if (!(amax > 0.0f)) return -kMaxScaleExp;
  int x;
  const float m = frexpf(amax, &x);  // amax = m 2^x, 1/2 <= m < 1
  const int e = x - 9 + (m > 0.875f ? 1 : 0);
  return e < -kMaxScaleExp ? -kMaxScaleExp : e > kMaxScaleExp ? kMaxScaleExp : e;
}

// 2^e for e in [-126, 127].
__device__ __forceinline__ float pow2i(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }
// The exponent of a scale (a power of two within the cache's range).
__device__ __forceinline__ int exponent_of(float scale) {
  const int e = (int)((__builtin_bit_cast(uint32_t, scale) >> 23) & 255u) - 127;
  return e < -kMaxScaleExp ? -kMaxScaleExp : e > kMaxScaleExp ? kMaxScaleExp : e;
}

// Values that e4m3 cannot hold under this scale, infinities and NaN become NaN.
__device__ __forceinline__ float storable(float y) { return __builtin_fabsf(y) <= 448.0f ? y : __builtin_nanf(""); }
// Four values to four bytes of e4m3, to nearest and even.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(storable(a), storable(b), 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(storable(c), storable(d), w, true);
  return (uint32_t)w;
}
// Bytes of a word that hold NaN (0x7f or 0xff), as 0x80 in each.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ void unpack_e4m3(uint32_t w, float* y) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  y[0] = lo[0], y[1] = lo[1], y[2] = hi[0], y[3] = hi[1];
}

// Eight bytes of e4m3 as eight values of T: exact in fp16 and bf16.
template <typename T>
struct From8;
template <>
struct From8<bf16> {
  typedef bf16 vec2 __attribute__((ext_vector_type(2)));
  __device__ static bf16x8 cvt(uint32_t lo, uint32_t hi) {
    const vec2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    const vec2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const vec2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    const vec2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
};
template <>
struct From8<f16> {
  typedef f16 vec2 __attribute__((ext_vector_type(2)));
  __device__ static f16x8 cvt(uint32_t lo, uint32_t hi) {
    const vec2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
    const vec2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const vec2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
    const vec2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
};
#endif

}  // namespace lcv
