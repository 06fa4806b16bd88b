// Attention over the 8-bit cache (cache_common.h): softmax(scale q k^T) v for any
// number of query rows, grouped heads, ragged lengths read on the device, and a
// causal mask among an item's queries.
//
// The stored bytes go to the matrix cores as T, exactly; a block's scales are powers
// of two and enter where they round nothing.  With u = score * log2(e), a block's key
// scale multiplies u, and its value scale 2^ev is added to the exponent:
//   P' = exp2(u + ev - m),  m the running maximum of u + ev,
//   O  = sum P' v8,         l = sum 2^-ev P',
// so P' <= 1 in any mix of scales, O holds the true sum over 2^m, and l the softmax's
// own denominator.  P' is rounded to T once (bf16 2^-9, fp16 2^-12 relative; an fp16
// P' below 2^-14 loses bits only where the block with the larger values has an e4m3
// step 2^16 times what is lost); sums, maxima and O stay in fp32.
//
// The rows of one key head are its group's queries, row r = query r % S of head
// r / S; a row sees the first `vis` tokens.  What a row does not see has P' = 0, and
// a NaN among the values of such tokens is taken out of its product.
#include "attn_common.h"
#include "cache_common.h"

namespace lcv {
namespace {

constexpr float kNegInf = -__builtin_inff();
constexpr float kLn2 = 0.69314718055994531f;

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

struct Few {
  int32_t tiles, splits;
  float* part_o;   // [work id][16][D]
  float* part_ml;  // [work id][16][2]
};

// The 16 rows of a tile, merged from `n` parts (strides in floats), and written.
template <typename T, int D>
__device__ __forceinline__ void merge_rows(const CacheAttn& a, int b, int kvh, int tile, const float* o, int64_t o_step,
                                           const float* ml, int64_t ml_step, int n, float* to_o, float* to_ml) {
  const int row = threadIdx.x / 16, d0 = threadIdx.x % 16 * (D / 16);
  float m = kNegInf;
  for (int i = 0; i < n; ++i) m = __builtin_elementwise_maximum(m, ml[i * ml_step + 2 * row]);
  const float base = m == kNegInf ? 0.0f : m;
  float l = 0.0f, acc[D / 16];
#pragma unroll
  for (int e = 0; e < D / 16; ++e) acc[e] = 0.0f;
  for (int i = 0; i < n; ++i) {
    const float f = fast_exp2(ml[i * ml_step + 2 * row] - base);
    l = __builtin_fmaf(ml[i * ml_step + 2 * row + 1], f, l);
    const float* src = o + i * o_step + row * D + d0;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) acc[e] = __builtin_fmaf(src[e], f, acc[e]);
  }
  if (to_o) {
#pragma unroll
    for (int e = 0; e < D / 16; ++e) to_o[row * D + d0 + e] = acc[e];
    if (d0 == 0) {
      to_ml[2 * row] = m;
      to_ml[2 * row + 1] = l;
    }
    return;
  }
  const int r = tile * 16 + row;
  if (r >= a.group * a.S) return;
  const int g = r / a.S, i = r - g * a.S;
  const int h = kvh * a.group + g;
  const bool empty = m == kNegInf;
  const float inv = 1.0f / l;
  T* out = reinterpret_cast<T*>(const_cast<void*>(a.out.ptr)) + (int64_t)b * a.out.sb + (int64_t)h * a.out.sh +
           (int64_t)i * a.out.ss + d0;
  T t[D / 16];
#pragma unroll
  for (int e = 0; e < D / 16; ++e) t[e] = from_f32<T>(empty ? 0.0f : acc[e] * inv);
  __builtin_memcpy(__builtin_assume_aligned(out, 2 * D / 16), t, sizeof(t));
  if (a.lse && d0 == 0)
    a.lse[((int64_t)b * a.c.H * a.group + h) * a.S + i] = empty ? kNegInf : (m + __builtin_log2f(l)) * kLn2;
}

// Few rows: one workgroup walks a part of one key head's blocks for 16 rows, its
// four waves taking every fourth block.  The operands come straight from memory in
// the layout the products want (16 x 16 x 32 MFMAs, P in registers): lane (G, gi) =
// (lane / 16, lane % 16) holds, of key tile t of a block, key 16 (gi / 4) + 4 t + gi % 4
// at D/4 contiguous values from G D / 4, so that the scores' accumulators hold keys
// 16 G + 4 t + i of row gi, which is the order of the 16 bytes that a lane reads of
// v8's row 16 dt + gi.
template <typename T, int D>
__global__ __launch_bounds__(256) void few_rows_kernel(CacheAttn a, Few f) {
  typedef typename Mfma<T>::vec8 vec8;
  __shared__ float part_o[4][16 * D];
  __shared__ float part_ml[4][32];
  const int wid = xcd_linear_work_id(blockIdx.x, gridDim.x);
  const int tile = wid % f.tiles;
  const int split = wid / f.tiles % f.splits;
  const int bh = wid / (f.tiles * f.splits);
  const int b = bh / a.c.H, kvh = bh - b * a.c.H;
  const int lane = threadIdx.x % 64, G = lane / 16, gi = lane % 16;
  const int wave = uniform_i32(threadIdx.x / 64);
  const Lens n = item_lens(a, b);
  const int rows = a.group * a.S;
  int r = tile * 16 + gi;
  const int vis = r < rows ? visible(a, n, r % a.S) : 0;
  r = r < rows ? r : 0;
  int most = vis;
  for (int o = 1; o < 16; o <<= 1) {
    const int x = __shfl_xor(most, o);
    most = x > most ? x : most;
  }
  most = uniform_i32(most);
  const int nblk = (most + 63) / 64;
  const int j0 = (int)((int64_t)split * nblk / f.splits), j1 = (int)((int64_t)(split + 1) * nblk / f.splits);

  const T* q = reinterpret_cast<const T*>(a.q.ptr) + (int64_t)b * a.q.sb +
               (int64_t)(kvh * a.group + r / a.S) * a.q.sh + (int64_t)(r % a.S) * a.q.ss + G * (D / 4);
  vec8 qf[D / 32];
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks)
    qf[ks] = __builtin_bit_cast(vec8, *reinterpret_cast<const u32x4*>(q + 8 * ks));

  const uint8_t* kb = a.c.k8 + (int64_t)bh * a.c.nb * (64 * D) + (16 * (gi / 4) + gi % 4) * D + G * (D / 4);
  const uint8_t* vb = a.c.v8 + (int64_t)bh * a.c.nb * (64 * D) + gi * 64 + 16 * G;
  const float* ksc = a.c.k_scale + (int64_t)bh * a.c.nb;
  const float* vsc = a.c.v_scale + (int64_t)bh * a.c.nb;

  f32x4 o[D / 16];
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = kNegInf, l = 0.0f;
  for (int j = j0 + wave; j < j1; j += 4) {
    u32x4 kw[4][D / 64], vw[D / 16];
    const uint8_t* kj = kb + (int64_t)j * (64 * D);
    const uint8_t* vj = vb + (int64_t)j * (64 * D);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int u = 0; u < D / 64; ++u) kw[t][u] = *reinterpret_cast<const u32x4*>(kj + 4 * t * D + 16 * u);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) vw[dt] = *reinterpret_cast<const u32x4*>(vj + dt * (16 * 64));
    const float c = a.scale_log2 * ksc[j];
    const int ev = exponent_of(vsc[j]);
    f32x4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks)
        s[t] = Mfma<T>::mma(From8<T>::cvt(kw[t][ks / 2][2 * (ks % 2)], kw[t][ks / 2][2 * (ks % 2) + 1]), qf[ks], s[t]);
    }
    const int left = vis - 64 * j - 16 * G;  // key 4 t + i of this lane is seen if below
    float mx = kNegInf;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] = 4 * t + i < left ? s[t][i] * c : kNegInf;
        mx = __builtin_elementwise_maximum(mx, s[t][i]);
      }
    mx = max_quarters(mx);
    const float fev = (float)ev;
    const float m_new = __builtin_elementwise_maximum(m, mx + fev);
    const float base = m_new == kNegInf ? 0.0f : m_new;
    const float down = fast_exp2(m - base);
    const float off = fev - base;
    vec8 pf[2];
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = fast_exp2(s[t][i] + off);
        sum += p;
        pf[t / 2][4 * (t % 2) + i] = from_f32<T>(p);
      }
    l = __builtin_fmaf(l, down, sum * pow2i(-ev));
    m = m_new;
    // A block that some row sees in part: NaN bytes count for the rows that see them alone.
    uint32_t bad = 0;
    if (__ballot(vis > 0 && vis < 64 * j + 64)) {
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= nan_bytes(vw[dt][e]);
    }
    if (__ballot(bad != 0)) {
      vec8 seen[2];
#pragma unroll
      for (int e = 0; e < 16; ++e) seen[e / 8][e % 8] = from_f32<T>(e < left ? 1.0f : 0.0f);
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        u32x4 is;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t nan = nan_bytes(vw[dt][e]);
          is[e] = nan >> 7 << 3;                        // 0x08: a positive number
          vw[dt][e] &= ~((nan - (nan >> 7)) | nan);     // zero
        }
        f32x4 hit = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < 2; ++u) hit = Mfma<T>::mma(From8<T>::cvt(is[2 * u], is[2 * u + 1]), seen[u], hit);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (hit[i] > 0.0f) o[dt][i] = __builtin_nanf("");
      }
    }
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[dt][i] *= down;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        o[dt] = Mfma<T>::mma(From8<T>::cvt(vw[dt][2 * u], vw[dt][2 * u + 1]), pf[u], o[dt]);
    }
  }
  l = sum_quarters(l);
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt)
    *reinterpret_cast<f32x4*>(&part_o[wave][gi * D + 16 * dt + 4 * G]) = o[dt];
  if (G == 0) {
    part_ml[wave][2 * gi] = m;
    part_ml[wave][2 * gi + 1] = l;
  }
  __syncthreads();
  merge_rows<T, D>(a, b, kvh, tile, part_o[0], 16 * D, part_ml[0], 32, 4,
                   f.splits > 1 ? f.part_o + (int64_t)wid * (16 * D) : nullptr, f.part_ml + (int64_t)wid * 32);
}

template <typename T, int D>
__global__ __launch_bounds__(256) void join_kernel(CacheAttn a, Few f) {
  const int tile = blockIdx.x % f.tiles, bh = blockIdx.x / f.tiles;
  const int64_t first = (int64_t)bh * f.tiles * f.splits + tile;
  merge_rows<T, D>(a, bh / a.c.H, bh % a.c.H, tile, f.part_o + first * (16 * D), (int64_t)f.tiles * (16 * D),
                   f.part_ml + first * 32, (int64_t)f.tiles * 32, f.splits, nullptr, nullptr);
}

Few plan_few(const CacheAttn& a) {
  Few f{};
  f.tiles = (a.group * a.S + 15) / 16;
  const int64_t work = (int64_t)a.c.B * a.c.H * f.tiles;
  const int64_t blocks = (a.max_len + 63) / 64;
  int64_t splits = (1024 + work - 1) / work;
  if (splits > blocks / 4) splits = blocks / 4;
  f.splits = (int)(splits < 1 ? 1 : splits);
  return f;
}

size_t few_bytes(const CacheAttn& a, const Few& f, int D) {
  return f.splits > 1 ? (size_t)a.c.B * a.c.H * f.tiles * f.splits * 16 * (D + 2) * sizeof(float) : 0;
}

template <typename T, int D>
hipError_t launch(const CacheAttn& a, hipStream_t stream) {
  Few f = plan_few(a);
  const int64_t parts = (int64_t)a.c.B * a.c.H * f.tiles * f.splits;
  f.part_o = reinterpret_cast<float*>(a.workspace);
  f.part_ml = f.part_o + parts * 16 * D;
  hipLaunchKernelGGL((few_rows_kernel<T, D>), dim3((uint32_t)parts), dim3(256), 0, stream, a, f);
  if (f.splits > 1)
    hipLaunchKernelGGL((join_kernel<T, D>), dim3((uint32_t)(parts / f.splits)), dim3(256), 0, stream, a, f);
  return hipGetLastError();
}

}  // namespace

size_t cache_attn_workspace(const CacheAttn& a, int D) { return few_bytes(a, plan_few(a), D); }

hipError_t launch_cache_attn(const CacheAttn& a, int dtype, int D, hipStream_t stream) {
  if (dtype == LCV_BSA_F16) return D == 64 ? launch<f16, 64>(a, stream) : launch<f16, 128>(a, stream);
  return D == 64 ? launch<bf16, 64>(a, stream) : launch<bf16, 128>(a, stream);
}

}  // namespace lcv
