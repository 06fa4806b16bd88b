// Attention weights per cached token: w_out[j] = w_in[j] + sum over the rows that see
// token j of exp(scale q.k_j - lse), the rows' lse as cached_attention gives it.  What
// an eviction ranks tokens by.
//
// Both kernels hold 64 keys (one block, one scale) per wave in registers as the B operand
// of S = Q K^T (16 x 16 x 32 MFMAs) and walk the rows: the accumulators hold 4 rows of
// one key, so that a key's sum over rows is a sum over registers.  Lane (G, gi) =
// (lane / 16, lane % 16) holds key 16 t + gi of tile t and D/4 contiguous values from
// G D / 4.  No atomics: the order of every sum is fixed.
#include "cache_attn.h"

namespace lcv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// lse in units of log2; where it is -inf every score is, and any finite number will do.
__device__ __forceinline__ float offset_of(float lse) { return lse == -__builtin_inff() ? 0.0f : lse * kLog2e; }

// What turns a block's products into scores: never zero, so that -inf stays -inf, as in the
// attention.
__device__ __forceinline__ float key_scale(const CacheAttn& a, int64_t block) {
  const float c = a.scale_log2 * a.c.k_scale[block];
  return c > 0x1p-126f ? c : 0x1p-126f;
}

template <typename T, int D>
__device__ __forceinline__ void load_keys(const CacheAttn& a, int64_t block, int lane, typename Mfma<T>::vec8 (&kf)[4][D / 32]) {
  const uint8_t* kb = a.c.k8 + block * (64 * D) + lane % 16 * D + lane / 16 * (D / 4);
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(kb + 16 * t * D + 16 * u);
      kf[t][2 * u] = From8<T>::cvt(w[0], w[1]);
      kf[t][2 * u + 1] = From8<T>::cvt(w[2], w[3]);
    }
}

// Few rows (up to kFewRows a key head, row r = query r / group of head r % group): a
// pass over the keys, one block a wave; the rows come from L2, 16 at a time.  Bound by the
// keys' bytes: one token of 4 requests over 45,480 tokens of 8 heads of 128 (49 MB) takes
// 14 to 15 us, 3.4 TB/s (four waves a SIMD; with the registers of five 5 us more): a wave
// waits for its one block with nothing beside it.
template <typename T, int D>
__global__ __launch_bounds__(256) void few_weights_kernel(CacheAttn a, const float* w_in, float* w_out) {
  typedef typename Mfma<T>::vec8 vec8;
  const int lane = threadIdx.x % 64, G = lane / 16, gi = lane % 16;
  const int64_t block = (int64_t)blockIdx.x * 4 + uniform_i32(threadIdx.x / 64);
  if (block >= (int64_t)a.c.B * a.c.H * a.c.nb) return;
  const int bh = (int)(block / a.c.nb), j = (int)(block % a.c.nb);
  const int b = bh / a.c.H, kvh = bh - b * a.c.H;
  const Lens n = item_lens(a, b);
  const int rows = a.group * a.S;
  const float before = w_in ? w_in[block * 64 + lane] : 0.0f;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (64 * j < n.len) {
    vec8 kf[4][D / 32];
    load_keys<T, D>(a, block, lane, kf);
    const float c = key_scale(a, block);
    for (int r0 = 0; r0 < rows; r0 += 16) {
      const int r = r0 + gi < rows ? r0 + gi : rows - 1;
      const T* q = reinterpret_cast<const T*>(a.q.ptr) + (int64_t)b * a.q.sb +
                   (int64_t)(kvh * a.group + r % a.group) * a.q.sh + (int64_t)(r / a.group) * a.q.ss + G * (D / 4);
      vec8 qf[D / 32];
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks)
        qf[ks] = __builtin_bit_cast(vec8, *reinterpret_cast<const u32x4*>(q + 8 * ks));
      int vis[4];
      float off[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int re = r0 + 4 * G + e < rows ? r0 + 4 * G + e : rows - 1;
        vis[e] = r0 + 4 * G + e < rows ? visible(a, n, re / a.group) - 64 * j - gi : 0;
        off[e] = offset_of(a.lse[((int64_t)b * a.c.H * a.group + kvh * a.group + re % a.group) * a.S + re / a.group]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4 s = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) s = Mfma<T>::mma(qf[ks], kf[t][ks], s);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sum[t] += 16 * t < vis[e] ? fast_exp2(__builtin_fmaf(s[e], c, -off[e])) : 0.0f;
      }
    }
  }
  float got = 0.0f;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const float all = sum_quarters(sum[t]);
    got = G == t ? all : got;  // lane 16 t + gi: key 16 t + gi
  }
  w_out[block * 64 + lane] = before + got;
}

// Many rows: four waves hold 256 keys of a head and walk its queries, head by head of
// the group, 32 rows at a time.  The rows and their lse go straight from memory into a
// ring of three LDS slots, two tiles ahead, one barrier a tile; LDS rows in chunks of 16
// bytes, chunk c of row r at c ^ kswz(r) (attn_common.h).  The exponentials (24 cycles an
// element against 8 of its MFMAs) are the bound: 3120 rows of 32 heads of 128 over 9360
// tokens take 250 us, 957 TFLOP/s, the adding of parts with them; for D = 64 they are twice
// as many for the same products (3000 rows of 16 heads over 9000 tokens 106 us, 520
// TFLOP/s).  Four waves a SIMD hide them (260 and 110 with three, against 256 and 103).
// Bank conflicts take 0.44 of the LDS's active cycles, waiting for it 0.6 % of the waves'.
template <typename T, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4, 4)))
void many_weights_kernel(CacheAttn a, const float* w_in, float* w_out, float* parts, int splits) {
  typedef typename Mfma<T>::vec8 vec8;
  typedef MfmaCfg<T, D> C;
  constexpr int kRows = 32, kRowBytes = 2 * D;
  constexpr int kTile = kRows * kRowBytes;
  constexpr int kLoads = kTile / 4096;                          // 1 KB loads of a wave
  __shared__ __attribute__((aligned(1024))) uint8_t ring[3 * kTile];
  __shared__ __attribute__((aligned(1024))) float ring_lse[3][64];

  const int wid = xcd_linear_work_id(blockIdx.x, gridDim.x);
  const int quads = (a.c.nb + 3) / 4;
  // The items of a head next to one another: an XCD's share is not one item's, which may be short.
  const int kvh = wid / (quads * splits) / a.c.B, b = wid / (quads * splits) % a.c.B, bh = b * a.c.H + kvh;
  const int split = wid / quads % splits;
  const int lane = threadIdx.x % 64, G = lane / 16, gi = lane % 16;
  const int wave = uniform_i32(threadIdx.x / 64);
  const int j = wid % quads * 4 + wave;
  const Lens n = item_lens(a, b);
  const int64_t block = (int64_t)bh * a.c.nb + j;
  const bool mine = j < a.c.nb && 64 * j < n.len;  // wave-uniform
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};

  // Tiles of a head that some row of may see a key of the workgroup; this part's of them.
  const int first_key = wid % quads * 256;
  int tiles = first_key < n.len ? (n.ql + kRows - 1) / kRows : 0, skip = 0;
  if (a.causal && tiles > 0) {  // query i sees first_key from i = first_key - (len - ql) on
    const int i = first_key - (n.len - n.ql);
    skip = i > 0 ? i / kRows : 0;
  }
  const int per_head = tiles - skip > 0 ? tiles - skip : 0;
  const int all = per_head * a.group;
  const int t0 = (int)((int64_t)split * all / splits), t1 = (int)((int64_t)(split + 1) * all / splits);
  if (t0 < t1) {  // workgroup-uniform
    vec8 kf[4][D / 32];
    float c = 0.0f;
    if (mine) {
      load_keys<T, D>(a, block, lane, kf);
      c = key_scale(a, block);
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) kf[t][ks] = __builtin_bit_cast(vec8, u32x4{0u, 0u, 0u, 0u});
    }
    int h = kvh * a.group + t0 / per_head, at_h = t0 % per_head;  // of the next tile to fetch
    auto fetch = [&](int slot) {
      const int i0 = (skip + at_h) * kRows;
      const T* q = reinterpret_cast<const T*>(a.q.ptr) + (int64_t)b * a.q.sb + (int64_t)h * a.q.sh + (int64_t)i0 * a.q.ss;
      const int last = a.S - 1 - i0;  // rows behind the last repeat it
      const __amdgpu_buffer_rsrc_t qrs = __builtin_amdgcn_make_buffer_rsrc((void*)q, (short)0, -1, kBufferFlags);
      const __amdgpu_buffer_rsrc_t lrs = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(a.lse + ((int64_t)b * a.c.H * a.group + h) * a.S + i0), (short)0, -1, kBufferFlags);
      const uint32_t m0 = lds_addr(ring + slot * kTile + 1024 * (kLoads * wave));
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int row = (kLoads * wave + u) * C::kRowsPerDma + lane / C::DC;
        const int src = row < last ? row : last;
        dma16_settled(qrs, (uint32_t)src * (uint32_t)a.q.ss * 2u + 16u * ((lane % C::DC) ^ C::kswz(row)), 0, m0 + 1024u * u);
      }
      const int row = lane % 32 < last ? lane % 32 : last;
      dma4_settled(lrs, 4u * row, lds_addr(ring_lse[slot]));
      if (++at_h == per_head) at_h = 0, ++h;
    };
    int kaddr[D / 32];
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) kaddr[ks] = gi * kRowBytes + 16 * ((G * (D / 32) + ks) ^ C::kswz(gi));
    auto tile = [&](const uint8_t* q, int slot, int i0, auto kind) {
      constexpr bool part = decltype(kind)::value;  // not every row of the tile sees the whole block
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
          const vec8 qf =
              __builtin_bit_cast(vec8, *reinterpret_cast<const u32x4*>(q + kaddr[ks] + rt * (16 * kRowBytes)));
#pragma unroll
          for (int t = 0; t < 4; ++t) s[t] = Mfma<T>::mma(qf, kf[t][ks], s[t]);
        }
        const f32x4 lse = *reinterpret_cast<const f32x4*>(&ring_lse[slot][16 * rt + 4 * G]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float off = __builtin_elementwise_maximum(lse[e], -0x1p100f) * -kLog2e;  // offset_of, an instruction less
          const int left = part ? visible(a, n, i0 + 16 * rt + 4 * G + e) - 64 * j - gi : 64;
#pragma unroll
          for (int t = 0; t < 4; ++t)
            sum[t] += 16 * t < left ? fast_exp2(__builtin_fmaf(s[t][e], c, off)) : 0.0f;
        }
      }
    };
    int slot = 0, tile_i = t0 % per_head;
    fetch(0);
    if (t0 + 1 < t1) fetch(1);
    for (int at = t0; at < t1; ++at) {
      if (at + 1 < t1) wait_vmcnt<kLoads + 1>();
      else wait_vmcnt<0>();
      __syncthreads();  // the tile has landed, and the one before it is read by all
      if (at + 2 < t1) fetch(slot == 0 ? 2 : slot - 1);
      const int i0 = (skip + tile_i) * kRows;
      tile_i = tile_i + 1 == per_head ? 0 : tile_i + 1;
      const int top = i0 + kRows - 1 < n.ql ? visible(a, n, i0 + kRows - 1) : n.len;  // of the tile's real rows, an upper bound
      if (mine && 64 * j < top) {
        const uint8_t* q = ring + slot * kTile;
        if (i0 + kRows > n.ql || 64 * j + 64 > visible(a, n, i0)) tile(q, slot, i0, Flag<true>{});
        else tile(q, slot, i0, Flag<false>{});
      }
      slot = slot == 2 ? 0 : slot + 1;
    }
  }
  float got = 0.0f;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const float s = sum_quarters(sum[t]);
    got = G == t ? s : got;
  }
  if (j >= a.c.nb) return;
  if (splits > 1)
    parts[(int64_t)split * a.c.B * a.c.H * a.c.nb * 64 + block * 64 + lane] = got;
  else
    w_out[block * 64 + lane] = (w_in ? w_in[block * 64 + lane] : 0.0f) + got;
}

__global__ __launch_bounds__(256) void add_parts_kernel(const float* w_in, const float* parts, int splits, int64_t total,
                                                        float* w_out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  float sum = parts[i];
  for (int p = 1; p < splits; ++p) sum += parts[(int64_t)p * total + i];
  w_out[i] = (w_in ? w_in[i] : 0.0f) + sum;
}

// A pass over the keys up to here, a walk over the rows above.  us, 8 key heads of 128: 64
// rows over 9000 tokens 9.3 against 10.7, over two items of 40,000 36 either way; 96 rows
// over these 48 against 36, 128 rows 60 against 32.
constexpr int kFewRows = 64;

// The rows are split over workgroups, to about kParts, where the keys are too few to fill
// the chip: 3120 rows of 32 heads over 9360 tokens 256 us, with 2048 271, with 1024 302; two
// causal prompts of 8 key heads over 2048 and 5000 tokens 109, 120, 138.
constexpr int64_t kParts = 4096;
int row_splits(const CacheAttn& a) {
  if ((int64_t)a.group * a.S <= kFewRows) return 1;
  const int64_t work = (int64_t)a.c.B * a.c.H * ((a.c.nb + 3) / 4), tiles = (int64_t)a.group * ((a.S + 31) / 32);
  int64_t splits = (kParts + work - 1) / work;
  if (splits > tiles / 4) splits = tiles / 4;
  return (int)(splits < 1 ? 1 : splits);
}

template <typename T, int D>
hipError_t launch(const CacheAttn& a, const float* w_in, float* w_out, hipStream_t stream) {
  const int64_t blocks = (int64_t)a.c.B * a.c.H * a.c.nb;
  if ((int64_t)a.group * a.S <= kFewRows) {
    hipLaunchKernelGGL((few_weights_kernel<T, D>), dim3((uint32_t)((blocks + 3) / 4)), dim3(256), 0, stream, a, w_in, w_out);
    return hipGetLastError();
  }
  const int splits = row_splits(a);
  float* parts = reinterpret_cast<float*>(a.workspace);
  hipLaunchKernelGGL((many_weights_kernel<T, D>), dim3((uint32_t)((int64_t)a.c.B * a.c.H * ((a.c.nb + 3) / 4) * splits)),
                     dim3(256), 0, stream, a, w_in, w_out, parts, splits);
  if (splits > 1)
    hipLaunchKernelGGL(add_parts_kernel, dim3((uint32_t)((blocks * 64 + 255) / 256)), dim3(256), 0, stream, w_in, parts,
                       splits, blocks * 64, w_out);
  return hipGetLastError();
}

}  // namespace

size_t cache_weights_workspace(const CacheAttn& a, int D) {
  const int splits = row_splits(a);
  return splits > 1 ? (size_t)splits * a.c.B * a.c.H * a.c.nb * 64 * sizeof(float) : 0;
}

hipError_t launch_cache_weights(const CacheAttn& a, int dtype, int D, const float* w_in, float* w_out,
                                hipStream_t stream) {
  if (dtype == LCV_BSA_F16)
    return D == 64 ? launch<f16, 64>(a, w_in, w_out, stream) : launch<f16, 128>(a, w_in, w_out, stream);
  return D == 64 ? launch<bf16, 64>(a, w_in, w_out, stream) : launch<bf16, 128>(a, w_in, w_out, stream);
}

}  // namespace lcv
