// Attention over the 8-bit cache (cache_common.h): softmax(scale q k^T) v for any
// number of query rows, grouped heads, ragged lengths read on the device, and a
// causal mask among an item's queries.
//
// The stored bytes go to the matrix cores exactly, as T or as they are; a block's scales
// are powers of two and enter where they round nothing: the key scale multiplies
// u = score * log2(e), the value scale 2^ev multiplies sums in fp32 or is added to u.
//
// P is rounded to T once, after its sum (bf16 2^-9, fp16 2^-12 relative), and fp16 holds
// nothing below 2^-25.  A block of a small value scale must not get there beside one of a
// large scale, however small its scale: what the large block stores may be zeros in all
// channels but one.  So fp16 products are formed under one scale, or scales at most
// kSpread apart, and P are powers above that limit.  Sums, maxima and O stay in fp32, in
// which no mix of scales in [2^-60, 2^60] leaves the range; a token whose weight is below
// 2^-40 of the heaviest's may be left out of the row's sum.
//
// The rows of one key head are its group's queries, row r = query r / group of the
// group's head r % group; a row sees the first `vis` tokens, rows in order no fewer.  What
// a row does not see has P' = 0, and a NaN among the values of such tokens is taken out of
// its product.  A row all of whose scores are -inf counts as one that sees nothing.
#include "cache_attn.h"

namespace lcv {
namespace {

constexpr float kNegInf = -__builtin_inff();
constexpr float kLn2 = 0.69314718055994531f;

// What the rows [r0, r1) of a key head see: the most of any, and the least of those that
// see any token.
struct Reach {
  int most, least;
};
__device__ __forceinline__ Reach reach(const CacheAttn& a, const Lens& n, int r0, int r1) {
  const int rows = a.group * a.S;
  if (r1 > rows) r1 = rows;
  const int i0 = r0 / a.group;
  if (r0 >= r1 || i0 >= n.ql) return {0, 0};
  int i1 = (r1 - 1) / a.group;
  if (i1 >= n.ql) i1 = n.ql - 1;
  const int least = visible(a, n, i0);
  return {visible(a, n, i1), least > 0 ? least : 1};
}

// How the walk over the blocks is split.  Many rows: into parts of `per` blocks, at most
// `splits` of an item, part s of item b in slot s B + b.  Few rows: per is 0, the parts go
// by the lengths (few_per), at most `splits` of all items, which take the slots one after
// another.  A part's sums and maxima lie in the workspace by (slot, key head, 16 rows).
struct Parts {
  int32_t tiles;  // of 16 rows, of one key head
  int32_t splits, per;
  float* o;       // [slots][H][tiles][16][D]
  float* ml;      // [slots][H][tiles][16][2]
  int32_t* items; // [B][2], few rows: an item's first slot, the blocks of its parts
};
__device__ __forceinline__ int64_t part_at(const CacheAttn& a, const Parts& p, int slot, int kvh, int tile) {
  return ((int64_t)slot * a.c.H + kvh) * p.tiles + tile;
}

__device__ __forceinline__ int item_blocks(const CacheAttn& a, int b) { return (item_lens(a, b).len + 63) / 64; }

// Few rows: the blocks of a part, so that all items together, `walks` times each, make
// about kFewParts parts, from the lengths, not from the bound on them: 4 requests of 3000
// tokens in a cache of 65,536 take 12.5 us against 19.5 (6 tokens over 8200, 4097, 1 and
// 12,000 22.2 against 21.6).  us: kFewParts 512 (640, 768): 8 requests over 168,716 tokens
// 68 (75, 76), 32 heads over 18,720 33 (37, 37).  kFewBlocks 8 (4, 16): one token over 30,000
// of one head 16 (21, 16), four over 2048 of 8 heads 15 (14, 17).  A walk of up to kOnePart
// blocks is not worth a second launch: 24 rows over 1000 tokens 14.0, in parts of 8 18.3.
constexpr int kFewParts = 512, kFewBlocks = 8, kOnePart = 16;
__device__ __forceinline__ int few_per(const CacheAttn& a, int walks, int blocks) {  // blocks: item `lane`'s
  for (int b = 64 + threadIdx.x % 64; b < a.c.B; b += 64) blocks += item_blocks(a, b);
  for (int o = 1; o < 64 && o < a.c.B; o <<= 1) blocks += __shfl_xor(blocks, o);
  const int64_t all = __builtin_amdgcn_readlane(blocks, 0);
  const int per = (int)((all * walks + 4 * kFewParts - 1) / (4 * kFewParts) * 4);
  return per < kFewBlocks ? kFewBlocks : per;
}
// An item's own: a short history is one part.
__device__ __forceinline__ int item_per(int blocks, int per) { return blocks <= kOnePart ? kOnePart : per; }
__device__ __forceinline__ int item_parts(int blocks, int per) {
  return blocks <= kOnePart ? 1 : (blocks + per - 1) / per;
}

template <typename T>
__device__ __forceinline__ T* out_row(const CacheAttn& a, int b, int kvh, int r) {
  return reinterpret_cast<T*>(const_cast<void*>(a.out.ptr)) + (int64_t)b * a.out.sb +
         (int64_t)(kvh * a.group + r % a.group) * a.out.sh + (int64_t)(r / a.group) * a.out.ss;
}
template <typename T>
__device__ __forceinline__ const T* q_row(const CacheAttn& a, int b, int kvh, int r) {
  return reinterpret_cast<const T*>(a.q.ptr) + (int64_t)b * a.q.sb + (int64_t)(kvh * a.group + r % a.group) * a.q.sh +
         (int64_t)(r / a.group) * a.q.ss;
}
__device__ __forceinline__ int64_t lse_at(const CacheAttn& a, int b, int kvh, int r) {
  return ((int64_t)b * a.c.H * a.group + kvh * a.group + r % a.group) * a.S + r / a.group;
}

// P of up to 2^kRoom: fp16 then loses what is below 2^-37 of the largest.
template <typename T>
constexpr int kRoom = 0;
template <>
constexpr int kRoom<f16> = 12;

// Few rows: one workgroup walks a part of one key head's blocks for 16 or 32 rows (NT
// tiles), its four waves taking every fourth block.  The operands come straight from
// memory in the layout the products want (16 x 16 x 32 MFMAs, P in registers): lane
// (G, gi) = (lane / 16, lane % 16) holds, of key tile t of a block, key
// 16 (gi / 4) + 4 t + gi % 4 at D/4 contiguous values from G D / 4, so that the scores'
// accumulators hold keys 16 G + 4 t + i of row gi, which is the order of the 16 bytes
// that a lane reads of v8's row 16 dt + gi.  Keys and values of a wave's next block are
// asked for as soon as those of this one are used.
//
// A block's P lie under its own maximum, and its product is added to O in fp32 under that
// of the walk and with the block's value scale: O holds the values' own size.
//
// Bound by the cache's bytes: a token each of 8 requests over 168,716 tokens in all, 8 heads
// of 128 (345 MB), takes 68 us with the join's 5, 5.1 TB/s (a copy of 1 GiB: 5.0); one over
// 501 tokens 5.3 us, its loads' latency.  The next block's operands need the registers of
// three waves a SIMD for 16 rows (74 us; two 79, four 111) and of two for 32 (24 rows of 8
// heads over 9000 tokens 17 us; three 27).  In the joining of the waves' parts all 16 rows
// of part_o lie in the same banks (0.8 of the LDS's active cycles): 1.4 % of the waves'
// cycles go by waiting for it over long histories, 12 % where a wave walks two blocks (6
// tokens of 4 requests, 17 us).
template <typename T, int D, int NT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(NT == 1 ? 3 : 2, NT == 1 ? 3 : 2)))
void few_rows_kernel(CacheAttn a, Parts p) {
  typedef typename Mfma<T>::vec8 vec8;
  __shared__ float part_o[4][16 * D];
  __shared__ float part_ml[4][32];
  // Work: (part, key head) u, whose tiles follow one another on one XCD (u % 8), the heads
  // next to one another.  Only the parts that an item has are counted: a long item beside
  // short ones then finds the chip free of workgroups that have nothing to do (22 us
  // against 16 for lengths of 8200, 4097, 1 and 12000).
  const int slot = blockIdx.x / kNumXcd, wide = p.tiles / NT;
  const int tile = slot % wide * NT;
  const int u = slot / wide * kNumXcd + blockIdx.x % kNumXcd;
  const int lane = threadIdx.x % 64, G = lane / 16, gi = lane % 16;
  const int kvh = u % a.c.H;
  const int slot_at = u / a.c.H;
  const int blocks = lane < a.c.B ? item_blocks(a, lane) : 0, few = few_per(a, a.c.H * (p.tiles / NT), blocks);
  int b = a.c.B == 1 ? 0 : -1, split = slot_at;
  for (int b0 = 0; b < 0 && b0 < a.c.B; b0 += 64) {  // wave-uniform
    const int parts = b0 + lane < a.c.B ? item_parts(b0 == 0 ? blocks : item_blocks(a, b0 + lane), few) : 0;
    int upto = parts;
    for (int o = 1; o < 64 && o < a.c.B; o <<= 1) {
      const int x = __shfl_up(upto, o);
      upto += lane >= o ? x : 0;
    }
    const uint64_t beyond = __ballot(split < upto);
    if (beyond) {
      const int l = __builtin_ctzll(beyond);
      b = b0 + l;
      split -= __builtin_amdgcn_readlane(upto - parts, l);
    } else {
      split -= __builtin_amdgcn_readlane(upto, 63);
    }
  }
  if (b < 0) return;
  const int bh = b * a.c.H + kvh;
  const int wave = uniform_i32(threadIdx.x / 64);
  const Lens n = item_lens(a, b);
  const int rows = a.group * a.S;
  const Reach all = reach(a, n, 16 * tile, 16 * tile + 16 * NT);
  const int nblk = (all.most + 63) / 64, per = item_per((n.len + 63) / 64, few);
  if (p.items && split == 0 && kvh == 0 && tile == 0 && threadIdx.x == 0)
    p.items[2 * b] = slot_at, p.items[2 * b + 1] = per;
  const int j0 = split * per;
  const int j1 = j0 + per < nblk ? j0 + per : nblk;
  if (split > 0 && j0 >= nblk) return;  // the first part of a tile always answers

  vec8 qf[NT][D / 32];
  int vis[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = 16 * (tile + nt) + gi;
    vis[nt] = r < rows ? visible(a, n, r / a.group) : 0;
    const T* q = q_row<T>(a, b, kvh, r < rows ? r : 0) + G * (D / 4);
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks)
      qf[nt][ks] = __builtin_bit_cast(vec8, *reinterpret_cast<const u32x4*>(q + 8 * ks));
  }
  const uint8_t* kb = a.c.k8 + (int64_t)bh * a.c.nb * (64 * D) + (16 * (gi / 4) + gi % 4) * D + G * (D / 4);
  const uint8_t* vb = a.c.v8 + (int64_t)bh * a.c.nb * (64 * D) + gi * 64 + 16 * G;
  const float* ksc = a.c.k_scale + (int64_t)bh * a.c.nb;
  const float* vsc = a.c.v_scale + (int64_t)bh * a.c.nb;

  f32x4 o[NT][D / 16];
  float m[NT], l[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = kNegInf, l[nt] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) o[nt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  u32x4 kw[4][D / 64], vw[D / 16];
  float ks_next = 0.0f, vs_next = 0.0f;
  auto ask_k = [&](int j, int t) {
#pragma unroll
    for (int u = 0; u < D / 64; ++u)
      kw[t][u] = *reinterpret_cast<const u32x4*>(kb + (int64_t)j * (64 * D) + 4 * t * D + 16 * u);
  };
  auto ask_v = [&](int j, int dt) {
    vw[dt] = *reinterpret_cast<const u32x4*>(vb + (int64_t)j * (64 * D) + dt * (16 * 64));
  };
  auto ask_scales = [&](int j) { ks_next = ksc[j], vs_next = vsc[j]; };
  int j = j0 + wave;
  if (j < j1) {
    ask_scales(j);
#pragma unroll
    for (int t = 0; t < 4; ++t) ask_k(j, t);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) ask_v(j, dt);
  }
  for (; j < j1; j += 4) {
    const int jn = j + 4 < j1 ? j + 4 : j;  // past the end: this block again, unused
    const float c = a.scale_log2 * ks_next > 0x1p-126f ? a.scale_log2 * ks_next : 0x1p-126f;
    const float unit = pow2i(exponent_of(vs_next));
    f32x4 s[NT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) {
        const vec8 k = From8<T>::cvt(kw[t][ks / 2][2 * (ks % 2)], kw[t][ks / 2][2 * (ks % 2) + 1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][t] = Mfma<T>::mma(k, qf[nt][ks], s[nt][t]);
      }
    }
    ask_scales(jn);
#pragma unroll
    for (int t = 0; t < 4; ++t) ask_k(jn, t);
    const bool part = 64 * j + 64 > all.least;  // some row sees the block in part
    vec8 pf[NT][2];
    float down[NT], up[NT];  // what is there, and what the block adds, to the new maximum
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (part) {
        const int left = here(vis[nt] - 64 * j - 16 * G);
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (x >= left) s[nt][x / 4][x % 4] = kNegInf;
      }
      float mx = s[nt][0][0];
#pragma unroll
      for (int x = 1; x < 16; ++x) mx = __builtin_elementwise_maximum(mx, s[nt][x / 4][x % 4]);
      const float top = max_quarters(mx) * c;  // the block's own, under which its P lie
      const float m_new = __builtin_elementwise_maximum(m[nt], top);
      const float base = m_new == kNegInf ? 0.0f : m_new;
      down[nt] = fast_exp2(m[nt] - base);
      up[nt] = fast_exp2(top - base) * pow2i(-kRoom<T>);
      const float off = (float)kRoom<T> - (top == kNegInf ? 0.0f : top);
      float sum = 0.0f;
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const float e = fast_exp2(__builtin_fmaf(s[nt][x / 4][x % 4], c, off));
        sum += e;
        pf[nt][x / 8][x % 8] = from_f32<T>(e);
      }
      l[nt] = __builtin_fmaf(l[nt], down[nt], sum * up[nt]);
      up[nt] *= unit;
      m[nt] = m_new;
    }
    // NaN bytes of a block that some row sees in part count for the rows that see them alone.
    uint32_t bad = 0;
    if (part) {
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= nan_bytes(vw[dt][e]);
    }
    if (__ballot(bad != 0)) {
      vec8 seen[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 16; ++x)
          seen[nt][x / 8][x % 8] = from_f32<T>(64 * j + 16 * G + x < vis[nt] ? 1.0f : 0.0f);
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        u32x4 is;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t nan = nan_bytes(vw[dt][e]);
          is[e] = nan >> 7 << 3;                     // a positive number for each
          vw[dt][e] &= ~((nan - (nan >> 7)) | nan);  // zero
        }
        const vec8 i0 = From8<T>::cvt(is[0], is[1]), i1 = From8<T>::cvt(is[2], is[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          f32x4 hit = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          hit = Mfma<T>::mma(i0, seen[nt][0], hit);
          hit = Mfma<T>::mma(i1, seen[nt][1], hit);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (hit[i] > 0.0f) o[nt][dt][i] = __builtin_nanf("");
        }
      }
    }
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      const vec8 v0 = From8<T>::cvt(vw[dt][0], vw[dt][1]), v1 = From8<T>::cvt(vw[dt][2], vw[dt][3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        f32x4 t = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        t = Mfma<T>::mma(v0, pf[nt][0], t);
        t = Mfma<T>::mma(v1, pf[nt][1], t);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][dt][i] = __builtin_fmaf(t[i], up[nt], o[nt][dt][i] * down[nt]);
      }
      ask_v(jn, dt);
    }
  }
  // The four waves' parts together: thread (row, 16th of D).
  const bool last = nblk <= per;  // nothing to join
  const int row = threadIdx.x / 16, d0 = threadIdx.x % 16 * (D / 16);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float sum = sum_quarters(l[nt]);
    __syncthreads();
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
      *reinterpret_cast<f32x4*>(&part_o[wave][gi * D + 16 * dt + 4 * G]) = o[nt][dt];
    if (G == 0) {
      part_ml[wave][2 * gi] = m[nt];
      part_ml[wave][2 * gi + 1] = sum;
    }
    __syncthreads();
    const int r = 16 * (tile + nt) + row;
    if (r >= rows) continue;
    float top = kNegInf;
    for (int w = 0; w < 4; ++w) top = __builtin_elementwise_maximum(top, part_ml[w][2 * row]);
    const float base = top == kNegInf ? 0.0f : top;
    float lsum = 0.0f, acc[D / 16];
#pragma unroll
    for (int e = 0; e < D / 16; ++e) acc[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = fast_exp2(part_ml[w][2 * row] - base);
      lsum = __builtin_fmaf(part_ml[w][2 * row + 1], f, lsum);
#pragma unroll
      for (int e = 0; e < D / 16; ++e) acc[e] = __builtin_fmaf(part_o[w][row * D + d0 + e], f, acc[e]);
    }
    if (last) {
      const bool empty = top == kNegInf || visible(a, n, r / a.group) == 0;
      const float inv = 1.0f / lsum;
      T t[D / 16];
#pragma unroll
      for (int e = 0; e < D / 16; ++e) t[e] = from_f32<T>(empty ? 0.0f : acc[e] * inv);
      __builtin_memcpy(__builtin_assume_aligned(out_row<T>(a, b, kvh, r) + d0, 2 * D / 16), t, sizeof(t));
      if (a.lse && d0 == 0) a.lse[lse_at(a, b, kvh, r)] = empty ? kNegInf : (top + __builtin_log2f(lsum)) * kLn2;
    } else {
      const int64_t at = part_at(a, p, slot_at, kvh, tile + nt);
      __builtin_memcpy(__builtin_assume_aligned(p.o + at * (16 * D) + row * D + d0, 4 * D / 16), acc, sizeof(acc));
      if (d0 == 0) {
        p.ml[at * 32 + 2 * row] = top;
        p.ml[at * 32 + 2 * row + 1] = lsum;
      }
    }
  }
}

// A row's parts together.  `wide` rows share a walk, whose reach says how many parts there
// are.  THREADS threads take a row: a wave where there are few rows, so that many loads
// are under way, 16 where there are many (kJoinRows).
template <typename T, int D, int THREADS>
__global__ __launch_bounds__(256) void join_kernel(CacheAttn a, Parts p, int wide, int64_t total) {
  constexpr int kN = D / THREADS;
  const int64_t id = (int64_t)blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS;
  if (id >= total) return;
  const int rows = a.group * a.S;
  const int r = (int)(id % rows), bh = (int)(id / rows);
  const int b = bh / a.c.H, kvh = bh - b * a.c.H;
  int slot = b, step = a.c.B, per = p.per;
  if (per == 0) {  // few rows: the items' parts one after another
    slot = p.items[2 * b], per = p.items[2 * b + 1];
    step = 1;
  }
  const Lens n = item_lens(a, b);
  const int first = r / wide * wide;
  const int nblk = (reach(a, n, first, first + wide).most + 63) / 64;
  if (nblk <= per) return;  // written already
  const int parts = (nblk + per - 1) / per;
  const int lane = threadIdx.x % THREADS;
  const int64_t stride = (int64_t)step * a.c.H * p.tiles;
  const int64_t at = part_at(a, p, slot, kvh, r / 16);
  const float* ml = p.ml + at * 32 + 2 * (r % 16);
  const float* o = p.o + at * (16 * D) + r % 16 * D + lane * kN;
  float top = kNegInf;
  for (int i = lane; i < parts; i += THREADS) top = __builtin_elementwise_maximum(top, ml[i * stride * 32]);
  for (int x = 1; x < THREADS; x <<= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, x));
  const float base = top == kNegInf ? 0.0f : top;
  float lsum = 0.0f, acc[kN];
#pragma unroll
  for (int e = 0; e < kN; ++e) acc[e] = 0.0f;
  // So many parts' loads are under way together (past the last part it again, unused): one
  // token of one head over 30,000 tokens 15.8 us with eight, 17.5 with four.
  constexpr int kBatch = THREADS == 64 ? 8 : 4;
  for (int i0 = 0; i0 < parts; i0 += kBatch) {
    float x[kBatch][kN], m[kBatch], l[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = i0 + k < parts ? i0 + k : parts - 1;
      m[k] = ml[i * stride * 32];
      l[k] = ml[i * stride * 32 + 1];
      __builtin_memcpy(x[k], __builtin_assume_aligned(o + i * stride * (16 * D), 4 * kN > 16 ? 16 : 4 * kN), sizeof(x[k]));
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const bool there = i0 + k < parts;
      const float f = fast_exp2(m[k] - base);
      lsum = there ? __builtin_fmaf(l[k], f, lsum) : lsum;
#pragma unroll
      for (int e = 0; e < kN; ++e) acc[e] = there ? __builtin_fmaf(x[k][e], f, acc[e]) : acc[e];
    }
  }
  const bool empty = top == kNegInf || visible(a, n, r / a.group) == 0;
  const float inv = 1.0f / lsum;
  T t[kN];
#pragma unroll
  for (int e = 0; e < kN; ++e) t[e] = from_f32<T>(empty ? 0.0f : acc[e] * inv);
  __builtin_memcpy(__builtin_assume_aligned(out_row<T>(a, b, kvh, r) + lane * kN, 2 * kN), t, sizeof(t));
  if (a.lse && lane == 0) a.lse[lse_at(a, b, kvh, r)] = empty ? kNegInf : (top + __builtin_log2f(lsum)) * kLn2;
}

// us: four prompts of 1 to 2048 queries over 391 to 5000 tokens 176 sorted, 233 in turn; four
// items of 700 to 4000 tokens 157 and 218; eight equal ones of 512 tokens 22.5 and 21.4;
// sixteen 27 and 23, as the search goes over the items.
constexpr int kSorted = 8;

// Which tile of 128 rows of which item a workgroup takes: the r-th of a key head's.
struct Turn {
  int b, tile;
};

// Items next to one another, of each the longest walk first.  A CU's workgroups, 32 apart,
// are not all one item's.
__device__ __forceinline__ Turn in_turn(const CacheAttn& a, int tiles, int r) {
  const int b = (r + r / a.c.B * a.c.B / 32) % a.c.B, at = r / a.c.B;
  return {b, a.causal ? tiles - 1 - at : at};
}

// The longest walk of all items first (up to kSorted of them).  Lane b holds item b's
// lengths; the walk of the r-th is the largest x that more than r tiles reach, looked for
// 64 numbers at a time.
__device__ __forceinline__ Turn by_length(const CacheAttn& a, int tiles, int r) {
  const int lane = threadIdx.x % 64;
  const Lens mine = item_lens(a, lane < a.c.B ? lane : 0);
  auto item = [&](int b) {
    return Lens{__builtin_amdgcn_readlane(mine.len, b), __builtin_amdgcn_readlane(mine.ql, b)};
  };
  auto real = [&](const Lens& n) { return (n.ql * a.group + 127) / 128; };  // tiles with queries
  auto reaching = [&](const Lens& n, int x) {  // how many of the item's tiles walk x blocks or more
    if (x == 0) return tiles;
    if (64 * (x - 1) >= n.len || n.ql == 0) return 0;
    const int t = real(n), i = 64 * (x - 1) - (n.len - n.ql);  // the first query to see the x-th block
    const int first = a.causal && i > 0 ? i * a.group / 128 : 0;
    return t - (first < t ? first : t - 1);
  };
  int lo = 0, hi = (a.max_len + 63) / 64 + 1;  // more than r reach lo, not so hi
  while (hi - lo > 1) {                        // wave-uniform
    const int step = (hi - lo + 64) / 65, x = lo + (lane + 1) * step;
    int all = 0;
    for (int b = 0; b < a.c.B; ++b) all += x < hi ? reaching(item(b), x) : 0;
    const int n = __popcll(__ballot(all > r));
    lo += n * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  // Lane b: the tiles of item b that walk lo blocks, behind those of the items before.
  const int from = reaching(mine, lo + 1), n = lane < a.c.B ? reaching(mine, lo) - from : 0;
  int longer = lane < a.c.B ? from : 0, upto = n;
  for (int o = 1; o < a.c.B; o <<= 1) {
    longer += __shfl_xor(longer, o);
    const int x = __shfl_up(upto, o);
    upto += lane >= o ? x : 0;
  }
  r -= __builtin_amdgcn_readlane(longer, 0);
  const int b = __builtin_ctzll(__ballot(upto > r));
  const int at = __builtin_amdgcn_readlane(from + n - upto, b) + r, t = __builtin_amdgcn_readlane(real(mine), b);
  return {b, at < t ? t - 1 - at : at};  // the tiles without queries last
}

// Many rows: one workgroup of four waves takes 128 rows of one key head, wave w rows
// 32 w .. 32 w + 31, and walks a part of the blocks.  A block's 8 KB of keys and 8 KB
// of values (D = 128) go straight from memory into a ring of three LDS slots, two
// blocks ahead, one barrier a block; every wave turns the bytes into T as it reads
// them.  Operands as in few_rows_kernel.  LDS rows are 64 or 128 bytes in chunks of 16,
// chunk c of row r at c ^ swz(r), which spreads the 16 rows that a lane group reads over
// the banks.  (Conflicts still take half of the LDS's active cycles, which access causes
// them is not known; the waves wait for it in 1 % of theirs.)
//
// Here the value scale 2^ev is added to the exponent,
//   P' = exp2(u + ev - m),  O = sum P' v8,  l = sum 2^(least - ev) P',  least the least ev,
// so that O holds the true sum over 2^m and l the softmax's denominator over 2^(m - least).
// A row's offset m comes from its first half block, and later halves need no maximum: in
// bf16 that of u + ev, in fp16 that of u plus least (or plus the largest ev less kLift, if
// that is more), so that P' is no less than a token's weight against the half's heaviest (or
// 2^-3 of it).  Where a half's sum passes a bound (fp16's largest number; 2^40 in bf16), or
// is NaN, or the half's scores are all -inf, or the value scales are more than 2^kSpread
// apart, the workgroup walks with care: band by band of scales so close, each walked once
// for the rows' maxima of u + ev and once for its products, and O and l brought from band
// to band.  The next band's offset lies no more than kFar below the largest so far, which
// leaves O room in fp32.  (Rescaling O inside the walk costs it 60 registers: 4310 us, below
// 3600.)  12,480 fp16 queries of 32 heads over 18,720 tokens take 3670 us, beside one value
// that is 2^16 times the others 6990, with scores that pass the bound 9390.
//
// Bound by instructions: a block costs a wave 64 MFMAs (1024 cycles), 32 exponentials with
// their sums and 128 conversions of bytes, about 2350 cycles with the MFMAs beside them.
// D = 128 leaves registers for three waves a SIMD (12,480 queries of 32 heads over 18,720
// tokens: two 3804 us, three 3580), D = 64 for four (4000 queries of 16 heads over 9000
// tokens: 195 us, three 200).
//
// kBytes (bf16, D = 128, long walks): the keys' bytes go to 16 x 16 x 128 MFMAs as they are,
// and a row's values as the sum of two e4m3 numbers under the row's 2^e and 2^(e - 4): two
// passes at twice bf16's rate, and 64 conversions less.  e4m3's 4 bits twice are bf16's 8,
// so that values from 2^(e - 6) on (2^-14.8 of the row's largest) are exact; one below is
// off by no more than 2^(e - 14).  What that adds up to in a score, if every key held its
// scale's largest number there, has to stay below kLost in u for all rows of the workgroup
// (normed rows of 128 against normed keys: 2^-20 for each such value, of which a row has
// 0.02), else it converts the keys: a row whose largest value is far above the rest, which
// its keys may not answer, or an infinite one.
// 12,480 queries of 32 heads over 18,720 tokens then take 3380 us, 1132 TFLOP/s, against
// 3710 (a product of 8192^3 makes 1214; 3250 to 3500 from card to card); 2048 over
// 2048 of 32 heads 80 against 83.
template <typename T>
constexpr float kMaxSum = 0x1p40f;
template <>
constexpr float kMaxSum<f16> = 65504.0f;
template <typename T>
constexpr int kSpread = 32;
template <>
constexpr int kSpread<f16> = 12;
constexpr int kLift = 9;
constexpr float kFar = 80.0f;

template <typename T>
constexpr bool kIsBf16 = false;
template <>
constexpr bool kIsBf16<bf16> = true;

// Of blocks j0 .. j1 - 1: the largest exponent of a value scale below `below`, and the
// least one; without any, one below and one above the range.  With KEYS, the largest key
// scale too.
struct Span {
  int top, least;
  float key;
};
template <bool KEYS>
__device__ __forceinline__ Span span_of(const float* ksc, const float* vsc, int j0, int j1, int below) {
  Span s = {-kMaxScaleExp - 1, kMaxScaleExp + 1, 0.0f};
  for (int j = j0 + threadIdx.x % 64; j < j1; j += 64) {
    const float key = KEYS ? ksc[j] : 0.0f;
    const int e = exponent_of(vsc[j]);
    s.top = e < below && e > s.top ? e : s.top;
    s.least = e < s.least ? e : s.least;
    s.key = fmaxf(s.key, key);
  }
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_xor(s.top, o), l = __shfl_xor(s.least, o);
    s.top = t > s.top ? t : s.top;
    s.least = l < s.least ? l : s.least;
    if constexpr (KEYS) s.key = fmaxf(s.key, __shfl_xor(s.key, o));
  }
  return {uniform_i32(s.top), uniform_i32(s.least), s.key};
}
typedef int i32x8 __attribute__((ext_vector_type(8)));
constexpr float kLost = 0x1p-14f;

// The least e >= -123 with |q| <= 448 2^e = 1.75 2^(e + 8) in the lane's row, of which it
// holds a quarter.
template <int D, typename V>
__device__ __forceinline__ int byte_exponent(const V (&q)[D / 32]) {
  float amax = 0.0f;
#pragma unroll
  for (int x = 0; x < D / 4; ++x) amax = fmaxf(amax, __builtin_fabsf(to_f32(q[x / 8][x % 8])));
  const int e = (int)((__builtin_bit_cast(uint32_t, max_quarters(amax)) + 0x1fffffu) >> 23) - 135;
  return e < -123 ? -123 : e;
}

template <int D>
struct Tile8 {
  static constexpr int kKeyChunks = D / 16;  // of a key's row
  __device__ static int kswz(int r) { return D == 128 ? ((r >> 4) << 1 | ((r >> 1) & 1)) : r >> 4; }
  __device__ static int vswz(int d) { return (d >> 2) & 3; }
};

template <typename T, int D, bool kBytes>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 128 ? 3 : 4, D == 128 ? 3 : 4)))
void many_rows_kernel(CacheAttn a, Parts p) {
  typedef typename Mfma<T>::vec8 vec8;
  typedef Tile8<D> C;
  constexpr int kHalf = 64 * D;      // bytes of a block's keys or values
  constexpr int kSlot = 2 * kHalf;
  constexpr int kLoads = kHalf / 4096;  // 1 KB loads of a wave for keys, and for values
  constexpr int kRows = 128;
  __shared__ __attribute__((aligned(1024))) uint8_t ring[3 * kSlot];
  static_assert(3 * kSlot >= kRows * 2 * D, "the ring stages the output rows");

  const int wid = xcd_linear_work_id(blockIdx.x, gridDim.x);
  const int tiles = p.tiles / 8;  // of 128 rows
  const int of_head = wid % (a.c.B * tiles), split = wid / (a.c.B * tiles) % p.splits;
  const int kvh = wid / (a.c.B * tiles * p.splits);
  const bool sorted = a.c.B > 1 && a.c.B <= kSorted && p.splits == 1;
  const Turn turn = sorted ? by_length(a, tiles, of_head) : in_turn(a, tiles, of_head);
  const int b = turn.b, tile = turn.tile;
  const int bh = b * a.c.H + kvh;
  const int tid = threadIdx.x, lane = tid % 64, G = lane / 16, gi = lane % 16;
  const int wave = uniform_i32(tid / 64);
  const Lens n = item_lens(a, b);
  const int rows = a.group * a.S;
  const int nblk = (reach(a, n, kRows * tile, kRows * tile + kRows).most + 63) / 64;
  const int j0 = split * p.per;
  const int j1 = j0 + p.per < nblk ? j0 + p.per : nblk;
  if (split > 0 && j0 >= nblk) return;  // the first part of a tile always answers
  // One wave's reading decides for all, as barriers go by it.
  __shared__ Span wave_span;
  if (tid < 64) {
    const Span s = span_of<kBytes>(a.c.k_scale + (int64_t)bh * a.c.nb, a.c.v_scale + (int64_t)bh * a.c.nb, j0, j1,
                                   kMaxScaleExp + 1);
    if (tid == 0) wave_span = s;
  }
  const Reach mine = reach(a, n, kRows * tile + 32 * wave, kRows * tile + 32 * wave + 32);
  const int own = uniform_i32(mine.most), least = uniform_i32(mine.least);

  int vis[2];
  vec8 qf[2][D / 32];
#pragma unroll
  for (int qt = 0; qt < 2; ++qt) {
    const int r = kRows * tile + 32 * wave + 16 * qt + gi;
    vis[qt] = r < rows ? visible(a, n, r / a.group) : 0;
    const T* q = q_row<T>(a, b, kvh, r < rows ? r : 0) + G * (D / 4);
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks)  // a row that sees nothing: no number of its own gets into a sum
      qf[qt][ks] = __builtin_bit_cast(
          vec8, vis[qt] > 0 ? *reinterpret_cast<const u32x4*>(q + 8 * ks) : u32x4{0u, 0u, 0u, 0u});
  }
  __syncthreads();
  const Span span = {uniform_i32(wave_span.top), uniform_i32(wave_span.least), wave_span.key};
  __shared__ int wave_dirty[4];
  auto rest = [&](auto form) __attribute__((always_inline)) {
    constexpr bool bytes = decltype(form)::value;
    i32x8 q8[2][2];  // [query tile][first, rest]
    int q8_scale[2];
    if constexpr (bytes) {
#pragma unroll
      for (int qt = 0; qt < 2; ++qt) {
        const int e = byte_exponent<D>(qf[qt]);
        const float inv = pow2i(-e);
#pragma unroll
        for (int w = 0; w < D / 16; ++w) {
          float x[4], y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = to_f32(qf[qt][w / 2][4 * (w % 2) + i]) * inv;
          const uint32_t word = pack_e4m3(x[0], x[1], x[2], x[3]);
          unpack_e4m3(word, y);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = (x[i] - y[i]) * 16.0f;
          q8[qt][0][w] = (int)word;
          q8[qt][1][w] = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3],
                                                        __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), true);
        }
        q8_scale[qt] = e + 127;
      }
    }

    const uint32_t head_bytes = (uint32_t)a.c.nb * (uint32_t)kHalf;  // capacities are limited so that this fits
    const uint8_t* vhead = a.c.v8 + (int64_t)bh * a.c.nb * kHalf;
    const __amdgpu_buffer_rsrc_t krs = __builtin_amdgcn_make_buffer_rsrc(
        a.c.k8 + (int64_t)bh * a.c.nb * kHalf, (short)0, (int)head_bytes, kBufferFlags);
    const __amdgpu_buffer_rsrc_t vrs =
        __builtin_amdgcn_make_buffer_rsrc((void*)vhead, (short)0, (int)head_bytes, kBufferFlags);
    uint32_t ko[kLoads], vo[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int slot = 64 * (kLoads * wave + u) + lane;  // 16-byte chunk of the block
      const int kr = slot / C::kKeyChunks, kc = slot % C::kKeyChunks;
      ko[u] = 16u * (uint32_t)(kr * C::kKeyChunks + (kc ^ C::kswz(kr)));
      const int vr = slot / 4, vc = slot % 4;
      vo[u] = 16u * (uint32_t)(vr * 4 + (vc ^ C::vswz(vr)));
    }
    auto fetch = [&](int j, int slot) {
      const uint32_t m0 = lds_addr(ring + slot * kSlot + 1024 * (kLoads * wave));
      const int off = (int)((uint32_t)j * (uint32_t)kHalf);
#pragma unroll
      for (int u = 0; u < kLoads; ++u) dma16_settled(krs, ko[u], off, m0 + 1024u * u);
#pragma unroll
      for (int u = 0; u < kLoads; ++u) dma16_settled(vrs, vo[u], off, m0 + kHalf + 1024u * u);
    };

    // The scales of 64 blocks at a time: lane l holds block base + l's.
    const float* ksc = a.c.k_scale + (int64_t)bh * a.c.nb;
    const float* vsc = a.c.v_scale + (int64_t)bh * a.c.nb;
    float ks64 = 0.0f, vs64 = 0.0f;
    auto scales = [&](int base) {
      const int j = base + lane < a.c.nb ? base + lane : a.c.nb - 1;
      ks64 = ksc[j];
      vs64 = vsc[j];
    };

    // A block's keys go in two halves: half h of lane group G is keys 16 G + 8 (h ^ G % 2)
    // .. + 7 (the groups alternate, so that the 8 bytes that a half reads of each of v8's
    // chunks lie in all banks), two key tiles of 4 a group.
    const int hk = 8 * (G & 1), hr = 8 * ((gi / 4) & 1);
    int kaddr[2][D / 64], vaddr[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = 16 * (gi / 4) + (hr ^ (8 * h)) + gi % 4;  // its swizzle is that of the lane, whatever the tile
#pragma unroll
      for (int u = 0; u < D / 64; ++u) kaddr[h][u] = row * D + 16 * ((G * (D / 64) + u) ^ C::kswz(row));
      vaddr[h] = kHalf + gi * 64 + 16 * (G ^ C::vswz(gi)) + (hk ^ (8 * h));
    }

    f32x4 o[D / 16][2];
    float m[2], l[2];
    bool nan_found = false;

    f32x4 s[2][2][2];  // [half][key tile][query tile]
    vec8 pf[2][2];     // [half][query tile]
    float sum[2];
    auto qk = [&](const uint8_t* tile8, int h) {
      constexpr int kReads = 2 * (D / 64);  // read r: key tile r / (D / 64), chunk r % (D / 64)
      u32x4 kw[kReads];
#pragma unroll
      for (int r = 0; r < kReads; ++r)
        kw[r] = *reinterpret_cast<const u32x4*>(tile8 + kaddr[h][r % (D / 64)] + 4 * (r / (D / 64)) * D);
#pragma unroll
      for (int t = 0; t < 2; ++t) s[h][t][0] = s[h][t][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (bytes) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          i32x8 k;
#pragma unroll
          for (int x = 0; x < 8; ++x) k[x] = (int)kw[2 * t + x / 4][x % 4];
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int qt = 0; qt < 2; ++qt)
              s[h][t][qt] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                  k, q8[qt][part], s[h][t][qt], 0, 0, 0, 127, 0, q8_scale[qt] - 4 * part);
        }
        return;
      }
#pragma unroll
      for (int r = 0; r < kReads; ++r) {
        const int t = r / (D / 64), u = r % (D / 64);
        const vec8 k0 = From8<T>::cvt(kw[r][0], kw[r][1]), k1 = From8<T>::cvt(kw[r][2], kw[r][3]);
        s[h][t][0] = Mfma<T>::mma(k0, qf[0][2 * u], s[h][t][0]);
        s[h][t][1] = Mfma<T>::mma(k0, qf[1][2 * u], s[h][t][1]);
        s[h][t][0] = Mfma<T>::mma(k1, qf[0][2 * u + 1], s[h][t][0]);
        s[h][t][1] = Mfma<T>::mma(k1, qf[1][2 * u + 1], s[h][t][1]);
      }
    };
    auto mask = [&](int j, int h) {
#pragma unroll
      for (int qt = 0; qt < 2; ++qt) {
        const int left = here(vis[qt] - 64 * j - 16 * G - (hk ^ (8 * h)));
#pragma unroll
        for (int x = 0; x < 8; ++x)
          if (x >= left) s[h][x / 4][qt][x % 4] = kNegInf;
      }
    };
    auto row_max = [&](int h, int qt) {
      float mx = s[h][0][qt][0];
#pragma unroll
      for (int x = 1; x < 8; ++x) mx = __builtin_elementwise_maximum(mx, s[h][x / 4][qt][x % 4]);
      return max_quarters(mx);
    };
    auto raise = [&](int h, float c, float ev) {
#pragma unroll
      for (int qt = 0; qt < 2; ++qt)
        m[qt] = __builtin_elementwise_maximum(m[qt], __builtin_fmaf(row_max(h, qt), c, ev));
    };
    auto key_scale = [&](int j) {
      const float c = a.scale_log2 * __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ks64), j & 63));
      return c > 0x1p-126f ? c : 0x1p-126f;  // so that a masked score of -inf times c is -inf
    };
    auto exps = [&](int h, float c, float ev) {
#pragma unroll
      for (int qt = 0; qt < 2; ++qt) {
        const float off = m[qt] == kNegInf ? ev : ev - m[qt];
        sum[qt] = 0.0f;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float p = fast_exp2(__builtin_fmaf(s[h][x / 4][qt][x % 4], c, off));
          sum[qt] += p;
          pf[h][qt][x] = from_f32<T>(p);
        }
      }
    };
    auto pv = [&](const uint8_t* tile8, int h) {
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(tile8 + vaddr[h] + dt * (16 * 64));
        const vec8 v = From8<T>::cvt(w[0], w[1]);
        o[dt][0] = Mfma<T>::mma(v, pf[h][0], o[dt][0]);
        o[dt][1] = Mfma<T>::mma(v, pf[h][1], o[dt][1]);
      }
    };
    // The same where some row sees the block in part: NaN count as zero here, and are put
    // where they belong at the end.
    auto pv_part = [&](const uint8_t* tile8, int h) {
      uint32_t bad = 0;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        u32x2 w = *reinterpret_cast<const u32x2*>(tile8 + vaddr[h] + dt * (16 * 64));
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t nan = nan_bytes(w[x]);
          bad |= nan;
          w[x] &= ~((nan - (nan >> 7)) | nan);
        }
        const vec8 v = From8<T>::cvt(w[0], w[1]);
        o[dt][0] = Mfma<T>::mma(v, pf[h][0], o[dt][0]);
        o[dt][1] = Mfma<T>::mma(v, pf[h][1], o[dt][1]);
      }
      if (__ballot(bad != 0)) nan_found = true;
    };

    auto value_exponent = [&](int j) {
      return exponent_of(__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vs64), j & 63)));
    };
    const float lifted = (float)(span.top - kLift > span.least ? span.top - kLift : span.least);
    bool dirty = false;
    // careful: the offsets are known.
    auto block = [&](int j, int slot, int e, auto kind, auto how) {
      constexpr bool part = decltype(kind)::value;  // some row of the wave sees the block in part
      constexpr bool careful = decltype(how)::value;
      const uint8_t* tile8 = ring + slot * kSlot;
      const float c = key_scale(j), ev = (float)e, unit = pow2i(span.least - e);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        qk(tile8, h);
        if constexpr (part) mask(j, h);
        if constexpr (!careful) {
          if (h == 0 && j == j0) {
            raise(h, c, kIsBf16<T> ? ev : lifted);
            if (__ballot((m[0] == kNegInf && vis[0] > 64 * j0) || (m[1] == kNegInf && vis[1] > 64 * j0))) dirty = true;
          }
        }
        exps(h, c, ev);
        if constexpr (!careful) {
          if (__ballot(!(sum[0] <= kMaxSum<T> && sum[1] <= kMaxSum<T>))) dirty = true;
        }
        l[0] = __builtin_fmaf(sum[0], unit, l[0]);
        l[1] = __builtin_fmaf(sum[1], unit, l[1]);
        if constexpr (part) pv_part(tile8, h);
        else pv(tile8, h);
      }
    };
    // Blocks before `whole` are seen whole by every row of the wave that sees any token.
    const int whole = own == 0 ? 0 : least / 64 < j1 ? least / 64 : j1;
    int j, slot;
    auto begin = [&] {
      j = j0, slot = 0;
      scales(j0 & ~63);
      fetch(j0, 0);
      if (j0 + 1 < j1) fetch(j0 + 1, 1);
    };
    auto next = [&] {
      if (j + 1 < j1) wait_vmcnt<2 * kLoads>();
      else wait_vmcnt<0>();
      __syncthreads();  // block j has landed, and the one before it is read by all
      if ((j & 63) == 0 && j > j0) scales(j);
      if (j + 2 < j1) fetch(j + 2, slot == 0 ? 2 : slot - 1);
    };
    auto clear = [&] {
      m[0] = m[1] = kNegInf;
      l[0] = l[1] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int qt = 0; qt < 2; ++qt) o[dt][qt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    };
    clear();
    bool careful = span.top - span.least > kSpread<T>;  // workgroup-uniform
    if (!careful && j0 < j1) {
      begin();
      for (; j < whole; ++j) {
        next();
        block(j, slot, value_exponent(j), Flag<false>{}, Flag<false>{});
        slot = slot == 2 ? 0 : slot + 1;
      }
      for (; j < j1; ++j) {
        next();
        if (64 * j < own) block(j, slot, value_exponent(j), Flag<true>{}, Flag<false>{});
        slot = slot == 2 ? 0 : slot + 1;
      }
      if (lane == 0) wave_dirty[wave] = dirty ? 1 : 0;
      __syncthreads();  // the ring is free, the flags are there
      careful = uniform_i32(wave_dirty[0] | wave_dirty[1] | wave_dirty[2] | wave_dirty[3]) != 0;
      if (careful) clear();
    }
    if (careful) {
      float reached[2] = {kNegInf, kNegInf};  // the largest u + ev so far
      for (int band = span.top;;) {           // value scales of kSpread exponents up to `band`
        auto mine = [&](int j, int e) { return 64 * j < own && e <= band && e >= band - kSpread<T>; };
        const float held[2] = {m[0], m[1]};
        m[0] = m[1] = kNegInf;
        begin();
        for (; j < j1; ++j, slot = slot == 2 ? 0 : slot + 1) {  // the rows' maxima
          next();
          const int e = value_exponent(j);
          if (!mine(j, e)) continue;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            qk(ring + slot * kSlot, h);
            if (j >= whole) mask(j, h);
            raise(h, key_scale(j), (float)e);
          }
        }
        __syncthreads();  // the ring is free
#pragma unroll
        for (int qt = 0; qt < 2; ++qt) {
          float f = 1.0f;
          if (m[qt] == kNegInf) {  // nothing of the band, or nothing that counts
            m[qt] = held[qt];
          } else {
            reached[qt] = __builtin_elementwise_maximum(reached[qt], m[qt]);
            m[qt] = __builtin_elementwise_maximum(m[qt], reached[qt] - kFar) - (float)kRoom<T>;
            if (held[qt] != kNegInf) f = fast_exp2(held[qt] - m[qt]);
          }
          l[qt] *= f;
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[dt][qt][i] *= f;
        }
        begin();
        for (; j < whole; ++j, slot = slot == 2 ? 0 : slot + 1) {
          next();
          const int e = value_exponent(j);
          if (mine(j, e)) block(j, slot, e, Flag<false>{}, Flag<true>{});
        }
        for (; j < j1; ++j, slot = slot == 2 ? 0 : slot + 1) {
          next();
          const int e = value_exponent(j);
          if (mine(j, e)) block(j, slot, e, Flag<true>{}, Flag<true>{});
        }
        const int lower = span_of<false>(ksc, vsc, j0, j1, band - kSpread<T>).top;
        if (tid == 0) wave_span.top = lower;
        __syncthreads();  // the ring is free
        band = uniform_i32(wave_span.top);
        if (band < span.least) break;
      }
    }
    if (nan_found) {  // wave-uniform, rare: rows that see a NaN among the values get one
      for (int j = whole > j0 ? whole : j0; j < j1 && 64 * j < own; ++j) {
        const uint8_t* vj = vhead + (int64_t)j * kHalf + gi * 64 + 16 * G;
        vec8 seen[2][2];
#pragma unroll
        for (int qt = 0; qt < 2; ++qt)
#pragma unroll
          for (int x = 0; x < 16; ++x)
            seen[x / 8][qt][x % 8] = from_f32<T>(64 * j + 16 * G + x < vis[qt] ? 1.0f : 0.0f);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
          u32x4 is = *reinterpret_cast<const u32x4*>(vj + dt * (16 * 64));
#pragma unroll
          for (int x = 0; x < 4; ++x) is[x] = nan_bytes(is[x]) >> 7 << 3;  // a positive number for each NaN
          const vec8 i0 = From8<T>::cvt(is[0], is[1]), i1 = From8<T>::cvt(is[2], is[3]);
#pragma unroll
          for (int qt = 0; qt < 2; ++qt) {
            f32x4 hit = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            hit = Mfma<T>::mma(i0, seen[0][qt], hit);
            hit = Mfma<T>::mma(i1, seen[1][qt], hit);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (hit[i] > 0.0f) o[dt][qt][i] = __builtin_nanf("");
          }
        }
      }
    }
    __syncthreads();  // the ring is free

    const float size = pow2i(span.least);
    if (nblk > p.per) {  // under the offset of l, as few_rows_kernel's
      const int64_t part = part_at(a, p, split * a.c.B + b, kvh, 8 * tile + 2 * wave);
#pragma unroll
      for (int qt = 0; qt < 2; ++qt) {
        float* po = p.o + (part + qt) * (16 * D) + gi * D + 4 * G;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) *reinterpret_cast<f32x4*>(po + 16 * dt) = o[dt][qt] * size;
        const float all = sum_quarters(l[qt]);
        if (G == 0) {
          float* ml = p.ml + (part + qt) * 32 + 2 * gi;
          ml[0] = vis[qt] > 64 * j0 ? m[qt] - (float)span.least : kNegInf;  // a row that saw none of this part
          ml[1] = vis[qt] > 64 * j0 ? all : 0.0f;
        }
      }
      return;
    }
#pragma unroll
    for (int qt = 0; qt < 2; ++qt) {
      const float all = sum_quarters(l[qt]);
      const bool empty = vis[qt] == 0 || all == 0.0f;
      const float inv = size / all;
      const int row = 32 * wave + 16 * qt + gi;
      uint8_t* orow = ring + row * (2 * D);
      const int swz = (row / (128 / D)) % (D / 8);
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        u32x2 w;
#pragma unroll
        for (int x = 0; x < 2; ++x)
          w[x] = bits16(from_f32<T>(empty ? 0.0f : o[dt][qt][2 * x] * inv)) |
                 (bits16(from_f32<T>(empty ? 0.0f : o[dt][qt][2 * x + 1] * inv)) << 16);
        *reinterpret_cast<u32x2*>(orow + 16 * ((2 * dt + G / 2) ^ swz) + 8 * (G % 2)) = w;
      }
      const int r = kRows * tile + row;
      if (a.lse && G == 0 && r < rows)
        a.lse[lse_at(a, b, kvh, r)] = empty ? kNegInf : (m[qt] - (float)span.least + __builtin_log2f(all)) * kLn2;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kRows * (D / 8) / 256; ++u) {
      const int piece = tid + 256 * u, row = piece / (D / 8), c = piece % (D / 8);
      const int r = kRows * tile + row;
      if (r >= rows) continue;
      *reinterpret_cast<u32x4*>(out_row<T>(a, b, kvh, r) + 8 * c) =
          *reinterpret_cast<const u32x4*>(ring + row * (2 * D) + 16 * (c ^ ((row / (128 / D)) % (D / 8))));
    }
  };
  if constexpr (kBytes) {
    bool fine = true;
#pragma unroll
    for (int qt = 0; qt < 2; ++qt) {
      const int e = byte_exponent<D>(qf[qt]);
      const float bound = 0x1p-6f * pow2i(e);
      float small = 0.0f;  // values that may be off
#pragma unroll
      for (int x = 0; x < D / 4; ++x) {
        const float y = __builtin_fabsf(to_f32(qf[qt][x / 8][x % 8]));
        small += y != 0.0f && y < bound ? 1.0f : 0.0f;
      }
      const float lost = sum_quarters(small) * (0x1p-8f * bound) * (448.0f * span.key) * a.scale_log2;
      fine = fine && e < 120 && lost <= kLost;  // false for an infinite value, and for a NaN
    }
    if (!__syncthreads_or(!fine)) {
      rest(Flag<true>{});
      return;
    }
  }
  rest(Flag<false>{});
}

// Tiles of 32 rows straight from memory up to here, of 128 through LDS above.  us, 8 heads
// over two items of 1000 (one of 9000, two of 40,000) tokens, bf16, D = 128: 64 rows 14 (23,
// 56) against 19 (25, 69), 96 rows 14 (25, 69) against 20 (26, 71), 128 rows 14 (31, 80)
// against 21 (29, 74).
constexpr int kFewRows = 96;
enum Kind { kFew16, kFew32, kMany };

Kind kind_of(const CacheAttn& a) {
  const int rows = a.group * a.S;
  return rows <= 16 ? kFew16 : rows <= kFewRows ? kFew32 : kMany;
}

// Many rows: parts are written and joined in fp32, 64 KB a tile, so walks are split only
// where there are fewer than two a CU.  us, D = 128, bf16: 512 walks of 32 blocks 78, in two
// parts each 96, in five 122; D = 64, 500 walks of 141 blocks 198 in two, 222 in one.  Parts
// of at least kManyBlocks 6 (4, 8): 128 rows of 8 heads over 9000 tokens 28 (28, 30), over
// two items of 1000 20 (20, 24), 2048 causal queries of 4 heads over one key head 30 (31,
// 29).  128 walks of up to kManyOnePart 8 blocks 20.5, in two parts 23.5.
constexpr int64_t kManyParts = 512, kManyBlocks = 6, kManyOnePart = 8;
// Walks of fewer blocks convert the keys (kBytes above): forming the two numbers takes 1.5 us
// a workgroup.  us, 2048 queries of 32 heads over 8 key heads: over 8 blocks 29.4, as bytes
// 31.1; over 16 45.3 and 45.5, over 32 77.9 and 74.6 (three causal prompts: 117 and 119).
constexpr int kLongWalk = 32;
// us, walk and join: 256 rows 73 with a wave a row, 78 with 16 threads; 64,000 rows 212, 192.
constexpr int64_t kJoinRows = 4096;

int wide_of(Kind kind) { return kind == kMany ? 128 : kind == kFew32 ? 32 : 16; }

Parts plan(const CacheAttn& a) {
  Parts p{};
  const Kind kind = kind_of(a);
  const int64_t rows = (int64_t)a.group * a.S, blocks = ((int64_t)a.max_len + 63) / 64;
  const int wide = wide_of(kind);
  const int64_t walks = (int64_t)a.c.H * ((rows + wide - 1) / wide);  // of an item
  p.tiles = (int)((rows + wide - 1) / wide * (wide / 16));
  if (kind == kMany) {
    int64_t per = blocks;
    if (blocks > kManyOnePart) {
      const int64_t splits = (kManyParts + a.c.B * walks - 1) / (a.c.B * walks);
      per = (blocks + splits - 1) / splits;
      if (per < kManyBlocks) per = kManyBlocks;
    }
    p.per = (int)(per < blocks ? per : blocks);
    p.splits = (int)((blocks + p.per - 1) / p.per);
  } else {  // a part holds at least kFewParts-th of all blocks, so each item adds one to kFewParts / walks
    const int64_t each = (blocks + kFewBlocks - 1) / kFewBlocks, more = kFewParts / walks;
    p.splits = (int)(blocks <= kOnePart ? a.c.B : a.c.B * each < a.c.B + more ? a.c.B * each : a.c.B + more);
  }
  return p;
}

// The slots of parts in the workspace; 0: no part is joined.
int64_t slots_of(const CacheAttn& a, const Parts& p) {
  if (p.per > 0) return p.splits > 1 ? (int64_t)p.splits * a.c.B : 0;
  return p.splits > a.c.B ? p.splits : 0;
}

template <typename T, int D>
hipError_t launch(const CacheAttn& a, hipStream_t stream) {
  Parts p = plan(a);
  const Kind kind = kind_of(a);
  const int64_t heads = (int64_t)a.c.B * a.c.H, total = heads * a.group * a.S, slots = slots_of(a, p);
  const int wide = wide_of(kind);
  p.o = reinterpret_cast<float*>(a.workspace);
  p.ml = p.o + slots * a.c.H * p.tiles * 16 * D;
  if (slots > 0) p.items = reinterpret_cast<int32_t*>(p.ml + slots * a.c.H * p.tiles * 32);
  const int64_t each = p.tiles / (wide / 16);
  const int64_t few = ((int64_t)p.splits * a.c.H + kNumXcd - 1) / kNumXcd * kNumXcd;  // in whole rounds of the XCDs
  const dim3 grid((uint32_t)((kind == kMany ? heads * p.splits : few) * each)), threads(256);
  constexpr bool bytes = kIsBf16<T> && D == 128;
  if (kind == kMany && bytes && p.per >= kLongWalk)
    hipLaunchKernelGGL((many_rows_kernel<T, D, bytes>), grid, threads, 0, stream, a, p);
  else if (kind == kMany)
    hipLaunchKernelGGL((many_rows_kernel<T, D, false>), grid, threads, 0, stream, a, p);
  else if (kind == kFew32)
    hipLaunchKernelGGL((few_rows_kernel<T, D, 2>), grid, threads, 0, stream, a, p);
  else
    hipLaunchKernelGGL((few_rows_kernel<T, D, 1>), grid, threads, 0, stream, a, p);
  if (slots > 0) {
    if (total <= kJoinRows)
      hipLaunchKernelGGL((join_kernel<T, D, 64>), dim3((uint32_t)((total + 3) / 4)), threads, 0, stream, a, p, wide, total);
    else
      hipLaunchKernelGGL((join_kernel<T, D, 16>), dim3((uint32_t)((total + 15) / 16)), threads, 0, stream, a, p, wide, total);
  }
  return hipGetLastError();
}

}  // namespace

size_t cache_attn_workspace(const CacheAttn& a, int D) {
  const Parts p = plan(a);
  const size_t slots = (size_t)slots_of(a, p);
  return slots > 0 ? slots * a.c.H * p.tiles * 16 * (D + 2) * sizeof(float) + (size_t)a.c.B * 2 * sizeof(int32_t) : 0;
}

hipError_t launch_cache_attn(const CacheAttn& a, int dtype, int D, hipStream_t stream) {
  if (dtype == LCV_BSA_F16) return D == 64 ? launch<f16, 64>(a, stream) : launch<f16, 128>(a, stream);
  return D == 64 ? launch<bf16, 64>(a, stream) : launch<bf16, 128>(a, stream);
}

}  // namespace lcv
