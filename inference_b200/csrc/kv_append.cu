// Rotation of queries and keys and the store of keys and values into a paged cache, one launch (no counterpart in the
// reference, whose caller rotates with rope_neox and copies rows into the cache by itself).
//
//   q [tokens, heads, dim], k / v [tokens, kv_heads, dim]: rows of a token contiguous, tokens at any stride (the three parts
//   of a fused projection's output); caches [blocks, block_size, kv_heads, dim] in the operands' type or in E4M3.
//
// Token i of a sequence whose n new tokens end at length len has position p = len - n + i; pairs (x_j, x_{j + r/2}) are
// turned by p base^(-2j/r) yarn, and K and V go to row p % block_size of block block_tables[b][p / block_size].
//
// Bound by HBM for many tokens (every byte is read once and written once), by latency for few.  So the loads of a thread's
// items are issued before anything is known about the token (its sequence, its angles), and both are worked out while they
// are on their way.  Angles: p times the frequency in turns, in fp64, of which only the fraction is kept: p f in fp32 has
// lost 6e-3 rad by position 1e5.  One fp64 product per token and pair, shared by all heads through shared memory.
//
// E4M3: a scale belongs to a cache block and a KV head, so the unit of work is a block, and all of a call's tokens in it
// belong to one CTA, a warp per head and kind (K, V).  Scales are powers of two: a floating format loses nothing by them
// (a scale that fits closer would move the values inside a binade), and when a later token needs a larger one, the
// tokens already there move to it without another rounding (but for E4M3's subnormals).  The values that are quantised
// are the rotated ones in fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "internal.h"
#include "ragged.cuh"

namespace ib200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kItems = 4;          // vector pairs of a thread in flight
constexpr int kMaxHalf = 128;      // rotary_dim up to 256, the largest head
constexpr int kMaxTile = 16;       // tokens of a CTA that share a table of angles
constexpr float kMinScale = 7.888609052210118e-31f;   // 2^-100: the scale of a block without a non-zero value

struct AppendParams {
  const void *q, *k, *v;
  void *q_out, *k_out;             // k_out may be null
  void *k_cache, *v_cache;
  float *k_scales, *v_scales;      // E4M3 caches only
  const int32_t *block_tables, *seq_lens, *cu;   // cu null: token i is sequence i's only one
  int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;   // of a token, in elements
  int64_t tokens;
  int batch, heads, kv_heads, dim, half, block_size, max_blocks, num_blocks;
  int pairs_log2;                  // log2 of the vector pairs of a head
  int tile;                        // tokens per CTA of the token role
  int kv_ctas;                     // E4M3: CTAs of the block role, in front of the others
  double turns[kMaxHalf];          // frequency of pair j in turns per position
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// V elements that are read and written together: 16 bytes, or one element where alignment or the rotary size ask for it
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};
template <int V>
struct alignas(V) Bytes {
  uint8_t e[V];
};

// where a token lies: its position (-1: nobody's token) and its cache row (-1: none)
struct Place {
  int pos;
  int64_t row;
};
__device__ __forceinline__ int64_t cache_row(const AppendParams& p, int b, int pos) {
  const int j = pos / p.block_size;
  if (j >= p.max_blocks) return -1;
  const int blk = __ldg(p.block_tables + static_cast<int64_t>(b) * p.max_blocks + j);
  return blk < 0 || blk >= p.num_blocks ? -1 : static_cast<int64_t>(blk) * p.block_size + (pos - j * p.block_size);
}
// (the whole warp)
__device__ __forceinline__ Place place_of(const AppendParams& p, int64_t t) {
  Place out = {-1, -1};
  int b;
  if (p.cu == nullptr) {
    b = static_cast<int>(t);
    out.pos = max(-1, __ldg(p.seq_lens + b) - 1);
  } else {
    b = last_at_or_below(t, p.batch, [&](int i) { return static_cast<int64_t>(__ldg(p.cu + i)); });
    if (b < 0) return out;
    const int64_t behind = __ldg(p.cu + b + 1) - t;
    if (behind <= 0) return out;
    out.pos = static_cast<int>(max(static_cast<int64_t>(-1), __ldg(p.seq_lens + b) - behind));
  }
  if (out.pos >= 0) out.row = cache_row(p, b, out.pos);
  return out;
}

// (cos, sin) of pair j at a position
__device__ __forceinline__ float2 turn_of(const AppendParams& p, int pos, int j) {
  const double turns = static_cast<double>(pos) * p.turns[j];
  float s, c;
  sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
  return make_float2(c, s);
}

// Pair i of a head of dim / (2 V): the vectors it consists of (in units of V elements) and whether it is turned.
// The first half / V pairs are (j, j + half / V); what lies behind the rotary part goes two by two.
struct PairOf {
  int a, b;
  bool turned;
};
template <int V>
__device__ __forceinline__ PairOf pair_of(const AppendParams& p, int i) {
  const int h = p.half / V;
  if (i < h) return {i, i + h, true};
  return {2 * i, 2 * i + 1, false};
}

// x0, x1 <- the pair turned; cs: this token's table
template <typename T, int V>
__device__ __forceinline__ void turn(const Vec<T, V>& a, const Vec<T, V>& b, bool turned, const float2* cs, int j, float (&x0)[V],
                                     float (&x1)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float f0 = to_f32<T>(a.e[e]), f1 = to_f32<T>(b.e[e]);
    if (turned) {
      const float2 c = cs[j * V + e];
      x0[e] = f0 * c.x - f1 * c.y;
      x1[e] = f1 * c.x + f0 * c.y;
    } else {
      x0[e] = f0;
      x1[e] = f1;
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> narrow(const float (&x)[V]) {
  Vec<T, V> out;
#pragma unroll
  for (int e = 0; e < V; ++e) out.e[e] = from_f32<T>(x[e]);
  return out;
}

// ---- a CTA of p.tile tokens: heads [0, heads) are q's, then kv_heads of k, then kv_heads of v (kStore; else q alone)
template <typename T, int V, bool kStore>
__device__ __forceinline__ void token_role(const AppendParams& p, int64_t cta, float2* cs) {
  __shared__ Place places[kMaxTile];
  const int64_t t0 = cta * p.tile;
  const int n = static_cast<int>(min(static_cast<int64_t>(p.tile), p.tokens - t0));
  const int per_token = p.heads + (kStore ? 2 * p.kv_heads : 0);
  const int total = (n * per_token) << p.pairs_log2;
  const int mask = (1 << p.pairs_log2) - 1;

  Vec<T, V> a[kItems], b[kItems];
  auto source = [&](int tok, int h) -> const T* {
    const int64_t t = t0 + tok;
    if (h < p.heads) return static_cast<const T*>(p.q) + t * p.q_stride + static_cast<int64_t>(h) * p.dim;
    h -= p.heads;
    if (h < p.kv_heads) return static_cast<const T*>(p.k) + t * p.k_stride + static_cast<int64_t>(h) * p.dim;
    return static_cast<const T*>(p.v) + t * p.v_stride + static_cast<int64_t>(h - p.kv_heads) * p.dim;
  };
  auto load = [&](int base) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int it = base + i * kThreads + threadIdx.x;
      if (it < total) {
        const int th = it >> p.pairs_log2, tok = th / per_token;
        const PairOf pr = pair_of<V>(p, it & mask);
        const Vec<T, V>* src = reinterpret_cast<const Vec<T, V>*>(source(tok, th - tok * per_token));
        a[i] = src[pr.a];
        b[i] = src[pr.b];
      }
    }
  };
  load(0);
  const int warp = threadIdx.x >> 5;
  for (int tok = warp; tok < n; tok += kWarps) {
    const Place at = place_of(p, t0 + tok);
    if ((threadIdx.x & 31) == 0) places[tok] = at;
    for (int j = threadIdx.x & 31; j < p.half; j += 32) cs[tok * p.half + j] = turn_of(p, at.pos, j);
  }
  __syncthreads();
  for (int base = 0; base < total; base += kItems * kThreads) {
    if (base > 0) load(base);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int it = base + i * kThreads + threadIdx.x;
      if (it >= total) continue;
      const int th = it >> p.pairs_log2, tok = th / per_token, j = it & mask;
      int h = th - tok * per_token;
      const Place at = places[tok];
      if (at.pos < 0) continue;
      const PairOf pr = pair_of<V>(p, j);
      const int64_t t = t0 + tok;
      if (h >= p.heads + p.kv_heads) {   // v: as it is
        if (at.row < 0) continue;
        h -= p.heads + p.kv_heads;
        Vec<T, V>* dst = reinterpret_cast<Vec<T, V>*>(static_cast<T*>(p.v_cache) + (at.row * p.kv_heads + h) * p.dim);
        dst[pr.a] = a[i];
        dst[pr.b] = b[i];
        continue;
      }
      float x0[V], x1[V];
      turn<T, V>(a[i], b[i], pr.turned, cs + tok * p.half, j, x0, x1);
      const Vec<T, V> y0 = narrow<T, V>(x0), y1 = narrow<T, V>(x1);
      T *first = nullptr, *second = nullptr;
      if (h < p.heads) {
        first = static_cast<T*>(p.q_out) + t * p.q_out_stride + static_cast<int64_t>(h) * p.dim;
      } else {
        h -= p.heads;
        if (at.row >= 0) first = static_cast<T*>(p.k_cache) + (at.row * p.kv_heads + h) * p.dim;
        if (p.k_out) second = static_cast<T*>(p.k_out) + t * p.k_out_stride + static_cast<int64_t>(h) * p.dim;
      }
      if (first) {
        reinterpret_cast<Vec<T, V>*>(first)[pr.a] = y0;
        reinterpret_cast<Vec<T, V>*>(first)[pr.b] = y1;
      }
      if (second) {
        reinterpret_cast<Vec<T, V>*>(second)[pr.a] = y0;
        reinterpret_cast<Vec<T, V>*>(second)[pr.b] = y1;
      }
    }
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
append_kernel(const __grid_constant__ AppendParams p) {
  extern __shared__ float2 cs[];
  token_role<T, V, true>(p, blockIdx.x, cs);
}

// ------------------------------------------------------------------------------------------------ E4M3 caches
// the smallest power of two s with amax <= 448 s (448 = 1.75 2^8), no less than kMinScale
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax) + 0x1FFFFFu;   // a mantissa above 1.75 carries into the exponent
  const int e = static_cast<int>(u >> 23) - 8;
  return fmaxf(e > 0 ? __uint_as_float(static_cast<uint32_t>(e) << 23) : 0.0f, kMinScale);
}
// x / s as an E4M3 byte (1 / s is exact): infinities become +-448, NaN stays NaN
__device__ __forceinline__ uint8_t quantised(float x, float inv) {
  return static_cast<uint8_t>(__nv_cvt_float_to_fp8(x * inv, __NV_SATFINITE, __NV_E4M3));
}
__device__ __forceinline__ float value_of(uint8_t byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(byte, __NV_E4M3)));
}

// ---- a CTA of one cache block of one sequence: its new tokens, rows [off, off + n) of the block, every KV head.
// Sequence b owns items [cu[b] / block_size + 2 b, cu[b + 1] / block_size + 2 (b + 1)): n tokens touch no more than
// floor(n / block_size) + 2 blocks, and the bound needs no sum over the sequences before.
template <typename T, int V>
__device__ __forceinline__ void block_role(const AppendParams& p, int64_t item, float2* cs) {
  __shared__ float amax_of[2][64];   // several chunks of tokens: maximum so far of (kind, head) of this round
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int b, first_pos, last_pos, j;     // the sequence's new positions [first_pos, last_pos], the block among its own
  int64_t t_first;
  if (p.cu == nullptr) {
    b = static_cast<int>(item);
    last_pos = first_pos = __ldg(p.seq_lens + b) - 1;
    if (first_pos < 0) return;
    j = first_pos / p.block_size;
    t_first = item;
  } else {
    b = last_at_or_below(item, p.batch, [&](int i) { return static_cast<int64_t>(__ldg(p.cu + i) / p.block_size) + 2 * i; });
    if (b < 0) return;
    const int c0 = __ldg(p.cu + b), c1 = __ldg(p.cu + b + 1);
    const int n = c1 - c0;
    if (n <= 0 || c0 < 0 || c1 > p.tokens) return;
    const int len = __ldg(p.seq_lens + b);
    last_pos = len - 1;
    first_pos = len - n;
    t_first = c0;
    if (first_pos < 0) {   // more new tokens than the sequence is long: the first of them have no position
      t_first -= first_pos;
      first_pos = 0;
    }
    if (last_pos < 0) return;
    j = first_pos / p.block_size + static_cast<int>(item - (c0 / p.block_size + 2 * b));
    if (static_cast<int64_t>(j) * p.block_size > last_pos) return;
  }
  const int pos0 = max(first_pos, j * p.block_size);
  const int n = static_cast<int>(min(static_cast<int64_t>(last_pos), static_cast<int64_t>(j + 1) * p.block_size - 1)) - pos0 + 1;
  const int64_t t0 = t_first + (pos0 - first_pos);
  const int64_t row0 = cache_row(p, b, pos0);
  if (row0 < 0 && p.k_out == nullptr) return;
  const int off = pos0 - j * p.block_size;
  const int64_t blk = row0 < 0 ? 0 : row0 / p.block_size;
  const int mask = (1 << p.pairs_log2) - 1;
  const int chunks = (n + kMaxTile - 1) / kMaxTile;

  auto table = [&](int c) {   // angles of a chunk's tokens
    const int rows = min(kMaxTile, n - c * kMaxTile);
    for (int i = threadIdx.x; i < rows * p.half; i += kThreads) {
      const int r = i / p.half;
      cs[i] = turn_of(p, pos0 + c * kMaxTile + r, i - r * p.half);
    }
  };
  // (rounds of 64 heads, so that the maxima have a place whatever the number of heads)
  for (int h0 = 0; h0 < p.kv_heads; h0 += 64) {
    const int jobs = 2 * min(64, p.kv_heads - h0);
    for (int step = 0; step < (chunks == 1 ? 1 : 2 * chunks); ++step) {
      const bool measure = step < chunks, store = chunks == 1 || step >= chunks;
      const int c = store && chunks > 1 ? step - chunks : step;
      const int rows = min(kMaxTile, n - c * kMaxTile), total = rows << p.pairs_log2;
      const int64_t tc = t0 + c * kMaxTile;
      if (step > 0 || h0 > 0) __syncthreads();
      table(c);
      __syncthreads();
      for (int job = warp; job < jobs; job += kWarps) {
        const bool is_k = (job & 1) == 0;
        const int hr = job >> 1, h = h0 + hr;
        const T* src = is_k ? static_cast<const T*>(p.k) + tc * p.k_stride : static_cast<const T*>(p.v) + tc * p.v_stride;
        const int64_t stride = is_k ? p.k_stride : p.v_stride;
        src += static_cast<int64_t>(h) * p.dim;
        Vec<T, V> a[kItems], bb[kItems];
        auto load = [&](int base) {
#pragma unroll
          for (int i = 0; i < kItems; ++i) {
            const int it = base + i * 32 + lane;
            if (it < total) {
              const PairOf pr = pair_of<V>(p, it & mask);
              const Vec<T, V>* s = reinterpret_cast<const Vec<T, V>*>(src + (it >> p.pairs_log2) * stride);
              a[i] = s[pr.a];
              bb[i] = s[pr.b];
            }
          }
        };
        load(0);
        float* scales = is_k ? p.k_scales : p.v_scales;
        const int64_t at = blk * p.kv_heads + h;
        const float old = off > 0 && row0 >= 0 ? scales[at] : 0.0f;
        float amax = 0.0f;
        if (measure) {
          for (int base = 0; base < total; base += 32 * kItems) {
            if (base > 0) load(base);
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
              const int it = base + i * 32 + lane;
              if (it < total) {
                const PairOf pr = pair_of<V>(p, it & mask);
                float x0[V], x1[V];
                turn<T, V>(a[i], bb[i], is_k && pr.turned, cs + (it >> p.pairs_log2) * p.half, it & mask, x0, x1);
#pragma unroll
                for (int e = 0; e < V; ++e) {   // (neither NaN nor an infinity sets a scale)
                  const float f0 = fabsf(x0[e]), f1 = fabsf(x1[e]);
                  amax = fmaxf(amax, fmaxf(f0 < INFINITY ? f0 : 0.0f, f1 < INFINITY ? f1 : 0.0f));
                }
              }
            }
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
          if (chunks > 1) {
            if (lane == 0) amax_of[is_k ? 0 : 1][hr] = step == 0 ? amax : fmaxf(amax_of[is_k ? 0 : 1][hr], amax);
            __syncwarp();
          }
          if (total > 32 * kItems && store) load(0);
        }
        if (!store) continue;
        if (chunks > 1) amax = amax_of[is_k ? 0 : 1][hr];
        const float scale = fmaxf(old, scale_for(amax)), inv = 1.0f / scale;
        uint8_t* cache = static_cast<uint8_t*>(is_k ? p.k_cache : p.v_cache);
        const int64_t row_bytes = static_cast<int64_t>(p.kv_heads) * p.dim;
        uint8_t* head = cache + row0 * row_bytes + static_cast<int64_t>(h) * p.dim;   // (row0 < 0: not written)
        if (row0 >= 0 && c == 0) {
          if (off > 0 && scale > old) {   // the tokens before move to the larger scale
            const float ratio = old / scale;
            constexpr int W = 8;
            const int per_row = p.dim / W;
            for (int it = lane; it < off * per_row; it += 32) {
              const int r = it / per_row;
              Bytes<W>* d = reinterpret_cast<Bytes<W>*>(head - (r + 1) * row_bytes) + (it - r * per_row);
              Bytes<W> y = *d;
#pragma unroll
              for (int e = 0; e < W; ++e) y.e[e] = quantised(value_of(y.e[e]), ratio);
              *d = y;
            }
          }
          if (off == 0 || scale > old) {
            __syncwarp();   // every lane has read the old one
            if (lane == 0) scales[at] = scale;
          }
        }
        for (int base = 0; base < total; base += 32 * kItems) {
          if (base > 0) load(base);
#pragma unroll
          for (int i = 0; i < kItems; ++i) {
            const int it = base + i * 32 + lane;
            if (it >= total) continue;
            const int r = it >> p.pairs_log2, i2 = it & mask;
            const PairOf pr = pair_of<V>(p, i2);
            float x0[V], x1[V];
            turn<T, V>(a[i], bb[i], is_k && pr.turned, cs + r * p.half, i2, x0, x1);
            if (row0 >= 0) {
              Bytes<V> y0, y1;
#pragma unroll
              for (int e = 0; e < V; ++e) {
                y0.e[e] = quantised(x0[e], inv);
                y1.e[e] = quantised(x1[e], inv);
              }
              Bytes<V>* d = reinterpret_cast<Bytes<V>*>(head + (c * kMaxTile + r) * row_bytes);
              d[pr.a] = y0;
              d[pr.b] = y1;
            }
            if (is_k && p.k_out) {
              Vec<T, V>* d = reinterpret_cast<Vec<T, V>*>(static_cast<T*>(p.k_out) + (tc + r) * p.k_out_stride +
                                                          static_cast<int64_t>(h) * p.dim);
              d[pr.a] = narrow<T, V>(x0);
              d[pr.b] = narrow<T, V>(x1);
            }
          }
        }
      }
    }
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
append_fp8_kernel(const __grid_constant__ AppendParams p) {
  extern __shared__ float2 cs[];
  if (static_cast<int64_t>(blockIdx.x) < p.kv_ctas) block_role<T, V>(p, blockIdx.x, cs);
  else token_role<T, V, false>(p, static_cast<int64_t>(blockIdx.x) - p.kv_ctas, cs);
}

template <typename T, int V>
int launch_tv(AppendParams p, bool fp8, cudaStream_t stream) {
  p.pairs_log2 = 0;
  while ((2 * V) << p.pairs_log2 < p.dim) ++p.pairs_log2;
  const int items = (p.heads + (fp8 ? 0 : 2 * p.kv_heads)) << p.pairs_log2;
  // as many tokens as give every thread its items
  p.tile = kItems * kThreads / items;
  p.tile = p.tile < 1 ? 1 : (p.tile > kMaxTile ? kMaxTile : p.tile);
  int64_t ctas = (p.tokens + p.tile - 1) / p.tile;
  if (fp8) {
    const int64_t kv = p.cu ? p.tokens / p.block_size + 2 * static_cast<int64_t>(p.batch) : p.tokens;
    if (kv > 0x3FFFFFFF) return INFEROP_ERR_LIMIT;
    p.kv_ctas = static_cast<int>(kv);
    ctas += kv;
  }
  if (ctas > 0x7FFFFFFF) return INFEROP_ERR_LIMIT;
  const size_t smem = static_cast<size_t>(fp8 ? kMaxTile : p.tile) * p.half * sizeof(float2);   // 16 KB at most
  const unsigned grid = static_cast<unsigned>(ctas);
  if (fp8) append_fp8_kernel<T, V><<<grid, kThreads, smem, stream>>>(p);
  else append_kernel<T, V><<<grid, kThreads, smem, stream>>>(p);
  return check_launch();
}

template <typename T>
int launch_t(const AppendParams& p, bool fp8, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
                       reinterpret_cast<uintptr_t>(p.q_out) | reinterpret_cast<uintptr_t>(p.k_out) |
                       reinterpret_cast<uintptr_t>(p.k_cache) | reinterpret_cast<uintptr_t>(p.v_cache);
  const int64_t strides = p.q_stride | p.k_stride | p.v_stride | p.q_out_stride | (p.k_out ? p.k_out_stride : 0);
  if ((at & 15u) == 0 && strides % V == 0 && p.half % V == 0) return launch_tv<T, V>(p, fp8, stream);
  return launch_tv<T, 1>(p, fp8, stream);
}

}  // namespace

int launch_kv_append(const KvAppendArgs& a, cudaStream_t stream) {
  AppendParams p;
  p.q = a.q, p.k = a.k, p.v = a.v;
  p.q_out = a.q_out, p.k_out = a.k_out;
  p.k_cache = a.k_cache, p.v_cache = a.v_cache;
  p.k_scales = a.k_scales, p.v_scales = a.v_scales;
  p.block_tables = a.block_tables, p.seq_lens = a.seq_lens, p.cu = a.cu_seqlens;
  p.q_stride = a.q_stride, p.k_stride = a.k_stride, p.v_stride = a.v_stride;
  p.q_out_stride = a.q_out_stride, p.k_out_stride = a.k_out_stride;
  p.tokens = a.tokens;
  p.batch = a.batch, p.heads = a.heads, p.kv_heads = a.kv_heads, p.dim = a.dim, p.half = a.rotary_dim / 2;
  p.block_size = a.block_size, p.max_blocks = a.max_blocks, p.num_blocks = a.num_blocks;
  p.kv_ctas = 0;
  // base^(-2 j / rotary_dim) as powers of one root: the product of 128 of them is off by 2e-14 at most, 2e-8 rad at 1e6
  const double root = p.half > 0 ? pow(a.base, -1.0 / p.half) : 1.0;
  double f = a.yarn_factor / 6.283185307179586476925;
  for (int j = 0; j < kMaxHalf; ++j, f *= root) p.turns[j] = j < p.half ? f : 0.0;
  switch (a.dt) {
    case 0: return launch_t<float>(p, a.k_scales != nullptr, stream);
    case 1: return launch_t<__half>(p, a.k_scales != nullptr, stream);
    case 2: return launch_t<__nv_bfloat16>(p, a.k_scales != nullptr, stream);
    default: return INFEROP_ERR_DTYPE;
  }
}

}  // namespace ib200
