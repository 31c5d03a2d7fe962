// Paged attention decode over 8-bit caches: E4M3 K and V with one fp32 scale per cache block and KV head (no counterpart in the
// reference).  The contract of attention_mma.cu otherwise; the work is cut and its parts are added as there
// (attention_split.cuh).
//
// The bytes are half of a 16-bit cache's, so what an SM does per row has to be half as much too:
//   * A warp's step is 32 tokens (16 at head size 256): two cache blocks or two halves of one (block sizes are multiples of 16).
//     One lane asks for its K and V rows by tiled TMA loads, into a ring of the warp's own; the blocks' scales come along by
//     cp.async, and multiply a block's scores and its sums once each.
//   * Both products are fp16 ones, in which E4M3 is exact.  (With E4M3 operands mma.sync counted twice as many products and a
//     conversion per operand register, and q needs two or three E4M3 parts: 150 us in the place of 133 at the time.)  Weights are
//     p = hi + lo, 22 bits of p 2^15, in rows 0-7 and 8-15 of one product; E4M3 has no infinity that a zero part could meet.
//   * A byte of K or V is converted once, straight from ldmatrix: K as it lies, four dims of a token in a register; V transposed
//     by bytes, four tokens of a dim.  The dims of q and the tokens of a score tile are ordered so that a register's halves
//     are the two halves of an operand, and a thread's four scores belong to the four tokens that it holds of V.
//
// Bound by instruction latency with twelve warps on an SM, as many as 168 registers allow: 387 instructions per 16 tokens (590 in
// the form of attention_mma.cu with rows copied by cp.async), 43 % of the issue slots while an SM is active.  Measured (bf16, 32 heads over 8 KV
// heads of 128, blocks of 16 in random order): 64 x 4096 tokens 120 us = 4.5 TB/s (133 us in that form; 173 us
// over a bf16 cache), 64 x 1000 43 us, one sequence of 777 10.8 us (15); 16 heads over 8 of 256, 64 x 4096: 220 us = 4.9 TB/s; one
// sequence of 65536, 8 heads over one of 64: 21 us.  A producer warp for all tiles was slower (250 us: its chain of loads
// is as long as a unit), and so were eight warps per CTA (150 us: 128 registers, spills).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "attention_split.cuh"
#include "internal.h"
#include "quant_math.cuh"

namespace ib200 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr float kUp = 15.0f;           // weights are 2^15 p, in their sum and in the denominator
constexpr float kBalance = 0.1f;       // of a unit's time and a part's (UnitList::begin)

template <int D>
struct FCfg {
  static constexpr int kHalves = D == 256 ? 1 : 2;                // 16-token blocks of a warp's step
  static constexpr int kTok = 16 * kHalves;
  static constexpr int kUnit = kWarps * kTok;                     // tokens of the CTA per step: the unit the work is cut in
  static constexpr int kRowBytes = D < 128 ? D : 128;             // of a tile's row; size 256: two tiles side by side
  static constexpr int kTiles = D / kRowBytes;
  static constexpr int kTileBytes = 16 * kRowBytes;
  static constexpr int kHalfBytes = kTiles * kTileBytes;          // K or V of 16 tokens
  static constexpr int kStageBytes = 2 * kHalves * kHalfBytes;    // K, then V
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr int kRec = D + 2;
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kMetaBytes = kWarps * kStages * kHalves * 8;   // the scales of a step's blocks
  // Up to four heads of a pair, whose states take little room: three CTAs per SM (size 256: two); else two.
  static constexpr int ctas_per_sm(int gt) { return D == 256 || gt > 4 ? 2 : 3; }
  static constexpr int merge_bytes(int gt) {
    return 4 * gt * (kWarps * kRec > kAttnSms * ctas_per_sm(gt) ? kWarps * kRec : kAttnSms * ctas_per_sm(gt));
  }
  static constexpr int smem_bytes(int gt) { return 1024 + kRingBytes + kMetaBytes + kWarps * kStages * 8 + merge_bytes(gt); }
  static constexpr int kRegCtas = D == 256 ? 2 : 3;
  static constexpr bool fits(int gt) { return ctas_per_sm(gt) * (smem_bytes(gt) + 1280) <= 233472 && smem_bytes(gt) + 256 <= 232448; }
  static_assert(fits(4) && fits(kAttnRows), "resident CTAs");
  static_assert(kAttnSms * 3 <= AttnSet::kCounters, "a counter per CTA");
  static constexpr size_t kWorkspaceBytes = static_cast<size_t>(kAttnSms) * kRegCtas * 2 * kAttnRows * kRec * sizeof(float);
};

struct Fp8AttnParams : AttnWork {
  void* out;
  const void* q;
  const int32_t* block_tables;
  const float* k_scales;   // [num_blocks][kv_heads]
  const float* v_scales;
  int num_heads, num_kv_heads, num_blocks, block_shift;   // block_shift: log2(block_size) or -1
  int q_words;             // q may be read in 32-bit words
  int wide;                // the tiles of a step's two blocks come as one: block sizes are multiples of 32
  float scale_log2e;       // what a product is multiplied by: to base 2 or, capped, to the cap's units
  float cap_log2e;         // kMod: the cap (0: none), to base 2
  const float* slopes;     // kMod: a head's loss per token of distance, or null
  int no_loads;            // test hook: no tile is asked for
  DeviceStatus* status;
};

constexpr uint32_t kSiteFp8Tiles = 0x351;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// two E4M3 values as fp16 (exact)
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t low_half) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(low_half)));
  return r;
}
__device__ __forceinline__ void mma_f16_add(float (&c)[4], uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(0u), "r"(a2), "r"(b0), "r"(b1));
}
// (the product alone)
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// two 16 x 16 byte matrices (rows: lanes 0-15, 16-31), transposed: columns lane / 4 (r[0], r[2]) and lane / 4 + 8 (r[1], r[3]),
// rows 4 (lane % 4) .. + 3
__device__ __forceinline__ void ldsm2_bytes_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// a += (b + c) f, two sums per instruction; f2: f twice
__device__ __forceinline__ void add_scaled(float2& a, const float (&d)[4], float2 f2) {
  a = __ffma2_rn(__fadd2_rn(make_float2(d[0], d[1]), make_float2(d[2], d[3])), f2, a);
}

template <typename T>
__device__ __forceinline__ T narrow16(float v);
template <>
__device__ __forceinline__ __half narrow16(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow16(float v) { return __float2bfloat16_rn(v); }

// Where 16-byte chunk c of row r of a tile lies: the TMA's swizzle moves it to c xor turn_of_row(r) inside the row (64-byte
// rows: two of them share 128 bytes).  With place = row_place(r, c0), chunk c0 xor c of the same row is chunk_place(place, c).
template <int D>
__device__ __forceinline__ uint32_t row_place(int r, int c0) {
  return r * FCfg<D>::kRowBytes + ((D == 64 ? (r >> 1) & 3 : r & 7) ^ c0) * 16;
}
template <int D>
__device__ __forceinline__ uint32_t chunk_place(uint32_t place, int c) {
  constexpr int kPer = FCfg<D>::kRowBytes / 16;
  return (place ^ (c % kPer * 16)) + c / kPer * FCfg<D>::kTileBytes;
}

// kMod: scores may be capped and / or fall with distance
template <typename T, int D, bool kMod>
__global__ void __launch_bounds__(kThreads, FCfg<D>::kRegCtas)
paged_attn_fp8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Fp8AttnParams p) {
  using C = FCfg<D>;
  using Units = UnitList<C::kUnit>;
  using Cursor = typename Units::Cursor;
  constexpr int kHalves = C::kHalves;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ int sh_last;
  __shared__ uint32_t sh_abort;
  const int lane = threadIdx.x & 31;
  const int warp = __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x >> 5), 0);
  const int row = lane >> 2;        // head row of this lane's accumulators
  const int quad = lane & 3;
  uint8_t* const ring = smem + warp * (C::kStages * C::kStageBytes);
  const uint32_t meta = smem_u32(smem + C::kRingBytes) + warp * (C::kStages * kHalves * 8);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + C::kRingBytes + C::kMetaBytes) + warp * C::kStages;
  float* states = reinterpret_cast<float*>(smem + C::kRingBytes + C::kMetaBytes + kWarps * C::kStages * 8);

  if (threadIdx.x == 0) sh_abort = 0u;
  if (lane == 0) {   // (a warp's barriers are its own)
    for (int s = 0; s < C::kStages; ++s) mbar_init(&bars[s], 1);
    mbar_init_fence();
    if (warp == 0) {
      tma_prefetch_desc(&map_k);
      tma_prefetch_desc(&map_v);
    }
  }
  __syncthreads();

  // q, the cache, the tables and the lengths may come from the kernel queued before this one; dependents are
  // not signalled early: the outputs are whole when a kernel behind this one starts, however it is launched
  pdl_wait();

  long long share, u0;
  Cursor use;
  if (!Units::template begin<true>(p, kBalance, use, share, u0)) return;
  const int my_units = use.left;
  const int gpk = (p.num_heads / p.num_kv_heads) / p.gt;   // head groups per KV head

  // ---- producer: a step's tiles.  Lane h looks up the block of half h, one step before it is asked for (-1: a hole, or nothing)
  Cursor pre = use;
  const int block_mask = (1 << (p.block_shift < 0 ? 0 : p.block_shift)) - 1;
  auto lookup = [&]() -> int {
    const int t = pre.t + warp * C::kTok + (lane & (kHalves - 1)) * 16;
    if (pre.left <= 0 || t >= pre.len) return -1;
    const int j = p.block_shift >= 0 ? t >> p.block_shift : t / p.block_size;
    const int blk = __ldg(p.block_tables + static_cast<int64_t>(pre.b) * p.max_blocks + j);
    return blk < p.num_blocks ? blk : -1;
  };
  int next_block = lookup();
  uint32_t holes = 0;               // halves of the ring's slots that nothing came for
  auto issue = [&](int slot) {
    const int t = pre.t + warp * C::kTok, kvh = pre.gi / gpk, mine = next_block;
    const bool any = pre.left > 0 && t < pre.len;   // warp-uniform
    if (pre.left > 0) {
      pre.next(p);
      next_block = lookup();
    }
    int blk[kHalves];
    uint32_t none = 0;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      blk[h] = __shfl_sync(0xFFFFFFFFu, mine, h);
      none |= (blk[h] < 0 ? 1u : 0u) << h;
    }
    holes = (holes & ~(((1u << kHalves) - 1u) << (slot * kHalves))) | none << (slot * kHalves);
    if (any) {
      if (lane == 0 && !p.no_loads) {
        uint8_t* dst = ring + slot * C::kStageBytes;
        const int off = p.block_shift >= 0 ? t & block_mask : t % p.block_size;
        if (kHalves == 2 && p.wide) {
          // (both halves lie in one block)
          if (blk[0] >= 0) {
            mbar_arrive_expect_tx(&bars[slot], C::kStageBytes);
            tma_load_2d(dst, &map_k, &bars[slot], kvh * D, blk[0] * p.block_size + off);
            tma_load_2d(dst + kHalves * C::kHalfBytes, &map_v, &bars[slot], kvh * D, blk[0] * p.block_size + off);
          } else {
            mbar_arrive(&bars[slot]);   // nothing comes
          }
        } else {
          mbar_arrive_expect_tx(&bars[slot], 2 * C::kHalfBytes * (kHalves - __popc(none)));
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            if (blk[h] < 0) continue;
            const int y = blk[h] * p.block_size + (h == 0 ? off : p.block_shift >= 0 ? (t + 16) & block_mask : (t + 16) % p.block_size);
#pragma unroll
            for (int x = 0; x < C::kTiles; ++x) {
              tma_load_2d(dst + h * C::kHalfBytes + x * C::kTileBytes, &map_k, &bars[slot], kvh * D + x * 128, y);
              tma_load_2d(dst + (kHalves + h) * C::kHalfBytes + x * C::kTileBytes, &map_v, &bars[slot], kvh * D + x * 128, y);
            }
          }
        }
      }
      if (lane < kHalves && mine >= 0) {
        const int64_t at = static_cast<int64_t>(mine) * p.num_kv_heads + kvh;
        const uint32_t to = meta + (slot * kHalves + lane) * 8;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(p.k_scales + at) : "memory");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + 4), "l"(p.v_scales + at) : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  // ---- the query rows of a pair as A operands: product kk takes dims 16 kk .. + 15, quad's four of them in two registers
  uint32_t qa[D / 16][2];
  float q_scale = 0.0f, slope = 0.0f;   // what this lane's row of products is multiplied by, before the block's scale
  auto load_q = [&](const Cursor& c) {
    const int kvh = c.gi / gpk;
    const int head0 = kvh * (p.num_heads / p.num_kv_heads) + (c.gi - kvh * gpk) * p.gt;
    const uint16_t* qrow = static_cast<const uint16_t*>(p.q) + (static_cast<int64_t>(c.b) * p.num_heads + head0 + row) * D;
    if constexpr (kMod) slope = p.slopes && row < p.gt ? __ldg(p.slopes + head0 + row) * 1.4426950408889634f : 0.0f;
    float mx = 0.0f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = kk * 16 + quad * 4 + h * 2;
        uint32_t x = 0;
        if (row < p.gt) {
          if (p.q_words) x = __ldg(reinterpret_cast<const uint32_t*>(qrow + e));
          else x = static_cast<uint32_t>(qrow[e]) | (static_cast<uint32_t>(qrow[e + 1]) << 16);
        }
        qa[kk][h] = x;
        const float2 f = widen2<T>(x);
        mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
    }
    q_scale = p.scale_log2e;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      // bf16 -> fp16 through a power of two that takes the row's maximum to 2^14 .. 2^15: every element down to 2^-28 of
      // it keeps its eight bits, smaller ones an absolute step of 2^-39 of it.  The power and its inverse are normal numbers for
      // every finite maximum; one below 2^-112 gets to 2^126 times itself, 1 at least if it is a normal number.
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
      int up = 127 + 14 - static_cast<int>(__float_as_uint(mx) >> 23);
      up = mx > 0.0f && mx < INFINITY ? min(126, up) : 0;   // (zeros, or an infinity: as they are)
      const float f = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
      q_scale *= __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 a = widen2<T>(qa[kk][h]);
          qa[kk][h] = pack_half2(a.x * f, a.y * f);
        }
      }
    }
  };

  load_q(use);
#pragma unroll
  for (int s = 0; s < C::kStages - 1; ++s) issue(s);

  // ldmatrix addresses.  K: row n of score tile h is token 4 (n / 2) + n % 2 + 2 (h xor n / 4): the eight rows of a matrix lie
  // in different banks, and quad's columns 2 quad, + 1 of the two tiles are tokens 4 quad .. + 3.
  const int mi = lane >> 3, mr = lane & 7;
  const int k_tok = 4 * (mr >> 1) + (mr & 1) + 2 * ((mi >> 1) ^ (mr >> 2));
  const bool swap = quad >= 2;      // tile 0 has tokens 4 quad + 2, + 3
  const uint32_t ring_at = smem_u32(ring);
  const uint32_t k_place = row_place<D>(k_tok, mi & 1);
  const uint32_t v_place = kHalves * C::kHalfBytes + row_place<D>(lane & 15, lane >> 4);

  int slot = 0;
  uint32_t phases = 0;
  bool dead = false;                // a wait ran out: nothing more is waited for or computed
  while (use.left > 0) {
    // ---- a pair (or the part of it that is this CTA's)
    const int b = use.b, gi = use.gi, len = use.len, t_first = use.t;
    const int kvh = gi / gpk;
    const int head0 = kvh * (p.num_heads / p.num_kv_heads) + (gi - kvh * gpk) * p.gt;
    float2 acc[D / 8];
#pragma unroll
    for (int j = 0; j < D / 8; ++j) acc[j] = make_float2(0.0f, 0.0f);
    float m = -INFINITY, l = 0.0f;
    const long long seg_u = u0 + (my_units - use.left);   // unit index of this segment's first unit
    int t_last;
    bool end;
    do {
      __syncwarp();   // every lane has read the slot that is filled next
      {
        int ahead = slot + C::kStages - 1;
        if (ahead >= C::kStages) ahead -= C::kStages;
        issue(ahead);
      }
      const int tw = use.t + warp * C::kTok;
      if (tw < len) {
        asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
        if (!dead) dead = !mbar_wait(&bars[slot], (phases >> slot) & 1u, &sh_abort, p.status, kSiteFp8Tiles);
        dead = __any_sync(0xFFFFFFFFu, dead);
        __syncwarp();                           // the scales are lane 0's and 1's copies: a vote orders no memory
        phases ^= 1u << slot;
        if (!dead) {
          const uint32_t at = ring_at + slot * C::kStageBytes;
          const uint32_t none = holes >> (slot * kHalves) & ((1u << kHalves) - 1u);
          float2 scales[kHalves];
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
            asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];"
                         : "=f"(scales[h].x), "=f"(scales[h].y)
                         : "r"(meta + (slot * kHalves + h) * 8)
                         : "memory");
          const bool partial = tw + C::kTok > len || none != 0u;
          if (partial) {
            // rows that are no token's: whatever is there, NaN perhaps, and 0 x NaN would reach the sums
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
              const int have = none >> h & 1u ? 0 : max(0, len - tw - 16 * h);
              if (none >> h & 1u) scales[h] = make_float2(0.0f, 0.0f);
              for (int i = have * (D / 16) + lane; i < 16 * (D / 16); i += 32)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(
                                 at + (kHalves + h) * C::kHalfBytes + chunk_place<D>(row_place<D>(i / (D / 16), 0), i % (D / 16))),
                             "r"(0u)
                             : "memory");
            }
            fence_proxy_async_smem();   // the slot's next tiles come by TMA
            __syncwarp();
          }
          float sc[kHalves][2][4] = {};
#pragma unroll
          for (int kk = 0; kk < D / 16; kk += 2) {
            uint32_t kf[kHalves][4];   // chunks kk and kk + 1 of tile 0's tokens, of tile 1's
#pragma unroll
            for (int h = 0; h < kHalves; ++h) ldsm4(at + h * C::kHalfBytes + chunk_place<D>(k_place, kk), kf[h]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int i = 0; i < 2 * kHalves; ++i) {   // (the chains of sums alternate)
                const uint32_t w = kf[i >> 1][2 * (i & 1) + e];
                mma_f16_add(sc[i >> 1][i & 1], qa[kk + e][0], qa[kk + e][1], e4m3x2_to_f16x2(w & 0xFFFFu), e4m3x2_to_f16x2(w >> 16));
              }
            }
          }
          float s[4 * kHalves];   // tokens 4 quad .. + 3 of either half
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            const float f = q_scale * scales[h].x;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * h + i] = (swap ? sc[h][1 - (i >> 1)][i & 1] : sc[h][i >> 1][i & 1]) * f;
          }
          const int behind = len - 1 - (tw + 4 * quad);   // tokens behind this lane's first
          if constexpr (kMod) {
#pragma unroll
            for (int i = 0; i < 4 * kHalves; ++i) s[i] = scored(s[i], p.cap_log2e, slope, behind - (i >> 2) * 16 - (i & 3));
          }
          if (partial) {
#pragma unroll
            for (int i = 0; i < 4 * kHalves; ++i)
              if (behind < (i >> 2) * 16 + (i & 3) || (none >> (i >> 2) & 1u)) s[i] = -INFINITY;
          }
          float mx = s[0];
#pragma unroll
          for (int i = 1; i < 4 * kHalves; ++i) mx = fmaxf(mx, s[i]);
          mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
          if (__any_sync(0xFFFFFFFFu, mx > m)) {
            // a new maximum (always in the first step, rare later): the state is rescaled
            const float m_new = fmaxf(m, mx);
            const float alpha = ex2(m - finite_max(m_new));
            m = m_new;
            l *= alpha;
            const float2 alpha2 = make_float2(alpha, alpha);
#pragma unroll
            for (int j = 0; j < D / 8; ++j) acc[j] = __fmul2_rn(acc[j], alpha2);
          }
          const float ref = finite_max(m) - kUp;
          uint32_t hi[2 * kHalves], lo[2 * kHalves];
#pragma unroll
          for (int h = 0; h < 2 * kHalves; ++h) {
            const float p0 = ex2(s[2 * h] - ref), p1 = ex2(s[2 * h + 1] - ref);   // 0 for a missing token
            l += p0 + p1;
            hi[h] = pack_half2(p0, p1);
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&hi[h]));
            lo[h] = pack_half2(p0 - a.x, p1 - a.y);
          }
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            const float2 v2 = make_float2(scales[h].y, scales[h].y);
#pragma unroll
            for (int c = 0; c < D / 16; c += 2) {
              uint32_t vf[4];
              ldsm2_bytes_trans(at + h * C::kHalfBytes + chunk_place<D>(v_place, c), vf);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float d[4];
                mma_f16(d, hi[2 * h], lo[2 * h], hi[2 * h + 1], lo[2 * h + 1], e4m3x2_to_f16x2(vf[i] & 0xFFFFu),
                        e4m3x2_to_f16x2(vf[i] >> 16));
                add_scaled(acc[2 * c + i], d, v2);
              }
            }
          }
        }
      }
      if (++slot == C::kStages) slot = 0;
      t_last = use.t;
      end = use.t + C::kUnit >= len || use.left == 1;
      use.next(p);
    } while (!end);

    if (use.left > 0) load_q(use);

    // ---- the warps' states -> one
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
    if (row < p.gt) {
      float* st = states + (warp * p.gt + row) * C::kRec;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(st + j * 8 + quad * 2) = acc[j];
      if (quad == 0) {
        st[D] = m;
        st[D + 1] = l;
      }
    }
    T* out = static_cast<T*>(p.out) + (static_cast<int64_t>(b) * p.num_heads + head0) * D;
    finish_pair<kWarps, D, C::kUnit, true>(p, states, p.gt, sh_last, out, len, t_first, t_last, use.left, share, seg_u,
                                           [](float v) { return narrow16<T>(v); });
    __syncthreads();   // the states may be overwritten now
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (dead) {
    // tiles that this warp asked for may still be on their way: give them time to land before the CTA ends
    const long long w0 = clock64();
    while (clock64() - w0 < (1LL << 22)) {
    }
  }
}

template <typename T, int D, bool kMod>
int launch_d(const CUtensorMap& mk, const CUtensorMap& mv, const Fp8AttnParams& p, int sm_count, bool pdl, cudaStream_t stream) {
  using C = FCfg<D>;
  constexpr int kUnit = C::kUnit;
  const auto kernel = paged_attn_fp8_kernel<T, D, kMod>;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem_bytes(kAttnRows));
    if (e != cudaSuccess) return note_cuda_error(e);
    attr_done[dev] = true;
  }
  const int64_t pairs = static_cast<int64_t>(p.batch) * p.groups;
  int64_t ctas = pairs;
  if (!p.whole) {
    // as many CTAs as are resident at once, but no more than the tables could fill
    const int64_t most = pairs * ((static_cast<int64_t>(p.max_blocks) * p.block_size + kUnit - 1) / kUnit);
    ctas = static_cast<int64_t>(sm_count < kAttnSms ? sm_count : kAttnSms) * C::ctas_per_sm(p.gt);
    if (ctas > most) ctas = most;
  }
  if (ctas > 0x7FFFFFFF) return INFEROP_ERR_LIMIT;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::smem_bytes(p.gt);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, mk, mv, p);
  if (e != cudaSuccess) return note_cuda_error(e);
  return check_launch();
}

template <typename T, bool kMod>
int launch_t(const CUtensorMap& mk, const CUtensorMap& mv, const Fp8AttnParams& p, int head_dim, int sm_count, bool pdl,
             cudaStream_t stream) {
  switch (head_dim) {
    case 64: return launch_d<T, 64, kMod>(mk, mv, p, sm_count, pdl, stream);
    case 128: return launch_d<T, 128, kMod>(mk, mv, p, sm_count, pdl, stream);
    case 256: return launch_d<T, 256, kMod>(mk, mv, p, sm_count, pdl, stream);
    default: return INFEROP_ERR_SHAPE;
  }
}

}  // namespace

size_t paged_attn_fp8_workspace_bytes() {
  constexpr size_t a = FCfg<64>::kWorkspaceBytes, b = FCfg<128>::kWorkspaceBytes, c = FCfg<256>::kWorkspaceBytes;
  return a > b ? (a > c ? a : c) : (b > c ? b : c);
}

int launch_paged_attn_fp8(DeviceCtx* ctx, void* out, const void* q, const void* k_cache, const void* v_cache, const Fp8Cache& cache,
                          const int32_t* block_tables, const int32_t* seq_lens, int32_t dt, int batch, int num_heads, int num_kv_heads,
                          int head_dim, int block_size, int max_blocks_per_seq, float scale, const ScoreMod& mod, float* workspace,
                          int* counters, bool pdl, cudaStream_t stream) {
  Fp8AttnParams p;
  p.out = out;
  p.q = q;
  p.block_tables = block_tables;
  p.k_scales = cache.k_scales;
  p.v_scales = cache.v_scales;
  p.num_blocks = cache.num_blocks;
  p.seq_lens = seq_lens;
  p.partial = workspace;
  p.counters = counters;
  p.batch = batch;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.block_size = block_size;
  p.block_shift = -1;
  for (int sh = 0; sh < 31; ++sh)
    if ((1 << sh) == block_size) p.block_shift = sh;
  p.max_blocks = max_blocks_per_seq;
  p.gt = heads_per_pair(num_heads / num_kv_heads);
  p.groups = num_heads / p.gt;
  p.whole = workspace == nullptr || batch > kMaxBatchCut ? 1 : 0;
  p.q_words = (reinterpret_cast<uintptr_t>(q) & 3u) == 0 ? 1 : 0;
  p.scale_log2e = mod.softcap > 0.0f ? scale / mod.softcap : scale * 1.4426950408889634f;
  p.cap_log2e = mod.softcap * 1.4426950408889634f;
  p.slopes = mod.slopes;
  p.no_loads = options().debug_no_loads;
  p.status = ctx->status;
  // (rows of a KV head are head_dim bytes of a token's num_kv_heads head_dim)
  const uint64_t rows = static_cast<uint64_t>(cache.num_blocks) * block_size, cols = static_cast<uint64_t>(num_kv_heads) * head_dim;
  const uint32_t box = head_dim < 128 ? head_dim : 128;
  p.wide = head_dim <= 128 && block_size % 32 == 0 ? 1 : 0;
  const uint32_t box_rows = p.wide ? 32 : 16;
  CUtensorMap mk, mv;
  int rc = make_tensor_map_2d_scattered(&mk, k_cache, 1, rows, cols, cols, box_rows, box, box);
  if (rc == INFEROP_OK) rc = make_tensor_map_2d_scattered(&mv, v_cache, 1, rows, cols, cols, box_rows, box, box);
  if (rc != INFEROP_OK) return rc;
  const int sms = ctx->sm_count;
  if (dt == 1)
    return mod.any() ? launch_t<__half, true>(mk, mv, p, head_dim, sms, pdl, stream)
                     : launch_t<__half, false>(mk, mv, p, head_dim, sms, pdl, stream);
  return mod.any() ? launch_t<__nv_bfloat16, true>(mk, mv, p, head_dim, sms, pdl, stream)
                   : launch_t<__nv_bfloat16, false>(mk, mv, p, head_dim, sms, pdl, stream);
}

}  // namespace ib200
