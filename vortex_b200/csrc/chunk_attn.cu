// Attention of chunks of new tokens over the paged KV cache, on the
// 5th-generation tensor cores.
//
//   O[r, h]   = sum_j exp(scale q_r . k_j - lse[r, h]) v_j,   j <= last(r)
//   lse[r, h] = log sum_j exp(scale q_r . k_j)
//
// with last(r) = len - n_queries + r (causal) or len - 1. Between one query
// per sequence (drafted tokens: the cache is read once, HBM-bound) and
// thousands (chunks of prompts: tensor- and exponential-bound).
//
// Rows. The G query heads of a kv head share its keys, so row t * G + g of a
// tile is head g of the chunk's token t: a tile of 128 rows holds 128 / G
// tokens, one TMA box of [tokens][G][64] per 64 columns. An item is (sequence,
// kv head, 256 rows); a key tile is 128 tokens, K and V of one kv head.
//
// Two streams. A CTA works on two tiles of scores at a time, each with its own
// S and O in tensor memory. An item of more than 128 rows gives each stream
// half of the rows and both the same key tiles; a smaller item gives both the
// same rows and every other key tile, and the streams are joined at the end.
// Either way the tensor core works on one stream while the other takes
// exponentials. P overwrites its own S: S, S, O, O fill the 512 columns.
//
// Work split. The key tiles of all items in a row are cut into equal runs, one
// per SM (the host gives each CTA its first item and tile), so ragged batches,
// long caches with few rows and causal triangles balance alike. A run that
// ends inside an item leaves its unnormalised sums in the caller's scratch and
// a second kernel joins an item's parts; where it costs few key tiles, items
// stay whole (cut_runs).
//
// Warps: 0-15 softmax (two warpgroups to a stream, each half of a tile's keys:
// thread = row = TMEM lane; the halves tell each other their maxima), 16 issues
// the MMAs, 17 the TMA copies; int8 caches use 18, which looks the V scales over,
// and add 20-27, which turn int8 pages into K tiles of bf16 and V tiles of f16
// (codes are exact in both). Pages come through one ring of tiles in the order K,
// V, K, V, ...; a page box is up to 128 tokens of one block, of which only those
// that hold tokens are copied.
//
// Keys behind the last token never count: S is masked by selection, the
// MMA stops at the last 16 keys with a token and the rest of those 16 V rows
// is zeroed. A key that only some rows of a tile see may hold inf or NaN: such
// elements of V are taken out of the tile before the product and added to the
// rows that see them (0 * inf would reach the others).
//
// Roundings. bf16 caches: P to bf16 once (2^-8 of a weight at most, as the
// output's own; decode attention keeps a second part of P, which here would be
// half as much tensor core work again), the sums l are of the f32 weights. int8 caches: the weights carry the V scale,
// log2(w) = log2(p) + log2(scale), the reference is the maximum of those, and w
// goes into P as f16 times 2^6: 2^-11 of a weight, and weights down to 2^-30 of
// the row's largest keep at least one bit; l is of w / scale in f32 or, beside
// scales out of 2^+-30, of the scores alone (kFarLog2). Value rows of zeros count
// for l alone: warp 18 finds them, a few scales at a time, while S is formed.
// Every wait is bounded, and a CTA ends behind its own copies and products.
//
// Measured: 4096 tokens behind 12288 (8 x 4 heads of 128) 810 us in a dozen
// calls (1965 MHz, 1.19 PFLOP/s of 1.6), 920 in thousands (1640 MHz, power cap
// of 1000 W, 1.05); 4 x 512 of 2048 (8 x 4 heads) 74 us, of 32 heads in int8 129
// (127 before zero rows and scales far apart were handled); 300 of 500 (8 x 4
// heads) 16 us; heads of 64, 4 x 512 of 2048 69 us, in int8 114. One zero row in
// each tile costs int8 90%. A step of both streams (256 rows x 128 keys)
// takes 3,400 to 4,000 cycles, of which the tensor core needs 2,100 and the 32
// thousand exponentials 2,050: the chain S, maximum, P, O of a stream hides
// only behind the other one's. A fourth of the exponentials on the FMA pipe
// (polynomial of degree 5) made short chunks 3% faster and long ones 6% slower.
// A call's fixed part is 11 us: 3 until the first scores, 2 at the end.
#include <atomic>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cuda.h>
#include <cuda_bf16.h>

#include <mutex>

#include "chunk_attn.h"

using namespace vxb;
using namespace vxb::tc;
using namespace vxb::chunk;

namespace {

template <int D, bool INT8>
struct Cfg {
  static constexpr int SLAB = BN * 128;             // 64 bf16 columns of 128 rows
  static constexpr int TILE = SLAB * (D / 64);      // one bf16 tile
  static constexpr int RAW = INT8 ? BN * D : 0;     // one int8 tile
  static constexpr int SLOTS = INT8 ? (D == 128 ? 3 : 6) : (D == 128 ? 5 : 10);
  static constexpr int RAWS = INT8 ? (D == 128 ? 3 : 6) : 0;
  static constexpr int OFF_KV = 2 * TILE;
  static constexpr int OFF_RAW = OFF_KV + SLOTS * TILE;
  // int8: three f32 per key of the last SLOTS tiles, K's scale times a.scale_log2, log2 of V's, 1 / V's;
  // then what is unusual about them (scale_role)
  static constexpr int KEYS = 3 * BN + 4;
  static constexpr int OFF_SCALE = OFF_RAW + RAWS * RAW;
  static constexpr int OFF_X = OFF_SCALE + (INT8 ? SLOTS * KEYS * 4 : 0);  // what the two halves of a row tell each other
  static constexpr int OFF_FAR = OFF_X + 4 * BM * 4;  // int8: the threads' maximum of scores (kFarLog2), +inf while they need none
  static constexpr int OFF_BARS = OFF_FAR + (INT8 ? 4 * BM * 4 : 0);
  static constexpr int SMEM = OFF_BARS + 768;
  // warpgroups: two of softmax for each stream, one of the MMA and TMA warps,
  // int8: two that convert; registers at launch and of each
  static constexpr int THREADS = INT8 ? 896 : 640, REGS = INT8 ? 72 : 96;
  static constexpr int REG_SOFT = INT8 ? 88 : 104, REG_PROD = INT8 ? 56 : 64, REG_CONV = 48;
  static_assert(4 * REG_SOFT + REG_PROD + (INT8 ? 2 * REG_CONV : 0) <= THREADS / 128 * REGS, "registers");
  static_assert(SMEM <= 232448, "shared memory");
};

template <int SLOTS, int RAWS>
struct Bars {
  uint64_t q_full, q_empty, o_free, drained, s_full[2], p_full[2], o_full[2], full[SLOTS], empty[SLOTS], keyed[SLOTS], scaled[SLOTS], raw_full[RAWS + 1],
      raw_empty[RAWS + 1];
  uint32_t tmem;
  int acc[2];  // the stream's O already holds values that its first product adds to
  // the softmax warps' run and its piece (of even and odd number): in shared
  // memory, to leave their registers to the scores
  Run run;
  Piece piece[2];
  int more[2];
};

// 16-byte chunk c (8 columns) of row r of a bf16 tile in shared memory
__device__ __forceinline__ uint32_t chunk_off(int r, int c) {
  return (uint32_t)((c >> 3) * (BN * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint64_t as_u64(float2 v) {
  uint64_t u;
  asm("mov.b64 %0, {%1, %2};" : "=l"(u) : "f"(v.x), "f"(v.y));
  return u;
}
__device__ __forceinline__ float2 as_f2(uint64_t u) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(u));
  return v;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(as_u64(a)), "l"(as_u64(b)), "l"(as_u64(c)));
  return as_f2(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(as_u64(a)), "l"(as_u64(b)));
  return as_f2(d);
}
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
               "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}

// four f32 of shared memory (the same for every lane) as two pairs
__device__ __forceinline__ void four_keys(const float *f, float2 &lo, float2 &hi) {
  const float4 x = *reinterpret_cast<const float4 *>(f);
  lo = make_float2(x.x, x.y);
  hi = make_float2(x.z, x.w);
}

// w[j] of lane q (of four) and w[q] of lane j change places
__device__ __forceinline__ void transpose4(uint4 (&w)[4], int lane) {
  auto swap = [&](uint4 &lo, uint4 &hi, int bit) {  // lanes with the bit give lo and get it, the others hi
    const bool up = lane & bit;
    const uint4 give = up ? lo : hi;
    const uint4 got = make_uint4(__shfl_xor_sync(0xffffffffu, give.x, bit), __shfl_xor_sync(0xffffffffu, give.y, bit),
                                 __shfl_xor_sync(0xffffffffu, give.z, bit), __shfl_xor_sync(0xffffffffu, give.w, bit));
    (up ? lo : hi) = got;
  };
  swap(w[0], w[1], 1);
  swap(w[2], w[3], 1);
  swap(w[0], w[2], 2);
  swap(w[1], w[3], 2);
}

// int8: what the sum of weights gets from a tile with unusual scales (scale_role),
// from N keys of S, the first `last` + 1 of them visible. The keys whose value row is
// zero (log2 scale -inf) add 2^(score + ref). Where the sum has a maximum of its own
// (`far`), and from here on where such a share is too large or the row has no unit
// but such keys, all keys add 2^(score - maximum). Rare: a function of its own leaves
// the softmax its registers. Called by whole warps; rows without a token (`token`)
// have no say.
template <int N>
__device__ __noinline__ float odd_tile(uint32_t tS, const float *keys, int last, float ref, float m, float l, bool token, bool far, float *far_s) {
  constexpr float SHIFT = 6.f;
  float v[8];
  if (!far) {
    float share = 0.f;
#pragma unroll 1
    for (int c = 0; c < N; c += 8) {
      tmem_ld8(tS + c, v);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 8; e++) share += c + e <= last && keys[BN + c + e] == -INFINITY ? ex2(fmaf(v[e], keys[c + e], ref)) : 0.f;
    }
    if (!__any_sync(0xffffffffu, token && (!(share <= kMostShare) || m == -INFINITY))) return l + share;
    *far_s = l == 0.f ? -INFINITY : fminf(m - SHIFT, FLT_MAX);
  }
  const float before = *far_s;
  float top = before;
#pragma unroll 1
  for (int c = 0; c < N; c += 8) {
    tmem_ld8(tS + c, v);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 8; e++) top = c + e <= last ? fmaxf(top, v[e] * keys[c + e]) : top;
  }
  const float own = top == -INFINITY ? 0.f : -top;
  l = before == -INFINITY ? l : l * ex2(before - top);
#pragma unroll 1
  for (int c = 0; c < N; c += 8) {
    tmem_ld8(tS + c, v);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 8; e++) l += c + e <= last ? ex2(fmaf(v[e], keys[c + e], own)) : 0.f;
  }
  // (a row without a token has what lies in shared memory for queries: no
  // maximum of its may read as "none", since whole warps have one or none)
  *far_s = fminf(top, FLT_MAX);
  return l;
}

// The end of a row whose sums have maxima of their own (+inf: a half that needed
// none, its sum is in O's unit m): O is divided by the sum, which then is 1. The
// factor of O, the row's maximum and the sum.
__device__ __noinline__ float3 far_join(float m, float l0, float l1, float top0, float top1) {
  top0 = top0 < INFINITY ? top0 : l0 == 0.f ? -INFINITY : m;
  top1 = top1 < INFINITY ? top1 : l1 == 0.f ? -INFINITY : m;
  const float t = fmaxf(top0, top1);
  const float l = (top0 == -INFINITY ? l0 : l0 * ex2(top0 - t)) + (top1 == -INFINITY ? l1 : l1 * ex2(top1 - t));
  return l > 0.f ? make_float3(ex2(m - t) / l, t + log2f(l), 1.f) : make_float3(0.f, -INFINITY, l);
}

// ------------------------------------------------------------------ softmax: thread = (stream, row, half of a tile's keys)
template <int D, bool INT8, class B>
__device__ __forceinline__ void softmax_role(const ChunkArgs &a, uint8_t *sm, B &bars) {
  using C = Cfg<D, INT8>;
  constexpr int N = BN / 2;
  constexpr float SHIFT = INT8 ? 6.f : 0.f;  // P, O and l hold 2^SHIFT times the weights
  const int st = threadIdx.x >> 8, half = (threadIdx.x >> 7) & 1, warp4 = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
  const int r = warp4 * 32 + lane, tid = threadIdx.x & 255;  // row of the tile; thread of the stream
  const uint32_t lane_off = (uint32_t)(warp4 * 32) << 16;
  const uint32_t tS = bars.tmem + st * 128 + half * N + lane_off;  // this half's scores, then (bf16) its weights
  const uint32_t tO = bars.tmem + 256 + st * 128 + lane_off, tO_other = bars.tmem + 256 + (st ^ 1) * 128 + lane_off;
  float *x_row = reinterpret_cast<float *>(sm + C::OFF_X) + r;  // [stream][half][row]
  float *x_mine = x_row + (st * 2 + half) * BM, *x_half = x_row + (st * 2 + (half ^ 1)) * BM;
  float *far_row_s = reinterpret_cast<float *>(sm + C::OFF_FAR) + r, *far_s = far_row_s + (st * 2 + half) * BM;  // int8
  const int pair = 4 + st * 4 + warp4;  // barrier of the two warps that share these rows
  Waiter wait{a.err};
  uint32_t step = 0, pieces = 0, ring = 0;  // this stream's steps; pieces; first ring index of the piece
  while (true) {
    if (threadIdx.x == 0) {
      Run run = bars.run;
      Piece next;
      bars.more[pieces & 1] = run.next(a, next);
      bars.piece[pieces & 1] = next;
      bars.run = run;
    }
    __syncwarp();
    bar_sync(1, 512);
    if (!bars.more[pieces & 1]) break;
    const Piece &p = bars.piece[pieces & 1];
    const int tile_tok = p.tok0 + (p.both ? st * a.sh.tpt : 0);  // first token of this stream's rows
    const int live = min(a.sh.tpt, p.tok0 + p.ntok - tile_tok) * a.G;
    // last visible key; rows that do not exist are never masked (nor read)
    const int lim = r < live ? (a.sh.causal ? p.s.len - p.s.rows + tile_tok + r / a.G : p.s.len - 1) : INT_MAX;
    // the same of the first row of this stream, and of both
    const int lim_first = a.sh.causal ? p.s.len - p.s.rows + tile_tok : p.s.len - 1, lim_item = a.sh.causal ? p.s.len - p.s.rows + p.tok0 : p.s.len - 1;
    const bool warp_live = warp4 * 32 < live;
    float m = -INFINITY, l = 0.f;
    if constexpr (INT8) *far_s = INFINITY;
    bool far = false;  // int8: the sum has a maximum of its own from here on
    const int steps = p.steps(st);
    for (int i = 0; i < steps; i++, step++) {
      const int t = p.tile(st, i), k0 = t * BN, kh = k0 + half * N;
      const uint32_t kv = ring + 2 * (uint32_t)(t - p.tb);  // ring index of K; V is the next
      wait(&bars.s_full[st], step & 1);
      tc_fence_after();
      // V elements that only some rows may see, and rows behind the last token
      bool odd = false;
      const bool both_here = p.both && i < p.n0;  // the other stream works on the same tile
      // the tile's first key that is hidden from some row of either stream that uses it
      const int hidden = max(0, (both_here ? lim_item : lim_first) + 1 - k0);
      const bool diagonal = hidden < min(BN, p.s.len - k0);
      if constexpr (!INT8) {
        if (diagonal || p.s.len - k0 < BN) {
          const int valid = min(BN, p.s.len - k0);
          uint8_t *sv_tile = sm + C::OFF_KV + ((kv + 1) % C::SLOTS) * C::TILE;
          wait(&bars.full[(kv + 1) % C::SLOTS], ((kv + 1) / C::SLOTS) & 1);
          if (valid < BN && !(both_here && st == 1)) {
            const int rows = (valid + 15) / 16 * 16 - valid;
            for (int c = tid; c < rows * (D / 8); c += 256)
              *reinterpret_cast<uint4 *>(sv_tile + chunk_off(valid + c / (D / 8), c % (D / 8))) = make_uint4(0u, 0u, 0u, 0u);
            fence_async_smem();
          }
          if (diagonal) {
            uint32_t found[2] = {0u, 0u};
#pragma unroll 4
            for (int c = hidden * (D / 8) + tid, n = 0; c < valid * (D / 8); c += 256, n ^= 1)
              found[n] = add_odd(found[n], *reinterpret_cast<const uint4 *>(sv_tile + chunk_off(c / (D / 8), c % (D / 8))));
            __syncwarp();
            odd = bar_or(2 + st, 256, (odd_bf16(found[0]) | odd_bf16(found[1])) != 0);
          }
        }
      }
      if (warp_live) {
        // int8 reads S twice, 32 columns at a time: its threads have too few
        // registers for 64 scores (spilled, they took twice as long)
        constexpr int KEEP = INT8 ? 32 : N;
        float s[KEEP];
        // what the scales of this tile's keys make: there until its V is released, after P
        const float *keys = reinterpret_cast<const float *>(sm + C::OFF_SCALE) + (kv / 2 % C::SLOTS) * C::KEYS + half * N;
        if constexpr (INT8) wait(&bars.scaled[kv / 2 % C::SLOTS], (kv / 2 / C::SLOTS) & 1);
        const bool masked = !__all_sync(0xffffffffu, kh + N - 1 <= lim);
        auto scores = [&](int c0) {
#pragma unroll
          for (int c = 0; c < KEEP; c += 32) tmem_ld32(tS + c0 + c, *reinterpret_cast<float(*)[32]>(s + c));
          tmem_wait_ld();
          if constexpr (INT8) {
#pragma unroll
            for (int c = 0; c < KEEP; c += 4) {
              float2 k[2], v[2];
              four_keys(keys + c0 + c, k[0], k[1]);
              four_keys(keys + BN + c0 + c, v[0], v[1]);
#pragma unroll
              for (int e = 0; e < 2; e++) {
                const float2 y = fma2(make_float2(s[c + 2 * e], s[c + 2 * e + 1]), k[e], v[e]);
                s[c + 2 * e] = y.x;
                s[c + 2 * e + 1] = y.y;
              }
            }
          }
          if (masked) {
#pragma unroll
            for (int c = 0; c < KEEP; c++) s[c] = kh + c0 + c <= lim ? s[c] : -INFINITY;
          }
        };
        // a scale of the tile (of both halves' keys), or of one before it
        uint32_t odd = 0;
        if constexpr (INT8) {
          odd = reinterpret_cast<const uint32_t *>(keys)[3 * BN - half * N];
          if ((odd & 1) && !far) {
            far = true;
            *far_s = l == 0.f ? -INFINITY : fminf(m - SHIFT, FLT_MAX);
          }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int c0 = 0; c0 < N; c0 += KEEP) {
          scores(c0);
          float mx4[4] = {mx, s[0], s[1], s[2]};
#pragma unroll
          for (int c = 3; c + 7 < KEEP; c += 8) {
#pragma unroll
            for (int e = 0; e < 4; e++) mx4[e] = max3(mx4[e], s[c + 2 * e], s[c + 2 * e + 1]);
          }
          mx4[0] = max3(mx4[0], s[KEEP - 5], s[KEEP - 4]);
          mx = max3(max3(mx4[0], mx4[1], mx4[2]), max3(mx4[3], s[KEEP - 3], s[KEEP - 2]), s[KEEP - 1]);
        }
        // the row's maximum over both halves (the next S, so the next write
        // here, waits for both halves' P)
        *x_mine = mx;
        bar_sync(pair, 64);
        mx = fmaxf(mx, *x_half) * (INT8 ? 1.f : a.scale_log2);
        const bool grow = mx > m + RESCALE_THRESHOLD;
        const float m_new = grow ? mx : m;
        const float mb = m_new == -INFINITY ? 0.f : m_new;
        float alpha = grow ? ex2(m - mb) : 1.f;
        m = m_new;
        if (i > 0 && __any_sync(0xffffffffu, grow)) {
          // s_full of this step came behind the products of the last: O is whole.
          // Each half takes half of its columns.
#pragma unroll 1
          for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 8) {
            float o[8];
            tmem_ld8(tO + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] *= alpha;
            tmem_st8(tO + c, o);
          }
        }
        const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), ref2 = make_float2(SHIFT - mb, SHIFT - mb);
        float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        if constexpr (INT8) {
          if (odd || far) {
            l = odd_tile<N>(tS, keys, lim - kh, ref2.x, m, l * (far ? 1.f : alpha), r < live, far, far_s);
            far = __any_sync(0xffffffffu, *far_s < INFINITY);  // (a warp's lanes agree)
            alpha = 1.f;
          }
        }
#pragma unroll
        for (int c = 0; c < N / 32; c++) {
          if constexpr (INT8) scores(c * 32);
          float *v = s + c * 32 % KEEP;
#pragma unroll
          for (int e0 = 0; e0 < 32; e0 += 4) {
            float2 inv[2];
            if constexpr (INT8) {
              four_keys(keys + 2 * BN + c * 32 + e0, inv[0], inv[1]);
              if (masked) {  // 0 * what is not finite
#pragma unroll
                for (int e = 0; e < 2; e++) {
                  inv[e].x = kh + c * 32 + e0 + 2 * e <= lim ? inv[e].x : 0.f;
                  inv[e].y = kh + c * 32 + e0 + 2 * e + 1 <= lim ? inv[e].y : 0.f;
                }
              }
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float *y = v + e0 + 2 * e;
              const float2 x = INT8 ? add2(make_float2(y[0], y[1]), ref2) : fma2(make_float2(y[0], y[1]), scale2, ref2);
              const float2 w = make_float2(ex2(x.x), ex2(x.y));
              y[0] = w.x;
              y[1] = w.y;
              sum2[e] = INT8 ? fma2(w, inv[e], sum2[e]) : add2(sum2[e], w);
            }
          }
          uint32_t h[16];
#pragma unroll
          for (int e = 0; e < 16; e++) {
            if constexpr (INT8) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h[e]) : "f"(v[2 * e + 1]), "f"(v[2 * e]));
            else h[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
          }
          tmem_st16u(tS + c * 16, h);
        }
        if (!far) l = l * alpha + ((sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y));
        tmem_wait_st();
      }
      if constexpr (!INT8) {
        if (odd) {
          // rare: every non-finite V element, added to the rows that see its
          // key (each half: its keys), one half after the other
          const int valid = min(BN, p.s.len - k0);
          uint8_t *sv_tile = sm + C::OFF_KV + ((ring + 2 * (uint32_t)(t - p.tb) + 1) % C::SLOTS) * C::TILE;
#pragma unroll 1
          for (int turn = 0; turn < 2; turn++) {
            if (warp_live && turn == half) {
              if (i == 0 && half == 0) {
                const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                for (int c = 0; c < D; c += 8) tmem_st8(tO + c, z);
                tmem_wait_st();
              }
              for (int k = max(hidden, half * N); k < min(valid, (half + 1) * N); k++)
                for (int c = 0; c < D / 8; c++) {
                  const uint4 w = *reinterpret_cast<const uint4 *>(sv_tile + chunk_off(k, c));
                  if (!(odd_bf16(w.x) | odd_bf16(w.y) | odd_bf16(w.z) | odd_bf16(w.w))) continue;
                  const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll 1
                  for (int e = 0; e < 8; e++) {
                    const uint32_t bits = (ww[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
                    if ((bits & 0x7F80u) != 0x7F80u) continue;
                    const uint32_t two = __float_as_uint(tmem_ld1(tS + ((k - half * N) >> 1)));
                    const float pk = __uint_as_float(k & 1 ? two & 0xFFFF0000u : two << 16), o = tmem_ld1(tO + c * 8 + e);
                    tmem_st1(tO + c * 8 + e, k0 + k <= lim ? fmaf(pk, __uint_as_float(bits << 16), o) : o);
                    tmem_wait_st();
                  }
                }
            }
            tc_fence_before();
            __syncwarp();
            bar_sync(2 + st, 256);
            tc_fence_after();
          }
          if (i == 0 && tid == 0) bars.acc[st] = 1;
          // every row has taken the odd elements: out of the tile with them
          if (both_here) bar_sync(1, 512);
          if (!(both_here && st == 1)) {
            for (int c = hidden * (D / 8) + tid; c < valid * (D / 8); c += 256) {
              uint4 *at = reinterpret_cast<uint4 *>(sv_tile + chunk_off(c / (D / 8), c % (D / 8)));
              *at = make_uint4(even_bf16(at->x), even_bf16(at->y), even_bf16(at->z), even_bf16(at->w));
            }
            fence_async_smem();
          }
          __syncwarp();
          if (both_here) bar_sync(1, 512);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.p_full[st]);
    }
    m -= SHIFT;
    // ---------------- end of the piece: l of both halves, of a shared row of
    // both streams, then O
    bar_sync(pair, 64);  // the last step's maxima have been read
    *x_mine = l;
    bar_sync(pair, 64);
    float own = 1.f;  // factor that brings this stream's O to the unit of l
    if (INT8 && (*far_s < INFINITY || far_row_s[(st * 2 + (half ^ 1)) * BM] < INFINITY)) {
      const float3 y = far_join(m, l, *x_half, *far_s, far_row_s[(st * 2 + (half ^ 1)) * BM]);
      own = y.x;
      m = y.y;
      l = y.z;
    } else {
      l += *x_half;
    }
    float f0 = own, f1 = 0.f;  // factors of this stream's and the other's O
    if (!p.both) {
      bar_sync(1, 512);
      *x_mine = half ? l : m;
      if (INT8 && half == 0) *far_s = own;
      bar_sync(1, 512);
      const float om = x_row[(st ^ 1) * 2 * BM], ol = x_row[((st ^ 1) * 2 + 1) * BM];
      const float top = fmaxf(m, om);
      f0 = m == -INFINITY ? 0.f : ex2(m - top);
      f1 = om == -INFINITY ? 0.f : ex2(om - top);
      // NaN sums stay: a stream with steps whose maximum is -inf has l = 0 or NaN
      l = (m == -INFINITY ? l : l * f0) + (om == -INFINITY ? ol : ol * f1);
      m = top;
      if constexpr (INT8) {
        f0 *= own;
        f1 *= far_row_s[(st ^ 1) * 2 * BM];
      }
      bar_sync(1, 512);  // read by all
      wait(&bars.o_full[st ^ 1], pieces & 1);
    } else {
      bar_sync(pair, 64);
    }
    wait(&bars.o_full[st], pieces & 1);
    tc_fence_after();
    const bool mine = r < live, whole = p.whole();
    const int tok = tile_tok + r / a.G;
    const size_t row = (size_t)(p.s.row0 + tok) * a.Hq + (size_t)p.head * a.G + r % a.G;
    // scratch of an unfinished item: the CTA's first or last part
    float *part = a.ws + (size_t)(blockIdx.x * 2 + (p.tb > 0 ? 0 : 1)) * (kRowsItem * (D + 2));
    const int prow = p.both ? st * BM + r : r;
    if (warp_live) {
      const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
      // the threads of a row take D / 2 columns each, or D / 4 but 32 at least
      const int width = p.both ? D / 2 : D / 4 > 32 ? D / 4 : 32, first = p.both ? half * width : (st * (D == 128 ? 2 : 1) + half) * width;
      const int tq0 = (r & ~3) / a.G, gq0 = (r & ~3) - tq0 * a.G;
      const bool has0 = steps > 0, has1 = !p.both && p.steps(st ^ 1) > 0;
      f0 *= inv;
      f1 *= inv;
#pragma unroll 1
      for (int c = first; c < (D == 64 && !p.both && half ? 0 : first + width); c += 32) {
        uint4 w[4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          float o[16], x[16];
#pragma unroll
          for (int e = 0; e < 16; e++) o[e] = x[e] = 0.f;
          if (has0) tmem_ld16(tO + c + h * 16, o);
          if (has1) tmem_ld16(tO_other + c + h * 16, x);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; e++) o[e] = has1 ? fmaf(x[e], f1, o[e] * f0) : o[e] * f0;
          if (!whole) {
            float4 *dst = reinterpret_cast<float4 *>(part + ((size_t)((c + h * 16) / 8) * kRowsItem + prow) * 8);
#pragma unroll
            for (int q = 0; q < 4; q++)
              if (mine) __stcg(dst + (q >> 1) * (kRowsItem * 2) + (q & 1), make_float4(o[q * 4], o[q * 4 + 1], o[q * 4 + 2], o[q * 4 + 3]));
          }
#pragma unroll
          for (int q = 0; q < 2; q++)
            w[h * 2 + q] = make_uint4(pack_bf16(o[q * 8], o[q * 8 + 1]), pack_bf16(o[q * 8 + 2], o[q * 8 + 3]),
                                      pack_bf16(o[q * 8 + 4], o[q * 8 + 5]), pack_bf16(o[q * 8 + 6], o[q * 8 + 7]));
        }
        if (whole) {
          // four lanes exchange their 64 bytes, so that they write one row at
          // a time (each its own row took twice as long: 32 lines a store)
          transpose4(w, lane);
          int tq = tq0, gq = gq0;
#pragma unroll
          for (int q = 0; q < 4; q++) {
            if ((r & ~3) + q < live)
              *reinterpret_cast<uint4 *>(a.out + (((size_t)(p.s.row0 + tile_tok + tq) * a.Hq) + (size_t)p.head * a.G + gq) * D + c + (r & 3) * 8) = w[q];
            if (++gq == a.G) {
              gq = 0;
              tq++;
            }
          }
        }
      }
      if (mine && half == 0 && (p.both || st == 0)) {
        if (!whole) __stcg(reinterpret_cast<float2 *>(part + (size_t)kRowsItem * D) + prow, make_float2(m, l));
        else if (a.lse) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
      }
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars.o_free);
    pieces++;
    ring += 2 * (uint32_t)max(0, p.te - p.tb);
  }
}

// ------------------------------------------------------------------ MMA warp
// A ring slot that walks on: K and V of a tile are neighbours, tiles two apart.
template <int SLOTS>
struct Slot {
  uint32_t slot, phase;
  __device__ __forceinline__ void skip(uint32_t n) {  // n <= SLOTS
    slot += n;
    if (slot >= SLOTS) {
      slot -= SLOTS;
      phase ^= 1;
    }
  }
};

template <int D, bool INT8, class B>
__device__ __forceinline__ void mma_role(const ChunkArgs &a, uint8_t *sm, B &bars) {
  using C = Cfg<D, INT8>;
  constexpr uint32_t ID_QK = idesc_bf16(BM, BN, false);
  // int8: P and V in f16 (bits 7 and 10 of the types say bf16)
  constexpr uint32_t ID_PV = INT8 ? idesc_bf16(BM, D, true) & ~((1u << 7) | (1u << 10)) : idesc_bf16(BM, D, true);
  constexpr uint64_t KMAJOR = desc_base(16, 1024), VMAJOR = desc_base(C::SLAB, 1024);
  const uint32_t s_q = smem_u32(sm) >> 4, s_kv = smem_u32(sm + C::OFF_KV) >> 4;
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars.tmem, 0);
  const uint32_t one = elect_one();
  Waiter wait{a.err};
  Run run(a);
  Piece p{};
  Slot<C::SLOTS> ring{0, 0};  // K of the piece's first tile
  uint32_t pieces = 0, p_phase = 0;  // p_phase: bit of each stream
  // S of a stream from the K tile in a slot
  auto qk = [&](uint32_t st, const Slot<C::SLOTS> &k, bool fresh, bool release) {
    if (fresh) wait(&bars.full[k.slot], k.phase);
    tc_fence_after();
    const uint64_t q = KMAJOR + (s_q + (p.both ? st : 0) * (C::TILE >> 4)), kd = KMAJOR + (s_kv + k.slot * (C::TILE >> 4));
#pragma unroll
    for (int x = 0; x < D / 16; x++) {
      const uint32_t off = ((x >> 2) * C::SLAB + (x & 3) * 32) >> 4;
      mma_ss(one, tmem + st * 128, q + off, kd + off, ID_QK, x > 0 ? 1u : 0u);
    }
    mma_commit(one, &bars.s_full[st]);
    if (release) mma_commit(one, &bars.empty[k.slot]);
  };
  // O of a stream plus its P times the V tile in a slot (k16: its 16s of keys)
  auto pv = [&](uint32_t st, const Slot<C::SLOTS> &v, bool first, int k16, bool fresh, bool release) {
    if (fresh) wait(&bars.full[v.slot], v.phase);
    wait(&bars.p_full[st], (p_phase >> st) & 1);
    p_phase ^= 1u << st;
    tc_fence_after();
    uint32_t acc = first ? 0u : 1u;
    if (!INT8 && first && __shfl_sync(0xffffffffu, *(volatile int *)&bars.acc[st], 0)) {
      acc = 1u;
      __syncwarp();
      *(volatile int *)&bars.acc[st] = 0;
    }
    const uint64_t vd = VMAJOR + (s_kv + v.slot * (C::TILE >> 4));
    const uint32_t t_o = tmem + 256 + st * 128, t_p = tmem + st * 128;
    // P of 64 keys is in the first 32 columns of each half of S
#pragma unroll
    for (int x = 0; x < BN / 16; x++)
      if (x < k16) mma_ts(one, t_o, t_p + (x >> 2) * 64 + (x & 3) * 8, vd + (x * 2048 >> 4), ID_PV, x > 0 ? 1u : acc);
    if (release) mma_commit(one, &bars.empty[v.slot]);
  };
  while (run.next(a, p)) {
    const int tiles = max(0, p.te - p.tb);
    // the last tile of the sequence holds fewer keys
    const int last = (p.s.len - 1) / BN - p.tb, last16 = (p.s.len - (p.tb + last) * BN + 15) / 16;
    Slot<C::SLOTS> k = ring, v = ring;
    v.skip(1);
    wait(&bars.q_full, pieces & 1);
    // the softmax warps have read the last piece's O before the first product
    if (tiles == 0 && pieces > 0) wait(&bars.o_free, (pieces - 1) & 1);
    if (p.both) {
      // both streams use a tile; stream 1 sees at least as many
      if (p.n0 > 0) qk(0, k, true, false);
      if (p.n1 > 0) qk(1, k, p.n0 == 0, true);
      if (tiles > 0 && pieces > 0) wait(&bars.o_free, (pieces - 1) & 1);
#pragma unroll 1
      for (int i = 0; i < p.n1; i++) {
        const int k16 = i == last ? last16 : BN / 16;
        k.skip(2);
        if (i < p.n0) {
          pv(0, v, i == 0, k16, true, false);
          if (i + 1 < p.n0) qk(0, k, true, false);
          else mma_commit(one, &bars.o_full[0]);
        }
        pv(1, v, i == 0, k16, i >= p.n0, true);
        if (i + 1 < p.n1) qk(1, k, i + 1 >= p.n0, true);
        else mma_commit(one, &bars.o_full[1]);
        v.skip(2);
      }
    } else {
      // tile i belongs to stream i & 1; S runs two tiles ahead
      for (int i = 0; i < 2 && i < tiles; i++) {
        qk(i, k, true, true);
        k.skip(2);
      }
      if (tiles > 0 && pieces > 0) wait(&bars.o_free, (pieces - 1) & 1);
#pragma unroll 1
      for (int i = 0; i < tiles; i++) {
        const uint32_t st = i & 1;
        pv(st, v, i < 2, i == last ? last16 : BN / 16, true, true);
        if (i + 2 < tiles) qk(st, k, true, true);
        else mma_commit(one, &bars.o_full[st]);
        k.skip(2);
        v.skip(2);
      }
    }
    mma_commit(one, &bars.q_empty);
    if (p.n0 == 0) mma_commit(one, &bars.o_full[0]);
    if (p.n1 == 0) mma_commit(one, &bars.o_full[1]);
    ring = v;
    ring.skip(C::SLOTS - 1);  // V of the tile behind the last, less one
    ring.phase ^= 1;
    pieces++;
  }
  // (behind a wait that has run out, products may be under way that nobody waits for)
  mma_commit(one, &bars.drained);
  wait.last(&bars.drained, 0);
}

// ------------------------------------------------------------------ TMA warp
template <int D, bool INT8, class B>
__device__ __forceinline__ void tma_role(const CUtensorMap *tq, const CUtensorMap *tk, const CUtensorMap *tv, const ChunkArgs &a,
                                         uint8_t *sm, B &bars) {
  using C = Cfg<D, INT8>;
  constexpr int SLABS = INT8 ? 1 : D / 64;
  constexpr int RING = INT8 ? C::RAWS : C::SLOTS;
  constexpr int ROW = INT8 ? D : 128;  // bytes of a box row
  const int lane = threadIdx.x & 31;
  const int per_tile = BN / a.box;  // boxes of a tile and slab
  uint8_t *tiles = sm + (INT8 ? C::OFF_RAW : C::OFF_KV);
  Waiter wait{a.err};
  Run run(a);
  Piece p{};
  uint32_t idx = 0, pieces = 0, issued = 0, queries = 0;
  while (run.next(a, p)) {
    const int32_t *table = a.tables + (size_t)p.s.slot * a.mbps;
    // pool rows of this lane's box in the tiles t .. t + 32 / per_tile - 1
    const int group = 32 / per_tile;
    int rows = 0;
    auto look_up = [&](int t) {
      const int tok = (t + lane / per_tile) * BN + lane % per_tile * a.box;
      if (tok < p.s.len && t + lane / per_tile < p.te) {
        const int b = tok / a.bs;
        rows = (int)(((long long)__ldcg(table + b) * a.Hkv + p.head) * a.bs + (tok - b * a.bs));
      }
    };
    auto load = [&](const CUtensorMap *map, int t) {
      const uint32_t slot = idx % RING;
      uint64_t *full = INT8 ? &bars.raw_full[slot] : &bars.full[slot], *empty = INT8 ? &bars.raw_empty[slot] : &bars.empty[slot];
      if (idx >= RING) wait(empty, (idx / RING - 1) & 1);
      const int boxes = (min(BN, p.s.len - t * BN) + a.box - 1) / a.box;
      // (behind a wait that has run out nothing is copied any more)
      if (lane == 0 && !wait.dead) mbar_expect_tx(full, (uint32_t)(boxes * SLABS * a.box * ROW));
      __syncwarp();
      const int row = __shfl_sync(0xffffffffu, rows, (t - p.tb) % group * per_tile + lane / SLABS % per_tile);
      if (lane < boxes * SLABS && !wait.dead) {
        const int b = lane / SLABS, sl = lane % SLABS;
        tma_load_2d(tiles + slot * (INT8 ? C::RAW : C::TILE) + sl * C::SLAB + b * a.box * ROW, map, sl * 64, row, full);
      }
      __syncwarp();
      idx++;
      if (!wait.dead) issued = idx;
    };
    auto load_q = [&]() {
      if (pieces > 0) wait(&bars.q_empty, (pieces - 1) & 1);
      if (lane == 0 && !wait.dead) {
        queries = pieces + 1;
        const int halves = p.both ? 2 : 1;
        mbar_expect_tx(&bars.q_full, (uint32_t)(halves * (D / 64) * a.sh.tpt * a.G * 128));
        for (int h = 0; h < halves; h++)
          for (int sl = 0; sl < D / 64; sl++)
            tma_load_3d(sm + h * C::TILE + sl * C::SLAB, tq, sl * 64, p.head * a.G, p.s.row0 + p.tok0 + h * a.sh.tpt, &bars.q_full);
      }
      __syncwarp();
    };
    if (p.te <= p.tb || pieces == 0) load_q();
    for (int t = p.tb; t < p.te; t++) {
      if ((t - p.tb) % group == 0) look_up(t);
      load(tk, t);
      if (t == p.tb && pieces > 0) load_q();  // behind the first keys: the last piece may still use Q
      load(tv, t);
    }
    pieces++;
  }
  // no copy is under way when the CTA ends, also behind a wait that has run out
  issued = __reduce_max_sync(0xffffffffu, issued);
  queries = __reduce_max_sync(0xffffffffu, queries);
  for (uint32_t i = issued > RING ? issued - RING : 0; i < issued; i++)
    wait.last(INT8 ? &bars.raw_full[i % RING] : &bars.full[i % RING], (i / RING) & 1);
  if (queries > 0) wait.last(&bars.q_full, (queries - 1) & 1);
}

// ------------------------------------------------------------------ scale warp (int8)
// Looks a tile's V scales over: bit 0 one out of 2^+-kFarLog2, bit 1 a value row of
// zeros. Such a row (only scale 1 can be one, so V is looked at in that rare case
// alone) gets the log2 scale -inf and the inverse 0.
template <int D, class B>
__device__ __forceinline__ void scale_role(const ChunkArgs &a, uint8_t *sm, B &bars) {
  using C = Cfg<D, true>;
  const int lane = threadIdx.x & 31;
  Waiter wait{a.err};
  Run run(a);
  Piece p{};
  uint32_t idx = 0;
  while (run.next(a, p)) {
    for (int t = p.tb; t < p.te; t++, idx++) {
      const uint32_t slot = idx % C::SLOTS, v = 2 * idx + 1;
      float *keys = reinterpret_cast<float *>(sm + C::OFF_SCALE) + slot * C::KEYS;
      wait(&bars.keyed[slot], (idx / C::SLOTS) & 1);
      auto far = [&](int k) { return !(keys[2 * BN + k] >= 1.f / kFarInverse && keys[2 * BN + k] <= kFarInverse); };
      uint32_t odd = 0;
      bool look = false;
      for (int k = lane; k < BN; k += 32) look |= far(k) || (keys[2 * BN + k] == 1.f && t * BN + k < p.s.len);
      if (__any_sync(0xffffffffu, look)) {
        wait(&bars.full[v % C::SLOTS], (v / C::SLOTS) & 1);
        const uint8_t *tile = sm + C::OFF_KV + v % C::SLOTS * C::TILE;
        for (int k = lane; k < BN; k += 32) {
          if (far(k)) odd |= 1u;
          if (keys[2 * BN + k] != 1.f || t * BN + k >= p.s.len) continue;
          uint32_t any = 0;
          for (int c = 0; c < D / 8 && !any; c++) {
            const uint4 x = *reinterpret_cast<const uint4 *>(tile + chunk_off(k, c));
            any = x.x | x.y | x.z | x.w;
          }
          if (any) continue;
          keys[BN + k] = -INFINITY;
          keys[2 * BN + k] = 0.f;
          odd |= 2u;
        }
        odd = __reduce_or_sync(0xffffffffu, odd);
      }
      if (lane == 0) reinterpret_cast<uint32_t *>(keys)[3 * BN] = odd;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.scaled[slot]);
    }
  }
}

// ------------------------------------------------------------------ converter warpgroup (int8)
template <int D, class B>
__device__ __forceinline__ void convert_role(const ChunkArgs &a, uint8_t *sm, B &bars) {
  using C = Cfg<D, true>;
  const int tid = threadIdx.x - 640, lane = threadIdx.x & 31;
  const int r = tid & 127, v_scale = tid >> 7;  // thread of K scales, or of V scales
  constexpr int N = BN * D / 16 / 256;
  Waiter wait{a.err};
  Run run(a);
  Piece p{};
  uint32_t idx = 0;
  while (run.next(a, p)) {
    const int32_t *table = a.tables + (size_t)p.s.slot * a.mbps;
    for (int t = p.tb; t < p.te; t++) {
      const int tok = t * BN + r, valid = min(BN, p.s.len - t * BN);
      size_t row = 0;
      if (r < valid) row = ((size_t)__ldcg(table + tok / a.bs) * a.Hkv + p.head) * a.bs + tok % a.bs;
      const float scale = r < valid ? __ldcg((v_scale ? a.sv : a.sk) + row) : 1.f;
#pragma unroll
      for (int v = 0; v < 2; v++, idx++) {
        const uint32_t raw = idx % C::RAWS, slot = idx % C::SLOTS;
        wait(&bars.raw_full[raw], (idx / C::RAWS) & 1);
        if (idx >= C::SLOTS) wait(&bars.empty[slot], (idx / C::SLOTS - 1) & 1);
        const uint8_t *src = sm + C::OFF_RAW + raw * C::RAW;
        uint8_t *dst = sm + C::OFF_KV + slot * C::TILE;
        // The slot was free: with 3 slots V of the tile before the last has
        // been used, with 6 K of the third last, whose S came behind P of the
        // tile before it. So the softmax is done with the tile SLOTS before
        // this one, and its place takes this tile's scales.
        if (!v) {
          float *keys = reinterpret_cast<float *>(sm + C::OFF_SCALE) + idx / 2 % C::SLOTS * C::KEYS + r;
          if (v_scale) {
            const float sv = scale < kLeastScale ? kLeastScale : scale;
            // (a factor 2^lv in the weight and 2^-lv in the sum: what the
            // approximate logarithm is off by, under 2^-16, is V's alone)
            const float lv = __log2f(sv);
            keys[BN] = lv;
            keys[2 * BN] = ex2(-lv);
          } else {
            keys[0] = scale * a.scale_log2;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.keyed[idx / 2 % C::SLOTS]);
        }
        // 16 codes at a time; rows behind the last token become zeros
        uint4 codes[N];
#pragma unroll
        for (int n = 0; n < N; n++) {
          const int c = tid + n * 256;
          codes[n] = c / (D / 16) < valid ? *reinterpret_cast<const uint4 *>(src + c * 16) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int n = 0; n < N; n++) {
          const int c = tid + n * 256, row_t = c / (D / 16), ch = c % (D / 16);
          const uint32_t in[4] = {codes[n].x, codes[n].y, codes[n].z, codes[n].w};
          uint32_t o[8];
#pragma unroll
          for (int e = 0; e < 4; e++)
#pragma unroll
            for (int half = 0; half < 2; half++) {
              uint32_t d;
              if (v) {
                // f16: (code ^ 0x80) under the magic 0x64 is 1024 + 128 + code
                const uint32_t x = __byte_perm(in[e] ^ 0x80808080u, 0x64646464u, half ? 0x4342u : 0x4140u);
                asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0x64806480u));
              } else {
                // bf16: the low 7 bits under the magic 0x43 are 128 + low7, the
                // sign bit alone 128 or 256; their difference is the code
                const uint32_t x = __byte_perm(in[e], 0x43434343u, half ? 0x4342u : 0x4140u);
                asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x & 0xFF7FFF7Fu), "r"(x & 0xFF80FF80u));
              }
              o[e * 2 + half] = d;
            }
          *reinterpret_cast<uint4 *>(dst + chunk_off(row_t, 2 * ch)) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4 *>(dst + chunk_off(row_t, 2 * ch + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bars.raw_empty[raw]);
          mbar_arrive(&bars.full[slot]);
        }
      }
    }
  }
}

template <int D, bool INT8>
__global__ void __launch_bounds__(Cfg<D, INT8>::THREADS, 1)
    chunk_attn_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                      const __grid_constant__ CUtensorMap tv, const __grid_constant__ ChunkArgs a) {
  using C = Cfg<D, INT8>;
  using B = Bars<C::SLOTS, C::RAWS>;
  static_assert(sizeof(B) <= 768, "barriers");
  extern __shared__ __align__(1024) uint8_t sm[];
  B &bars = *reinterpret_cast<B *>(sm + C::OFF_BARS);
  const int warp = threadIdx.x >> 5;
  if (warp == 0) {
    // no tensor memory is taken that a CTA of the last kernel may still ask for
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 17 * 32) {
    for (const CUtensorMap *map : {&tq, &tk, &tv}) asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  }
  if (threadIdx.x == 32) {
    bars.run = Run(a);
    mbar_init(&bars.q_full, 1);
    mbar_init(&bars.q_empty, 1);
    mbar_init(&bars.o_free, 16);
    mbar_init(&bars.drained, 1);
    for (int i = 0; i < 2; i++) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 8);
      mbar_init(&bars.o_full[i], 1);
      bars.acc[i] = 0;
    }
    for (int i = 0; i < C::SLOTS; i++) {
      mbar_init(&bars.full[i], INT8 ? 8 : 1);
      mbar_init(&bars.empty[i], 1);
      mbar_init(&bars.keyed[i], 8);  // int8: the tile's scales
      mbar_init(&bars.scaled[i], 1);
    }
    for (int i = 0; i < C::RAWS; i++) {
      mbar_init(&bars.raw_full[i], 1);
      mbar_init(&bars.raw_empty[i], 8);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;");      // the next kernel may start; it waits for this grid's end
  asm volatile("griddepcontrol.wait;" ::: "memory");  // what the last kernels wrote is there, and what they read is free
  const uint32_t tmem = bars.tmem;
  if (warp < 16) {
    regs_inc<C::REG_SOFT>();
    softmax_role<D, INT8>(a, sm, bars);
  } else if (warp < 20) {
    regs_dec<C::REG_PROD>();
    if (warp == 16) {
      mma_role<D, INT8>(a, sm, bars);
    } else if (warp == 17) {
      tma_role<D, INT8>(&tq, &tk, &tv, a, sm, bars);
    } else if (INT8 && warp == 18) {
      if constexpr (INT8) scale_role<D>(a, sm, bars);
    }
  } else {
    if constexpr (INT8) {
      regs_dec<C::REG_CONV>();
      convert_role<D>(a, sm, bars);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

// Joins the parts of the items that CTA boundaries cut: block x belongs to the
// boundary before CTA x + 1 and takes the item if that boundary is its first.
// O = sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i. Up to 38 MB of parts, which the
// L2 holds; about 5 us behind the many-row kernel, 3 us behind the few-row one.
constexpr int kJoinThreads = 128;
// A part's sums lie [row][D] (few rows) or [D / 8][256 rows][8], as their writers' lanes run.
template <int D, bool FEW>
__global__ void __launch_bounds__(kJoinThreads) chunk_join_kernel(const __grid_constant__ ChunkArgs a) {
  constexpr int COLS = FEW ? 4 : 8, ACROSS = D / COLS, ROWS = kJoinThreads / ACROSS;  // columns of a thread, threads of a row
  const int c = (int)blockIdx.x + 1;
  const Start it = a.start[c], before = a.start[c - 1];
  auto same = [&](const Start &x) { return x.seq == it.seq && x.head == it.head && x.pair == it.pair && x.tile > 0; };
  if (it.tile == 0 || same(before)) return;
  const ChunkSeq s = a.seq[it.seq];
  const int tok0 = it.pair * 2 * a.sh.tpt, ntok = min(2 * a.sh.tpt, s.rows - tok0);
  const bool both = ntok > a.sh.tpt;
  const int rows = ntok * a.G;
  int last = c;  // CTAs c - 1 .. last hold parts
  while (last + 1 < a.n_ctas && same(a.start[last + 1])) last++;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x;
  const int col = FEW ? tid % ACROSS : tid / 8 % ACROSS, first = FEW ? tid / ACROSS : tid / (8 * ACROSS) * 8 + tid % 8;
  for (int r = (int)blockIdx.y * ROWS + first; r < rows; r += gridDim.y * ROWS) {
    // row r of the item in the scratch: the second tile starts at 128
    const int tile_rows = a.sh.tpt * a.G, prow = both && r >= tile_rows ? BM + r - tile_rows : r;
    auto part = [&](int x) { return a.ws + (size_t)(x * 2 + (x == c - 1 ? 1 : 0)) * (kRowsItem * (D + 2)); };
    const size_t at = FEW ? (size_t)prow * D + col * 4 : ((size_t)col * kRowsItem + prow) * 8;
    float m = -INFINITY, l = 0.f, o[COLS];
#pragma unroll
    for (int e = 0; e < COLS; e++) o[e] = 0.f;
    for (int x = c - 1; x <= last; x += 2) {  // two parts at a time are mostly all of them: every load before its first use
      float2 ml[2];
      float4 y[2][COLS / 4];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float *from = part(min(x + h, last));
        ml[h] = __ldcg(reinterpret_cast<const float2 *>(from + (size_t)kRowsItem * D) + prow);
#pragma unroll
        for (int e = 0; e < COLS / 4; e++) y[h][e] = __ldcg(reinterpret_cast<const float4 *>(from + at) + e);
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        if (x + h > last) break;
        const float top = fmaxf(m, ml[h].x);
        // without a maximum l and O are 0, or NaN
        const float f0 = m == -INFINITY ? 1.f : ex2(m - top), f1 = ml[h].x == -INFINITY ? 1.f : ex2(ml[h].x - top);
        m = top;
        l = fmaf(ml[h].y, f1, l * f0);
#pragma unroll
        for (int e = 0; e < COLS / 4; e++) {
          o[e * 4] = fmaf(y[h][e].x, f1, o[e * 4] * f0);
          o[e * 4 + 1] = fmaf(y[h][e].y, f1, o[e * 4 + 1] * f0);
          o[e * 4 + 2] = fmaf(y[h][e].z, f1, o[e * 4 + 2] * f0);
          o[e * 4 + 3] = fmaf(y[h][e].w, f1, o[e * 4 + 3] * f0);
        }
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int tok = tok0 + r / a.G;
    const size_t row = (size_t)(s.row0 + tok) * a.Hq + (size_t)it.head * a.G + r % a.G;
#pragma unroll
    for (int e = 0; e < COLS; e += 4)
      *reinterpret_cast<uint2 *>(a.out + row * D + col * COLS + e) =
          make_uint2(pack_bf16(o[e] * inv, o[e + 1] * inv), pack_bf16(o[e + 2] * inv, o[e + 3] * inv));
    if (col == 0 && a.lse) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
  }
}

// ------------------------------------------------------------------ host
using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn(vxb_ctx *ctx) {
  static std::mutex mu;
  static EncodeTiledFn fn = nullptr;
  std::lock_guard<std::mutex> lk(mu);
  if (!fn) {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess || !p) {
      cudaGetLastError();
      set_error(ctx, VXB_ECUDA, "vxb_chunk_attention: cuTensorMapEncodeTiled is not available from the driver");
      return nullptr;
    }
    fn = reinterpret_cast<EncodeTiledFn>(p);
  }
  return fn;
}

int encode(vxb_ctx *ctx, EncodeTiledFn fn, CUtensorMap *map, CUtensorMapDataType type, int rank, const void *base,
           const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box, CUtensorMapSwizzle swizzle) {
  const cuuint32_t one[3] = {1, 1, 1};
  const CUresult r = fn(map, type, (cuuint32_t)rank, const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return VXB_OK;
}

template <int D, bool INT8>
int launch_many(vxb_kv *kv, const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, const ChunkArgs &a, cudaStream_t st) {
  using C = Cfg<D, INT8>;
  static std::atomic<bool> configured[64];  // kernel attributes set on this device (zero-initialized)
  if (!configured[kv->ctx->device & 63]) {
    VXB_CUDA_TRY(kv->ctx, cudaFuncSetAttribute(chunk_attn_kernel<D, INT8>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    configured[kv->ctx->device & 63] = true;
  }
  return launch_early(kv->ctx, "chunk_attn_kernel", chunk_attn_kernel<D, INT8>, dim3((unsigned)a.n_ctas), C::THREADS, C::SMEM, st, q, k, v, a);
}

int launch_many(vxb_kv *kv, const ChunkArgs &a, int64_t rows, cudaStream_t st) {
  vxb_ctx *ctx = kv->ctx;
  const int D = kv->head_dim;
  const bool i8 = kv->dtype == VXB_I8;
  EncodeTiledFn fn = encode_fn(ctx);
  if (!fn) return VXB_ECUDA;
  CUtensorMap mq, mk, mv;
  {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)a.Hq, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)a.Hq * D * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)a.G, (cuuint32_t)a.sh.tpt};
    if (int rc = encode(ctx, fn, &mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, a.q, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  }
  for (int v = 0; v < 2; v++) {
    const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)kv->max_blocks * a.Hkv * a.bs};
    const cuuint64_t strides[1] = {(cuuint64_t)D * kv->elem_bytes};
    const cuuint32_t box[2] = {i8 ? (cuuint32_t)D : 64u, (cuuint32_t)a.box};
    if (int rc = encode(ctx, fn, v ? &mv : &mk, i8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                        v ? a.pool_v : a.pool_k, dims, strides, box, i8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B))
      return rc;
  }
  if (D == 128) return i8 ? launch_many<128, true>(kv, mq, mk, mv, a, st) : launch_many<128, false>(kv, mq, mk, mv, a, st);
  return i8 ? launch_many<64, true>(kv, mq, mk, mv, a, st) : launch_many<64, false>(kv, mq, mk, mv, a, st);
}

int launch_join(vxb_kv *kv, const ChunkArgs &a, bool few, int max_rows, cudaStream_t st) {
  const int rows = kJoinThreads / (kv->head_dim / (few ? 4 : 8));
  auto *kernel = kv->head_dim == 128 ? (few ? chunk_join_kernel<128, true> : chunk_join_kernel<128, false>)
                                     : (few ? chunk_join_kernel<64, true> : chunk_join_kernel<64, false>);
  return launch_early(kv->ctx, "chunk_join_kernel", kernel, dim3((unsigned)(a.n_ctas - 1), (unsigned)((max_rows + rows - 1) / rows)), kJoinThreads,
                      0, st, a);
}

int ctas_of(const vxb_ctx *ctx) {
  const int sms = ctx->num_sms > 0 ? ctx->num_sms : 148;
  return sms < kMaxCtas ? sms : kMaxCtas;
}

// Items in their order, whole, one or more to a CTA, none with more than `most`
// key tiles; false if that takes more than `ctas` CTAs.
// (units: of each sequence's pairs, one sequence after another)
bool whole_runs(ChunkArgs &a, const int *units, long long most, int ctas) {
  a.n_ctas = 0;
  long long sum = most;
  int pairs = 0;
  for (int sq = 0; sq < a.n; sq++, units += pairs) {
    pairs = (a.seq[sq].rows + 2 * a.sh.tpt - 1) / (2 * a.sh.tpt);
    for (int hd = 0; hd < a.Hkv; hd++)
      for (int pr = 0; pr < pairs; pr++) {
        const int w = units[pr];
        sum += w;
        if (sum > most) {
          if (a.n_ctas == ctas || w > most) return false;
          a.start[a.n_ctas++] = {sq, hd, pr, 0, 0};
          sum = w;
        }
        a.start[a.n_ctas - 1].units = (int32_t)sum;
      }
  }
  return true;
}

// Cuts the key tiles of a.seq[0 .. a.n) into one run per CTA; whether a cut
// falls inside an item. Equal runs cut items, and the cut ones' parts are
// written, read and joined by a second launch: where whole items make the
// longest run no more than `slack` key tiles longer, they stay whole. Measured
// with cuts and whole: few rows, 32 heads x 333 keys 8.7 and 7.5 us (2 tiles
// longer), 600 keys 10.7 and 9.2 (3 longer), int8 8 heads x 1000 keys 12.3 and
// 18.0 (7 longer); many rows, 2 x 32 heads x 700 of 1500 tokens 69.7 and 61.0,
// 8 x 4 heads x 1000 of 6000 104.7 and 99.2 (12 longer), 2 x 8 heads x 600 of
// 2048 at D 64 54 and 60 (12 longer).
constexpr int kSlackFew = 4, kSlackMany = 8;
int cut_runs(const vxb_ctx *ctx, ChunkArgs &a, int slack, bool *cut) {
  long long per_head[kSeqs], units = 0, items = 0;
  int largest = 0, known = 0, unit[4 * kMaxCtas];  // units of the first pairs
  for (int i = 0; i < a.n; i++) {
    per_head[i] = 0;
    const int pairs = (a.seq[i].rows + 2 * a.sh.tpt - 1) / (2 * a.sh.tpt);
    for (int p = 0; p < pairs; p++) {
      const int w = units_of(a.seq[i], a.sh, p);
      if (known < 4 * kMaxCtas) unit[known++] = w;
      per_head[i] += w;
      largest = w > largest ? w : largest;
    }
    units += per_head[i] * a.Hkv;
    items += (long long)pairs * a.Hkv;
  }
  const int ctas = ctas_of(ctx);
  *cut = false;
  if (items <= 4 * ctas) {
    const long long equal = (units + ctas - 1) / ctas;
    for (long long most = equal > largest ? equal : largest; most <= equal + slack; most++)
      if (whole_runs(a, unit, most, ctas)) return VXB_OK;
  }
  a.n_ctas = (int)(units < ctas ? units : ctas);
  if (units / a.n_ctas >= INT_MAX / 4) return VXB_EINVAL;
  int sq = 0, hd = 0, pr = 0;
  long long at = 0;  // first unit of (sq, hd, pr)
  for (int c = 0; c < a.n_ctas; c++) {
    const long long u = units * c / a.n_ctas;
    while (true) {
      if (pr == 0 && u - at >= per_head[sq]) {  // whole heads at a time
        const long long fit = (u - at) / per_head[sq], skip = fit < a.Hkv - hd ? fit : a.Hkv - hd;
        at += skip * per_head[sq];
        hd += (int)skip;
      } else {
        const int w = units_of(a.seq[sq], a.sh, pr);
        if (u - at < w) break;
        at += w;
        pr++;
        if (pr * 2 * a.sh.tpt >= a.seq[sq].rows) {
          pr = 0;
          hd++;
        }
      }
      if (hd == a.Hkv) {
        hd = 0;
        sq++;
      }
    }
    a.start[c] = {sq, hd, pr, (int32_t)(u - at), (int32_t)(units * (c + 1) / a.n_ctas - u)};
    *cut |= u > at;
  }
  return VXB_OK;
}

int chunk_attention(vxb_kv *kv, int layer, int n, const int64_t *ids, const int32_t *counts, const uint16_t *d_q, int Hq,
                    float scale, int causal, uint16_t *d_out, float *d_lse, float *ws, cudaStream_t st) {
  vxb_ctx *ctx = kv->ctx;
  const int Hkv = kv->num_kv_heads, bs = kv->block_size;
  int64_t total = 0;
  for (int i = 0; i < n; i++) {
    if (counts[i] < 0) return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: sequence %lld has %d queries", (long long)ids[i], counts[i]);
    total += counts[i];
  }
  if (total > INT_MAX - kRowsItem) return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: %lld rows", (long long)total);
  if (total == 0) return VXB_OK;
  if (!d_q || !d_out || ((uintptr_t)d_q | (uintptr_t)d_out) % 16)
    return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: d_q and d_out must be 16-byte aligned device pointers");
  if ((int64_t)kv->max_blocks * Hkv * bs > INT_MAX)  // token rows of the pool are counted in 32 bits
    return set_error(ctx, VXB_EUNSUPPORTED, "vxb_chunk_attention: a pool of more than 2^31 token rows");
  ChunkArgs a;
  a.q = d_q;
  a.pool_k = kv->pool_k;
  a.pool_v = kv->pool_v;
  a.out = d_out;
  a.lse = d_lse;
  a.ws = ws;
  a.err = ctx->d_err;
  a.sk = kv->scale_k;
  a.sv = kv->scale_v;
  a.tables = kv->d_tables + (size_t)layer * kv->max_seqs * kv->max_blocks_per_seq;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.bs = bs;
  a.mbps = kv->max_blocks_per_seq;
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.box = bs % 128 == 0 ? 128 : bs % 64 == 0 ? 64 : bs % 32 == 0 ? 32 : 16;  // tokens of a page copy: within a block
  // Chunks of few rows and the others go to a kernel each; a few of the former
  // beside the latter stay with them (a launch of its own has a fixed part of
  // about 8 us, and leaves most SMs idle when it has few tiles).
  auto is_few = [&](int i) { return (int64_t)counts[i] * a.G <= kFewRows; };
  std::vector<int> lens(n, 0);
  bool all_few = true;
  int64_t few_tiles = 0;
  TableFinder find(kv, layer);
  for (int i = 0; i < n; i++) {
    if (counts[i] == 0) continue;
    auto it = find(ids[i]);
    if (it != kv->tables.end()) lens[i] = (int)it->second.len;
    if (is_few(i)) few_tiles += (int64_t)(lens[i] + BN - 1) / BN * Hkv;
    else all_few = false;
  }
  const bool together = !all_few && few_tiles < 8 * ctas_of(ctx);
  for (int few = 0; few < 2; few++) {
    a.sh = {few ? kFewRows : BM / a.G, causal != 0};
    int row = 0;
    for (int i = 0; i < n;) {
      a.n = 0;
      int max_rows = 0;
      for (; i < n && a.n < kSeqs; i++) {
        const int at = row;
        row += counts[i];
        if (counts[i] == 0 || (!together && is_few(i)) != (few == 1)) continue;
        a.seq[a.n++] = {lens[i] > 0 ? kv->slot_of.at(ids[i]) : 0, at, counts[i], lens[i]};
        max_rows = max_rows > counts[i] ? max_rows : counts[i];
      }
      if (a.n == 0) continue;
      bool cut = false;
      if (cut_runs(ctx, a, few ? kSlackFew : kSlackMany, &cut)) return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: too much work for one call");
      max_rows = (max_rows < 2 * a.sh.tpt ? max_rows : 2 * a.sh.tpt) * a.G;
      if (int rc = few ? launch_few(kv, a, max_rows, st) : launch_many(kv, a, total, st)) return rc;
      if (cut)
        if (int rc = launch_join(kv, a, few, max_rows, st)) return rc;
    }
  }
  return VXB_OK;
}

int check_heads(const vxb_kv *kv, int Hq) {
  if (Hq <= 0 || Hq % kv->num_kv_heads || Hq / kv->num_kv_heads > 128)
    return set_error(kv->ctx, VXB_EINVAL, "vxb_chunk_attention: num_q_heads %d must be a multiple (<= 128x) of the %d kv heads", Hq,
                     kv->num_kv_heads);
  return VXB_OK;
}

}  // namespace

VXB_API int vxb_chunk_attention_ws(const vxb_kv *kv, int num_q_heads, size_t *ws_bytes) {
  if (!kv || !kv->ctx) return set_error(nullptr, VXB_EINVAL, "vxb_chunk_attention_ws: null cache");
  if (!ws_bytes) return set_error(kv->ctx, VXB_EINVAL, "vxb_chunk_attention_ws: null output");
  if (int rc = check_heads(kv, num_q_heads)) return rc;
  *ws_bytes = (size_t)2 * ctas_of(kv->ctx) * part_floats(kv->head_dim) * sizeof(float);
  return VXB_OK;
}

VXB_API int vxb_chunk_attention(vxb_kv *kv, int layer, int n, const int64_t *h_seq_ids, const int32_t *h_n_queries,
                                const uint16_t *d_q, int num_q_heads, float softmax_scale, int causal, uint16_t *d_out,
                                float *d_lse, void *d_ws, size_t ws_bytes, void *stream) {
  if (!kv || !kv->ctx) return set_error(nullptr, VXB_EINVAL, "vxb_chunk_attention: null cache");
  vxb_ctx *ctx = kv->ctx;
  if (layer < 0 || layer >= kv->num_layers) return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: layer %d out of range", layer);
  if (n < 0 || (n > 0 && (!h_seq_ids || !h_n_queries))) return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: bad arguments");
  if (!(softmax_scale > 0.f) || std::isinf(softmax_scale * 1.44269504088896340736f))  // (times log2 e: as the kernels use it)
    return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: scale must be positive and finite");
  size_t need = 0;
  if (int rc = vxb_chunk_attention_ws(kv, num_q_heads, &need)) return rc;
  if (n == 0) return VXB_OK;
  if (!d_ws || (uintptr_t)d_ws % 16 || ws_bytes < need)
    return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: %zu bytes of 16-byte aligned scratch needed, %zu given", need, d_ws ? ws_bytes : 0);
  DeviceScope dev(ctx);
  if (dev.rc) return dev.rc;
  try {
    return chunk_attention(kv, layer, n, h_seq_ids, h_n_queries, d_q, num_q_heads, softmax_scale, causal, d_out, d_lse, (float *)d_ws,
                           (cudaStream_t)stream);
  } catch (...) {
    return set_error(ctx, VXB_ENOMEM, "vxb_chunk_attention: out of host memory");
  }
}
