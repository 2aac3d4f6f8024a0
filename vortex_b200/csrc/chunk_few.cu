// Chunk attention for few rows: the drafted tokens of a request, up to 64 rows
// (tokens x query heads of a kv head). Bound by reading the cache once, so the
// keys take the tensor core's 128 rows and the queries its N = 16, 32 or 64
// columns:
//
//   S^T = K Q^T         A = the K tile, B = the query rows
//   P^T = 2^(S^T - m)   thread = key and some of the rows
//   O^T += V^T P^T      A = the V tile read MN-major, B = P from shared memory
//
// With the queries as rows (chunk_attn.cu) a tile costs 128 exponentials per
// lane however few rows are live; here it costs N, and a per-key scale (int8)
// is one register of the key's thread. The reference maximum m of a row moves
// only when a score passes it by 2^8, so a tile needs one vote of the
// warpgroup and no reduction; l is summed per thread and reduced at the end.
//
// Loader warps bring tiles of 128 keys into two rings, one of K and one of V
// (K is used up as soon as its S is done, three tiles ahead of V): bf16 rows
// with cp.async (a 16-token page is only 4 KB: as many TMA boxes reach 5.6
// TB/s, 16-byte copies the memory rate), int8 rows by cp.async into a place of
// the thread that then converts them, K to bf16 and V to f16 (codes are exact
// in both). Rows behind the last token become zeros. Two warpgroups take the
// softmax of up to 32 rows, four of more (int8, 64 rows: 295 and 262 us then).
//
// int8 weights carry the V scale, w = p * scale, with the reference maximum
// taken over log2(w), and go into P as f16 times 2^6: off by 2^-11 at most, and
// weights down to 2^-30 of the row's largest keep at least one bit. bf16 P is off
// by 2^-8 (the type of V decides; decode attention keeps a second part of P). A
// value row of zeros counts for the sum alone (chunk_attn.h): its key's thread
// keeps it out of the reference. A row takes its reference from its first tile
// with a finite score (kUnset).
//
// Values of V that only some rows may see and that are not finite are taken
// out of the tile and added to the rows that see them, as in chunk_attn.cu.
//
// Measured: 32 x 32 heads, ctx 2k, 4 rows 162 us (6.6 TB/s); 32 x 8 heads, ctx
// 8k, 24 rows 164 us (6.6 TB/s), 64 rows 176, int8 16 rows 161 (3.4 TB/s), 64
// rows 229; heads of 64, ctx 8k, 16 rows 93 us (5.7 TB/s), 64 rows 146, int8 131
// and 188; 32 heads, 333 keys, 4 rows 6.6 us. bf16 tiles of 128 columns wait for
// memory. int8 halves the bytes and fills 61% of the issue slots with conversions
// and softmax; tiles of 64 columns wait for the chain vote, exponentials, P to
// shared memory, announcement (up to 1.3 us a tile against 0.75 us of memory).
// Looking for value rows of zeros and scales far apart costs int8 1 to 3%, heads
// of 64 and launches of 32 rows 3 to 6%; a row of zeros in every tile 30 to 40%.
#include <atomic>
#include <climits>
#include <cmath>
#include <cuda_fp16.h>
#include <type_traits>

#include "chunk_attn.h"

using namespace vxb;
using namespace vxb::tc;
using namespace vxb::chunk;

namespace {

template <int D, bool INT8, int NR>
struct Cfg {
  static constexpr int SLAB = BN * 128;         // 64 columns of 128 keys
  static constexpr int TILE = SLAB * (D / 64);
  static constexpr int AHEAD = 3;               // tiles whose S may be computed before the oldest one's P is there
  // int8: tiles of codes on their way, in shared memory of the thread that will
  // convert them (RAWS each of K and V; K's bring the scales of both)
  static constexpr int RAWS = INT8 ? 2 : 0, RAW_V = BN * D, RAW_K = RAW_V + BN * 8;
  // ring slots of K and of V
  static constexpr int KS = D == 64 ? (INT8 ? 4 : 5) : INT8 ? (NR == 64 ? 1 : 2) : NR == 64 ? 2 : 3;
  static constexpr int VS = D == 64 ? (INT8 ? 4 : 5) : INT8 ? 2 : 3;
  static constexpr int QBUFS = INT8 && D == 128 && NR > 16 ? 1 : 2;
  static constexpr int Q = NR * D * 2, P = NR * BN * 2;
  static constexpr int OFF_V = KS * TILE, OFF_Q = OFF_V + VS * TILE;
  static constexpr int OFF_P = OFF_Q + QBUFS * Q;  // two tiles
  static constexpr int OFF_RAW = OFF_P + 2 * P;
  static constexpr int OFF_SCALE = OFF_RAW + RAWS * (RAW_K + RAW_V);
  // Tiles whose K and V scales are kept: K of tile t is written when S of tile
  // t - KS is done, for which the softmax of the tile AHEAD before it is.
  static constexpr int SCALES = INT8 ? AHEAD + KS : 0;
  static constexpr int OFF_RED = OFF_SCALE + SCALES * 2 * BN * 4;  // per-warp results and per-row values of the softmax
  static constexpr int PER_ROW = INT8 ? 15 : 7;
  static constexpr int OFF_BARS = OFF_RED + PER_ROW * NR * 4;
  static constexpr int SMEM = OFF_BARS + 320;
  // Warpgroups: SOFT of softmax (up to 16 rows each), PER_SLOT each that load K
  // and V (int8 converts as it loads), one with the MMA and Q warps; registers
  // at launch and of each.
  static constexpr int SOFT = NR == 64 ? 4 : 2, PER_SLOT = INT8 && NR < 64 ? 2 : 1;
  static constexpr int THREADS = (SOFT + 2 * PER_SLOT + 1) * 128, REGS = THREADS == 640 ? 96 : 72;
  static constexpr int REG_SOFT = NR == 64 ? 72 : 96, REG_LOAD = NR == 64 ? 80 : INT8 ? 64 : 96, REG_MMA = 56;
  static_assert(SOFT * REG_SOFT + 2 * PER_SLOT * REG_LOAD + REG_MMA <= THREADS / 128 * REGS, "registers");
  static constexpr int COLS = (AHEAD + 2) * NR <= 128 ? 128 : (AHEAD + 2) * NR <= 256 ? 256 : 512;  // TMEM: S x AHEAD, O, O
  static_assert(SMEM <= 232448, "shared memory");
};

template <int KS, int VS>
struct Bars {
  uint64_t k_full[KS], k_empty[KS], v_full[VS], v_empty[VS], q_full[2], q_empty[2], s_full[3], p_full[2], pv_done[2], o_full[2], o_free[2], drained;
  uint32_t tmem;
  int acc;  // O already holds values that the piece's first product adds to
};
template <int D, bool INT8, int NR>
using BarsOf = Bars<Cfg<D, INT8, NR>::KS, Cfg<D, INT8, NR>::VS>;

// A ring's next slot, and how often it has gone around.
template <int SLOTS>
struct Ring {
  uint32_t slot = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == SLOTS) {
      slot = 0;
      phase ^= 1;
    }
  }
};

// 16-byte chunk c of row r of a tile, 128-byte swizzle
__device__ __forceinline__ uint32_t chunk_off(int r, int c) {
  return (uint32_t)((c >> 3) * (BN * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Instruction descriptor of kind::f16 with f32 sums: M = 128, N columns, B
// K-major, A K- or MN-major, both f16 or both bf16.
__host__ __device__ constexpr uint32_t idesc(int N, bool a_mn_major, bool f16) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | ((a_mn_major ? 1u : 0u) << 15) | ((uint32_t)(N >> 3) << 17) | (8u << 24);
}

// Column of a query row, or of V, that 16-byte chunk c of a tile's row holds.
// int8 rows of 128: a lane converts 16 codes, and its two chunks go to the same
// place of the two slabs (neighbouring chunks of one row would meet in the
// same banks), so the head dimension is permuted alike in Q, K, V and O.
template <int D, bool INT8>
__device__ __forceinline__ int chunk_of(int c) {
  return INT8 && D == 128 ? (c & 7) * 2 + (c >> 3) : c;
}

// Sums of each of N values over the lanes: lane i gets that of value i / (32 / N) in v[0].
template <int N, int OFF>
__device__ __forceinline__ void halve(float *v, int lane) {
  if constexpr (OFF > 0) {
    if constexpr (N > 1) {
      const bool up = (lane & OFF) != 0;
#pragma unroll
      for (int n = 0; n < N / 2; n++) {
        const float send = up ? v[n] : v[n + N / 2];
        v[n] = (up ? v[n + N / 2] : v[n]) + __shfl_xor_sync(0xffffffffu, send, OFF);
      }
      halve<N / 2, OFF / 2>(v, lane);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], OFF);
      halve<1, OFF / 2>(v, lane);
    }
  }
}

// Negated reference of a row that has seen no finite score yet: the first one
// passes it, and the vote for new references is called. The exponents of that
// tile were formed with it and have lost the score's last bits. bf16 forms them
// anew behind every vote (1% of a call for heads of 64). In int8 that, or a branch
// to it, took 3 to 9% of a call: there the unit is less far away, so that the
// weights of that one tile are off by 2^-14 ln 2 at most (f16 rounds at 2^-11),
// and scores are told from none down to -700 (nats).
template <bool INT8>
constexpr float kUnset = INT8 ? 1024.f : 1048576.f;

// int8: a tile's scores alone, added to each row's maximum and sum of 2^(score -
// maximum) over the warp's keys. Rare (kFarLog2): a function of its own leaves the
// softmax its registers. Row e of group j is row first + j * step + e of the item,
// its scores in column j * step + e.
__device__ __noinline__ void far_rows(uint32_t tS, int groups, int step, int first, float sc, int n_min, float *top, float *sum) {
#pragma unroll 1
  for (int j = 0; j < groups; j++)
#pragma unroll 1
    for (int e = 0; e < 8; e++) {
      const int n = j * 8 + e;
      const float s = tmem_ld1(tS + j * step + e);
      const bool sees = first + j * step + e >= n_min;
      float most;
      asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(most) : "f"(sees ? s * sc : -INFINITY));
      const float before = top[n], m = fmaxf(before, most), ref = m == -INFINITY ? 0.f : m;
      const float w = warp_sum(sees ? ex2(fmaf(s, sc, -ref)) : 0.f);
      __syncwarp();
      if ((threadIdx.x & 31) == 0) {
        sum[n] = (before == -INFINITY ? sum[n] : sum[n] * ex2(before - m)) + w;
        top[n] = m;
      }
      __syncwarp();
    }
}

// A key's row of the V tile is zero. Rare (only scale 1 can be such a row).
template <int D>
__device__ __noinline__ bool zero_row(const uint8_t *tile, int key) {
  for (int c = 0; c < D / 8; c++) {
    const uint4 x = *reinterpret_cast<const uint4 *>(tile + chunk_off(key, c));
    if (x.x | x.y | x.z | x.w) return false;
  }
  return true;
}

// ------------------------------------------------------------------ softmax: thread = (key, the warpgroup's rows)
// Rows go to the warpgroups in groups of eight in turn; groups without a live
// row are passed over.
template <int D, bool INT8, int NR>
__device__ __forceinline__ void softmax_role(const ChunkArgs &a, uint8_t *sm, BarsOf<D, INT8, NR> &bars) {
  using C = Cfg<D, INT8, NR>;
  constexpr int W = C::SOFT, N = NR / W, GROUPS = N / 8;  // warpgroups; rows of this one
  constexpr float SHIFT = INT8 ? 6.f : 0.f;  // P (and l) hold 2^SHIFT times the weights
  const int wg = threadIdx.x >> 7, key = threadIdx.x & 127, warp = key >> 5, lane = key & 31;
  const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
  // row n of the warpgroup's N is row row_of(n) of the item
  auto row_of = [&](int n) { return ((n >> 3) * W + wg) * 8 + (n & 7); };
  // this warpgroup's: per-warp results [4][N]; per row the negated reference, a factor, a change of the reference
  float *red = reinterpret_cast<float *>(sm + C::OFF_RED) + wg * C::PER_ROW * N, *ref_s = red + 4 * N, *f_s = ref_s + N, *d_s = f_s + N;
  float *far_top = d_s + N, *far_sum = far_top + 4 * N;  // int8: of each warp, see far_rows
  const float *scales = reinterpret_cast<const float *>(sm + C::OFF_SCALE);
  const int bar = 1 + wg;
  Waiter wait{a.err};
  Run run(a);
  Piece p{};
  uint32_t g = 0, pieces = 0;  // tiles and pieces so far
  if (key < N) ref_s[key] = 0.f;
  bar_sync(bar, 128);
  while (run.next(a, p)) {
    const int T = max(0, p.te - p.tb), live = p.ntok * a.G;
    const int groups = live > wg * 8 ? (live - wg * 8 + W * 8 - 1) / (W * 8) : 0;  // of this warpgroup's, with a live row
    const int base = p.s.len - p.s.rows + p.tok0;  // last key that the first token sees
    const uint32_t tO = bars.tmem + lane_off + (C::AHEAD + (pieces & 1)) * NR + wg * 8;
    float l[N];
#pragma unroll
    for (int n = 0; n < N; n++) l[n] = 0.f;
    auto own_sums = [&]() {  // int8: the sums so far become each warp's own (far_rows)
      halve<N, 16>(l, lane);
      if (lane % (32 / N) == 0) {
        const int n = lane / (32 / N);
        far_top[warp * N + n] = l[0] == 0.f ? -INFINITY : -ref_s[n] - SHIFT;
        far_sum[warp * N + n] = l[0];
      }
      __syncwarp();
    };
    bool own = false;  // int8: the sums have maxima of their own (far_rows)
    for (int t = 0; t < T; t++, g++) {
      const int k0 = (p.tb + t) * BN, k = k0 + key;
      const uint32_t tS = bars.tmem + lane_off + (g % C::AHEAD) * NR + wg * 8;
      wait(&bars.s_full[g % C::AHEAD], (g / C::AHEAD) & 1);
      tc_fence_after();
      // the first row that sees this thread's key
      const int n_min = k >= p.s.len ? INT_MAX : a.sh.causal && k > base ? (k - base) * a.G : 0;
      const bool masked = k0 + BN > p.s.len || (a.sh.causal && k0 + BN - 1 > base);
      float sc = a.scale_log2, add = SHIFT, isv = 1.f;
      bool far_key = false, zero = false;  // zero: the key's value row is
      if constexpr (INT8) {
        const float *tile = scales + g % C::SCALES * 2 * BN;
        sc *= tile[key];
        const float sv = tile[BN + key] < kLeastScale ? kLeastScale : tile[BN + key];
        if (__any_sync(0xffffffffu, sv == 1.f && k < p.s.len)) {
          wait(&bars.v_full[g % C::VS], (g / C::VS) & 1);
          zero = sv == 1.f && zero_row<D>(sm + C::OFF_V + g % C::VS * C::TILE, key);
          __syncwarp();
        }
        const float lv = __log2f(sv);  // off by under 2^-16, in V's factor alone
        add += lv;
        isv = ex2(-lv);
        far_key = !(fabsf(lv) <= kFarLog2);
      }
      float x[N];  // log2 of what goes into P
      // (the usual case of only live groups has code without their branches,
      // which keep the rows' chains apart)
      float top = -INFINITY;
      auto load = [&](auto all) {
#pragma unroll
        for (int j = 0; j < GROUPS; j++)
          if (decltype(all)::value || j < groups) tmem_ld8(tS + j * W * 8, *reinterpret_cast<float(*)[8]>(x + j * 8));
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < GROUPS; j++)
          if (decltype(all)::value || j < groups) {
#pragma unroll
            for (int n = j * 8; n < j * 8 + 8; n += 4) {
              const float4 r4 = *reinterpret_cast<const float4 *>(ref_s + n);
              const float ref[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
              for (int e = 0; e < 4; e++) x[n + e] = fmaf(x[n + e], sc, INT8 ? add + ref[e] : ref[e]);
            }
            if (masked) {
#pragma unroll
              for (int n = j * 8; n < j * 8 + 8; n++) x[n] = row_of(n) >= n_min ? x[n] : -INFINITY;
            }
#pragma unroll
            for (int n = j * 8; n < j * 8 + 8; n++) top = fmaxf(top, x[n]);
          }
      };
      if (groups == GROUPS) load(std::true_type{});
      else load(std::false_type{});
      if (INT8 && zero) {  // (w is p then: its share of the sum)
        far_key = top > kMostShareLog2;
        top = -INFINITY;
      }
      if (t == 0 || bar_or(bar, 128, top > RESCALE_THRESHOLD + SHIFT || far_key)) {
        bool odd = false;  // a key to look at
        if constexpr (INT8) {
          odd = bar_or(bar, 128, far_key || zero);
          if (odd && bar_or(bar, 128, far_key) && !own) {
            own_sums();
            own = true;
          }
        }
        // New references: a first tile's maximum, later the maximum of the rows
        // that passed it, becomes 2^SHIFT.
        float most = -INFINITY;
#pragma unroll
        for (int j = 0; j < GROUPS; j++)
          if (j < groups) {
#pragma unroll
            for (int n = j * 8; n < j * 8 + 8; n++) {
              float y;
              asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(INT8 && zero ? -INFINITY : x[n]));
              most = lane == n ? y : most;
            }
          }
        if (lane < N) red[warp * N + lane] = most;
        bar_sync(bar, 128);
        if (key < N) {
          const float m = fmaxf(fmaxf(red[key], red[N + key]), fmaxf(red[2 * N + key], red[3 * N + key]));
          const float d = t == 0 ? (m > -INFINITY ? SHIFT - m : kUnset<INT8>) : fminf(SHIFT - m, 0.f);
          ref_s[key] += d;
          d_s[key] = d;
          f_s[key] = ex2(d);
        }
        bar_sync(bar, 128);
        if constexpr (INT8) {
#pragma unroll
          for (int n = 0; n < N; n++) x[n] += d_s[n];
        } else {
          load(std::false_type{});
        }
        if (t > 0) {
          wait(&bars.pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1);
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < GROUPS; j++)
            if (j < groups) {
              float o[8];
              tmem_ld8(tO + j * W * 8, o);
              tmem_wait_ld();
#pragma unroll
              for (int n = 0; n < 8; n++) {
                const float f = f_s[j * 8 + n];
                o[n] *= f;
                l[j * 8 + n] *= f;
              }
              tmem_st8(tO + j * W * 8, o);
            }
          tmem_wait_st();
        }
        if (INT8 && odd && !own) {  // a row of zeros whose share of the sum is too large in the new unit
          float share = -INFINITY;
#pragma unroll
          for (int n = 0; n < N; n++) share = n / 8 < groups ? fmaxf(share, x[n]) : share;
          if (bar_or(bar, 128, zero && share > kMostShareLog2)) {
            own_sums();
            own = true;
          }
        }
      }
      // P of two tiles ago has been used
      uint8_t *P = sm + C::OFF_P + (g & 1) * C::P;
      if (g >= 2) wait(&bars.pv_done[g & 1], ((g - 2) >> 1) & 1);
      uint8_t *prow = P + (key >> 6) * (NR * 128) + wg * 8 * 128 + (key & 7) * 2;
      const uint32_t chunk = (uint32_t)(key & 63) >> 3;
      if (INT8 && own) {
        far_rows(tS, groups, W * 8, wg * 8, sc, n_min, far_top + warp * N, far_sum + warp * N);
        isv = 0.f;
      }
      auto weights = [&](auto all) {
#pragma unroll
        for (int j = 0; j < GROUPS; j++)
          if (decltype(all)::value || j < groups) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const int n = j * 8 + e;
              const float w0 = ex2(x[n]), w1 = ex2(x[n + 1]);
              uint32_t pair;
              if constexpr (INT8) {
                // a row without this key: no product with a scale that is not finite
                l[n] = !masked || row_of(n) >= n_min ? fmaf(w0, isv, l[n]) : l[n];
                l[n + 1] = !masked || row_of(n + 1) >= n_min ? fmaf(w1, isv, l[n + 1]) : l[n + 1];
                // (finite beside a row of zeros, whose weight has no bound)
                asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(pair) : "f"(w1), "f"(w0));
              } else {
                l[n] += w0;
                l[n + 1] += w1;
                pair = pack_bf16(w0, w1);
              }
              *reinterpret_cast<uint16_t *>(prow + j * W * 1024 + e * 128 + ((chunk ^ e) << 4)) = (uint16_t)pair;
              *reinterpret_cast<uint16_t *>(prow + j * W * 1024 + (e + 1) * 128 + ((chunk ^ (e + 1)) << 4)) = (uint16_t)(pair >> 16);
            }
          }
      };
      if (groups == GROUPS) weights(std::true_type{});
      else weights(std::false_type{});
      if constexpr (!INT8) {
        const int valid = min(BN, p.s.len - k0), hidden = a.sh.causal ? max(0, base + 1 - k0) : valid;
        if (hidden < valid) {  // some row does not see the keys from here on
          wait(&bars.v_full[g % C::VS], (g / C::VS) & 1);
          uint8_t *V = sm + C::OFF_V + (g % C::VS) * C::TILE;
          uint32_t found = 0;
          for (int c = hidden * (D / 8) + (int)threadIdx.x; c < valid * (D / 8); c += W * 128)
            found = add_odd(found, *reinterpret_cast<const uint4 *>(V + chunk_off(c / (D / 8), c % (D / 8))));
          __syncwarp();
          if (bar_or(W + 1, W * 128, odd_bf16(found) != 0)) {
            // rare: lane d of O^T takes every non-finite value of column d of V
            if (t > 0) {
              wait(&bars.pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1);
              tc_fence_after();
            } else {
              const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
              for (int j = 0; j < GROUPS; j++) tmem_st8(tO + j * W * 8, z);
              tmem_wait_st();
              if (threadIdx.x == 0) bars.acc = 1;
            }
            const int d = key % D;
            for (int i = hidden; i < valid; i++) {
              const uint32_t bits = *reinterpret_cast<const uint16_t *>(V + chunk_off(i, d >> 3) + (d & 7) * 2);
              const bool odd = (bits & 0x7F80u) == 0x7F80u;
              if (!__any_sync(0xffffffffu, odd)) continue;
              const int first = k0 + i > base ? (k0 + i - base) * a.G : 0;
              for (int n = 0; n < groups * 8; n++) {
                const int r = row_of(n);
                if (r < first) continue;
                const uint32_t off = (uint32_t)(i >> 6) * (NR * 128) + (uint32_t)r * 128 + ((((uint32_t)(i & 63) >> 3) ^ ((uint32_t)n & 7)) << 4) + (i & 7) * 2;
                const float w = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t *>(P + off) << 16);
                const uint32_t at = tO + (n >> 3) * W * 8 + (n & 7);
                const float o = tmem_ld1(at);
                tmem_st1(at, odd ? fmaf(w, __uint_as_float(bits << 16), o) : o);
                tmem_wait_st();
              }
            }
            bar_sync(W + 1, W * 128);
            for (int c = hidden * (D / 8) + (int)threadIdx.x; c < valid * (D / 8); c += W * 128) {
              uint4 *at = reinterpret_cast<uint4 *>(V + chunk_off(c / (D / 8), c % (D / 8)));
              *at = make_uint4(even_bf16(at->x), even_bf16(at->y), even_bf16(at->z), even_bf16(at->w));
            }
          }
        }
      }
      fence_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.p_full[g & 1]);
    }
    // ---------------- end of the piece (its code runs once a piece: kept short,
    // since it comes from beyond the instruction cache)
    bar_sync(bar, 128);  // red is free
    {
      // l of every row over the lanes: halves are exchanged until a lane has one row
      halve<N, 16>(l, lane);
      if (lane % (32 / N) == 0) red[warp * N + lane / (32 / N)] = l[0];
    }
    bar_sync(bar, 128);
    const bool whole = p.whole();
    float *part = a.ws + (size_t)(blockIdx.x * 2 + (p.tb > 0 ? 0 : 1)) * (kRowsItem * (D + 2));
    const size_t row0 = (size_t)(p.s.row0 + p.tok0) * a.Hq + (size_t)p.head * a.G;
    if (key < N) {
      float L = red[key] + red[N + key] + red[2 * N + key] + red[3 * N + key];
      const float unit = -ref_s[key] - SHIFT;  // of O (log2)
      float m = L == 0.f ? -INFINITY : unit, f = whole ? (L == 0.f ? 0.f : 1.f / L) : 1.f;
      if (INT8 && own) {
        // O and the sum have units of their own: O is divided by the sum here,
        // also in a part, whose sum then is 1
        const float *tops = far_top + key, *sums = far_sum + key;
        const float top = fmaxf(fmaxf(tops[0], tops[N]), fmaxf(tops[2 * N], tops[3 * N]));
        L = 0.f;
        for (int w = 0; w < 4; w++) L += tops[w * N] == -INFINITY ? sums[w * N] : sums[w * N] * ex2(tops[w * N] - top);
        f = L > 0.f ? ex2(unit - top) / L : L;
        m = top;
        if (!whole) {
          m = L > 0.f ? top + log2f(L) : -INFINITY;
          L = L > 0.f ? 1.f : L;
        }
      }
      f_s[key] = f;
      ref_s[key] = 0.f;
      const int r = row_of(key);
      if (r < live) {
        if (!whole) __stcg(reinterpret_cast<float2 *>(part + (size_t)kRowsItem * D) + r, make_float2(m, L));
        else if (a.lse) a.lse[row0 + (size_t)(r / a.G) * a.Hq + r % a.G] = (m + log2f(L)) * 0.69314718055994531f;
      }
    }
    bar_sync(bar, 128);
    wait(&bars.o_full[pieces & 1], (pieces >> 1) & 1);
    tc_fence_after();
    const int d = key < D ? chunk_of<D, INT8>(key >> 3) * 8 + (key & 7) : 0;
#pragma unroll 1
    for (int j = 0; j < groups; j++) {
      float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (T > 0) {
        tmem_ld8(tO + j * W * 8, o);
        tmem_wait_ld();
      }
      const int r0 = (j * W + wg) * 8, count = key < D ? live - r0 : 0;
      const float *f8 = f_s + j * 8;
      if (whole) {
        int h = r0 % a.G;
        uint16_t *to = a.out + (row0 + (size_t)(r0 / a.G) * a.Hq + h) * D + d;
        const size_t over = (size_t)(a.Hq - a.G) * D;  // from a token's last head of the group to the next token's first
#pragma unroll
        for (int e = 0; e < 8; e++) {
          if (e < count) *to = (uint16_t)pack_bf16(o[e] * f8[e], 0.f);
          to += D;
          if (++h == a.G) {
            h = 0;
            to += over;
          }
        }
      } else {
        float *to = part + (size_t)r0 * D + d;
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (e < count) __stcg(to + e * D, INT8 ? o[e] * f8[e] : o[e]);
      }
      __syncwarp();
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars.o_free[pieces & 1]);
    pieces++;
  }
}

// ------------------------------------------------------------------ MMA warp
template <int D, bool INT8, int NR>
__device__ __forceinline__ void mma_role(const ChunkArgs &a, uint8_t *sm, BarsOf<D, INT8, NR> &bars) {
  using C = Cfg<D, INT8, NR>;
  constexpr uint64_t KMAJOR = desc_base(16, 1024);
  // heads of 64: the second 64 rows of A are the first again, and are not read back
  constexpr uint64_t VMAJOR = desc_base(D == 128 ? C::SLAB : 0, 1024);
  const uint32_t s_k = smem_u32(sm) >> 4, s_v = smem_u32(sm + C::OFF_V) >> 4, s_q = smem_u32(sm + C::OFF_Q) >> 4, s_p = smem_u32(sm + C::OFF_P) >> 4;
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars.tmem, 0);
  const uint32_t one = elect_one();
  Waiter wait{a.err};
  Run run(a);
  Piece p{};
  uint32_t g = 0, pieces = 0;
  Ring<C::KS> kr;
  Ring<C::VS> vr;
  uint32_t s_buf = 0;  // S of the next tile
  auto filled = [&](uint64_t *full, uint32_t phase) {
    wait(full, phase);
    fence_async_smem();  // the loaders' cp.async (bf16) are announced without one
    tc_fence_after();
  };
  while (run.next(a, p)) {
    const int T = max(0, p.te - p.tb);
    const uint32_t pb = pieces & 1, qb = pieces % C::QBUFS;
    const int cols = (p.ntok * a.G + 15) / 16 * 16;  // of the NR, those with live rows
    const uint32_t id_s = idesc(cols, false, false), id_o = idesc(cols, true, INT8);
    const uint64_t q = KMAJOR + (s_q + qb * (C::Q >> 4));
    const uint32_t t_o = tmem + (C::AHEAD + pb) * NR;
    wait(&bars.q_full[qb], (pieces / C::QBUFS) & 1);
    auto issue_s = [&]() {
      filled(&bars.k_full[kr.slot], kr.phase);
      const uint64_t k = KMAJOR + (s_k + kr.slot * (C::TILE >> 4));
#pragma unroll
      for (int x = 0; x < D / 16; x++)
        mma_ss(one, tmem + s_buf * NR, k + (((x >> 2) * C::SLAB + (x & 3) * 32) >> 4), q + (((x >> 2) * (NR * 128) + (x & 3) * 32) >> 4), id_s,
               x > 0 ? 1u : 0u);
      mma_commit(one, &bars.s_full[s_buf]);
      mma_commit(one, &bars.k_empty[kr.slot]);
      kr.next();
      s_buf = s_buf + 1 == C::AHEAD ? 0 : s_buf + 1;
    };
    for (int t = 0; t < C::AHEAD && t < T; t++) issue_s();
    if (pieces >= 2) wait(&bars.o_free[pb], ((pieces >> 1) - 1) & 1);
    for (int t = 0; t < T; t++, g++) {
      const uint32_t buf = g & 1;
      wait(&bars.p_full[buf], (g >> 1) & 1);
      if (t + C::AHEAD < T) issue_s();  // S of tile t has been read
      filled(&bars.v_full[vr.slot], vr.phase);
      const uint64_t v = VMAJOR + (s_v + vr.slot * (C::TILE >> 4)), pp = KMAJOR + (s_p + buf * (C::P >> 4));
      uint32_t acc = t > 0 ? 1u : 0u;
      if (!INT8 && t == 0 && __shfl_sync(0xffffffffu, *(volatile int *)&bars.acc, 0)) {
        acc = 1u;
        __syncwarp();
        *(volatile int *)&bars.acc = 0;
      }
#pragma unroll
      for (int x = 0; x < BN / 16; x++)
        mma_ss(one, t_o, v + (x * 2048 >> 4), pp + (((x >> 2) * (NR * 128) + (x & 3) * 32) >> 4), id_o, x > 0 ? 1u : acc);
      mma_commit(one, &bars.v_empty[vr.slot]);
      mma_commit(one, &bars.pv_done[buf]);
      vr.next();
    }
    mma_commit(one, &bars.q_empty[qb]);
    mma_commit(one, &bars.o_full[pb]);
    pieces++;
  }
  // (behind a wait that has run out, products may be under way that nobody waits for)
  mma_commit(one, &bars.drained);
  wait.last(&bars.drained, 0);
}

// ------------------------------------------------------------------ loaders
// What a loader warp knows of a tile: lane i < 8 has the pool row of the tile's
// 16-token group i (of a block: block_size is a multiple of 16). The table's
// entry is read a tile ahead and used only then.
__device__ __forceinline__ int group_block(const ChunkArgs &a, const Piece &p, int tile) {
  const int tok = tile * BN + (threadIdx.x & 7) * 16;
  if (tok >= p.s.len) return 0;
  return __ldcg(a.tables + (size_t)p.s.slot * a.mbps + (a.bs == 16 ? tok >> 4 : tok / a.bs));
}
__device__ __forceinline__ int group_row(const ChunkArgs &a, const Piece &p, int tile, int block) {
  const int tok = tile * BN + (threadIdx.x & 7) * 16;
  if (tok >= p.s.len) return 0;
  return (block * a.Hkv + p.head) * a.bs + (a.bs == 16 ? 0 : tok % a.bs);
}

// Q warp: the query rows of each piece (zeros behind the last)
template <int D, bool INT8, int NR>
__device__ __forceinline__ void q_role(const ChunkArgs &a, uint8_t *sm, BarsOf<D, INT8, NR> &bars) {
  using C = Cfg<D, INT8, NR>;
  const int lane = threadIdx.x & 31;
  Waiter wait{a.err};
  Run run(a);
  Piece p{};
  uint32_t pieces = 0;
  while (run.next(a, p)) {
    const uint32_t qb = pieces % C::QBUFS;
    if (pieces >= C::QBUFS) wait(&bars.q_empty[qb], (pieces / C::QBUFS - 1) & 1);
    const uint32_t dst = smem_u32(sm + C::OFF_Q) + qb * C::Q;
    const int live = p.ntok * a.G;
#pragma unroll 4
    for (int c = lane; c < NR * (D / 8); c += 32) {
      const int n = c / (D / 8), ch = c % (D / 8), tok = n < live ? n / a.G : 0, h = n < live ? n - tok * a.G : 0;  // ch: chunk of the tile's row
      const uint16_t *src = a.q + ((size_t)(p.s.row0 + p.tok0 + tok) * a.Hq + (size_t)p.head * a.G + h) * D + chunk_of<D, INT8>(ch) * 8;
      cp16(dst + (ch >> 3) * (NR * 128) + n * 128 + (((ch & 7) ^ (n & 7)) << 4), src, n < live);
    }
    cp_wait_all();
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars.q_full[qb]);
    pieces++;
  }
}

// A loader group's tiles, one after another over the pieces of the run.
struct Tiles {
  Run run;
  Piece p;
  int t, T;
  bool more;
  __device__ __forceinline__ Tiles(const ChunkArgs &a) : run(a), p{}, t(0), T(0), more(true) { next(a); }
  __device__ __forceinline__ void next(const ChunkArgs &a) {
    if (++t < T) return;
    t = 0;
    do {
      more = run.next(a, p);
      T = max(0, p.te - p.tb);
    } while (more && T == 0);
  }
  __device__ __forceinline__ int tile() const { return p.tb + t; }
  __device__ __forceinline__ int block(const ChunkArgs &a) const { return more ? group_block(a, p, tile()) : 0; }
  __device__ __forceinline__ int rows(const ChunkArgs &a, int block) const { return group_row(a, p, tile(), block); }
};

// One group of four warps loads K, the other V.
template <int D, int NR, bool V>
__device__ __forceinline__ void load_role(const ChunkArgs &a, uint8_t *sm, BarsOf<D, false, NR> &bars) {
  using C = Cfg<D, false, NR>;
  const int tid = threadIdx.x & 127;
  constexpr int CHUNKS = D / 8, STEP = 128 / CHUNKS;  // rows per round of the 128 threads
  const int ch = tid % CHUNKS, r0 = tid / CHUNKS;
  uint64_t *full = V ? bars.v_full : bars.k_full, *empty = V ? bars.v_empty : bars.k_empty;
  const uint32_t ring = smem_u32(sm + (V ? C::OFF_V : 0));
  const uint16_t *pool = reinterpret_cast<const uint16_t *>(V ? a.pool_v : a.pool_k) + ch * 8;
  Waiter wait{a.err};
  Tiles c(a);
  Ring<V ? C::VS : C::KS> at;
  int next = c.block(a);
  for (bool first = true; c.more; at.next()) {
    const int valid = c.p.s.len - c.tile() * BN, rows = c.rows(a, next);
    c.next(a);
    next = c.block(a);  // the table's answer comes while this tile is copied
    if (!first) wait(&empty[at.slot], at.phase ^ 1);
    if (at.slot + 1 == (V ? C::VS : C::KS)) first = false;
    const uint32_t dst = ring + at.slot * C::TILE;
#pragma unroll
    for (int i = 0; i < BN / STEP; i++) {
      const int r = r0 + i * STEP;
      const int row = __shfl_sync(0xffffffffu, rows, r >> 4) + (r & 15);
      cp16(dst + chunk_off(r, ch), pool + (size_t)row * D, r < valid);
    }
    // arrives when this thread's copies have landed; the MMA warp, behind all
    // of them, orders them before its reads (fence.proxy.async)
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[at.slot])) : "memory");
  }
  cp_wait_all();
}

// int8: a thread copies the codes that it will convert RAWS tiles ahead into
// its own part of shared memory (loads into registers would not survive the
// fences between them).
template <int D, int NR, bool V>
__device__ __forceinline__ void load_role_i8(const ChunkArgs &a, uint8_t *sm, BarsOf<D, true, NR> &bars) {
  using C = Cfg<D, true, NR>;
  constexpr int THREADS = 128 * C::PER_SLOT, RAW = V ? C::RAW_V : C::RAW_K;
  const int tid = threadIdx.x % THREADS, lane = threadIdx.x & 31;
  constexpr int CHUNKS = D / 16, STEP = THREADS / CHUNKS, N = BN / STEP;
  const int ch = tid % CHUNKS, r0 = tid / CHUNKS;
  uint64_t *full = V ? bars.v_full : bars.k_full, *empty = V ? bars.v_empty : bars.k_empty;
  uint8_t *ring = sm + (V ? C::OFF_V : 0), *raw = sm + C::OFF_RAW + (V ? C::RAWS * C::RAW_K : 0);
  const uint8_t *pool = reinterpret_cast<const uint8_t *>(V ? a.pool_v : a.pool_k) + ch * 16;
  Waiter wait{a.err};
  Tiles f(a), c(a);  // what is fetched, what is converted
  int next = f.block(a);
  auto fetch = [&](uint32_t stage) {
    if (f.more) {
      const int valid = f.p.s.len - f.tile() * BN, rows = f.rows(a, next);
      f.next(a);
      next = f.block(a);
      const uint32_t dst = smem_u32(raw + stage * RAW) + tid * 16;
#pragma unroll
      for (int i = 0; i < N; i++) {
        const int r = r0 + i * STEP;
        const int row = __shfl_sync(0xffffffffu, rows, r >> 4) + (r & 15);
        cp16(dst + i * (THREADS * 16), pool + (size_t)row * D, r < valid);
      }
      if (!V && tid < 64) {  // both scales come with K: four keys' of K, or of V, a thread
        const int k = lane * 4, row = __shfl_sync(0xffffffffu, rows, k >> 4) + (k & 15);
        cp16(smem_u32(raw + stage * RAW + BN * D) + tid * 16, (tid < 32 ? a.sk : a.sv) + row, k < valid);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < C::RAWS; i++) fetch(i);
  Ring<V ? C::VS : C::KS> at;
  Ring<C::RAWS> stage;
  Ring<V ? 1 : C::SCALES> scales;
  for (bool first = true; c.more; at.next(), stage.next(), scales.next(), c.next(a)) {
    cp_wait<C::RAWS - 1>();
    const uint8_t *src = raw + stage.slot * RAW;
    uint4 x[N];
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = *reinterpret_cast<const uint4 *>(src + i * (THREADS * 16) + tid * 16);
    if (!first) wait(&empty[at.slot], at.phase ^ 1);
    if (at.slot + 1 == (V ? C::VS : C::KS)) first = false;
    if (!V && tid < 64) {
      const int k = lane * 4, live = c.p.s.len - c.tile() * BN - k;  // a key that does not exist has scale 1
      const float4 f = *reinterpret_cast<const float4 *>(src + BN * D + tid * 16);
      float *to = reinterpret_cast<float *>(sm + C::OFF_SCALE) + scales.slot * 2 * BN + (tid < 32 ? 0 : BN) + k;
      *reinterpret_cast<float4 *>(to) = make_float4(live > 0 ? f.x : 1.f, live > 1 ? f.y : 1.f, live > 2 ? f.z : 1.f, live > 3 ? f.w : 1.f);
    }
    uint8_t *dst = ring + at.slot * C::TILE;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int r = r0 + i * STEP;
      const uint32_t in[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      uint32_t o[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const uint32_t word = in[e >> 1], sel = e & 1 ? 0x4342u : 0x4140u;
        if constexpr (V) {
          // f16: (code ^ 0x80) under the magic 0x64 is 1024 + 128 + code
          const uint32_t h = __byte_perm(word ^ 0x80808080u, 0x64646464u, sel);
          asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(o[e]) : "r"(h), "r"(0x64806480u));
        } else {
          // bf16: the low 7 bits under the magic 0x43 are 128 + low7, the sign
          // bit alone 128 or 256; their difference is the code
          const uint32_t h = __byte_perm(word, 0x43434343u, sel);
          asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(o[e]) : "r"(h & 0xFF7FFF7Fu), "r"(h & 0xFF80FF80u));
        }
      }
      // columns 16 ch .. + 7 and .. + 15 (chunk_of)
      *reinterpret_cast<uint4 *>(dst + chunk_off(r, D == 128 ? ch : 2 * ch)) = make_uint4(o[0], o[1], o[2], o[3]);
      *reinterpret_cast<uint4 *>(dst + chunk_off(r, D == 128 ? ch + 8 : 2 * ch + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&full[at.slot]);
    fetch(stage.slot);  // its codes have been used
  }
  cp_wait_all();
}

template <int D, bool INT8, int NR>
__global__ void __launch_bounds__(Cfg<D, INT8, NR>::THREADS, 1) chunk_few_kernel(const __grid_constant__ ChunkArgs a) {
  using C = Cfg<D, INT8, NR>;
  using B = BarsOf<D, INT8, NR>;
  static_assert(sizeof(B) <= 320, "barriers");
  extern __shared__ __align__(1024) uint8_t sm[];
  B &bars = *reinterpret_cast<B *>(sm + C::OFF_BARS);
  const int warp = threadIdx.x >> 5;
  if (warp == 0) {
    // no tensor memory is taken that a CTA of the last kernel may still ask for
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem)), "r"((uint32_t)C::COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 32) {
    constexpr uint32_t LOADING = INT8 ? 4 * C::PER_SLOT : 128;
    for (int i = 0; i < C::KS; i++) {
      mbar_init(&bars.k_full[i], LOADING);
      mbar_init(&bars.k_empty[i], 1);
    }
    for (int i = 0; i < C::VS; i++) {
      mbar_init(&bars.v_full[i], LOADING);
      mbar_init(&bars.v_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&bars.q_full[i], 1);
      mbar_init(&bars.q_empty[i], 1);
      mbar_init(&bars.p_full[i], C::SOFT * 4);
      mbar_init(&bars.pv_done[i], 1);
      mbar_init(&bars.o_full[i], 1);
      mbar_init(&bars.o_free[i], C::SOFT * 4);
    }
    for (int i = 0; i < C::AHEAD; i++) mbar_init(&bars.s_full[i], 1);
    mbar_init(&bars.drained, 1);
    bars.acc = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;");  // the next kernel may start; it waits for this grid's end
  asm volatile("griddepcontrol.wait;" ::: "memory");  // what the last kernels wrote is there, and what they read is free
  const uint32_t tmem = bars.tmem;
  constexpr int SOFT_WARPS = C::SOFT * 4, LOAD_WARPS = C::PER_SLOT * 4;
  if (warp < SOFT_WARPS) {
    if constexpr (C::REG_SOFT > C::REGS) regs_inc<C::REG_SOFT>();
    softmax_role<D, INT8, NR>(a, sm, bars);
  } else if (warp < SOFT_WARPS + 2 * LOAD_WARPS) {
    if constexpr (C::REG_LOAD < C::REGS) regs_dec<C::REG_LOAD>();
    if constexpr (C::REG_LOAD > C::REGS) regs_inc<C::REG_LOAD>();
    const bool v = warp >= SOFT_WARPS + LOAD_WARPS;
    if constexpr (INT8) {
      if (v) load_role_i8<D, NR, true>(a, sm, bars);
      else load_role_i8<D, NR, false>(a, sm, bars);
    } else {
      if (v) load_role<D, NR, true>(a, sm, bars);
      else load_role<D, NR, false>(a, sm, bars);
    }
  } else {
    regs_dec<C::REG_MMA>();
    if (warp == SOFT_WARPS + 2 * LOAD_WARPS) {
      mma_role<D, INT8, NR>(a, sm, bars);
    } else if (warp == SOFT_WARPS + 2 * LOAD_WARPS + 1) {
      q_role<D, INT8, NR>(a, sm, bars);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::COLS));
}

template <int D, bool INT8, int NR>
int launch(vxb_kv *kv, const ChunkArgs &a, cudaStream_t st) {
  using C = Cfg<D, INT8, NR>;
  static std::atomic<bool> configured[64];  // kernel attributes set on this device (zero-initialized)
  if (!configured[kv->ctx->device & 63]) {
    VXB_CUDA_TRY(kv->ctx, cudaFuncSetAttribute(chunk_few_kernel<D, INT8, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    configured[kv->ctx->device & 63] = true;
  }
  return launch_early(kv->ctx, "chunk_few_kernel", chunk_few_kernel<D, INT8, NR>, dim3((unsigned)a.n_ctas), C::THREADS, C::SMEM, st, a);
}

template <int D, bool INT8>
int launch(vxb_kv *kv, const ChunkArgs &a, int max_rows, cudaStream_t st) {
  if (max_rows <= 16) return launch<D, INT8, 16>(kv, a, st);
  if (max_rows <= 32) return launch<D, INT8, 32>(kv, a, st);
  return launch<D, INT8, 64>(kv, a, st);
}

}  // namespace

int vxb::chunk::launch_few(vxb_kv *kv, const ChunkArgs &a, int max_rows, cudaStream_t st) {
  const bool i8 = kv->dtype == VXB_I8;
  if (kv->head_dim == 128) return i8 ? launch<128, true>(kv, a, max_rows, st) : launch<128, false>(kv, a, max_rows, st);
  return i8 ? launch<64, true>(kv, a, max_rows, st) : launch<64, false>(kv, a, max_rows, st);
}
