// Chunk attention for few rows: the drafted tokens of a request, up to 64 rows
// (tokens x query heads of a kv head). Bound by reading the cache once, so the
// keys take the tensor core's 128 rows and the queries its N = 16, 32 or 64
// columns:
//
//   S^T = K Q^T         A = the K tile, B = the query rows
//   P^T = 2^(S^T - m)   thread = key: N values each
//   O^T += V^T P^T      A = the V tile read MN-major, B = P from shared memory
//
// With the queries as rows (chunk_attn.cu) a tile costs 128 exponentials per
// lane however few rows are live; here it costs N, and a per-key scale (int8)
// is one register of the key's thread. The reference maximum m of a row moves
// only when a score passes it by 2^8, so a tile needs one vote of the
// warpgroup and no reduction; l is summed per thread and reduced at the end.
//
// Loader warps bring tiles of 128 keys into a ring in the order they are used
// (K0, K1, V0, K2, V1, ...): bf16 rows with cp.async (a 16-token page is only
// 4 KB: as many TMA boxes reach 5.6 TB/s, 16-byte copies the memory rate),
// int8 rows through registers, K to bf16 and V to f16 (codes are exact in
// both). Rows behind the last token become zeros.
//
// int8 weights carry the V scale, w = p * scale, with the reference maximum
// taken over log2(w), and go into P as f16 times 2^6: 11 significant bits, and
// weights down to 2^-30 of the row's largest keep at least one. bf16 P rounds
// at 2^-8 (the type of V decides).
//
// Values of V that only some rows may see and that are not finite are taken
// out of the tile and added to the rows that see them, as in chunk_attn.cu.
#include <atomic>
#include <climits>
#include <cmath>
#include <cuda_fp16.h>

#include "chunk_attn.h"

using namespace vxb;
using namespace vxb::tc;
using namespace vxb::chunk;

namespace {

template <int D, bool INT8, int NR>
struct Cfg {
  static constexpr int SLAB = BN * 128;         // 64 columns of 128 keys
  static constexpr int TILE = SLAB * (D / 64);
  // fewer where Q, P and the scales of int8 leave less room (int8 loads run ahead in registers)
  static constexpr int SLOTS = D == 128 ? (INT8 ? (NR == 64 ? 4 : NR == 32 ? 5 : 6) : NR == 64 ? 5 : 6) : 10;
  static constexpr int LAG = D == 128 ? 3 : 6;  // slots whose copies are in flight before the oldest is waited for
  static constexpr int Q = NR * D * 2, P = NR * BN * 2;
  static constexpr int OFF_Q = SLOTS * TILE;    // two pieces
  static constexpr int OFF_P = OFF_Q + 2 * Q;   // two tiles
  static constexpr int OFF_SCALE = OFF_P + 2 * P;
  static constexpr int SCALES = 8;              // tiles whose K and V scales are kept
  static constexpr int OFF_RED = OFF_SCALE + (INT8 ? SCALES * 2 * BN * 4 : 0);  // [4][NR] per warp, m, reference, factor [NR]
  static constexpr int OFF_BARS = OFF_RED + 7 * NR * 4;
  static constexpr int SMEM = OFF_BARS + 512;
  static constexpr int LOADERS = INT8 ? 8 : 4;  // warps
  static constexpr int THREADS = 128 + LOADERS * 32 + 32;
  static constexpr int COLS = 4 * NR;           // TMEM: S, S, O, O
  static_assert(SMEM <= 232448, "shared memory");
  static_assert(LAG < SLOTS && SCALES >= (SLOTS + 3 + 1) / 2, "ring");
};

template <int SLOTS>
struct Bars {
  uint64_t full[SLOTS], empty[SLOTS], q_empty[2], s_full[2], p_full[2], pv_done[2], o_full[2], o_free[2];
  uint32_t tmem;
  int acc;  // O already holds values that the piece's first product adds to
};

// ring index, within a piece of T tiles, of K and V of tile t
__device__ __forceinline__ uint32_t k_at(int t) { return t == 0 ? 0u : 2u * (uint32_t)t - 1u; }
__device__ __forceinline__ uint32_t v_at(int t, int T) { return t < T - 1 ? 2u * (uint32_t)t + 2u : 2u * (uint32_t)T - 1u; }

// 16-byte chunk c of row r of a tile, 128-byte swizzle
__device__ __forceinline__ uint32_t chunk_off(int r, int c) {
  return (uint32_t)((c >> 3) * (BN * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[N]);
template <>
__device__ __forceinline__ void tmem_ld<32>(uint32_t taddr, float (&v)[32]) { tmem_ld32(taddr, v); }
template <>
__device__ __forceinline__ void tmem_ld<16>(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t taddr, const float (&v)[N]);
template <>
__device__ __forceinline__ void tmem_st<16>(uint32_t taddr, const float (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
               "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
               "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])),
               "r"(__float_as_uint(v[8])), "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
               "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])), "r"(__float_as_uint(v[15]))
               : "memory");
}

// Instruction descriptor of kind::f16 with f32 sums: M = 128, N columns, B
// K-major, A K- or MN-major, both f16 or both bf16.
__host__ __device__ constexpr uint32_t idesc(int N, bool a_mn_major, bool f16) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | ((a_mn_major ? 1u : 0u) << 15) | ((uint32_t)(N >> 3) << 17) | (8u << 24);
}

// ------------------------------------------------------------------ softmax: thread = key
template <int D, bool INT8, int NR>
__device__ __forceinline__ void softmax_role(const ChunkArgs &a, uint8_t *sm, Bars<Cfg<D, INT8, NR>::SLOTS> &bars) {
  using C = Cfg<D, INT8, NR>;
  constexpr int CH = NR < 32 ? NR : 32;  // columns in registers at a time
  constexpr float SHIFT = INT8 ? 6.f : 0.f;  // P (and l) hold 2^SHIFT times the weights
  const int key = threadIdx.x, warp = key >> 5, lane = key & 31;
  const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
  float *red = reinterpret_cast<float *>(sm + C::OFF_RED), *m_s = red + 4 * NR, *ref_s = m_s + NR, *f_s = ref_s + NR;
  const float *scales = reinterpret_cast<const float *>(sm + C::OFF_SCALE);
  Waiter<true> wait{a.err};
  Run run(a);
  Piece p{};
  uint32_t g = 0, pieces = 0, ring = 0;  // tiles and pieces so far; first ring index of the piece
  while (run.next(a, p)) {
    const int T = max(0, p.te - p.tb), live = p.ntok * a.G;
    const int base = p.s.len - p.s.rows + p.tok0;  // last key that the first token sees
    const uint32_t tO = bars.tmem + lane_off + (2 + (pieces & 1)) * NR;
    float l[NR];
#pragma unroll
    for (int n = 0; n < NR; n++) l[n] = 0.f;
    for (int t = 0; t < T; t++, g++) {
      const int k0 = (p.tb + t) * BN, k = k0 + key;
      const uint32_t tS = bars.tmem + lane_off + (g & 1) * NR;
      wait(&bars.s_full[g & 1], (g >> 1) & 1);
      tc_fence_after();
      // the first row that sees this thread's key
      const int n_min = k >= p.s.len ? INT_MAX : a.sh.causal && k > base ? (k - base) * a.G : 0;
      const bool masked = k0 + BN > p.s.len || (a.sh.causal && k0 + BN - 1 > base);
      float sc = a.scale_log2, add = 0.f, isv = 1.f;
      if constexpr (INT8) {
        const float *tile = scales + g % C::SCALES * 2 * BN;
        sc *= tile[key];
        const float sv = tile[BN + key];
        add = log2f(sv);
        isv = 1.f / sv;
      }
      float s[CH];
      // log2 of the weight, without the reference
      auto load = [&](int c0) {
        tmem_ld<CH>(tS + c0, s);
        tmem_wait_ld();
#pragma unroll
        for (int n = 0; n < CH; n++) {
          s[n] = INT8 ? fmaf(s[n], sc, add) : s[n] * sc;
          if (masked) s[n] = c0 + n >= n_min ? s[n] : -INFINITY;
        }
      };
      bool over = t == 0;
#pragma unroll
      for (int c0 = 0; c0 < NR; c0 += CH) {
        load(c0);
        if (t > 0) {
#pragma unroll
          for (int n = 0; n < CH; n += 4) {
            const float4 m = *reinterpret_cast<const float4 *>(ref_s + c0 + n);
            over |= s[n] > m.x + RESCALE_THRESHOLD || s[n + 1] > m.y + RESCALE_THRESHOLD || s[n + 2] > m.z + RESCALE_THRESHOLD ||
                    s[n + 3] > m.w + RESCALE_THRESHOLD;
          }
        }
      }
      over = t == 0 || bar_or(1, 128, over);
      if (over) {
        // new references: the rows' maxima over this tile and before
#pragma unroll 1
        for (int c0 = 0; c0 < NR; c0 += CH) {
          if (NR > CH) load(c0);
          float top = -INFINITY;
#pragma unroll
          for (int n = 0; n < CH; n++) {
            const float x = warp_max(s[n]);
            top = lane == n ? x : top;
          }
          if (lane < CH) red[warp * NR + c0 + lane] = top;
        }
        bar_sync(1, 128);
        if (key < NR) {
          const float old = t == 0 ? -INFINITY : m_s[key];
          const float m = fmaxf(fmaxf(fmaxf(red[key], red[NR + key]), fmaxf(red[2 * NR + key], red[3 * NR + key])), old);
          m_s[key] = m;
          ref_s[key] = m == -INFINITY ? -1e30f : m;  // no score yet: any one passes it
          f_s[key] = m == old ? 1.f : ex2(old - m);
        }
        bar_sync(1, 128);
        if (t > 0) {
          wait(&bars.pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1);
          tc_fence_after();
#pragma unroll
          for (int c0 = 0; c0 < NR; c0 += 16) {
            float o[16];
            tmem_ld<16>(tO + c0, o);
            tmem_wait_ld();
#pragma unroll
            for (int n = 0; n < 16; n++) {
              const float f = f_s[c0 + n];
              o[n] *= f;
              l[c0 + n] *= f;
            }
            tmem_st<16>(tO + c0, o);
          }
          tmem_wait_st();
        }
      }
      // P of two tiles ago has been used
      uint8_t *P = sm + C::OFF_P + (g & 1) * C::P;
      if (g >= 2) wait(&bars.pv_done[g & 1], ((g - 2) >> 1) & 1);
      uint8_t *prow = P + (key >> 6) * (NR * 128) + (key & 7) * 2;
      const uint32_t chunk = (uint32_t)(key & 63) >> 3 << 4;
#pragma unroll
      for (int c0 = 0; c0 < NR; c0 += CH) {
        if (NR > CH) load(c0);
#pragma unroll
        for (int n = 0; n < CH; n += 4) {
          const float4 ref = *reinterpret_cast<const float4 *>(ref_s + c0 + n);
          const float m4[4] = {ref.x, ref.y, ref.z, ref.w};
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int r = c0 + n + e;
            const float w = ex2(INT8 ? s[n + e] - (m4[e] - SHIFT) : s[n + e] - m4[e]);
            uint16_t bits;
            if constexpr (INT8) {
              // a row without this key: no product with a scale that is not finite
              l[r] = !masked || r >= n_min ? fmaf(w, isv, l[r]) : l[r];
              bits = __half_as_ushort(__float2half_rn(w));
            } else {
              l[r] += w;
              bits = (uint16_t)pack_bf16(w, 0.f);
            }
            *reinterpret_cast<uint16_t *>(prow + r * 128 + (chunk ^ ((uint32_t)(r & 7) << 4))) = bits;
          }
        }
      }
      if constexpr (!INT8) {
        if (a.sh.causal && min(k0 + BN, p.s.len) - 1 > base) {
          // some row does not see all of this tile's keys
          const int valid = min(BN, p.s.len - k0);
          const uint32_t vi = ring + v_at(t, T);
          wait(&bars.full[vi % C::SLOTS], (vi / C::SLOTS) & 1);
          uint8_t *V = sm + (vi % C::SLOTS) * C::TILE;
          uint32_t found = 0;
          for (int c = key; c < valid * (D / 8); c += 128) {
            const uint4 w = *reinterpret_cast<const uint4 *>(V + chunk_off(c / (D / 8), c % (D / 8)));
            found |= odd_bf16(w.x) | odd_bf16(w.y) | odd_bf16(w.z) | odd_bf16(w.w);
          }
          __syncwarp();
          if (bar_or(1, 128, found != 0)) {
            // rare: lane d of O^T takes every non-finite value of column d of V
            if (t > 0) {
              wait(&bars.pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1);
              tc_fence_after();
            } else {
              float z[16];
#pragma unroll
              for (int n = 0; n < 16; n++) z[n] = 0.f;
#pragma unroll
              for (int c0 = 0; c0 < NR; c0 += 16) tmem_st<16>(tO + c0, z);
              tmem_wait_st();
              if (key == 0) bars.acc = 1;
            }
            const int d = key % D;
            for (int j = 0; j < valid; j++) {
              const uint32_t bits = *reinterpret_cast<const uint16_t *>(V + chunk_off(j, d >> 3) + (d & 7) * 2);
              const bool odd = (bits & 0x7F80u) == 0x7F80u;
              if (!__any_sync(0xffffffffu, odd)) continue;
              const int first = a.sh.causal && k0 + j > base ? (k0 + j - base) * a.G : 0;
              for (int n = first; n < NR; n++) {
                const uint32_t off = (uint32_t)(j >> 6) * (NR * 128) + (uint32_t)n * 128 + ((((uint32_t)(j & 63) >> 3) ^ ((uint32_t)n & 7)) << 4) + (j & 7) * 2;
                const float w = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t *>(P + off) << 16);
                const float o = tmem_ld1(tO + n);
                tmem_st1(tO + n, odd ? fmaf(w, __uint_as_float(bits << 16), o) : o);
                tmem_wait_st();
              }
            }
            bar_sync(1, 128);
            for (int c = key; c < valid * (D / 8); c += 128) {
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
    // ---------------- end of the piece
    // l of every row: over the lanes, then the warps
    bar_sync(1, 128);  // red is free
#pragma unroll
    for (int n = 0; n < NR; n++) {
      const float x = warp_sum(l[n]);
      if (lane == (n & 31)) red[warp * NR + n] = x;
    }
    bar_sync(1, 128);
    if (key < NR) f_s[key] = red[key] + red[NR + key] + red[2 * NR + key] + red[3 * NR + key];
    bar_sync(1, 128);
    const bool whole = p.whole();
    float *part = a.ws + (size_t)(blockIdx.x * 2 + (p.tb > 0 ? 0 : 1)) * (kRowsItem * (D + 2));
    const size_t row0 = (size_t)(p.s.row0 + p.tok0) * a.Hq + (size_t)p.head * a.G;
    if (key < live) {
      const float m = T > 0 ? m_s[key] : -INFINITY, L = f_s[key];
      if (!whole) {
        __stcg(reinterpret_cast<float2 *>(part + (size_t)kRowsItem * D) + key, make_float2(m - SHIFT, L));
      } else if (a.lse) {
        a.lse[row0 + (size_t)(key / a.G) * a.Hq + key % a.G] = L == 0.f ? -INFINITY : (m - SHIFT + log2f(L)) * 0.69314718055994531f;
      }
    }
    wait(&bars.o_full[pieces & 1], (pieces >> 1) & 1);
    tc_fence_after();
#pragma unroll 1
    for (int c0 = 0; c0 < NR && c0 < live; c0 += 16) {
      float o[16];
#pragma unroll
      for (int n = 0; n < 16; n++) o[n] = 0.f;
      if (T > 0) {
        tmem_ld<16>(tO + c0, o);
        tmem_wait_ld();
      }
      int tok = c0 / a.G, h = c0 - tok * a.G;
      if (key < D) {
#pragma unroll
        for (int n = 0; n < 16; n++) {
          if (c0 + n < live) {
            if (whole) {
              const float L = f_s[c0 + n];
              a.out[(row0 + (size_t)tok * a.Hq + h) * D + key] = (uint16_t)pack_bf16(L == 0.f ? 0.f : o[n] * (1.f / L), 0.f);
            } else {
              __stcg(part + (size_t)(c0 + n) * D + key, o[n]);
            }
          }
          if (++h == a.G) {
            h = 0;
            tok++;
          }
        }
      }
      __syncwarp();
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars.o_free[pieces & 1]);
    pieces++;
    ring += 2 * (uint32_t)T;
  }
}

// ------------------------------------------------------------------ MMA thread
template <int D, bool INT8, int NR>
__device__ __forceinline__ void mma_role(const ChunkArgs &a, uint8_t *sm, Bars<Cfg<D, INT8, NR>::SLOTS> &bars) {
  using C = Cfg<D, INT8, NR>;
  constexpr uint32_t ID_S = idesc(NR, false, false), ID_O = idesc(NR, true, INT8);
  const uint32_t s_kv = smem_u32(sm), s_q = smem_u32(sm + C::OFF_Q), s_p = smem_u32(sm + C::OFF_P), tmem = bars.tmem;
  Waiter<false> wait{a.err};
  Run run(a);
  Piece p{};
  uint32_t g = 0, pieces = 0, ring = 0;
  while (run.next(a, p)) {
    const int T = max(0, p.te - p.tb);
    const uint32_t pb = pieces & 1;
    auto issue_s = [&](int t) {
      const uint32_t i = ring + k_at(t), slot = i % C::SLOTS, buf = (g + t) & 1;
      wait(&bars.full[slot], (i / C::SLOTS) & 1);
      tc_fence_after();
      const uint32_t k = s_kv + slot * C::TILE, q = s_q + pb * C::Q;
#pragma unroll
      for (int x = 0; x < D / 16; x++)
        umma_bf16(tmem + buf * NR, sw128_desc(k + (x >> 2) * C::SLAB + (x & 3) * 32, 16, 1024),
                  sw128_desc(q + (x >> 2) * (NR * 128) + (x & 3) * 32, 16, 1024), ID_S, x > 0 ? 1u : 0u);
      umma_commit(&bars.s_full[buf]);
      umma_commit(&bars.empty[slot]);
    };
    if (T > 0) issue_s(0);
    if (T > 1) issue_s(1);
    if (pieces >= 2) wait(&bars.o_free[pb], ((pieces >> 1) - 1) & 1);
    for (int t = 0; t < T; t++) {
      const uint32_t i = ring + v_at(t, T), slot = i % C::SLOTS, buf = (g + t) & 1;
      wait(&bars.p_full[buf], ((g + t) >> 1) & 1);
      wait(&bars.full[slot], (i / C::SLOTS) & 1);
      tc_fence_after();
      uint32_t acc = t > 0 ? 1u : 0u;
      if (!INT8 && t == 0 && *(volatile int *)&bars.acc) {
        acc = 1u;
        *(volatile int *)&bars.acc = 0;
      }
      const uint32_t v = s_kv + slot * C::TILE, pp = s_p + buf * C::P;
      // heads of 64: the second 64 rows of A are the first again, and are not read back
#pragma unroll
      for (int x = 0; x < BN / 16; x++)
        umma_bf16(tmem + (2 + pb) * NR, sw128_desc(v + x * 2048, D == 128 ? C::SLAB : 0, 1024),
                  sw128_desc(pp + (x >> 2) * (NR * 128) + (x & 3) * 32, 16, 1024), ID_O, x > 0 ? 1u : acc);
      umma_commit(&bars.empty[slot]);
      umma_commit(&bars.pv_done[buf]);
      if (t + 2 < T) issue_s(t + 2);
    }
    umma_commit(&bars.q_empty[pb]);
    umma_commit(&bars.o_full[pb]);
    g += (uint32_t)T;
    ring += 2 * (uint32_t)T;
    pieces++;
  }
}

// ------------------------------------------------------------------ loaders
// What a loader warp knows of a tile: lane i < 8 has the pool row of the tile's
// 16-token group i (of a block: block_size is a multiple of 16).
__device__ __forceinline__ int group_row(const ChunkArgs &a, const Piece &p, const int32_t *table, int tile) {
  const int tok = tile * BN + (threadIdx.x & 7) * 16;
  if (tok >= p.s.len) return 0;
  const int b = a.bs == 16 ? tok >> 4 : tok / a.bs;
  return (__ldg(table + b) * a.Hkv + p.head) * a.bs + (tok - b * a.bs);
}

// Query rows of the piece into its buffer (zeros behind the last), by `threads` threads
template <int D, int NR>
__device__ __forceinline__ void load_q(const ChunkArgs &a, const Piece &p, uint32_t dst, int tid, int threads) {
  const int live = p.ntok * a.G;
  for (int c = tid; c < NR * (D / 8); c += threads) {
    const int n = c / (D / 8), ch = c % (D / 8), tok = n / a.G;
    const uint16_t *src = a.q + ((size_t)(p.s.row0 + p.tok0 + (n < live ? tok : 0)) * a.Hq + (size_t)p.head * a.G + (n < live ? n - tok * a.G : 0)) * D + ch * 8;
    cp16(dst + (ch >> 3) * (NR * 128) + n * 128 + (((ch & 7) ^ (n & 7)) << 4), src, n < live);
  }
}

template <int D, int NR>
__device__ __forceinline__ void load_role(const ChunkArgs &a, uint8_t *sm, Bars<Cfg<D, false, NR>::SLOTS> &bars) {
  using C = Cfg<D, false, NR>;
  const int tid = threadIdx.x - 128, lane = threadIdx.x & 31;
  const uint32_t s_kv = smem_u32(sm), s_q = smem_u32(sm + C::OFF_Q);
  constexpr int CHUNKS = D / 8, STEP = 128 / CHUNKS;  // rows per round of the 128 threads
  const int ch = tid % CHUNKS, r0 = tid / CHUNKS;
  Waiter<true> wait{a.err};
  Run run(a);
  Piece p{};
  uint32_t idx = 0, told = 0, pieces = 0;  // copied and announced slots
  auto tell = [&](uint32_t upto) {  // their copies have landed
    fence_async_smem();
    __syncwarp();
    if (lane == 0)
      for (uint32_t i = told; i < upto; i++) mbar_arrive(&bars.full[i % C::SLOTS]);
    told = upto;
  };
  // waiting for the MMA side: the tiles that it may need first are announced first
  auto wait_told = [&](uint64_t *bar, uint32_t ph) {
    if (__all_sync(0xffffffffu, mbar_try(smem_u32(bar), ph))) return;
    cp_wait<0>();
    tell(idx);
    wait(bar, ph);
  };
  auto copy = [&](const void *pool, int rows, int tile) {
    const uint32_t slot = idx % C::SLOTS;
    if (idx >= C::SLOTS) wait_told(&bars.empty[slot], (idx / C::SLOTS - 1) & 1);
    const uint32_t dst = s_kv + slot * C::TILE;
    const int valid = p.s.len - tile * BN;
    const uint16_t *src = reinterpret_cast<const uint16_t *>(pool) + ch * 8;
#pragma unroll
    for (int i = 0; i < BN / STEP; i++) {
      const int r = r0 + i * STEP;
      const int row = __shfl_sync(0xffffffffu, rows, r >> 4) + (r & 15);
      cp16(dst + chunk_off(r, ch), src + (size_t)row * D, r < valid);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    idx++;
    if (idx - told > C::LAG) {
      cp_wait<C::LAG>();
      tell(idx - C::LAG);
    }
  };
  while (run.next(a, p)) {
    const int32_t *table = a.tables + (size_t)p.s.slot * a.mbps;
    const int T = max(0, p.te - p.tb);
    if (pieces >= 2) wait_told(&bars.q_empty[pieces & 1], ((pieces >> 1) - 1) & 1);
    if (T > 0) {
      load_q<D, NR>(a, p, s_q + (pieces & 1) * C::Q, tid, 128);  // lands with the first K
      int next = group_row(a, p, table, p.tb);
      copy(a.pool_k, next, p.tb);
      for (int t = 0; t < T; t++) {
        const int now = next;
        if (t + 1 < T) {
          next = group_row(a, p, table, p.tb + t + 1);
          copy(a.pool_k, next, p.tb + t + 1);
        }
        copy(a.pool_v, now, p.tb + t);
      }
    }
    pieces++;
  }
  cp_wait<0>();
  tell(idx);
}

// int8: two groups of four warps take the slots in turn; the codes of a group's
// next slot are on their way in registers while it converts this one's.
template <int D, int NR>
__device__ __forceinline__ void load_role_i8(const ChunkArgs &a, uint8_t *sm, Bars<Cfg<D, true, NR>::SLOTS> &bars) {
  using C = Cfg<D, true, NR>;
  const int tid = (threadIdx.x - 128) & 127, lane = threadIdx.x & 31;
  const uint32_t half = (threadIdx.x - 128) >> 7;
  constexpr int CHUNKS = D / 16, STEP = 128 / CHUNKS, N = BN / STEP;
  const int ch = tid % CHUNKS, r0 = tid / CHUNKS;
  Waiter<true> wait{a.err};
  // this group's next slot: j (of parity `half`) of the 2 T slots of piece p
  Run run(a);
  Piece p{};
  uint32_t ring = 0, tiles = 0, pieces = 0, q_seen = 0;  // ring and tiles: before p; pieces: with p
  int T = 0, j = 0;
  auto next_piece = [&]() {
    do {
      ring += 2 * (uint32_t)T;
      tiles += (uint32_t)T;
      if (!run.next(a, p)) return false;
      pieces++;
      T = max(0, p.te - p.tb);
    } while (T == 0);
    j = (int)half;
    return true;
  };
  uint4 w[N];
  float scale_k = 1.f, scale_v = 1.f;
  // slot j: K of tile 0, then K of the next tile and V in turn, V of the last at the end
  auto tile_of = [&]() { return j == 0 ? 0 : j == 2 * T - 1 ? T - 1 : j & 1 ? (j + 1) / 2 : j / 2 - 1; };
  auto is_v = [&]() { return j == 2 * T - 1 || (j > 0 && !(j & 1)); };
  auto fetch = [&]() {
    const bool v = is_v();
    const int tile = p.tb + tile_of(), valid = p.s.len - tile * BN;
    const int rows = group_row(a, p, a.tables + (size_t)p.s.slot * a.mbps, tile);
    const uint8_t *src = reinterpret_cast<const uint8_t *>(v ? a.pool_v : a.pool_k) + ch * 16;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int r = r0 + i * STEP;
      const int row = __shfl_sync(0xffffffffu, rows, r >> 4) + (r & 15);
      w[i] = r < valid ? __ldcg(reinterpret_cast<const uint4 *>(src + (size_t)row * D)) : make_uint4(0u, 0u, 0u, 0u);
    }
    const int row = __shfl_sync(0xffffffffu, rows, tid >> 4) + (tid & 15);
    if (!v) {  // both scales come with K; a key that does not exist has scale 1
      scale_k = tid < valid ? __ldcg(a.sk + row) : 1.f;
      scale_v = tid < valid ? __ldcg(a.sv + row) : 1.f;
    }
  };
  bool more = next_piece();
  if (more) fetch();
  while (more) {
    const bool v = is_v(), first = j == 0;
    const uint32_t idx = ring + (uint32_t)j, slot = idx % C::SLOTS, tile = tiles + (uint32_t)tile_of();
    const float sk = scale_k, sv = scale_v;
    if (first) {
      // Q lands with the first K. Every piece's buffer is waited for in turn,
      // also of pieces without tiles: a phase must not be missed.
      for (; q_seen < pieces; q_seen++)
        if (q_seen >= 2) wait(&bars.q_empty[q_seen & 1], ((q_seen >> 1) - 1) & 1);
      load_q<D, NR>(a, p, smem_u32(sm + C::OFF_Q) + ((pieces - 1) & 1) * C::Q, tid, 128);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    uint4 x[N];
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = w[i];
    j += 2;
    more = j < 2 * T || next_piece();
    if (more) fetch();
    if (idx >= C::SLOTS) wait(&bars.empty[slot], (idx / C::SLOTS - 1) & 1);
    if (!v) {
      // read before tile + 2's K is used up, and this K is at most SLOTS behind
      float *at = reinterpret_cast<float *>(sm + C::OFF_SCALE) + tile % C::SCALES * 2 * BN + tid;
      at[0] = sk;
      at[BN] = sv;
    }
    uint8_t *dst = sm + slot * C::TILE;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int r = r0 + i * STEP;
      const uint32_t in[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      uint32_t o[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const uint32_t word = in[e >> 1], sel = e & 1 ? 0x4342u : 0x4140u;
        if (v) {
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
      *reinterpret_cast<uint4 *>(dst + chunk_off(r, 2 * ch)) = make_uint4(o[0], o[1], o[2], o[3]);
      *reinterpret_cast<uint4 *>(dst + chunk_off(r, 2 * ch + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
    }
    if (first) cp_wait<0>();
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars.full[slot]);
  }
}

template <int D, bool INT8, int NR>
__global__ void __launch_bounds__(Cfg<D, INT8, NR>::THREADS, 1) chunk_few_kernel(const __grid_constant__ ChunkArgs a) {
  using C = Cfg<D, INT8, NR>;
  using B = Bars<C::SLOTS>;
  static_assert(sizeof(B) <= 512, "barriers");
  extern __shared__ __align__(1024) uint8_t sm[];
  B &bars = *reinterpret_cast<B *>(sm + C::OFF_BARS);
  const int warp = threadIdx.x >> 5;
  asm volatile("griddepcontrol.launch_dependents;");  // the kernel that joins the parts waits for this grid's end
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem)), "r"((uint32_t)C::COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 32) {
    for (int i = 0; i < C::SLOTS; i++) {
      mbar_init(&bars.full[i], 4);
      mbar_init(&bars.empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&bars.q_empty[i], 1);
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 4);
      mbar_init(&bars.pv_done[i], 1);
      mbar_init(&bars.o_full[i], 1);
      mbar_init(&bars.o_free[i], 4);
    }
    bars.acc = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  if (warp < 4) {
    softmax_role<D, INT8, NR>(a, sm, bars);
  } else if (warp < 4 + C::LOADERS) {
    if constexpr (INT8) load_role_i8<D, NR>(a, sm, bars);
    else load_role<D, NR>(a, sm, bars);
  } else {
    if ((threadIdx.x & 31) == 0) mma_role<D, INT8, NR>(a, sm, bars);
    __syncwarp();
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
  chunk_few_kernel<D, INT8, NR><<<a.n_ctas, C::THREADS, C::SMEM, st>>>(a);
  return launch_check(kv->ctx, "chunk_few_kernel");
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
