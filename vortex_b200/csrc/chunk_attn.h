// What the kernels of the chunk attention share: a launch's record, the cut of
// its key tiles into one run per CTA, bounded waits.
#pragma once

#include "kv_cache.h"
#include "tc_common.h"

namespace vxb {
namespace chunk {

constexpr int BM = 128, BN = 128;
constexpr int kSeqs = 128;    // sequences of one launch (their record is a kernel parameter)
constexpr int kMaxCtas = 160;
constexpr int kRowsItem = 2 * BM;
constexpr float RESCALE_THRESHOLD = 8.f;  // O is rescaled when a row's maximum grows by more (log2)

// int8: weights carry the V scale, and a row's unit follows the largest of them.
// The sum l takes the weight times the scale's inverse, as long as all scales of
// the tiles so far are within 2^+-kFarLog2: a weight that f32 flushes then is
// under 2^-50 of the row's largest p. From the first tile with another scale on,
// l is formed from the scores alone, with their own maximum, and meets O at the
// end: it knows nothing of the values' sizes, infinite ones included. A scale
// under 2^-100 (values under 1e-28) counts as that.
//
// The cache gives a row of zeros the scale 1. Its weight, which the output has no
// use for, would set the unit and leave smaller values' weights few bits, or none:
// such a key counts for the sum alone. While its share is under 2^60 of the unit
// that is one more term, else the sum takes its own maximum as above.
constexpr float kMostShareLog2 = 60.f, kMostShare = 1152921504606846976.f;
constexpr float kLeastScale = 7.8886091e-31f, kFarLog2 = 30.f, kFarInverse = 1073741824.f;  // 2^-100, 2^30
struct ChunkSeq {
  int32_t slot, row0, rows, len;
};
struct Start {  // a CTA's first item, the first of its key tiles, and the key tiles of the run
  int32_t seq, head, pair, tile, units;
};
struct Shape {
  int tpt;  // tokens of a 128-row tile
  int causal;
};
struct ChunkArgs {
  const uint16_t *q;
  const void *pool_k, *pool_v;
  uint16_t *out;
  float *lse;
  float *ws;
  int *err;
  const float *sk, *sv;
  const int32_t *tables;  // of the layer
  int n, Hq, Hkv, G, bs, mbps, box, n_ctas;
  Shape sh;
  float scale_log2;
  ChunkSeq seq[kSeqs];
  Start start[kMaxCtas];
};
static_assert(sizeof(ChunkArgs) <= 8192, "kernel parameters");

// Key tiles that the tokens before tok_end of a chunk see
__host__ __device__ inline int tiles_of(const ChunkSeq &s, const Shape &sh, int tok_end) {
  const int seen = sh.causal ? s.len - s.rows + tok_end : s.len;
  return seen > 0 ? (seen + BN - 1) / BN : 0;
}
// Units of an item: its key tiles, one at least
__host__ __device__ inline int units_of(const ChunkSeq &s, const Shape &sh, int pair) {
  const int end = (pair + 1) * 2 * sh.tpt;
  const int t = tiles_of(s, sh, end < s.rows ? end : s.rows);
  return t > 0 ? t : 1;
}

#ifdef __CUDACC__
using namespace vxb::tc;

// Bounded wait of a whole warp; once one has run out, the following ones do not
// wait again, and the kernel ends.
struct Waiter {
  int *err;
  bool dead = false;
  __device__ __forceinline__ void operator()(uint64_t *bar, uint32_t parity) {
    if (!mbar_wait(bar, parity, dead ? 0 : kWaitBudget)) {
      dead = true;
      atomicExch(err, 1);
    }
    __syncwarp();
  }
  // For what the warp itself has under way, at its end: waited for in any case.
  __device__ __forceinline__ void last(uint64_t *bar, uint32_t parity) {
    if (!mbar_wait(bar, parity)) atomicExch(err, 1);
    __syncwarp();
  }
};

// The run of a CTA as pieces: consecutive key tiles of one item.
struct Piece {
  ChunkSeq s;
  int head, tok0, ntok, tb, te, units, te_u;
  bool both;   // two tiles of rows, the same keys; else one tile, every other key tile
  int n0, n1;  // steps of the streams
  __device__ __forceinline__ int tile(int stream, int i) const { return both ? tb + i : tb + 2 * i + stream; }
  __device__ __forceinline__ int steps(int stream) const { return stream ? n1 : n0; }
  __device__ __forceinline__ bool whole() const { return tb == 0 && te_u == units; }
};
struct Run {
  Start at;
  int left;
  Run() = default;
  __device__ Run(const ChunkArgs &a) {
    at = a.start[blockIdx.x];
    left = at.units;
  }
  __device__ __forceinline__ bool next(const ChunkArgs &a, Piece &p) {
    if (left <= 0) return false;
    p.s = a.seq[at.seq];
    p.head = at.head;
    p.tok0 = at.pair * 2 * a.sh.tpt;
    p.ntok = min(2 * a.sh.tpt, p.s.rows - p.tok0);
    p.both = p.ntok > a.sh.tpt;
    const int n = tiles_of(p.s, a.sh, p.tok0 + p.ntok);
    p.units = max(1, n);
    p.tb = at.tile;
    p.te_u = min(p.units, p.tb + left);
    p.te = min(p.te_u, n);
    const int count = max(0, p.te - p.tb);
    if (p.both) {
      p.n0 = max(0, min(p.te, tiles_of(p.s, a.sh, p.tok0 + a.sh.tpt)) - p.tb);
      p.n1 = count;
    } else {
      p.n0 = (count + 1) / 2;
      p.n1 = count / 2;
    }
    left -= p.te_u - p.tb;
    at.tile = 0;
    at.pair++;
    if (at.pair * 2 * a.sh.tpt >= p.s.rows) {
      at.pair = 0;
      if (++at.head == a.Hkv) {
        at.head = 0;
        at.seq++;
      }
    }
    return true;
  }
};

__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ bool bar_or(int id, int threads, bool p) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, %3, p;\n selp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"((uint32_t)p), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
  tmem_wait_ld();
  return __uint_as_float(r);
}
__device__ __forceinline__ void tmem_st1(uint32_t taddr, float v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(__float_as_uint(v)) : "memory");
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[8]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const float (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(__float_as_uint(v[0])),
               "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])),
               "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7]))
               : "memory");
}

// MMA issue. A whole warp runs the issuing loop and one elected lane's
// instructions take effect: the operands are then uniform over the warp and
// stay in uniform registers. (One lane alone in the loop took 80 cycles per
// instruction to move them there.)
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r;
}
// 128-byte-swizzled matrix descriptor without its address; adding (address >> 4) gives the whole
__device__ __forceinline__ constexpr uint64_t desc_base(uint32_t lbo, uint32_t sbo) {
  return ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(id), "r"(acc), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t bdesc, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(id), "r"(acc), "r"(one)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t one, uint64_t *bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar)),
      "r"(one)
      : "memory");
}

// A warpgroup's share of the block's registers.
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// Adds 0 * x of every element: NaN in a lane of acc once an element was inf or NaN
__device__ __forceinline__ uint32_t add_odd(uint32_t acc, const uint4 &x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; i++) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(w[i]), "r"(0u));
  return acc;
}
__device__ __forceinline__ uint32_t odd_bf16(uint32_t w) {  // a non-finite element in a pair
  return (uint32_t)((w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u);
}

__device__ __forceinline__ uint32_t even_bf16(uint32_t w) {  // the pair with zeros for those
  if ((w & 0x7F80u) == 0x7F80u) w &= 0xFFFF0000u;
  if ((w & 0x7F800000u) == 0x7F800000u) w &= 0xFFFFu;
  return w;
}
#endif

#ifdef __CUDACC__
// Launches a kernel that may start its CTAs before the stream's last kernel has
// ended; it waits for that itself (griddepcontrol.wait) before it touches memory,
// and reads through L2 alone: a line in L1 may be one that an earlier kernel
// read on this SM, before a kernel in between wrote it.
template <typename T>
struct Same {
  using type = T;
};
template <typename... P>
int launch_early(vxb_ctx *ctx, const char *what, void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t st,
                 const typename Same<P>::type &...args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VXB_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, kernel, args...));
  return launch_check(ctx, what);
}
#endif

// Scratch of an item's part: 256 rows of D sums, then (maximum, sum) pairs.
inline size_t part_floats(int D) { return (size_t)kRowsItem * (D + 2); }

// Chunks of up to kFewRows rows per kv head (chunk_few.cu); everything else goes
// to the kernel in chunk_attn.cu.
constexpr int kFewRows = 64;
int launch_few(vxb_kv *kv, const ChunkArgs &a, int max_rows, cudaStream_t st);

}  // namespace chunk
}  // namespace vxb
