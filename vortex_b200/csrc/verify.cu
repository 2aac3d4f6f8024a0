// Token probabilities and verification of drafted tokens.
//
// vxb_token_probs: p = exp((x - max) / t) / sum per row of logits: the row is
// read once from HBM and written once. Few rows: a cluster of up to 8 CTAs
// keeps its row in registers (latency: 4.4 us for 5 rows of 32,000). Many rows:
// one pass for the running maximum and sum and a second over the row, which
// the L2 (and a quarter of it shared memory) still holds; few registers are
// tied up, so the SMs stay full of loads: 160 rows of 131,071 in 38 us, 4.4 TB/s
// (the register form reached 2.0). DRAM carries the floor's bytes, the two
// passes do not overlap. Maximum and sum go through distributed shared memory.
//
// vxb_verify_drafts: the accept tests are a handful of gathers; the token that
// is drawn needs one row of p (and q): a cluster per request sums its slices
// in f64, finds the slice, the warp and at last the index where the cumulative
// sum passes the drawn share. One request of 32,000 6.9 us: a chain of eight
// dependent reads and cluster barriers; 64 of 131,072 21 us (3.1 TB/s), 16 us
// of it the two rows.
#include <climits>
#include <cmath>
#include <cooperative_groups.h>

#include "vxb_internal.h"

using namespace vxb;
namespace cg = cooperative_groups;

namespace {

constexpr int kMaxCluster = 8;
constexpr int kMaxVocab = 1 << 30;  // indices and the steps over a row stay within 32 bits

// ------------------------------------------------------------------ probabilities
constexpr int kProbThreads = 512, kRowThreads = 256;  // of the two forms

struct ProbArgs {
  const float *x, *temp;
  float *p;
  int vocab, slice;  // a CTA's share of a row
  double t;
};

// max over a CTA (every thread gets it); NaN passed over
template <int THREADS>
__device__ float block_max(float v, float *s) {
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = s[0];
  for (int i = 1; i < THREADS / 32; i++) r = fmaxf(r, s[i]);
  __syncthreads();
  return r;
}

template <int THREADS>
__device__ float block_sum(float v, float *s) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = 0.f;
  for (int i = 0; i < THREADS / 32; i++) r += s[i];
  __syncthreads();
  return r;
}

template <int THREADS>
__device__ int block_min(int v, int *s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = min(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  int r = s[0];
  for (int i = 1; i < THREADS / 32; i++) r = min(r, s[i]);
  __syncthreads();
  return r;
}

// exp(d / t) with d = x - max <= 0 and c = log2(e) / t: the roundings of d, of c
// and of the product cost up to 2^-24 of |d| / t each, the special-function unit
// 2 ulp.
__device__ __forceinline__ float exp_scaled(float d, float c) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * c));
  return e;
}
// (never 0: -inf, a banned token, stays -inf at any temperature)
__device__ __forceinline__ float log2e_over(double t) { return fmaxf((float)(1.4426950408889634074 / t), 1e-37f); }

// The cluster's maximum (NaN passed over), and its first index: 1 there, 0
// elsewhere. Ranks take [begin, end) of the row; every thread's `m` is the
// maximum of what it has seen.
template <int THREADS>
__device__ void one_hot(cg::cluster_group &cl, const float *x, float *p, int begin, int end, float m, int *s_redi, int *s_first) {
  int first = INT_MAX;
  for (int c = begin + (int)threadIdx.x; c < end && first == INT_MAX; c += THREADS)
    if (x[c] == m && m != -INFINITY) first = c;
  first = block_min<THREADS>(first, s_redi);
  if (threadIdx.x == 0) *s_first = first;
  cl.sync();  // every rank has read its part: p may be x
  for (int i = 0; i < (int)cl.num_blocks(); i++) first = min(first, *cl.map_shared_rank(s_first, i));
  for (int c = begin + (int)threadIdx.x; c < end; c += THREADS) p[c] = c == first ? 1.f : 0.f;
  cl.sync();  // the others' shared memory stays until they have read it
}

// PER: values of a row that a thread keeps
template <int PER>
__global__ void __launch_bounds__(kProbThreads) token_probs_kernel(const ProbArgs a) {
  cg::cluster_group cl = cg::this_cluster();
  __shared__ float s_red[kProbThreads / 32];
  __shared__ int s_redi[kProbThreads / 32];
  __shared__ float s_max, s_sum;
  __shared__ int s_first;
  const int ranks = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int row = (int)(blockIdx.x / ranks);
  const int begin = min(rank * a.slice, a.vocab), end = min(begin + a.slice, a.vocab);
  const float *x = a.x + (size_t)row * a.vocab;
  float *p = a.p + (size_t)row * a.vocab;
  const double t = a.temp ? (double)a.temp[row] : a.t;
  float v[PER];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int c = begin + i * kProbThreads + (int)threadIdx.x;
    v[i] = c < end ? __ldcs(x + c) : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < PER; i++) m = fmaxf(m, v[i]);
  m = block_max<kProbThreads>(m, s_red);
  if (threadIdx.x == 0) s_max = m;
  cl.sync();
  for (int i = 0; i < ranks; i++) m = fmaxf(m, *cl.map_shared_rank(&s_max, i));
  if (!(t >= 0.01)) {
    one_hot<kProbThreads>(cl, x, p, begin, end, m, s_redi, &s_first);
    return;
  }
  const float c = log2e_over(t);
  const float ref = m == -INFINITY ? 0.f : m;  // -inf alone gives zeros, NaN beside it NaN
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    v[i] = exp_scaled(v[i] - ref, c);
    sum += v[i];
  }
  sum = block_sum<kProbThreads>(sum, s_red);
  if (threadIdx.x == 0) s_sum = sum;
  cl.sync();
  sum = 0.f;
  for (int i = 0; i < ranks; i++) sum += *cl.map_shared_rank(&s_sum, i);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int k = begin + i * kProbThreads + (int)threadIdx.x;
    if (k < end) p[k] = v[i] * inv;
  }
  cl.sync();
}

constexpr int kKeep = 8;  // fours of a thread that the second pass finds in shared memory, not in L2 (39.3 -> 38.0 us)

// Two passes over the row. Four values a load where x and p have the same
// place within 16 bytes (VEC): `head` single ones lead to the first boundary,
// the cluster's ranks share the fours, the last rank takes the rest.
template <bool VEC>
__global__ void __launch_bounds__(kRowThreads, 5) token_probs_rows_kernel(const ProbArgs a) {
  cg::cluster_group cl = cg::this_cluster();
  __shared__ float s_red[kRowThreads / 32];
  __shared__ int s_redi[kRowThreads / 32];
  __shared__ float s_max, s_sum;
  __shared__ int s_first;
  const int ranks = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int row = (int)(blockIdx.x / ranks);
  const float *x = a.x + (size_t)row * a.vocab;
  float *p = a.p + (size_t)row * a.vocab;
  const double t = a.temp ? (double)a.temp[row] : a.t;
  const int head = VEC ? min((int)((16 - ((uintptr_t)x & 15)) & 15) / 4, a.vocab) : 0;
  const int fours = VEC ? (a.vocab - head) / 4 : 0, share = (fours + ranks - 1) / ranks;
  const int b4 = min(rank * share, fours), e4 = min(b4 + share, fours);
  const float4 *x4 = reinterpret_cast<const float4 *>(x + head);
  float4 *p4 = reinterpret_cast<float4 *>(p + head);
  // single values of this rank: VEC the head (rank 0) and the rest (last rank), else a slice
  const int rest = head + 4 * fours;
  const int s0 = VEC ? (rank == ranks - 1 ? rest : a.vocab) : min(rank * a.slice, a.vocab);
  const int s1 = VEC ? a.vocab : min(s0 + a.slice, a.vocab);
  if (!(t >= 0.01)) {
    const int begin = min(rank * a.slice, a.vocab), end = min(begin + a.slice, a.vocab);
    float m = -INFINITY;
    for (int k = begin + (int)threadIdx.x; k < end; k += kRowThreads) m = fmaxf(m, x[k]);
    m = block_max<kRowThreads>(m, s_red);
    if (threadIdx.x == 0) s_max = m;
    cl.sync();
    for (int i = 0; i < ranks; i++) m = fmaxf(m, *cl.map_shared_rank(&s_max, i));
    one_hot<kRowThreads>(cl, x, p, begin, end, m, s_redi, &s_first);
    return;
  }
  const float c = log2e_over(t);
  // running maximum and sum of this thread
  float m = -INFINITY, sum = 0.f;
  auto take = [&](float top, auto &&weights) {  // weights(ref): sum of exp of the new values
    if (top > m) {
      sum *= exp_scaled(m - top, c);
      m = top;
    }
    sum += weights(m == -INFINITY ? 0.f : m);
  };
  auto e = [&](float y) { return exp_scaled(y, c); };
  constexpr int U = 4;  // loads under way
  // the first of the share stay in shared memory (each thread's own)
  __shared__ float4 s_keep[VEC ? kKeep : 1][kRowThreads];
  int n = 0;
  for (int k = b4 + (int)threadIdx.x; k < e4; k += U * kRowThreads, n += U) {
    float4 u[U];
#pragma unroll
    for (int i = 0; i < U; i++)
      u[i] = k + i * kRowThreads < e4 ? x4[k + i * kRowThreads] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
#pragma unroll
    for (int i = 0; i < U; i++)
      if (n + i < kKeep) s_keep[n + i][threadIdx.x] = u[i];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < U; i++) top = fmaxf(top, fmaxf(fmaxf(u[i].x, u[i].y), fmaxf(u[i].z, u[i].w)));
    take(top, [&](float r) {
      float w[U];
#pragma unroll
      for (int i = 0; i < U; i++) w[i] = (e(u[i].x - r) + e(u[i].y - r)) + (e(u[i].z - r) + e(u[i].w - r));
      return (w[0] + w[1]) + (w[2] + w[3]);
    });
  }
  auto single = [&](auto &&f) {
    if (VEC && rank == 0)
      for (int k = (int)threadIdx.x; k < head; k += kRowThreads) f(k);
    for (int k = s0 + (int)threadIdx.x; k < s1; k += kRowThreads) f(k);
  };
  single([&](int k) {
    const float y = x[k];
    take(y, [&](float r) { return e(y - r); });
  });
  // the row's, from those of the threads
  float top = block_max<kRowThreads>(m, s_red);
  if (threadIdx.x == 0) s_max = top;
  cl.sync();
  for (int i = 0; i < ranks; i++) top = fmaxf(top, *cl.map_shared_rank(&s_max, i));
  sum = block_sum<kRowThreads>(m == -INFINITY ? sum : sum * e(m - top), s_red);
  if (threadIdx.x == 0) s_sum = sum;
  cl.sync();
  sum = 0.f;
  for (int i = 0; i < ranks; i++) sum += *cl.map_shared_rank(&s_sum, i);
  const float inv = sum == 0.f ? 0.f : 1.f / sum, ref = top == -INFINITY ? 0.f : top;
  n = 0;
  for (int k = b4 + (int)threadIdx.x; k < e4; k += U * kRowThreads, n += U) {
    float4 u[U];
#pragma unroll
    for (int i = 0; i < U; i++)
      if (k + i * kRowThreads < e4) u[i] = n + i < kKeep ? s_keep[n + i][threadIdx.x] : __ldcs(x4 + k + i * kRowThreads);
#pragma unroll
    for (int i = 0; i < U; i++)
      if (k + i * kRowThreads < e4)
        __stcs(p4 + k + i * kRowThreads, make_float4(e(u[i].x - ref) * inv, e(u[i].y - ref) * inv, e(u[i].z - ref) * inv, e(u[i].w - ref) * inv));
  }
  single([&](int k) { p[k] = e(x[k] - ref) * inv; });
  cl.sync();
}

// ------------------------------------------------------------------ verification
constexpr int kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32;
constexpr int kRequests = 512;  // of one launch

struct VerifyArgs {
  const int32_t *drafts;
  const float *target, *draft, *u_accept, *u_sample;
  int32_t *tokens, *accepted;
  int n, req0, vocab, slice;  // req0: first request of the launch
  int32_t first[kRequests + 1];  // first draft of each request
};
static_assert(sizeof(VerifyArgs) <= 4096, "kernel parameters");

// Mass of an index: max(p - q, 0) in f64, p alone without q; NaN counts as 0.
// (`point`: the index whose q is 1 when the drafts were not drawn.)
__device__ __forceinline__ double mass(float p, float q) {
  return p > q ? (double)p - (double)q : 0.0;
}
struct Row {
  const float *p, *q;
  int point, end;
  // masses of the indices v + 32 u, u < N: all loads before the arithmetic
  template <int N>
  __device__ __forceinline__ void get(int v, double (&m)[N]) const {
    float a[N], b[N];
    if (q) {
#pragma unroll
      for (int u = 0; u < N; u++) {
        const bool in = v + u * 32 < end;
        a[u] = in ? __ldg(p + v + u * 32) : 0.f;
        b[u] = in ? __ldg(q + v + u * 32) : 0.f;
      }
    } else {
#pragma unroll
      for (int u = 0; u < N; u++) {
        a[u] = v + u * 32 < end ? __ldg(p + v + u * 32) : 0.f;
        b[u] = v + u * 32 == point ? 1.f : 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < N; u++) m[u] = mass(a[u], b[u]);
  }
};

__global__ void __launch_bounds__(kVerifyThreads) verify_drafts_kernel(const __grid_constant__ VerifyArgs a) {
  cg::cluster_group cl = cg::this_cluster();
  __shared__ double s_warp[kVerifyWarps], s_all[kMaxCluster * kVerifyWarps];
  __shared__ int s_refused;
  const int ranks = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int i = (int)(blockIdx.x / ranks), req = a.req0 + i;
  const int d0 = a.first[i], g = a.first[i + 1] - d0;
  const size_t row0 = (size_t)d0 + req;  // the target has one row more for each request before this one
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) s_refused = g;
  __syncthreads();
  for (int j = threadIdx.x; j < g; j += kVerifyThreads) {
    const int tok = a.drafts[d0 + j];
    bool ok = tok >= 0 && tok < a.vocab;
    if (ok) {
      const double p = (double)a.target[(row0 + j) * a.vocab + tok];
      const double q = a.draft ? (double)a.draft[(size_t)(d0 + j) * a.vocab + tok] : 1.0;
      ok = (double)a.u_accept[d0 + j] * q < p;
    }
    if (!ok) atomicMin(&s_refused, j);
  }
  __syncthreads();
  const int r = s_refused;
  Row row;
  row.p = a.target + (row0 + r) * a.vocab;
  row.q = r < g && a.draft ? a.draft + (size_t)(d0 + r) * a.vocab : nullptr;
  row.point = r < g && !a.draft ? a.drafts[d0 + r] : -1;
  // run k = rank * kVerifyWarps + warp of the cluster: a.slice consecutive indices
  const int begin = (int)min((long long)(rank * kVerifyWarps + warp) * a.slice, (long long)a.vocab);
  const int end = (int)min((long long)begin + a.slice, (long long)a.vocab);
  row.end = end;
  // sums of two runs per lane, and the sums up to and with each: the same
  // operations in the same order in every warp, so all agree on them
  constexpr int EACH = kMaxCluster * kVerifyWarps / 32;
  double sum[EACH], upto[EACH], total = 0.0;
  for (int pass = 0; pass < 2; pass++) {
    // four sums a lane: f64 additions take their time
    double part[4] = {0.0, 0.0, 0.0, 0.0};
    for (int v = begin + lane; v < end; v += 512) {
      double m[16];
      row.get(v, m);
#pragma unroll
      for (int u = 0; u < 16; u++) part[u & 3] += m[u];
    }
    double mine = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) s_warp[warp] = mine;
    cl.sync();
    for (int k = threadIdx.x; k < kMaxCluster * kVerifyWarps; k += kVerifyThreads)
      s_all[k] = k < ranks * kVerifyWarps ? cl.map_shared_rank(s_warp, k / kVerifyWarps)[k % kVerifyWarps] : 0.0;
    cl.sync();  // s_all is whole, and nobody reads this CTA's s_warp any more
    double carry = 0.0;
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      sum[e] = upto[e] = s_all[e * 32 + lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, upto[e], o);
        if (lane >= o) upto[e] += y;
      }
      upto[e] += carry;
      carry = __shfl_sync(0xffffffffu, upto[e], 31);
    }
    total = carry;
    // differences without mass (p and q equal but for rounding): p itself
    if (total > 0.0 || (!row.q && row.point < 0)) break;
    row.q = nullptr;
    row.point = -1;
    __syncthreads();  // s_warp and s_all are written again
  }
  const double want = (double)a.u_sample[req] * total;
  // the first run whose sum passes `want`; if rounding leaves `want` at the
  // very end, the last run with mass
  int pick = -1, last_run = -1;
#pragma unroll
  for (int e = 0; e < EACH; e++) {
    const unsigned hit = __ballot_sync(0xffffffffu, sum[e] > 0.0 && upto[e] > want);
    const unsigned any = __ballot_sync(0xffffffffu, sum[e] > 0.0);
    if (pick < 0 && hit) pick = e * 32 + __ffs(hit) - 1;
    if (any) last_run = e * 32 + 31 - __clz(any);
  }
  if (pick < 0) pick = last_run;
  int32_t *out = a.tokens + row0;
  if (pick == rank * kVerifyWarps + warp) {
    double run = 0.0;  // the sum before this run
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      const double y = __shfl_sync(0xffffffffu, upto[e], (pick - 1) & 31);
      if (pick > 0 && (pick - 1) / 32 == e) run = y;
    }
    // in steps of 32 blocks of 32 indices: the blocks' sums (eight reductions at
    // a time: their chains overlap), the block that passes `want`, the index in it
    int found = -1, last = begin;
    for (int v0 = begin; v0 < end && found < 0; v0 += 1024) {
      double block = 0.0;  // lane b: sum of block b
      for (int b0 = 0; b0 < 32; b0 += 8) {
        double t[8];
        row.get(v0 + b0 * 32 + lane, t);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
          for (int u = 0; u < 8; u++) t[u] += __shfl_xor_sync(0xffffffffu, t[u], o);
#pragma unroll
        for (int u = 0; u < 8; u++) block = lane == b0 + u ? t[u] : block;
      }
      double sum = block;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, block > 0.0 && run + sum > want);
      const unsigned any = __ballot_sync(0xffffffffu, block > 0.0);
      if (hit || any) {
        // inside the block that passes, or the last with mass
        const int b = hit ? __ffs(hit) - 1 : 31 - __clz(any);
        const double before = run + __shfl_sync(0xffffffffu, sum, b) - __shfl_sync(0xffffffffu, block, b);
        double m[1];
        row.get(v0 + b * 32 + lane, m);
        const double x = m[0];
        double upto_v = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, upto_v, o);
          if (lane >= o) upto_v += y;
        }
        const unsigned in = __ballot_sync(0xffffffffu, x > 0.0 && before + upto_v > want);
        last = v0 + b * 32 + 31 - __clz(__ballot_sync(0xffffffffu, x > 0.0));
        if (hit) found = in ? v0 + b * 32 + __ffs(in) - 1 : last;
      }
      run += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) out[r] = found >= 0 ? found : last;
  }
  if (rank == 0) {
    if (threadIdx.x == 0) {
      a.accepted[req] = r;
      if (!(total > 0.0)) out[r] = 0;
    }
    for (int j = threadIdx.x; j <= g; j += kVerifyThreads)
      if (j != r) out[j] = j < r ? a.drafts[d0 + j] : -1;
  }
}

template <typename K, typename A>
int launch_clusters(vxb_ctx *ctx, K kernel, const A &a, long long items, int cluster, int threads, cudaStream_t st, const char *what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(items * cluster));
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VXB_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, kernel, a));
  return launch_check(ctx, what);
}

}  // namespace

VXB_API int vxb_token_probs(vxb_ctx *ctx, const float *d_logits, int rows, int vocab, const float *d_temperature,
                            double temperature, float *d_probs, void *stream) {
  if (!ctx) return set_error(nullptr, VXB_EINVAL, "vxb_token_probs: null context");
  if (rows < 0 || vocab < 1) return set_error(ctx, VXB_EINVAL, "vxb_token_probs: bad shape rows=%d vocab=%d", rows, vocab);
  if (!d_temperature && !std::isfinite(temperature)) return set_error(ctx, VXB_EINVAL, "vxb_token_probs: temperature must be finite");
  if (vocab > kMaxVocab) return set_error(ctx, VXB_EUNSUPPORTED, "vxb_token_probs: vocab %d > %d", vocab, kMaxVocab);
  if (rows == 0) return VXB_OK;
  if (!d_logits || !d_probs) return set_error(ctx, VXB_EINVAL, "vxb_token_probs: null pointer");
  DeviceScope dev(ctx);
  if (dev.rc) return dev.rc;
  if (rows > INT_MAX / kMaxCluster) return set_error(ctx, VXB_EINVAL, "vxb_token_probs: %d rows", rows);
  ProbArgs a{d_logits, d_temperature, d_probs, vocab, 0, temperature};
  const int sms = ctx->num_sms > 0 ? ctx->num_sms : 148;
  cudaStream_t st = (cudaStream_t)stream;
  // Rows that fit the SMs' registers at once (two CTAs of up to 16 values a
  // thread, or one of 32) stay there; others are read twice.
  int cluster = 1;
  while (cluster < kMaxCluster && vocab > cluster * kProbThreads * 4) cluster *= 2;
  const int per = ((vocab + cluster - 1) / cluster + kProbThreads - 1) / kProbThreads;
  if (per <= 32 && (long long)rows * cluster <= (per <= 16 ? 2 : 1) * sms) {
    a.slice = (vocab + cluster - 1) / cluster;
    if (per <= 4) return launch_clusters(ctx, token_probs_kernel<4>, a, rows, cluster, kProbThreads, st, "token_probs_kernel");
    if (per <= 8) return launch_clusters(ctx, token_probs_kernel<8>, a, rows, cluster, kProbThreads, st, "token_probs_kernel");
    if (per <= 16) return launch_clusters(ctx, token_probs_kernel<16>, a, rows, cluster, kProbThreads, st, "token_probs_kernel");
    return launch_clusters(ctx, token_probs_kernel<32>, a, rows, cluster, kProbThreads, st, "token_probs_kernel");
  }
  // as many ranks to a row as keep one wave of resident CTAs (5 per SM), with a
  // round of loads a thread at least: a second wave of a few CTAs costs as much
  // as the first (400 rows of 32,000: 1 rank 22.3 us, 2 ranks 25.8)
  cluster = 1;
  while (cluster < kMaxCluster && (long long)rows * cluster * 2 <= 5 * sms && vocab > cluster * kRowThreads * 16) cluster *= 2;
  a.slice = (vocab + cluster - 1) / cluster;
  if (((uintptr_t)d_logits & 15) == ((uintptr_t)d_probs & 15))
    return launch_clusters(ctx, token_probs_rows_kernel<true>, a, rows, cluster, kRowThreads, st, "token_probs_rows_kernel");
  return launch_clusters(ctx, token_probs_rows_kernel<false>, a, rows, cluster, kRowThreads, st, "token_probs_rows_kernel");
}

VXB_API int vxb_verify_drafts(vxb_ctx *ctx, int n, const int32_t *h_n_drafts, int vocab, const int32_t *d_drafts,
                              const float *d_target_probs, const float *d_draft_probs, const float *d_u_accept,
                              const float *d_u_sample, int32_t *d_tokens, int32_t *d_n_accepted, void *stream) {
  if (!ctx) return set_error(nullptr, VXB_EINVAL, "vxb_verify_drafts: null context");
  if (n < 0 || vocab < 1 || (n > 0 && !h_n_drafts)) return set_error(ctx, VXB_EINVAL, "vxb_verify_drafts: bad arguments");
  if (vocab > kMaxVocab) return set_error(ctx, VXB_EUNSUPPORTED, "vxb_verify_drafts: vocab %d > %d", vocab, kMaxVocab);
  if (n == 0) return VXB_OK;
  long long total = 0;
  for (int i = 0; i < n; i++) {
    if (h_n_drafts[i] < 0) return set_error(ctx, VXB_EINVAL, "vxb_verify_drafts: request %d has %d drafts", i, h_n_drafts[i]);
    total += h_n_drafts[i];
  }
  if (total + n > INT_MAX) return set_error(ctx, VXB_EINVAL, "vxb_verify_drafts: %lld rows", total + n);
  if (!d_target_probs || !d_u_sample || !d_tokens || !d_n_accepted || (total > 0 && (!d_drafts || !d_u_accept)))
    return set_error(ctx, VXB_EINVAL, "vxb_verify_drafts: null pointer");
  DeviceScope dev(ctx);
  if (dev.rc) return dev.rc;
  VerifyArgs a;
  a.drafts = d_drafts;
  a.target = d_target_probs;
  a.draft = d_draft_probs;
  a.u_accept = d_u_accept;
  a.u_sample = d_u_sample;
  a.tokens = d_tokens;
  a.accepted = d_n_accepted;
  a.vocab = vocab;
  int cluster = 1;
  // (two CTAs fit an SM: a cluster size that needs a second wave is too large)
  const int sms = ctx->num_sms > 0 ? ctx->num_sms : 148;
  while (cluster < kMaxCluster && vocab > cluster * kVerifyThreads * 4 && (long long)n * cluster * 2 <= 2 * sms) cluster *= 2;
  a.slice = (int)(((long long)vocab + cluster * kVerifyThreads - 1) / (cluster * kVerifyThreads) * 32);
  long long at = 0;
  for (int i = 0; i < n; i += kRequests) {
    a.req0 = i;
    a.n = n - i < kRequests ? n - i : kRequests;
    for (int j = 0; j < a.n; j++) {
      a.first[j] = (int32_t)at;
      at += h_n_drafts[i + j];
    }
    a.first[a.n] = (int32_t)at;
    if (int rc = launch_clusters(ctx, verify_drafts_kernel, a, a.n, cluster, kVerifyThreads, (cudaStream_t)stream, "verify_drafts_kernel")) return rc;
  }
  return VXB_OK;
}
