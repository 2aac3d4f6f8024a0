// Token probabilities and verification of drafted tokens.
//
// vxb_token_probs: p = exp((x - max) / t) / sum per row of logits. Bound by
// reading the row once and writing it once, so a row stays in registers
// between the two: a cluster of up to 8 CTAs takes a row (32 values a thread
// at most), its maximum and its sum go through distributed shared memory.
//
// vxb_verify_drafts: the accept tests are a handful of gathers; the token that
// is drawn needs one row of p (and q): a cluster per request sums its slices
// in f64, finds the slice, the warp and at last the index where the cumulative
// sum passes the drawn share.
#include <climits>
#include <cmath>
#include <cooperative_groups.h>

#include "vxb_internal.h"

using namespace vxb;
namespace cg = cooperative_groups;

namespace {

constexpr int kMaxCluster = 8;

// ------------------------------------------------------------------ probabilities
constexpr int kProbThreads = 512;

struct ProbArgs {
  const float *x, *temp;
  float *p;
  int vocab, slice;  // a CTA's share of a row
  double t;
};

// max over a CTA (every thread gets it); NaN passed over
__device__ float block_max(float v, float *s) {
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = s[0];
  for (int i = 1; i < kProbThreads / 32; i++) r = fmaxf(r, s[i]);
  __syncthreads();
  return r;
}

__device__ float block_sum(float v, float *s) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = 0.f;
  for (int i = 0; i < kProbThreads / 32; i++) r += s[i];
  __syncthreads();
  return r;
}

__device__ int block_min(int v, int *s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = min(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  int r = s[0];
  for (int i = 1; i < kProbThreads / 32; i++) r = min(r, s[i]);
  __syncthreads();
  return r;
}

// exp(d) with d = (x - max) / t <= 0. c + c_lo = log2(e) / t: the rounding of
// d * c and the low part of c enter to first order, so the result keeps the
// special-function unit's 2 ulp however far d is from 0.
__device__ __forceinline__ float exp_scaled(float d, float c, float c_lo) {
  const float y = d * c;
  const float rest = fmaf(d, c_lo, fmaf(d, c, -y));
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
  return d == -INFINITY ? 0.f : fmaf(e, rest * 0.69314718055994531f, e);
}

// PER: values of a row that a thread holds (0: rows too long for a cluster's
// registers, read a second time)
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
  const bool greedy = !(t >= 0.01);
  float v[PER > 0 ? PER : 1];
  float m = -INFINITY;
  if constexpr (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int c = begin + i * kProbThreads + (int)threadIdx.x;
      v[i] = c < end ? __ldcs(x + c) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) m = fmaxf(m, v[i]);
  } else {
    for (int c = begin + (int)threadIdx.x; c < end; c += kProbThreads) m = fmaxf(m, x[c]);
  }
  m = block_max(m, s_red);
  if (threadIdx.x == 0) s_max = m;
  cl.sync();
  for (int i = 0; i < ranks; i++) m = fmaxf(m, *cl.map_shared_rank(&s_max, i));
  if (greedy) {
    int first = INT_MAX;
    if constexpr (PER > 0) {
#pragma unroll
      for (int i = PER - 1; i >= 0; i--)
        if (v[i] == m && m != -INFINITY) first = begin + i * kProbThreads + (int)threadIdx.x;
    } else {
      for (int c = begin + (int)threadIdx.x; c < end && first == INT_MAX; c += kProbThreads)
        if (x[c] == m && m != -INFINITY) first = c;
    }
    first = block_min(first, s_redi);
    if (threadIdx.x == 0) s_first = first;
    cl.sync();
    for (int i = 0; i < ranks; i++) first = min(first, *cl.map_shared_rank(&s_first, i));
    for (int c = begin + (int)threadIdx.x; c < end; c += kProbThreads) p[c] = c == first ? 1.f : 0.f;
    cl.sync();  // the others' shared memory stays until they have read it
    return;
  }
  const double c64 = 1.4426950408889634074 / t;
  const float c = (float)c64, c_lo = (float)(c64 - (double)c);
  float sum = 0.f;
  if (m != -INFINITY) {
    if constexpr (PER > 0) {
#pragma unroll
      for (int i = 0; i < PER; i++) {
        v[i] = exp_scaled(v[i] - m, c, c_lo);
        sum += v[i];
      }
    } else {
      for (int i = begin + (int)threadIdx.x; i < end; i += kProbThreads) sum += exp_scaled(x[i] - m, c, c_lo);
    }
  }
  sum = block_sum(sum, s_red);
  if (threadIdx.x == 0) s_sum = sum;
  cl.sync();
  sum = 0.f;
  for (int i = 0; i < ranks; i++) sum += *cl.map_shared_rank(&s_sum, i);
  const float inv = m == -INFINITY ? 0.f : 1.f / sum;
  if constexpr (PER > 0) {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int k = begin + i * kProbThreads + (int)threadIdx.x;
      if (k < end) p[k] = m == -INFINITY ? 0.f : v[i] * inv;
    }
  } else {
    for (int k = begin + (int)threadIdx.x; k < end; k += kProbThreads)
      p[k] = m == -INFINITY ? 0.f : exp_scaled(x[k] - m, c, c_lo) * inv;
  }
  cl.sync();
}

// ------------------------------------------------------------------ verification
constexpr int kVerifyThreads = 256, kVerifyWarps = kVerifyThreads / 32;
constexpr int kRequests = 512;  // of one launch

struct VerifyArgs {
  const int32_t *drafts;
  const float *target, *draft, *u_accept, *u_sample;
  int32_t *tokens, *accepted;
  int n, req0, vocab, slice;  // req0: first request of the launch
  int32_t first[kRequests + 1];  // first draft of each request
};
static_assert(sizeof(VerifyArgs) <= 4096, "kernel parameters");

// mass of index v: max(p - q, 0) in f64, p alone without q; NaN counts as 0
__device__ __forceinline__ double mass(const float *p, const float *q, int point, int v) {
  double r = (double)__ldg(p + v);
  if (q) r -= (double)__ldg(q + v);
  else if (v == point) r -= 1.0;
  return r > 0.0 ? r : 0.0;
}

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
  const float *p = a.target + (row0 + r) * a.vocab;
  const float *q = r < g && a.draft ? a.draft + (size_t)(d0 + r) * a.vocab : nullptr;
  int point = r < g && !a.draft ? a.drafts[d0 + r] : -1;
  // run k = rank * kVerifyWarps + warp of the cluster: a.slice consecutive indices
  const int begin = (int)min((long long)(rank * kVerifyWarps + warp) * a.slice, (long long)a.vocab);
  const int end = (int)min((long long)begin + a.slice, (long long)a.vocab);
  // sums of two runs per lane, and the sums up to and with each: the same
  // operations in the same order in every warp, so all agree on them
  constexpr int EACH = kMaxCluster * kVerifyWarps / 32;
  double sum[EACH], upto[EACH], total = 0.0;
  for (int pass = 0; pass < 2; pass++) {
    double mine = 0.0;
#pragma unroll 8
    for (int v = begin + lane; v < end; v += 32) mine += mass(p, q, point, v);
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
    if (total > 0.0 || (!q && point < 0)) break;
    q = nullptr;
    point = -1;
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
    int found = -1, last = begin;
    for (int v0 = begin; v0 < end && found < 0; v0 += 32) {
      const int v = v0 + lane;
      const double x = v < end ? mass(p, q, point, v) : 0.0;
      double s = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, x > 0.0 && run + s > want);
      const unsigned any = __ballot_sync(0xffffffffu, x > 0.0);
      if (any) last = v0 + 31 - __clz(any);
      if (hit) found = v0 + __ffs(hit) - 1;
      run += __shfl_sync(0xffffffffu, s, 31);
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
  if (rows == 0) return VXB_OK;
  if (!d_logits || !d_probs) return set_error(ctx, VXB_EINVAL, "vxb_token_probs: null pointer");
  DeviceScope dev(ctx);
  if (dev.rc) return dev.rc;
  if (rows > INT_MAX / kMaxCluster) return set_error(ctx, VXB_EINVAL, "vxb_token_probs: %d rows", rows);
  ProbArgs a{d_logits, d_temperature, d_probs, vocab, 0, temperature};
  const int sms = ctx->num_sms > 0 ? ctx->num_sms : 148;
  // the smallest cluster that holds a row in registers, a larger one while SMs are idle
  int cluster = 1;
  while (cluster < kMaxCluster && (long long)cluster * kProbThreads * 32 < vocab) cluster *= 2;
  while (cluster < kMaxCluster && (long long)rows * cluster * 2 <= sms && vocab > cluster * kProbThreads) cluster *= 2;
  a.slice = (vocab + cluster - 1) / cluster;
  const int per = (a.slice + kProbThreads - 1) / kProbThreads;
  cudaStream_t st = (cudaStream_t)stream;
  if (per <= 4) return launch_clusters(ctx, token_probs_kernel<4>, a, rows, cluster, kProbThreads, st, "token_probs_kernel");
  if (per <= 8) return launch_clusters(ctx, token_probs_kernel<8>, a, rows, cluster, kProbThreads, st, "token_probs_kernel");
  if (per <= 16) return launch_clusters(ctx, token_probs_kernel<16>, a, rows, cluster, kProbThreads, st, "token_probs_kernel");
  if (per <= 32) return launch_clusters(ctx, token_probs_kernel<32>, a, rows, cluster, kProbThreads, st, "token_probs_kernel");
  return launch_clusters(ctx, token_probs_kernel<0>, a, rows, cluster, kProbThreads, st, "token_probs_kernel");
}

VXB_API int vxb_verify_drafts(vxb_ctx *ctx, int n, const int32_t *h_n_drafts, int vocab, const int32_t *d_drafts,
                              const float *d_target_probs, const float *d_draft_probs, const float *d_u_accept,
                              const float *d_u_sample, int32_t *d_tokens, int32_t *d_n_accepted, void *stream) {
  if (!ctx) return set_error(nullptr, VXB_EINVAL, "vxb_verify_drafts: null context");
  if (n < 0 || vocab < 1 || (n > 0 && !h_n_drafts)) return set_error(ctx, VXB_EINVAL, "vxb_verify_drafts: bad arguments");
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
  while (cluster < kMaxCluster && vocab > cluster * kVerifyThreads * 4) cluster *= 2;
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
