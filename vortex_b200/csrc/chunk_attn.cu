// Attention of chunks of new tokens over the paged KV cache: several queries
// of a sequence at once, each seeing the cached tokens up to its own.
//
//   O[r, h]   = sum_j exp(scale q_r . k_j - lse[r, h]) v_j,   j <= last(r)
//   lse[r, h] = log sum_j exp(scale q_r . k_j)
//
// with last(r) = len - n_queries + r (causal) or len - 1. One warp per (row,
// query head): the lanes share the head dimension, one pass over the visible
// keys with the running maximum and sum of the softmax in f32.
#include <climits>
#include <cmath>

#include <cuda_bf16.h>

#include "kv_cache.h"

using namespace vxb;

namespace {

constexpr int kSeqs = 128;  // sequences of one launch (their record is a kernel parameter)
struct ChunkSeq {
  int32_t slot, row0, rows, len;
};
struct ChunkArgs {
  const uint16_t *q;
  uint16_t *out;
  float *lse;
  const void *pool_k, *pool_v;
  const float *sk, *sv;
  const int32_t *tables;  // of the layer
  int n, rows, Hq, Hkv, G, bs, mbps, causal;
  float scale_log2;
  ChunkSeq seq[kSeqs];
};
static_assert(sizeof(ChunkArgs) <= 4096, "kernel parameters");

template <int D, bool INT8>
__global__ void __launch_bounds__(128) chunk_attn_kernel(const __grid_constant__ ChunkArgs a) {
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= (long long)a.rows * a.Hq) return;
  const int row = a.seq[0].row0 + (int)(item / a.Hq), head = (int)(item % a.Hq), hk = head / a.G;
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.seq[mid].row0 <= row) lo = mid;
    else hi = mid - 1;
  }
  const ChunkSeq s = a.seq[lo];
  const int keys = a.causal ? s.len - s.rows + (row - s.row0) + 1 : s.len;
  const int32_t *table = a.tables + (size_t)s.slot * a.mbps;
  const size_t at = ((size_t)row * a.Hq + head) * D + lane * PER;
  float q[PER], o[PER];
#pragma unroll
  for (int e = 0; e < PER; e++) {
    q[e] = bf16_bits_to_f32(a.q[at + e]);
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < keys; j++) {
    const size_t token = ((size_t)table[j / a.bs] * a.Hkv + hk) * a.bs + j % a.bs;
    float k[PER], v[PER], dot = 0.f;
#pragma unroll
    for (int e = 0; e < PER; e++) {
      if (INT8) {
        k[e] = (float)((const int8_t *)a.pool_k)[token * D + lane * PER + e] * a.sk[token];
        v[e] = (float)((const int8_t *)a.pool_v)[token * D + lane * PER + e] * a.sv[token];
      } else {
        k[e] = bf16_bits_to_f32(((const uint16_t *)a.pool_k)[token * D + lane * PER + e]);
        v[e] = bf16_bits_to_f32(((const uint16_t *)a.pool_v)[token * D + lane * PER + e]);
      }
      dot = fmaf(q[e], k[e], dot);
    }
    const float x = warp_sum(dot) * a.scale_log2;
    const float top = fmaxf(m, x);
    const float f = top == -INFINITY ? 1.f : exp2f(m - top), p = top == -INFINITY ? 0.f : exp2f(x - top);
    m = top;
    l = l * f + p;
#pragma unroll
    for (int e = 0; e < PER; e++) o[e] = o[e] * f + p * v[e];
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
  for (int e = 0; e < PER; e++) a.out[at + e] = __bfloat16_as_ushort(__float2bfloat16_rn(o[e] * inv));
  if (a.lse && lane == 0) a.lse[(size_t)row * a.Hq + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

int chunk_attention(vxb_kv *kv, int layer, int n, const int64_t *ids, const int32_t *counts, const uint16_t *d_q, int Hq,
                    float scale, int causal, uint16_t *d_out, float *d_lse, cudaStream_t st) {
  vxb_ctx *ctx = kv->ctx;
  int64_t total = 0;
  for (int i = 0; i < n; i++) {
    if (counts[i] < 0) return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: sequence %lld has %d queries", (long long)ids[i], counts[i]);
    total += counts[i];
  }
  if (total > INT_MAX) return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: %lld rows", (long long)total);
  if (total == 0) return VXB_OK;
  if (!d_q || !d_out || ((uintptr_t)d_q | (uintptr_t)d_out) % 16)
    return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: d_q and d_out must be 16-byte aligned device pointers");
  ChunkArgs a;
  a.q = d_q;
  a.out = d_out;
  a.lse = d_lse;
  a.pool_k = kv->pool_k;
  a.pool_v = kv->pool_v;
  a.sk = kv->scale_k;
  a.sv = kv->scale_v;
  a.tables = kv->d_tables + (size_t)layer * kv->max_seqs * kv->max_blocks_per_seq;
  a.Hq = Hq;
  a.Hkv = kv->num_kv_heads;
  a.G = Hq / kv->num_kv_heads;
  a.bs = kv->block_size;
  a.mbps = kv->max_blocks_per_seq;
  a.causal = causal;
  a.scale_log2 = scale * 1.44269504088896340736f;
  const bool i8 = kv->dtype == VXB_I8;
  int row = 0;
  for (int i = 0; i < n;) {
    a.n = 0;
    a.rows = -row;
    for (; i < n && a.n < kSeqs; i++) {
      if (counts[i] == 0) continue;
      auto it = kv->tables.find(std::make_pair(layer, ids[i]));
      const int len = it == kv->tables.end() ? 0 : (int)it->second.len;
      a.seq[a.n++] = {len > 0 ? kv->slot_of.at(ids[i]) : 0, row, counts[i], len};
      row += counts[i];
    }
    a.rows += row;
    if (a.n == 0) continue;
    const unsigned grid = (unsigned)(((long long)a.rows * Hq + 3) / 4);
    if (kv->head_dim == 128) {
      if (i8) chunk_attn_kernel<128, true><<<grid, 128, 0, st>>>(a);
      else chunk_attn_kernel<128, false><<<grid, 128, 0, st>>>(a);
    } else {
      if (i8) chunk_attn_kernel<64, true><<<grid, 128, 0, st>>>(a);
      else chunk_attn_kernel<64, false><<<grid, 128, 0, st>>>(a);
    }
    if (int rc = launch_check(ctx, "chunk_attn_kernel")) return rc;
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
  *ws_bytes = 256;
  return VXB_OK;
}

VXB_API int vxb_chunk_attention(vxb_kv *kv, int layer, int n, const int64_t *h_seq_ids, const int32_t *h_n_queries,
                                const uint16_t *d_q, int num_q_heads, float softmax_scale, int causal, uint16_t *d_out,
                                float *d_lse, void *d_ws, size_t ws_bytes, void *stream) {
  if (!kv || !kv->ctx) return set_error(nullptr, VXB_EINVAL, "vxb_chunk_attention: null cache");
  vxb_ctx *ctx = kv->ctx;
  if (layer < 0 || layer >= kv->num_layers) return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: layer %d out of range", layer);
  if (n < 0 || (n > 0 && (!h_seq_ids || !h_n_queries))) return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: bad arguments");
  if (!(softmax_scale > 0.f) || std::isinf(softmax_scale)) return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: scale must be positive and finite");
  size_t need = 0;
  if (int rc = vxb_chunk_attention_ws(kv, num_q_heads, &need)) return rc;
  if (n == 0) return VXB_OK;
  if (!d_ws || (uintptr_t)d_ws % 16 || ws_bytes < need)
    return set_error(ctx, VXB_EINVAL, "vxb_chunk_attention: %zu bytes of 16-byte aligned scratch needed, %zu given", need, d_ws ? ws_bytes : 0);
  DeviceScope dev(ctx);
  if (dev.rc) return dev.rc;
  try {
    return chunk_attention(kv, layer, n, h_seq_ids, h_n_queries, d_q, num_q_heads, softmax_scale, causal, d_out, d_lse, (cudaStream_t)stream);
  } catch (...) {
    return set_error(ctx, VXB_ENOMEM, "vxb_chunk_attention: out of host memory");
  }
}
