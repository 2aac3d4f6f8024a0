// Paged KV cache on the device.
//
// Follows PagedKVCache (src/kv_cache.rs:29-93): a fixed pool of max_blocks
// blocks of block_size tokens, a block table per (layer, seq_id), a free-block
// stack initialised to (0..max_blocks).rev() so blocks are handed out 0, 1, 2,
// ...; append_kv pops a block when the sequence's last block is full;
// free_seq returns every block of the sequence (all layers) to the stack.
// The reference stores one f64 vector per token and never uses num_heads; here
// a token holds [num_kv_heads, head_dim] keys and values in bf16, or int8 with
// one f32 scale per (token, head) computed by calibrate_minmax
// (src/quantize.rs:585-591: absmax/127, all-zero -> 1.0) and codes
// round-half-away(v/scale) clamped to [-128, 127] (src/quantize.rs:105-108).
#include <algorithm>
#include <climits>
#include <cmath>

#include "kv_cache.h"

using namespace vxb;

namespace {

__device__ __forceinline__ void append_token(const KVPlace &p, int i, int layer, int H, int D, int bs, int max_seqs,
                                             int mbps, int is_int8, const uint16_t *__restrict__ k,
                                             const uint16_t *__restrict__ v, void *pool_k, void *pool_v,
                                             float *scale_k, float *scale_v, int32_t *tables, int32_t *lens) {
  const size_t row = (size_t)H * D;
  if (!is_int8) {
    // 16-byte pieces of the token's [H, D] keys and values
    const int pieces = (int)(row / 8);
    for (int c = threadIdx.x; c < 2 * pieces; c += blockDim.x) {
      const bool isv = c >= pieces;
      const int cc = isv ? c - pieces : c;
      const int h = (cc * 8) / D, dd = (cc * 8) % D;
      const uint4 val = *reinterpret_cast<const uint4 *>((isv ? v : k) + (size_t)i * row + (size_t)cc * 8);
      uint16_t *dst = reinterpret_cast<uint16_t *>(isv ? pool_v : pool_k) +
                      (((size_t)p.block * H + h) * bs + p.offset) * D + dd;
      *reinterpret_cast<uint4 *>(dst) = val;
    }
  } else {
    // one warp per (head, k|v) row: f64 absmax/127 scale, round-half-away codes
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    for (int r = warp; r < 2 * H; r += nw) {
      const bool isv = r >= H;
      const int h = isv ? r - H : r;
      const uint16_t *src = (isv ? v : k) + (size_t)i * row + (size_t)h * D;
      double m = 0.0;
      for (int dd = lane; dd < D; dd += 32) m = fmax(m, fabs((double)bf16_bits_to_f32(src[dd])));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
      const double scale = m == 0.0 ? 1.0 : m / 127.0;
      int8_t *dst = reinterpret_cast<int8_t *>(isv ? pool_v : pool_k) + (((size_t)p.block * H + h) * bs + p.offset) * D;
      for (int dd = lane; dd < D; dd += 32) {
        const double q = round((double)bf16_bits_to_f32(src[dd]) / scale);
        dst[dd] = (int8_t)(isnan(q) ? 0.0 : fmin(fmax(q, -128.0), 127.0));
      }
      if (lane == 0) (isv ? scale_v : scale_k)[((size_t)p.block * H + h) * bs + p.offset] = (float)scale;
    }
  }
  if (threadIdx.x == 0) {
    if (p.offset == 0) tables[((size_t)layer * max_seqs + p.slot) * mbps + p.pos / bs] = p.block;
    atomicMax(lens + (size_t)layer * max_seqs + p.slot, p.pos + 1);
  }
}

__global__ void kv_append_kernel(const KVPlace *__restrict__ places, int layer, int H, int D, int bs, int max_seqs,
                                 int mbps, int is_int8, const uint16_t *__restrict__ k, const uint16_t *__restrict__ v,
                                 void *pool_k, void *pool_v, float *scale_k, float *scale_v, int32_t *tables,
                                 int32_t *lens) {
  const int i = blockIdx.x;
  const KVPlace p = places[i];
  append_token(p, i, layer, H, D, bs, max_seqs, mbps, is_int8, k, v, pool_k, pool_v, scale_k, scale_v, tables, lens);
}

// ---- ragged chunks (vxb_kv_append_chunks)
//
// A launch covers consecutive packed rows of the call: `n` pieces, piece i the
// rows [row0_i, row0_{i+1}) that become tokens pos0_i, pos0_i + 1, ... of one
// sequence; ids lists the pool blocks of its positions from block pos0_i /
// block_size on, starting at ids[blk0_i]. The record travels by value (a kernel
// has up to 32,764 bytes of parameters), so an append needs no host-to-device
// copy and no staging buffer that a later call could overwrite.
struct ChunkPiece {
  int32_t slot, pos0, row0, blk0;
};
template <int PIECES, int IDS>
struct ChunkArgsOf {
  static constexpr int kPieces = PIECES, kIds = IDS;
  const uint16_t *k, *v;
  void *pool_k, *pool_v;
  float *scale_k, *scale_v;
  int32_t *tables, *lens;  // of the layer
  int H, bs, mbps, n, row_end, tokens;
  ChunkPiece piece[PIECES];
  int32_t ids[IDS];
};
// A record of 4 KB for drafts (an append for 40 sequences and its truncate take
// 17.3 us, 19.5 us with the large one), one of 32 KB for prompts (15,300 tokens of
// 8 heads of 128: 34.5 us in launches of 640 blocks, 27.6 us in one).
using FewChunks = ChunkArgsOf<64, 640>;
using ManyChunks = ChunkArgsOf<256, 6912>;
static_assert(sizeof(FewChunks) <= 4096 && sizeof(ManyChunks) <= 32764, "kernel parameters");

constexpr int kChunkThreads = 256;
constexpr int kChunkTokens = 64;  // most tokens of a CTA

// One (token, K or V, head) row of D values per D / 8 lanes, 16 bytes a lane;
// every thread loads four pieces before it stores them. Memory-bound: the
// rows are read once and written once (bf16), and the destination of a row is
// 2 D contiguous bytes. A CTA takes `tokens` tokens, enough for two rounds of
// loads at few heads. 15,300 tokens of 8 heads of 128 21 us (5.9 TB/s), 14,000
// of 32 heads 73 us (6.2 TB/s); drafts of 32 sequences 2 us, the launch.
template <int D, bool INT8, class Args>
__global__ void __launch_bounds__(kChunkThreads) kv_append_chunks_kernel(const __grid_constant__ Args a) {
  __shared__ int32_t s_block[kChunkTokens], s_off[kChunkTokens];
  const int first = a.piece[0].row0 + (int)blockIdx.x * a.tokens;
  const int count = min(a.tokens, a.row_end - first);
  for (int t = threadIdx.x; t < count; t += kChunkThreads) {
    const int row = first + t;
    int lo = 0, hi = a.n - 1;  // the last piece whose row0 <= row
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.piece[mid].row0 <= row) lo = mid;
      else hi = mid - 1;
    }
    const ChunkPiece p = a.piece[lo];
    const int pos = p.pos0 + (row - p.row0);
    const int index = pos / a.bs;
    const int block = a.ids[p.blk0 + index - p.pos0 / a.bs];
    s_block[t] = block;
    s_off[t] = pos - index * a.bs;
    if (s_off[t] == 0) a.tables[(size_t)p.slot * a.mbps + index] = block;
    const int end = lo + 1 < a.n ? a.piece[lo + 1].row0 : a.row_end;
    if (row + 1 == end) a.lens[p.slot] = pos + 1;
  }
  __syncthreads();
  constexpr int LANES = D / 8, ROWS = kChunkThreads / LANES, UNROLL = 4;
  const int lane = threadIdx.x % LANES, r0 = threadIdx.x / LANES;
  const int rows = count * 2 * a.H;  // (token, K | V, head)
  for (int first_row = 0; first_row < rows; first_row += ROWS * UNROLL) {  // the same rounds for every thread: warps shuffle below
    const int base = first_row + r0;
    uint4 val[UNROLL];
    size_t dst[UNROLL];
    bool isv[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const int r = base + u * ROWS;
      if (r >= rows) break;
      const int t = r / (2 * a.H), h2 = r - t * 2 * a.H;
      isv[u] = h2 >= a.H;
      const int h = isv[u] ? h2 - a.H : h2;
      val[u] = __ldcs(reinterpret_cast<const uint4 *>((isv[u] ? a.v : a.k) + (((size_t)(first + t) * a.H + h) * D + lane * 8)));
      dst[u] = ((size_t)s_block[t] * a.H + h) * a.bs + s_off[t];  // token row of the pool
    }
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const bool live = base + u * ROWS < rows;
      if constexpr (!INT8) {
        if (live) *reinterpret_cast<uint4 *>((uint16_t *)(isv[u] ? a.pool_v : a.pool_k) + dst[u] * D + lane * 8) = val[u];
      } else {
        // calibrate_minmax: scale = absmax / 127 in f64 (1 for a row of
        // zeros), code = v / scale rounded half away from zero. The f32
        // quotient is within 1e-4 of the f64 one (|code| <= 127, two
        // roundings and the reciprocal's), so only quotients within 1e-3 of
        // a half need the f64 division.
        const uint32_t w[4] = {live ? val[u].x : 0u, live ? val[u].y : 0u, live ? val[u].z : 0u, live ? val[u].w : 0u};
        float x[8], m = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[2 * e] = __uint_as_float(w[e] << 16);
          x[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
          m = fmaxf(m, fmaxf(fabsf(x[2 * e]), fabsf(x[2 * e + 1])));
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const double scale = m == 0.f ? 1.0 : (double)m / 127.0;
        const float inv = m == 0.f ? 1.f : 127.f / m;
        // a tiny or non-finite maximum leaves the f32 quotient's error bound
        const bool plain = m == 0.f || (m > 1e-30f && m < 1e30f);
        uint32_t out[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float q = x[e] * inv, aq = fabsf(q);
          const float n = floorf(aq + 0.5f);
          int code;
          if (plain && fabsf(aq - floorf(aq) - 0.5f) > 1e-3f) {
            code = (int)copysignf(n, q);
          } else {
            const double e64 = round((double)x[e] / scale);
            code = isnan(e64) ? 0 : (int)fmin(fmax(e64, -128.0), 127.0);
          }
          out[e >> 2] |= ((uint32_t)code & 0xFFu) << (8 * (e & 3));
        }
        if (live) {
          *reinterpret_cast<uint2 *>((int8_t *)(isv[u] ? a.pool_v : a.pool_k) + dst[u] * D + lane * 8) = make_uint2(out[0], out[1]);
          if (lane == 0) (isv[u] ? a.scale_v : a.scale_k)[dst[u]] = (float)scale;
        }
      }
    }
  }
}

// lens[layer][slot] = min(lens[layer][slot], len) for consecutive layers
constexpr int kCutSeqs = 256;
struct CutArgs {
  int32_t *lens;
  int n, max_seqs;
  int32_t slot[kCutSeqs], len[kCutSeqs];
};
__global__ void kv_cut_lens_kernel(const __grid_constant__ CutArgs a) {
  int32_t *row = a.lens + (size_t)blockIdx.x * a.max_seqs;
  for (int i = threadIdx.x; i < a.n; i += blockDim.x) row[a.slot[i]] = min(row[a.slot[i]], a.len[i]);
}

__global__ void kv_set_entry_kernel(int32_t *entry, int32_t block) { *entry = block; }

// get_kv (src/kv_cache.rs:69-80) for tests: dequantized f32 [len, H, D].
__global__ void kv_gather_kernel(const int32_t *__restrict__ table, int len, int H, int D, int bs, int is_int8,
                                 const void *pool_k, const void *pool_v, const float *scale_k, const float *scale_v,
                                 float *__restrict__ k_out, float *__restrict__ v_out) {
  const int pos = blockIdx.x;
  if (pos >= len) return;
  const int block = table[pos / bs], off = pos % bs;
  for (int e = threadIdx.x; e < H * D; e += blockDim.x) {
    const int h = e / D, dd = e % D;
    const size_t idx = (((size_t)block * H + h) * bs + off) * D + dd;
    const size_t o = (size_t)pos * H * D + e;
    if (!is_int8) {
      k_out[o] = bf16_bits_to_f32(reinterpret_cast<const uint16_t *>(pool_k)[idx]);
      v_out[o] = bf16_bits_to_f32(reinterpret_cast<const uint16_t *>(pool_v)[idx]);
    } else {
      const size_t si = ((size_t)block * H + h) * bs + off;
      k_out[o] = (float)reinterpret_cast<const int8_t *>(pool_k)[idx] * scale_k[si];
      v_out[o] = (float)reinterpret_cast<const int8_t *>(pool_v)[idx] * scale_v[si];
    }
  }
}

// The first `rows` token rows of every head of block `src` into block `dst`
// (keys, values and, for int8, their scales): the private copy of a forked
// sequence's partly filled last block.
__global__ void kv_copy_rows_kernel(uint8_t *pool_k, uint8_t *pool_v, float *scale_k, float *scale_v, int src, int dst,
                                    int H, int bs, int D, int elem, int rows) {
  const int h = blockIdx.x;
  const size_t row_bytes = (size_t)D * elem;
  const size_t so = ((size_t)src * H + h) * bs * row_bytes, d0 = ((size_t)dst * H + h) * bs * row_bytes;
  const size_t n = (size_t)rows * row_bytes;
  for (size_t i = threadIdx.x * 4; i < n; i += (size_t)blockDim.x * 4) {
    *reinterpret_cast<uint32_t *>(pool_k + d0 + i) = *reinterpret_cast<const uint32_t *>(pool_k + so + i);
    *reinterpret_cast<uint32_t *>(pool_v + d0 + i) = *reinterpret_cast<const uint32_t *>(pool_v + so + i);
  }
  if (scale_k)
    for (int r = threadIdx.x; r < rows; r += blockDim.x) {
      scale_k[((size_t)dst * H + h) * bs + r] = scale_k[((size_t)src * H + h) * bs + r];
      scale_v[((size_t)dst * H + h) * bs + r] = scale_v[((size_t)src * H + h) * bs + r];
    }
}

int kv_check(vxb_kv *kv, const char *who) {
  if (!kv || !kv->ctx) return set_error(nullptr, VXB_EINVAL, "%s: null cache", who);
  return VXB_OK;
}

}  // namespace

namespace vxb {

int kv_place(vxb_kv *kv, int layer, int64_t seq_id, KVPlace *out) {
  auto key = std::make_pair(layer, seq_id);
  auto it = kv->tables.find(key);
  int slot;
  auto si = kv->slot_of.find(seq_id);
  if (si == kv->slot_of.end()) {
    if (kv->free_slots.empty())
      return set_error(kv->ctx, VXB_ENOBLOCKS, "KV cache has no free sequence slot (max_seqs=%d)", kv->max_seqs);
    slot = kv->free_slots.back();
    kv->free_slots.pop_back();
    kv->slot_of[seq_id] = slot;
  } else {
    slot = si->second;
  }
  vxb_kv::Table &t = it == kv->tables.end() ? kv->tables[key] : it->second;
  const bool needs_block = t.blocks.empty() || t.len % kv->block_size == 0;
  if (needs_block) {
    if ((int)t.blocks.size() >= kv->max_blocks_per_seq)
      return set_error(kv->ctx, VXB_ENOBLOCKS, "sequence %lld exceeds max_blocks_per_seq=%d", (long long)seq_id,
                       kv->max_blocks_per_seq);
    if (kv->free_blocks.empty()) return set_error(kv->ctx, VXB_ENOBLOCKS, "KV cache out of blocks");
    t.blocks.push_back(kv->free_blocks.back());
    kv->refs[kv->free_blocks.back()] = 1;
    kv->free_blocks.pop_back();
  }
  out->block = t.blocks.back();
  out->offset = (int32_t)(t.len % kv->block_size);
  out->slot = slot;
  out->pos = (int32_t)t.len;
  t.len++;
  return VXB_OK;
}

void kv_release_block(vxb_kv *kv, int32_t b) {
  if (--kv->refs[b] <= 0) {
    kv->refs[b] = 0;
    kv->free_blocks.push_back(b);
  }
}

void kv_unplace(vxb_kv *kv, int layer, int64_t seq_id, int n) {
  auto it = kv->tables.find(std::make_pair(layer, seq_id));
  if (it == kv->tables.end()) return;
  vxb_kv::Table &t = it->second;
  for (int i = 0; i < n && t.len > 0; i++) {
    t.len--;
    if (t.len % kv->block_size == 0 && !t.blocks.empty()) {
      kv_release_block(kv, t.blocks.back());
      t.blocks.pop_back();
    }
  }
}

int kv_append_launch(vxb_kv *kv, int layer, int n, const KVPlace *d_places, const uint16_t *d_k, const uint16_t *d_v,
                     cudaStream_t st) {
  if (n <= 0) return VXB_OK;
  kv_append_kernel<<<n, 128, 0, st>>>(d_places, layer, kv->num_kv_heads, kv->head_dim, kv->block_size, kv->max_seqs,
                                      kv->max_blocks_per_seq, kv->dtype == VXB_I8, d_k, d_v, kv->pool_k, kv->pool_v,
                                      kv->scale_k, kv->scale_v, kv->d_tables, kv->d_lens);
  return launch_check(kv->ctx, "kv_append_kernel");
}

}  // namespace vxb

VXB_API int vxb_kv_create(vxb_ctx *ctx, int num_layers, int num_kv_heads, int head_dim, int block_size,
                          int max_blocks, int max_seqs, int max_blocks_per_seq, int kv_dtype, vxb_kv **out) {
  if (!ctx || !out) return set_error(ctx, VXB_EINVAL, "vxb_kv_create: null argument");
  *out = nullptr;
  if (num_layers <= 0 || num_kv_heads <= 0 || max_blocks <= 0 || max_seqs <= 0 || max_blocks_per_seq <= 0)
    return set_error(ctx, VXB_EINVAL, "vxb_kv_create: sizes must be positive");
  if (head_dim != 64 && head_dim != 128)
    return set_error(ctx, VXB_EUNSUPPORTED, "vxb_kv_create: head_dim %d (supported: 64, 128)", head_dim);
  if (block_size <= 0 || block_size % 16)
    return set_error(ctx, VXB_EINVAL, "vxb_kv_create: block_size %d must be a positive multiple of 16", block_size);
  if (kv_dtype != VXB_BF16 && kv_dtype != VXB_I8)
    return set_error(ctx, VXB_EINVAL, "vxb_kv_create: kv_dtype must be VXB_BF16 or VXB_I8");
  if (int rc = use_device(ctx)) return rc;
  if (int rc = ws_reserve(ctx, 0, 0)) return rc;  // device error word: later calls allocate nothing
  vxb_kv *kv = new vxb_kv();
  kv->ctx = ctx;
  kv->num_layers = num_layers;
  kv->num_kv_heads = num_kv_heads;
  kv->head_dim = head_dim;
  kv->block_size = block_size;
  kv->max_blocks = max_blocks;
  kv->max_seqs = max_seqs;
  kv->max_blocks_per_seq = max_blocks_per_seq;
  kv->dtype = kv_dtype;
  kv->elem_bytes = kv_dtype == VXB_I8 ? 1 : 2;
  const size_t pool = (size_t)max_blocks * num_kv_heads * block_size * head_dim * kv->elem_bytes;
  const size_t tbl = (size_t)num_layers * max_seqs * max_blocks_per_seq * sizeof(int32_t);
  const size_t lens = (size_t)num_layers * max_seqs * sizeof(int32_t);
  bool ok = cudaMalloc(&kv->pool_k, pool) == cudaSuccess && cudaMalloc(&kv->pool_v, pool) == cudaSuccess &&
            cudaMalloc((void **)&kv->d_tables, tbl) == cudaSuccess && cudaMalloc((void **)&kv->d_lens, lens) == cudaSuccess;
  if (ok && kv_dtype == VXB_I8) {
    const size_t sc = (size_t)max_blocks * num_kv_heads * block_size * sizeof(float);
    ok = cudaMalloc((void **)&kv->scale_k, sc) == cudaSuccess && cudaMalloc((void **)&kv->scale_v, sc) == cudaSuccess;
  }
  if (ok) ok = cudaMemset(kv->d_tables, 0xFF, tbl) == cudaSuccess && cudaMemset(kv->d_lens, 0, lens) == cudaSuccess;
  if (!ok) {
    cudaGetLastError();
    vxb_kv_destroy(kv);
    return set_error(ctx, VXB_ENOMEM, "vxb_kv_create: device allocation failed (pool %zu bytes x2)", pool);
  }
  kv->free_blocks.reserve(max_blocks);
  for (int b = max_blocks - 1; b >= 0; b--) kv->free_blocks.push_back(b);
  kv->refs.assign(max_blocks, 0);
  for (int s = max_seqs - 1; s >= 0; s--) kv->free_slots.push_back(s);
  *out = kv;
  return VXB_OK;
}

VXB_API int vxb_kv_destroy(vxb_kv *kv) {
  if (!kv) return VXB_OK;
  if (kv->ctx) use_device(kv->ctx);
  cudaFree(kv->pool_k);
  cudaFree(kv->pool_v);
  cudaFree(kv->scale_k);
  cudaFree(kv->scale_v);
  cudaFree(kv->d_tables);
  cudaFree(kv->d_lens);
  delete kv;
  return VXB_OK;
}

static int upload_places(vxb_kv *kv, const std::vector<KVPlace> &pl, cudaStream_t st, KVPlace **d_out) {
  const size_t bytes = pl.size() * sizeof(KVPlace);
  if (int rc = ws_reserve(kv->ctx, bytes, 0)) return rc;
  VXB_CUDA_TRY(kv->ctx, cudaMemcpyAsync(kv->ctx->ws, pl.data(), bytes, cudaMemcpyHostToDevice, st));
  *d_out = (KVPlace *)kv->ctx->ws;
  return VXB_OK;
}

VXB_API int vxb_kv_append(vxb_kv *kv, int layer, int n, const int64_t *h_seq_ids, const uint16_t *d_k,
                          const uint16_t *d_v, void *stream) {
  if (int rc = kv_check(kv, "vxb_kv_append")) return rc;
  if (layer < 0 || layer >= kv->num_layers) return set_error(kv->ctx, VXB_EINVAL, "vxb_kv_append: layer %d out of range", layer);
  if (n < 0 || (n > 0 && (!h_seq_ids || !d_k || !d_v))) return set_error(kv->ctx, VXB_EINVAL, "vxb_kv_append: bad arguments");
  if (n == 0) return VXB_OK;
  for (int i = 0; i < n; i++)
    for (int j = 0; j < i; j++)
      if (h_seq_ids[i] == h_seq_ids[j])
        return set_error(kv->ctx, VXB_EINVAL, "vxb_kv_append: sequence %lld listed twice", (long long)h_seq_ids[i]);
  if (int rc = use_device(kv->ctx)) return rc;
  std::vector<KVPlace> pl(n);
  for (int i = 0; i < n; i++) {
    if (int rc = kv_place(kv, layer, h_seq_ids[i], &pl[i])) {
      for (int j = i - 1; j >= 0; j--) kv_unplace(kv, layer, h_seq_ids[j], 1);
      return rc;
    }
  }
  KVPlace *d_pl = nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  if (int rc = upload_places(kv, pl, st, &d_pl)) return rc;
  return kv_append_launch(kv, layer, n, d_pl, d_k, d_v, st);
}

VXB_API int vxb_kv_append_seq(vxb_kv *kv, int layer, int64_t seq_id, int n_tokens, const uint16_t *d_k,
                              const uint16_t *d_v, void *stream) {
  if (int rc = kv_check(kv, "vxb_kv_append_seq")) return rc;
  if (layer < 0 || layer >= kv->num_layers) return set_error(kv->ctx, VXB_EINVAL, "vxb_kv_append_seq: layer out of range");
  if (n_tokens < 0 || (n_tokens > 0 && (!d_k || !d_v))) return set_error(kv->ctx, VXB_EINVAL, "vxb_kv_append_seq: bad arguments");
  if (n_tokens == 0) return VXB_OK;
  if (int rc = use_device(kv->ctx)) return rc;
  std::vector<KVPlace> pl(n_tokens);
  for (int i = 0; i < n_tokens; i++) {
    if (int rc = kv_place(kv, layer, seq_id, &pl[i])) {
      kv_unplace(kv, layer, seq_id, i);
      return rc;
    }
  }
  KVPlace *d_pl = nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  if (int rc = upload_places(kv, pl, st, &d_pl)) return rc;
  return kv_append_launch(kv, layer, n_tokens, d_pl, d_k, d_v, st);
}

namespace {

// A sequence listed twice in one call (the calls below change each sequence once)
bool listed_twice(const int64_t *ids, int n) {
  int rising = 1;
  while (rising < n && ids[rising - 1] < ids[rising]) rising++;
  if (rising >= n) return false;
  std::vector<int64_t> sorted(ids, ids + n);
  std::sort(sorted.begin(), sorted.end());
  return std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end();
}

// Drop the tokens of one table behind `len` (host side): emptied blocks go
// back to the free stack, the last one first, so that the same appends get the
// same blocks again.
void cut_table(vxb_kv *kv, vxb_kv::Table &t, int64_t len) {
  const int64_t keep = (len + kv->block_size - 1) / kv->block_size;
  while ((int64_t)t.blocks.size() > keep) {
    kv_release_block(kv, t.blocks.back());
    t.blocks.pop_back();
  }
  t.len = len;
}

// The device's lengths of (slot, length) pairs, in `layers` layers from one on
int cut_lens(vxb_kv *kv, int layer, int layers, const std::vector<std::pair<int, int64_t>> &cuts, cudaStream_t st) {
  CutArgs a;
  a.lens = kv->d_lens + (size_t)layer * kv->max_seqs;
  a.max_seqs = kv->max_seqs;
  for (size_t i = 0; i < cuts.size();) {
    a.n = 0;
    for (; i < cuts.size() && a.n < kCutSeqs; i++) {
      a.slot[a.n] = cuts[i].first;
      a.len[a.n++] = (int32_t)std::min<int64_t>(cuts[i].second, INT_MAX);
    }
    kv_cut_lens_kernel<<<layers, std::min(128, (a.n + 31) / 32 * 32), 0, st>>>(a);
    if (int rc = launch_check(kv->ctx, "kv_cut_lens_kernel")) return rc;
  }
  return VXB_OK;
}

struct AppendSeq {
  vxb_kv::Table *table;  // null: not there yet, or no tokens
  int64_t len;           // tokens before the call
  int slot;              // -1: none yet
};

// The launches of an append whose tables already hold the new tokens' blocks
template <class Args>
int write_chunks(vxb_kv *kv, int layer, const std::vector<AppendSeq> &seqs, const int32_t *counts, const uint16_t *d_k,
                 const uint16_t *d_v, cudaStream_t st) {
  vxb_ctx *ctx = kv->ctx;
  const int bs = kv->block_size, n = (int)seqs.size();
  Args a;
  a.k = d_k;
  a.v = d_v;
  a.pool_k = kv->pool_k;
  a.pool_v = kv->pool_v;
  a.scale_k = kv->scale_k;
  a.scale_v = kv->scale_v;
  a.tables = kv->d_tables + (size_t)layer * kv->max_seqs * kv->max_blocks_per_seq;
  a.lens = kv->d_lens + (size_t)layer * kv->max_seqs;
  a.H = kv->num_kv_heads;
  a.bs = bs;
  a.mbps = kv->max_blocks_per_seq;
  a.n = 0;
  int used = 0, row = 0, rc = VXB_OK;
  auto flush = [&]() {
    if (a.n == 0 || rc) return;
    a.row_end = row;
    const int rows = row - a.piece[0].row0;
    // two rounds of 4 x 16 bytes per thread at least, but CTAs for every SM first
    const int per_token = 2 * a.H * (kv->head_dim / 8);
    int tokens = (2 * 4 * kChunkThreads + per_token - 1) / per_token;
    const int sms = kv->ctx->num_sms > 0 ? kv->ctx->num_sms : 148;
    while (tokens > 1 && (rows + tokens - 1) / tokens < 2 * sms) tokens = (tokens + 1) / 2;
    a.tokens = std::min(tokens, kChunkTokens);
    const unsigned grid = (unsigned)((rows + a.tokens - 1) / a.tokens);
    const bool i8 = kv->dtype == VXB_I8;
    if (kv->head_dim == 128) {
      if (i8) kv_append_chunks_kernel<128, true, Args><<<grid, kChunkThreads, 0, st>>>(a);
      else kv_append_chunks_kernel<128, false, Args><<<grid, kChunkThreads, 0, st>>>(a);
    } else {
      if (i8) kv_append_chunks_kernel<64, true, Args><<<grid, kChunkThreads, 0, st>>>(a);
      else kv_append_chunks_kernel<64, false, Args><<<grid, kChunkThreads, 0, st>>>(a);
    }
    rc = launch_check(ctx, "kv_append_chunks_kernel");
    a.n = 0;
    used = 0;
  };
  for (int i = 0; i < n && !rc; i++) {
    int64_t pos = seqs[i].len;
    int left = counts[i];
    while (left > 0 && !rc) {
      if (a.n == Args::kPieces || used == Args::kIds) flush();
      // as many of the chunk's tokens as the remaining ids reach
      const int64_t b0 = pos / bs;
      const int64_t room = (int64_t)(Args::kIds - used) * bs - pos % bs;
      const int take = (int)std::min<int64_t>(left, room);
      const int64_t b1 = (pos + take + bs - 1) / bs;
      a.piece[a.n++] = {seqs[i].slot, (int32_t)pos, row, used};
      for (int64_t b = b0; b < b1; b++) a.ids[used++] = seqs[i].table->blocks[(size_t)b];
      pos += take;
      row += take;
      left -= take;
    }
  }
  flush();
  return rc;
}

int append_chunks(vxb_kv *kv, int layer, int n, const int64_t *ids, const int32_t *counts, const uint16_t *d_k,
                  const uint16_t *d_v, cudaStream_t st) {
  vxb_ctx *ctx = kv->ctx;
  const int bs = kv->block_size;
  int64_t total = 0, need = 0, spanned = 0;  // rows; new blocks; blocks that take rows
  size_t new_slots = 0;
  for (int i = 0; i < n; i++) {
    if (counts[i] < 0) return set_error(ctx, VXB_EINVAL, "vxb_kv_append_chunks: sequence %lld has %d tokens", (long long)ids[i], counts[i]);
    total += counts[i];
  }
  if (total > INT_MAX) return set_error(ctx, VXB_EINVAL, "vxb_kv_append_chunks: %lld rows", (long long)total);
  if (total == 0) return VXB_OK;
  if (!d_k || !d_v || ((uintptr_t)d_k | (uintptr_t)d_v) % 16)
    return set_error(ctx, VXB_EINVAL, "vxb_kv_append_chunks: d_k and d_v must be 16-byte aligned device pointers");
  if (listed_twice(ids, n))
    return set_error(ctx, VXB_EINVAL, "vxb_kv_append_chunks: a sequence is listed twice");
  // everything is checked before anything is taken
  std::vector<AppendSeq> seqs(n, AppendSeq{nullptr, 0, -1});
  TableFinder find(kv, layer);
  for (int i = 0; i < n; i++) {
    if (counts[i] == 0) continue;
    auto it = find(ids[i]);
    auto si = kv->slot_of.find(ids[i]);
    AppendSeq &q = seqs[i];
    if (it != kv->tables.end()) {
      q.table = &it->second;
      q.len = it->second.len;
    }
    if (si == kv->slot_of.end()) new_slots++;
    else q.slot = si->second;
    const int64_t have = (q.len + bs - 1) / bs, want = (q.len + counts[i] + bs - 1) / bs;
    if (want > kv->max_blocks_per_seq || q.len + counts[i] > INT_MAX)
      return set_error(ctx, VXB_ENOBLOCKS, "sequence %lld exceeds max_blocks_per_seq=%d", (long long)ids[i], kv->max_blocks_per_seq);
    need += want - have;
    spanned += want - q.len / bs;
  }
  if (need > (int64_t)kv->free_blocks.size()) return set_error(ctx, VXB_ENOBLOCKS, "KV cache out of blocks");
  if (new_slots > kv->free_slots.size())
    return set_error(ctx, VXB_ENOBLOCKS, "KV cache has no free sequence slot (max_seqs=%d)", kv->max_seqs);

  // host tables: blocks and lengths, remembered for the launches. What may
  // throw comes before what takes blocks.
  for (int i = 0; i < n; i++) {
    if (counts[i] == 0) continue;
    AppendSeq &q = seqs[i];
    if (!q.table) q.table = &kv->tables[std::make_pair(layer, ids[i])];
    const int64_t want = (q.len + counts[i] + bs - 1) / bs;
    if ((int64_t)q.table->blocks.capacity() < want) q.table->blocks.reserve((size_t)std::max<int64_t>(want, 2 * q.len / bs));
    if (q.slot < 0) {
      q.slot = kv->slot_of[ids[i]] = kv->free_slots.back();
      kv->free_slots.pop_back();
    }
  }
  for (int i = 0; i < n; i++) {
    if (counts[i] == 0) continue;
    vxb_kv::Table &t = *seqs[i].table;
    const int64_t want = (t.len + counts[i] + bs - 1) / bs;
    while ((int64_t)t.blocks.size() < want) {
      t.blocks.push_back(kv->free_blocks.back());
      kv->refs[kv->free_blocks.back()] = 1;
      kv->free_blocks.pop_back();
    }
    t.len += counts[i];
  }

  const int rc = n <= FewChunks::kPieces && spanned <= FewChunks::kIds ? write_chunks<FewChunks>(kv, layer, seqs, counts, d_k, d_v, st)
                                                                      : write_chunks<ManyChunks>(kv, layer, seqs, counts, d_k, d_v, st);
  if (rc) {
    // nothing was launched behind the failed launch: the tokens are taken back,
    // on the host and, as far as the stream still takes launches, in the lengths
    // that the launches before it wrote
    for (int i = n - 1; i >= 0; i--)
      if (seqs[i].table) cut_table(kv, *seqs[i].table, seqs[i].len);
    const std::string what = ctx->err;
    std::vector<std::pair<int, int64_t>> cuts;
    for (const AppendSeq &q : seqs)
      if (q.table) cuts.emplace_back(q.slot, q.len);
    if (cut_lens(kv, layer, 1, cuts, st)) set_error(ctx, rc, "%s", what.c_str());
  }
  return rc;
}

int truncate(vxb_kv *kv, int n, const int64_t *ids, const int64_t *lens, cudaStream_t st) {
  vxb_ctx *ctx = kv->ctx;
  const int bs = kv->block_size;
  for (int i = 0; i < n; i++)
    if (lens[i] < 0) return set_error(ctx, VXB_EINVAL, "vxb_kv_truncate: sequence %lld to %lld tokens", (long long)ids[i], (long long)lens[i]);
  if (listed_twice(ids, n)) return set_error(ctx, VXB_EINVAL, "vxb_kv_truncate: a sequence is listed twice");
  struct Cut {
    vxb_kv::Table *table;
    int64_t len;
    int layer, slot;
  };
  std::vector<Cut> cuts, moves;  // moves: cuts inside a shared block
  std::vector<int> slots(n, -1);
  for (int i = 0; i < n; i++) {
    auto si = kv->slot_of.find(ids[i]);
    if (si != kv->slot_of.end()) slots[i] = si->second;
  }
  for (int layer = 0; layer < kv->num_layers; layer++) {
    TableFinder find(kv, layer);
    for (int i = 0; i < n; i++) {
      if (slots[i] < 0) continue;
      auto it = find(ids[i]);
      if (it == kv->tables.end() || it->second.len <= lens[i]) continue;
      vxb_kv::Table &t = it->second;
      cuts.push_back({&t, lens[i], layer, slots[i]});
      if (lens[i] % bs && kv->refs[t.blocks[(size_t)(lens[i] / bs)]] > 1) moves.push_back(cuts.back());
    }
  }
  if (cuts.empty()) return VXB_OK;
  if (moves.size() > kv->free_blocks.size()) {
    // Do the blocks suffice that the cuts themselves free? Of every block: the
    // references that cuts in front of it take, and the cuts inside it, each of
    // which needs a copy, but for the last where no other sequence keeps the block.
    struct Use {
      int taken = 0, inside = 0;
    };
    std::map<int32_t, Use> uses;
    for (const Cut &c : cuts) {
      const std::vector<int32_t> &blocks = c.table->blocks;
      if (c.len % bs) uses[blocks[(size_t)(c.len / bs)]].inside++;
      for (size_t b = (size_t)((c.len + bs - 1) / bs); b < blocks.size(); b++) uses[blocks[b]].taken++;
    }
    int64_t left = (int64_t)kv->free_blocks.size();
    for (const auto &[block, use] : uses) {
      const int kept = kv->refs[block] - use.taken;  // references behind the cuts
      left += kept == 0;
      if (use.inside) left -= use.inside - (kept == use.inside);
    }
    if (left < 0) return set_error(ctx, VXB_ENOBLOCKS, "KV cache out of blocks");
  }
  std::vector<std::pair<int, int64_t>> kept;  // (what may throw comes before what changes)
  for (int i = 0; i < n; i++)
    if (slots[i] >= 0) kept.emplace_back(slots[i], lens[i]);
  // in the opposite order of the appends, so that they get the same blocks again
  for (auto c = cuts.rbegin(); c != cuts.rend(); ++c) cut_table(kv, *c->table, c->len);
  for (const Cut &c : moves) {
    const size_t index = (size_t)(c.len / bs);
    const int32_t from = c.table->blocks[index];
    if (kv->refs[from] <= 1) continue;  // the other holders were cut in this call
    const int32_t to = kv->free_blocks.back();
    kv->free_blocks.pop_back();
    kv->refs[to] = 1;
    kv->refs[from]--;
    c.table->blocks[index] = to;
    kv_copy_rows_kernel<<<kv->num_kv_heads, 256, 0, st>>>((uint8_t *)kv->pool_k, (uint8_t *)kv->pool_v, kv->scale_k, kv->scale_v, from, to,
                                                          kv->num_kv_heads, bs, kv->head_dim, (int)kv->elem_bytes, (int)(c.len % bs));
    if (int rc = launch_check(ctx, "kv_copy_rows_kernel")) return rc;
    kv_set_entry_kernel<<<1, 1, 0, st>>>(kv->d_tables + ((size_t)c.layer * kv->max_seqs + c.slot) * kv->max_blocks_per_seq + index, to);
    if (int rc = launch_check(ctx, "kv_set_entry_kernel")) return rc;
  }
  return cut_lens(kv, 0, kv->num_layers, kept, st);
}

}  // namespace

VXB_API int vxb_kv_append_chunks(vxb_kv *kv, int layer, int n, const int64_t *h_seq_ids, const int32_t *h_n_tokens,
                                 const uint16_t *d_k, const uint16_t *d_v, void *stream) {
  if (int rc = kv_check(kv, "vxb_kv_append_chunks")) return rc;
  if (layer < 0 || layer >= kv->num_layers) return set_error(kv->ctx, VXB_EINVAL, "vxb_kv_append_chunks: layer %d out of range", layer);
  if (n < 0 || (n > 0 && (!h_seq_ids || !h_n_tokens))) return set_error(kv->ctx, VXB_EINVAL, "vxb_kv_append_chunks: bad arguments");
  if (n == 0) return VXB_OK;
  DeviceScope dev(kv->ctx);
  if (dev.rc) return dev.rc;
  try {
    return append_chunks(kv, layer, n, h_seq_ids, h_n_tokens, d_k, d_v, (cudaStream_t)stream);
  } catch (...) {
    return set_error(kv->ctx, VXB_ENOMEM, "vxb_kv_append_chunks: out of host memory");
  }
}

VXB_API int vxb_kv_truncate(vxb_kv *kv, int n, const int64_t *h_seq_ids, const int64_t *h_lens, void *stream) {
  if (int rc = kv_check(kv, "vxb_kv_truncate")) return rc;
  if (n < 0 || (n > 0 && (!h_seq_ids || !h_lens))) return set_error(kv->ctx, VXB_EINVAL, "vxb_kv_truncate: bad arguments");
  if (n == 0) return VXB_OK;
  DeviceScope dev(kv->ctx);
  if (dev.rc) return dev.rc;
  try {
    return truncate(kv, n, h_seq_ids, h_lens, (cudaStream_t)stream);
  } catch (...) {
    return set_error(kv->ctx, VXB_ENOMEM, "vxb_kv_truncate: out of host memory");
  }
}

VXB_API int vxb_kv_pages(const vxb_kv *kv, void **d_k, void **d_v, float **d_k_scale, float **d_v_scale,
                         int32_t **d_tables, int32_t **d_lens) {
  if (!kv) return set_error(nullptr, VXB_EINVAL, "vxb_kv_pages: null cache");
  if (d_k) *d_k = kv->pool_k;
  if (d_v) *d_v = kv->pool_v;
  if (d_k_scale) *d_k_scale = kv->scale_k;
  if (d_v_scale) *d_v_scale = kv->scale_v;
  if (d_tables) *d_tables = kv->d_tables;
  if (d_lens) *d_lens = kv->d_lens;
  return VXB_OK;
}

VXB_API int vxb_kv_free_seq(vxb_kv *kv, int64_t seq_id) {
  if (int rc = kv_check(kv, "vxb_kv_free_seq")) return rc;
  bool any = false;
  for (int layer = 0; layer < kv->num_layers; layer++) {
    auto it = kv->tables.find(std::make_pair(layer, seq_id));
    if (it == kv->tables.end()) continue;
    any = true;
    for (int32_t b : it->second.blocks) kv_release_block(kv, b);
    kv->tables.erase(it);
  }
  auto si = kv->slot_of.find(seq_id);
  if (si != kv->slot_of.end()) {
    const int slot = si->second;
    kv->free_slots.push_back(slot);
    kv->slot_of.erase(si);
    if (int rc = use_device(kv->ctx)) return rc;
    // lengths of the freed slot go back to zero (tables are rewritten on reuse)
    for (int layer = 0; layer < kv->num_layers; layer++)
      VXB_CUDA_TRY(kv->ctx, cudaMemsetAsync(kv->d_lens + (size_t)layer * kv->max_seqs + slot, 0, sizeof(int32_t), 0));
    VXB_CUDA_TRY(kv->ctx, cudaStreamSynchronize(0));
  }
  (void)any;
  return VXB_OK;
}

VXB_API int vxb_kv_stats(const vxb_kv *kv, int64_t *out6) {
  if (!kv || !out6) return set_error(nullptr, VXB_EINVAL, "vxb_kv_stats: null argument");
  out6[0] = kv->max_blocks - (int64_t)kv->free_blocks.size();  // used_blocks
  out6[1] = (int64_t)kv->free_blocks.size();                   // free_blocks
  out6[2] = kv->block_size;                                    // block_size
  out6[3] = (int64_t)kv->tables.size();                        // num_seqs (tables, as the reference counts)
  out6[4] = out6[0] * kv->num_kv_heads * kv->block_size * kv->head_dim * (int64_t)kv->elem_bytes * 2;  // device bytes
  out6[5] = (int64_t)kv->slot_of.size();                       // distinct sequences
  return VXB_OK;
}

VXB_API int vxb_kv_seq_len(const vxb_kv *kv, int layer, int64_t seq_id, int64_t *len) {
  if (!kv || !len) return set_error(nullptr, VXB_EINVAL, "vxb_kv_seq_len: null argument");
  auto it = kv->tables.find(std::make_pair(layer, seq_id));
  *len = it == kv->tables.end() ? 0 : it->second.len;
  return VXB_OK;
}

VXB_API int vxb_kv_block_table(const vxb_kv *kv, int layer, int64_t seq_id, int32_t *h_out, int cap, int *n) {
  if (!kv || !n) return set_error(nullptr, VXB_EINVAL, "vxb_kv_block_table: null argument");
  auto it = kv->tables.find(std::make_pair(layer, seq_id));
  *n = it == kv->tables.end() ? 0 : (int)it->second.blocks.size();
  if (it != kv->tables.end() && h_out)
    for (int i = 0; i < *n && i < cap; i++) h_out[i] = it->second.blocks[i];
  return VXB_OK;
}

VXB_API int vxb_kv_gather(vxb_kv *kv, int layer, int64_t seq_id, float *d_k_out, float *d_v_out, void *stream) {
  if (int rc = kv_check(kv, "vxb_kv_gather")) return rc;
  auto it = kv->tables.find(std::make_pair(layer, seq_id));
  if (it == kv->tables.end() || it->second.len == 0) return VXB_OK;
  if (!d_k_out || !d_v_out) return set_error(kv->ctx, VXB_EINVAL, "vxb_kv_gather: null output");
  if (int rc = use_device(kv->ctx)) return rc;
  const int slot = kv->slot_of.at(seq_id);
  const int32_t *table = kv->d_tables + ((size_t)layer * kv->max_seqs + slot) * kv->max_blocks_per_seq;
  kv_gather_kernel<<<(unsigned)it->second.len, 128, 0, (cudaStream_t)stream>>>(
      table, (int)it->second.len, kv->num_kv_heads, kv->head_dim, kv->block_size, kv->dtype == VXB_I8, kv->pool_k,
      kv->pool_v, kv->scale_k, kv->scale_v, d_k_out, d_v_out);
  return launch_check(kv->ctx, "kv_gather_kernel");
}

// Prefix reuse: sequence dst_seq starts as the first n_tokens tokens of
// src_seq in every layer. Full blocks are shared (each block counts the
// tables holding it; a shared block is never written again: appends go to
// a sequence's own last block or to a new one), a partly filled last block is
// copied into a block of dst's own. The reference only declares a
// prefix_cache map (src/kv_cache.rs:37, 44) and never fills it.
VXB_API int vxb_kv_fork(vxb_kv *kv, int64_t src_seq, int64_t dst_seq, int64_t n_tokens, void *stream) {
  if (int rc = kv_check(kv, "vxb_kv_fork")) return rc;
  if (src_seq == dst_seq) return set_error(kv->ctx, VXB_EINVAL, "vxb_kv_fork: source and target are the same sequence");
  if (n_tokens < 0) return set_error(kv->ctx, VXB_EINVAL, "vxb_kv_fork: negative token count");
  for (int l = 0; l < kv->num_layers; l++) {
    auto d = kv->tables.find(std::make_pair(l, dst_seq));
    if (d != kv->tables.end() && d->second.len > 0)
      return set_error(kv->ctx, VXB_EINVAL, "vxb_kv_fork: sequence %lld already holds tokens", (long long)dst_seq);
    auto sit = kv->tables.find(std::make_pair(l, src_seq));
    const int64_t have = sit == kv->tables.end() ? 0 : sit->second.len;
    if (n_tokens > have)
      return set_error(kv->ctx, VXB_EINVAL, "vxb_kv_fork: sequence %lld holds %lld tokens in layer %d, %lld asked",
                       (long long)src_seq, (long long)have, l, (long long)n_tokens);
  }
  if (n_tokens == 0) return VXB_OK;
  const int bs = kv->block_size;
  const int64_t full = n_tokens / bs, rem = n_tokens % bs;
  if (full + (rem > 0) > kv->max_blocks_per_seq)
    return set_error(kv->ctx, VXB_ENOBLOCKS, "sequence %lld exceeds max_blocks_per_seq=%d", (long long)dst_seq,
                     kv->max_blocks_per_seq);
  if (rem > 0 && (int64_t)kv->free_blocks.size() < kv->num_layers)
    return set_error(kv->ctx, VXB_ENOBLOCKS, "KV cache out of blocks");
  int slot;
  auto si = kv->slot_of.find(dst_seq);
  if (si == kv->slot_of.end()) {
    if (kv->free_slots.empty())
      return set_error(kv->ctx, VXB_ENOBLOCKS, "KV cache has no free sequence slot (max_seqs=%d)", kv->max_seqs);
    slot = kv->free_slots.back();
    kv->free_slots.pop_back();
    kv->slot_of[dst_seq] = slot;
  } else {
    slot = si->second;
  }
  if (int rc = use_device(kv->ctx)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  std::vector<int32_t> tab;
  for (int l = 0; l < kv->num_layers; l++) {
    const vxb_kv::Table &s = kv->tables.at(std::make_pair(l, src_seq));
    vxb_kv::Table &t = kv->tables[std::make_pair(l, dst_seq)];
    t.blocks.assign(s.blocks.begin(), s.blocks.begin() + full);
    for (int32_t b : t.blocks) kv->refs[b]++;
    if (rem > 0) {
      const int32_t b = kv->free_blocks.back();
      kv->free_blocks.pop_back();
      kv->refs[b] = 1;
      kv_copy_rows_kernel<<<kv->num_kv_heads, 256, 0, st>>>(
          (uint8_t *)kv->pool_k, (uint8_t *)kv->pool_v, kv->scale_k, kv->scale_v, s.blocks[full], b, kv->num_kv_heads,
          bs, kv->head_dim, (int)kv->elem_bytes, (int)rem);
      if (int rc = launch_check(kv->ctx, "kv_copy_rows_kernel")) return rc;
      t.blocks.push_back(b);
    }
    t.len = n_tokens;
    tab = t.blocks;
    const size_t row = ((size_t)l * kv->max_seqs + slot);
    VXB_CUDA_TRY(kv->ctx, cudaMemcpyAsync(kv->d_tables + row * kv->max_blocks_per_seq, tab.data(),
                                          tab.size() * sizeof(int32_t), cudaMemcpyHostToDevice, st));
    const int32_t len = (int32_t)n_tokens;
    VXB_CUDA_TRY(kv->ctx, cudaMemcpyAsync(kv->d_lens + row, &len, sizeof(int32_t), cudaMemcpyHostToDevice, st));
    VXB_CUDA_TRY(kv->ctx, cudaStreamSynchronize(st));  // tab and len are host temporaries
  }
  return VXB_OK;
}
