"""Paged KV cache and decode attention: host-side mirror of the reference's
PagedKVCache / paged_attention interface (src/kv_cache.rs:29-112) over
libvxb.so. Keys/values live in HBM; queries and outputs are torch CUDA tensors.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from . import _native as N
from .quant import _dptr, _stream_on, _stream_ptr, context

BF16 = N.BF16
I8 = N.I8


_I64 = np.dtype(np.int64)


def _whole_numbers(who: str, name: str, values, dtype, least=None):
    """values as a contiguous 1-D host array of dtype (itself where it is one);
    refused: fractions, other shapes, numbers that dtype does not hold and, in
    an array of another type, numbers under `least`."""
    if type(values) is np.ndarray and values.dtype == dtype and values.ndim == 1:
        return values if values.flags.c_contiguous else np.ascontiguousarray(values)
    a = np.atleast_1d(np.asarray(values))
    lo, hi = np.iinfo(dtype).min if least is None else least, np.iinfo(dtype).max
    if a.ndim != 1 or (a.size and (not np.issubdtype(a.dtype, np.integer) or int(a.min()) < lo or int(a.max()) > hi)):
        raise N.VxbError(N.VXB_EINVAL, f"{who}: {name} must be one list of whole numbers from {lo} to {hi}")
    return a.astype(dtype)


def _ids_counts(who: str, seq_ids, counts, dtype=np.dtype(np.int32)):
    """Host arrays of one sequence id and one count (or length) each."""
    ids = _whole_numbers(who, "seq_ids", seq_ids, _I64)
    c = _whole_numbers(who, "the counts", counts, dtype, least=0)  # (a negative one in an array of dtype is refused by the call)
    if ids.size != c.size:
        raise N.VxbError(N.VXB_EINVAL, f"{who}: {ids.size} sequences and {c.size} counts")
    return ids, c


def _device_rows(who: str, name: str, t, shape, device: int):
    """t as a contiguous, 16-byte aligned bf16 tensor of this shape on the cache's device."""
    import torch
    if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16 or not t.is_cuda or t.get_device() != device:
        raise N.VxbError(N.VXB_EINVAL, f"{who}: {name} must be a bf16 tensor on cuda:{device}")
    if t.shape != shape:
        raise N.VxbError(N.VXB_EINVAL, f"{who}: {name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _DeviceArray:
    """Device memory of a cache for torch.as_tensor; the tensor keeps the cache alive."""

    def __init__(self, owner, ptr: int, shape, typestr: str):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": tuple(shape), "typestr": typestr, "version": 3}


class PagedKVCache:
    """PagedKVCache::new(num_layers, num_heads, head_dim, block_size, max_blocks)
    (src/kv_cache.rs:41-45); num_heads are the KV heads of a token."""

    def __init__(self, num_layers: int, num_heads: int, head_dim: int, block_size: int = 16,
                 max_blocks: int = 256, max_seqs: int = 64, max_blocks_per_seq: int | None = None,
                 kv_dtype: int = BF16, device=None):
        self.ctx = context(device)
        self.num_layers, self.num_heads, self.head_dim = num_layers, num_heads, head_dim
        self.block_size, self.max_blocks = block_size, max_blocks
        self.kv_dtype = kv_dtype
        mbps = max_blocks_per_seq or max_blocks
        self.max_seqs, self.max_blocks_per_seq = max_seqs, mbps
        self._chunk_ws = {}  # num_q_heads -> scratch bytes of chunk_attention
        p = ctypes.c_void_p()
        N.check(N.lib().vxb_kv_create(self.ctx.ptr, num_layers, num_heads, head_dim, block_size, max_blocks,
                                      max_seqs, mbps, kv_dtype, ctypes.byref(p)), self.ctx.ptr)
        self.ptr = p

    def __del__(self):
        try:
            if getattr(self, "ptr", None):
                N.lib().vxb_kv_destroy(self.ptr)
                self.ptr = None
        except Exception:
            pass

    def _check(self, rc):
        if rc != N.VXB_OK:
            raise N.VxbError(rc, N.last_error(self.ctx.ptr))

    def append_kv(self, layer: int, seq_ids, k, v):
        """One token per listed sequence: k, v bf16 [n, H, D] on the device."""
        ids = np.ascontiguousarray(np.atleast_1d(seq_ids), dtype=np.int64)
        k = k.contiguous()
        v = v.contiguous()
        self._check(N.lib().vxb_kv_append(self.ptr, layer, ids.size, ids.ctypes.data_as(ctypes.c_void_p),
                                          _dptr(k), _dptr(v), _stream_ptr()))

    def append_seq(self, layer: int, seq_id: int, k, v):
        """Many tokens of one sequence: k, v bf16 [T, H, D]."""
        k = k.contiguous()
        v = v.contiguous()
        T = k.shape[0]
        self._check(N.lib().vxb_kv_append_seq(self.ptr, layer, int(seq_id), T, _dptr(k), _dptr(v), _stream_ptr()))

    def append_chunks(self, layer: int, seq_ids, n_tokens, k, v):
        """Ragged chunks: n_tokens[i] consecutive tokens of each listed
        sequence, their rows packed one sequence after another: k, v bf16
        [sum(n_tokens), H, D]."""
        ids, counts = _ids_counts("append_chunks", seq_ids, n_tokens)
        want = (sum(counts.tolist()), self.num_heads, self.head_dim)
        k = _device_rows("append_chunks", "k", k, want, self.ctx.device)
        v = _device_rows("append_chunks", "v", v, want, self.ctx.device)
        self._check(N.lib().vxb_kv_append_chunks(self.ptr, layer, ids.size, ids.tobytes(), counts.tobytes(),
                                                 k.data_ptr(), v.data_ptr(), _stream_on(self.ctx.device)))

    def truncate(self, seq_ids, lengths):
        """Takes appended tokens back: every layer of seq_ids[i] holds at most
        lengths[i] tokens afterwards."""
        ids, lens = _ids_counts("truncate", seq_ids, lengths, _I64)
        self._check(N.lib().vxb_kv_truncate(self.ptr, ids.size, ids.tobytes(), lens.tobytes(),
                                            _stream_on(self.ctx.device)))

    def pages(self) -> dict:
        """The cache's device memory as tensors that share it: k, v
        [max_blocks, H, block_size, D], tables [layers, max_seqs,
        max_blocks_per_seq] and lens [layers, max_seqs] (int32); int8 caches
        also k_scale, v_scale [max_blocks, H, block_size]."""
        import torch
        p = [ctypes.c_void_p() for _ in range(6)]
        self._check(N.lib().vxb_kv_pages(self.ptr, *(ctypes.addressof(x) for x in p)))
        page = (self.max_blocks, self.num_heads, self.block_size, self.head_dim)
        seqs = (self.num_layers, self.max_seqs, self.max_blocks_per_seq)

        def view(ptr, shape, typestr):
            return torch.as_tensor(_DeviceArray(self, ptr.value, shape, typestr), device=f"cuda:{self.ctx.device}")

        int8 = self.kv_dtype == I8
        out = {}
        for name, ptr in (("k", p[0]), ("v", p[1])):
            t = view(ptr, page, "|i1" if int8 else "<i2")
            out[name] = t if int8 else t.view(torch.bfloat16)
        if int8:
            out["k_scale"], out["v_scale"] = view(p[2], page[:3], "<f4"), view(p[3], page[:3], "<f4")
        out["tables"], out["lens"] = view(p[4], seqs, "<i4"), view(p[5], seqs[:2], "<i4")
        return out

    def get_kv(self, layer: int, seq_id: int):
        """PagedKVCache::get_kv: (keys, values) as f32 [len, H, D] tensors."""
        import torch
        n = self.seq_len(layer, seq_id)
        k = torch.empty((n, self.num_heads, self.head_dim), dtype=torch.float32, device="cuda")
        v = torch.empty_like(k)
        if n:
            self._check(N.lib().vxb_kv_gather(self.ptr, layer, int(seq_id), _dptr(k), _dptr(v), _stream_ptr()))
        return k, v

    def free_seq(self, seq_id: int):
        self._check(N.lib().vxb_kv_free_seq(self.ptr, int(seq_id)))

    def fork(self, src_seq: int, dst_seq: int, n_tokens: int):
        """Prefix reuse: dst_seq starts as the first n_tokens tokens of
        src_seq (full blocks shared, a partial last block copied)."""
        self._check(N.lib().vxb_kv_fork(self.ptr, int(src_seq), int(dst_seq), int(n_tokens), _stream_ptr()))

    def stats(self) -> dict:
        out = (ctypes.c_int64 * 6)()
        self._check(N.lib().vxb_kv_stats(self.ptr, out))
        return {"used_blocks": out[0], "free_blocks": out[1], "block_size": out[2], "num_seqs": out[3],
                "device_bytes": out[4], "sequences": out[5]}

    def used_blocks(self) -> int:
        return self.stats()["used_blocks"]

    def free_block_count(self) -> int:
        return self.stats()["free_blocks"]

    def seq_len(self, layer: int, seq_id: int) -> int:
        n = ctypes.c_int64()
        self._check(N.lib().vxb_kv_seq_len(self.ptr, layer, int(seq_id), ctypes.byref(n)))
        return n.value

    def block_table(self, layer: int, seq_id: int) -> list[int]:
        n = ctypes.c_int()
        self._check(N.lib().vxb_kv_block_table(self.ptr, layer, int(seq_id), None, 0, ctypes.byref(n)))
        buf = (ctypes.c_int32 * max(n.value, 1))()
        self._check(N.lib().vxb_kv_block_table(self.ptr, layer, int(seq_id), buf, n.value, ctypes.byref(n)))
        return list(buf[:n.value])

    def attention(self, layer: int, seq_ids, q, softmax_scale: float | None = None, out=None, lse=None):
        """paged_attention for one new query per sequence: q bf16 [n, Hq, D]
        -> bf16 [n, Hq, D] (and the natural-log sum-exp if lse is given)."""
        import torch
        ids = np.ascontiguousarray(np.atleast_1d(seq_ids), dtype=np.int64)
        q = q.contiguous()
        Hq = q.shape[1]
        if out is None:
            out = torch.empty_like(q)
        scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(self.head_dim)
        self._check(N.lib().vxb_decode_attention(self.ptr, layer, ids.size, ids.ctypes.data_as(ctypes.c_void_p),
                                                 _dptr(q), Hq, ctypes.c_float(scale), _dptr(out),
                                                 _dptr(lse) if lse is not None else None, _stream_ptr()))
        return out

    def chunk_attention(self, layer: int, seq_ids, n_queries, q, softmax_scale: float | None = None,
                        causal: bool = True, out=None, lse=None):
        """Attention of several queries per sequence: the n_queries[i] rows of
        seq_ids[i] (packed, q bf16 [sum(n_queries), Hq, D]) are its last
        n_queries[i] cached tokens; each sees the tokens up to its own (all of
        them with causal=False). Returns bf16 like q (and fills lse f32 [rows,
        Hq] if given). Rows that see nothing are zeros with lse -inf. Softmax
        weights are rounded once, to bf16 (int8 caches: f16); attention() keeps
        more bits of them."""
        import torch
        ids, counts = _ids_counts("chunk_attention", seq_ids, n_queries)
        rows, dev = sum(counts.tolist()), self.ctx.device
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise N.VxbError(N.VXB_EINVAL, "chunk_attention: q must be [rows, Hq, D]")
        Hq = q.shape[1]
        shape = (rows, Hq, self.head_dim)
        q = _device_rows("chunk_attention", "q", q, shape, dev)
        if out is None:
            out = torch.empty_like(q)
        elif out is not _device_rows("chunk_attention", "out", out, shape, dev):
            raise N.VxbError(N.VXB_EINVAL, "chunk_attention: out must be contiguous and 16-byte aligned")
        if lse is not None and (not isinstance(lse, torch.Tensor) or lse.dtype != torch.float32 or lse.get_device() != dev or not lse.is_contiguous()
                                or lse.shape != shape[:2]):
            raise N.VxbError(N.VXB_EINVAL, f"chunk_attention: lse must be contiguous f32 {shape[:2]} on cuda:{dev}")
        need = self._chunk_ws.get(Hq)
        if need is None:
            n = ctypes.c_size_t()
            self._check(N.lib().vxb_chunk_attention_ws(self.ptr, Hq, ctypes.byref(n)))
            need = self._chunk_ws[Hq] = n.value
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(self.head_dim)
        self._check(N.lib().vxb_chunk_attention(self.ptr, layer, ids.size, ids.tobytes(), counts.tobytes(),
                                                q.data_ptr(), Hq, scale, int(causal), out.data_ptr(),
                                                lse.data_ptr() if lse is not None else None, ws.data_ptr(), need,
                                                _stream_on(dev)))
        return out
