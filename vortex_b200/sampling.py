"""Sampling and continuous batching over libvxb.so: host-side mirror of the
reference's argmax / sample_top_p (stdlib/ai/transformer.vx:1163-1260) and of
ContinuousBatcher with the batcher_* builtins (src/kv_cache.rs:117-154,
255-290). Logits are torch CUDA tensors; the sampling runs on the device.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _native as N
from .kv_cache import _whole_numbers
from .quant import _dptr, _stream_on, _stream_ptr, context

_I32 = np.dtype(np.int32)


def argmax(logits):
    """Greedy token per row (first index of the maximum): f32 [rows, vocab]."""
    import torch
    lg = logits.reshape(-1, logits.shape[-1]).contiguous()
    out = torch.empty(lg.shape[0], dtype=torch.int32, device=lg.device)
    context(lg.device.index).call("vxb_argmax", _dptr(lg), lg.shape[0], lg.shape[1], _dptr(out), _stream_ptr())
    return out


def sample_top_p(logits, temperature: float, top_p: float, seeds):
    """sample_top_p per row of f32 logits [rows, vocab] with one seed per row;
    returns int32 tokens on the device (bit-matched to the reference)."""
    import torch
    lg = logits.reshape(-1, logits.shape[-1]).contiguous().float()
    rows, vocab = lg.shape
    sd = np.ascontiguousarray(np.broadcast_to(np.asarray(seeds, dtype=np.int64), (rows,)))
    out = torch.empty(rows, dtype=torch.int32, device=lg.device)
    context(lg.device.index).call("vxb_sample_top_p", _dptr(lg), rows, vocab, ctypes.c_double(temperature),
                                  ctypes.c_double(top_p), sd.ctypes.data_as(ctypes.c_void_p), _dptr(out),
                                  _stream_ptr())
    return out


def _f32_rows(who: str, name: str, t, shape=None, device=None):
    """t as a contiguous f32 CUDA tensor (of this shape, on this device)."""
    import torch
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float32:
        raise N.VxbError(N.VXB_EINVAL, f"{who}: {name} must be an f32 tensor on the GPU")
    if shape is not None and t.shape != shape:
        raise N.VxbError(N.VXB_EINVAL, f"{who}: {name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if device is not None and t.get_device() != device:
        raise N.VxbError(N.VXB_EINVAL, f"{who}: {name} is on {t.device}, not on cuda:{device}")
    return t if t.is_contiguous() else t.contiguous()


def token_probs(logits, temperature=1.0, out=None):
    """Probabilities of f32 logits [..., vocab] at a temperature (one number,
    or an f32 tensor with one per row on the logits' device): exp((x - max) /
    t) / sum; below 0.01 1 at the first maximum. -inf logits (banned tokens)
    get 0, a row of nothing else zeros. out may be logits."""
    import torch
    lg = _f32_rows("token_probs", "logits", logits)
    if lg.dim() == 0 or lg.shape[-1] == 0:
        raise N.VxbError(N.VXB_EINVAL, "token_probs: logits must be [..., vocab]")
    vocab = lg.shape[-1]
    rows = lg.numel() // vocab
    if out is None:
        out = torch.empty_like(lg)
    elif _f32_rows("token_probs", "out", out, lg.shape, lg.get_device()) is not out:
        raise N.VxbError(N.VXB_EINVAL, "token_probs: out must be contiguous")
    per_row = None
    if isinstance(temperature, torch.Tensor):
        per_row = _f32_rows("token_probs", "temperature", temperature.reshape(-1), (rows,), lg.get_device())
    dev = lg.get_device()
    N.Context.get(dev).call("vxb_token_probs", lg.data_ptr(), rows, vocab, per_row.data_ptr() if per_row is not None else None,
                      1.0 if per_row is not None else float(temperature), out.data_ptr(),
                      _stream_on(dev))
    return out


def verify_drafts(drafts, n_drafts, target_probs, draft_probs, u_accept, u_sample):
    """Speculative sampling: accepts each request's drafts in order while
    u_accept * q(draft) < p(draft), then draws one token, from max(p - q, 0) of
    the first refused draft's row or from p of the row behind the last draft.

    drafts int32 [D] with n_drafts[i] (host counts) for request i, packed;
    target_probs f32 [D + n, vocab] (one row more per request than drafts);
    draft_probs f32 [D, vocab], or None where the drafts were not drawn (q is 1
    at the draft); u_accept f32 [D] and u_sample f32 [n] uniform in [0, 1).
    Returns (tokens int32 [D + n]: accepted drafts, the drawn token, then -1,
    per request; accepted int32 [n])."""
    import torch
    counts = _whole_numbers("verify_drafts", "n_drafts", n_drafts, _I32, least=0)
    per = counts.tolist()
    if per and min(per) < 0:
        raise N.VxbError(N.VXB_EINVAL, "verify_drafts: n_drafts must not be negative")
    n, total = len(per), sum(per)
    if not isinstance(target_probs, torch.Tensor) or target_probs.dim() != 2 or target_probs.shape[1] == 0:
        raise N.VxbError(N.VXB_EINVAL, "verify_drafts: target_probs must be [rows, vocab]")
    vocab = target_probs.shape[1]
    p = _f32_rows("verify_drafts", "target_probs", target_probs, (total + n, vocab))
    dev = p.get_device()
    q = None if draft_probs is None else _f32_rows("verify_drafts", "draft_probs", draft_probs, (total, vocab), dev)
    ua = _f32_rows("verify_drafts", "u_accept", u_accept, (total,), dev)
    us = _f32_rows("verify_drafts", "u_sample", u_sample, (n,), dev)
    if not isinstance(drafts, torch.Tensor) or drafts.dtype != torch.int32 or drafts.get_device() != dev or drafts.shape != (total,):
        raise N.VxbError(N.VXB_EINVAL, f"verify_drafts: drafts must be int32 ({total},) on cuda:{dev}")
    if not drafts.is_contiguous():
        drafts = drafts.contiguous()
    tokens, accepted = drafts.new_empty(total + n), drafts.new_empty(n)
    N.Context.get(dev).call("vxb_verify_drafts", n, counts.tobytes(), vocab, drafts.data_ptr(), p.data_ptr(),
                      q.data_ptr() if q is not None else None, ua.data_ptr(), us.data_ptr(), tokens.data_ptr(),
                      accepted.data_ptr(), _stream_on(dev))
    return tokens, accepted


class ContinuousBatcher:
    """ContinuousBatcher::new(max_batch_size) (src/kv_cache.rs:128-154)."""

    def __init__(self, max_batch_size: int = 32):
        p = ctypes.c_void_p()
        N.check(N.lib().vxb_batcher_create(int(max_batch_size), ctypes.byref(p)))
        self.ptr = p
        self.max_batch_size = int(max_batch_size)

    def __del__(self):
        try:
            if getattr(self, "ptr", None):
                N.lib().vxb_batcher_destroy(self.ptr)
                self.ptr = None
        except Exception:
            pass

    def add_request(self, tokens) -> int | None:
        """The slot taken, or None when every slot is busy (the batcher_add
        builtin turns that into the error "batcher full")."""
        t = np.ascontiguousarray(tokens, dtype=np.uint64)
        slot = ctypes.c_int(-1)
        rc = N.lib().vxb_batcher_add(self.ptr, t.ctypes.data_as(ctypes.c_void_p), t.size, ctypes.byref(slot))
        if rc == N.VXB_ENOBLOCKS:
            return None
        N.check(rc)
        return slot.value

    def remove_request(self, slot_id: int):
        N.check(N.lib().vxb_batcher_remove(self.ptr, int(slot_id)))

    def num_active(self) -> int:
        n = ctypes.c_int()
        N.check(N.lib().vxb_batcher_num_active(self.ptr, ctypes.byref(n)))
        return n.value

    def slot(self, slot_id: int) -> dict:
        sid, pos, pre, done = ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int(), ctypes.c_int()
        nt = ctypes.c_size_t()
        N.check(N.lib().vxb_batcher_slot(self.ptr, int(slot_id), ctypes.byref(sid), ctypes.byref(pos),
                                         ctypes.byref(pre), ctypes.byref(done), ctypes.byref(nt)))
        return {"seq_id": sid.value, "position": pos.value, "is_prefill": bool(pre.value),
                "is_done": bool(done.value), "n_tokens": nt.value}

    def advance(self, slot_id: int, n: int, done: bool = False):
        N.check(N.lib().vxb_batcher_advance(self.ptr, int(slot_id), int(n), int(done)))


def batcher_add(b: ContinuousBatcher, tokens) -> int:
    """The batcher_add builtin (src/kv_cache.rs:260-268): the slot, or the
    error "batcher full"."""
    slot = b.add_request(tokens)
    if slot is None:
        raise N.VxbError(N.VXB_ENOBLOCKS, "batcher full")
    return slot
