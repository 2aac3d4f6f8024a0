"""Refusals of the chunk and draft operators that need no GPU: null handles at
the C ABI, and the argument checks of the Python mirror before any device
call."""
import ctypes

import numpy as np
import pytest

from vortex_b200 import _native as N
from vortex_b200 import kv_cache, sampling

torch = pytest.importorskip("torch")


def test_null_handles_are_refused():
    L = N.lib()
    n = ctypes.c_size_t()
    assert L.vxb_kv_append_chunks(None, 0, 0, None, None, None, None, None) == N.VXB_EINVAL
    assert "vxb_kv_append_chunks" in N.last_error(None)
    assert L.vxb_kv_truncate(None, 0, None, None, None) == N.VXB_EINVAL
    assert L.vxb_kv_pages(None, None, None, None, None, None, None) == N.VXB_EINVAL
    assert L.vxb_chunk_attention_ws(None, 8, ctypes.byref(n)) == N.VXB_EINVAL
    assert L.vxb_chunk_attention(None, 0, 0, None, None, None, 8, 1.0, 1, None, None, None, 0, None) == N.VXB_EINVAL
    assert "vxb_chunk_attention" in N.last_error(None)
    assert L.vxb_token_probs(None, None, 0, 1, None, 1.0, None, None) == N.VXB_EINVAL
    assert L.vxb_verify_drafts(None, 0, None, 1, None, None, None, None, None, None, None, None) == N.VXB_EINVAL
    assert "vxb_verify_drafts" in N.last_error(None)


def test_ids_and_counts():
    ids, counts = kv_cache._ids_counts("f", [3, 1], [2, 0])
    assert ids.dtype == np.int64 and counts.dtype == np.int32 and list(counts) == [2, 0]
    ids, counts = kv_cache._ids_counts("f", 7, 4)
    assert list(ids) == [7] and list(counts) == [4]
    ids, counts = kv_cache._ids_counts("f", [], [])
    assert ids.size == 0 and counts.size == 0
    for bad in ([1], [1, -1], [1.5, 2.0], [1, 2 ** 31], [[1, 2]]):
        with pytest.raises(N.VxbError):
            kv_cache._ids_counts("f", [3, 1], bad)


def test_rows_must_be_bf16_on_the_caches_device():
    for t in (np.zeros((2, 1, 64)), torch.zeros(2, 1, 64), torch.zeros(2, 1, 64, dtype=torch.bfloat16)):
        with pytest.raises(N.VxbError):
            kv_cache._device_rows("f", "k", t, (2, 1, 64), 0)


def test_token_probs_and_verify_drafts_refuse_host_tensors():
    with pytest.raises(N.VxbError):
        sampling.token_probs(torch.zeros(2, 8))
    with pytest.raises(N.VxbError):
        sampling.token_probs(np.zeros((2, 8), np.float32))
    p, u = torch.full((3, 8), 0.125), torch.zeros(3)
    with pytest.raises(N.VxbError):
        sampling.verify_drafts(torch.zeros(2, dtype=torch.int32), [2], p, None, u[:2], u[:1])
    with pytest.raises(N.VxbError):
        sampling.verify_drafts(torch.zeros(2, dtype=torch.int32), [-2], p, None, u[:2], u[:1])
    with pytest.raises(N.VxbError):
        sampling.verify_drafts(torch.zeros(2, dtype=torch.int32), [1.0, 1.0], p, None, u[:2], u[:1])
