"""Host arguments of the chunk and draft operators that no cast may change:
fractions, and numbers that the C ABI's types do not hold."""
import numpy as np
import pytest

from vortex_b200 import _native as N
from vortex_b200 import kv_cache, sampling

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("ids", [[1.7, 2], [1.0, 2.0], np.array([0.5, 3.0]), [2 ** 63, 1], np.array([2 ** 64 - 1, 1], np.uint64), [2 ** 70, 1],
                                 ["1", "2"], [[1, 2]], [True, False], [None, 1]])
def test_sequence_ids_are_whole_numbers_of_64_bits(ids):
    with pytest.raises(N.VxbError) as e:
        kv_cache._ids_counts("f", ids, [1, 1])
    assert e.value.code == N.VXB_EINVAL


@pytest.mark.parametrize("counts", [[-2 ** 32 + 5, 1], [-1, 1], np.array([-2 ** 31 - 1, 1]), [2 ** 31, 1], [2 ** 32 + 1, 1], [2 ** 70, 1], [0.5, 1]])
def test_counts_are_whole_numbers_of_32_bits(counts):
    with pytest.raises(N.VxbError):
        kv_cache._ids_counts("f", [1, 2], counts)
    p, u = torch.full((4, 8), 0.125), torch.zeros(3)
    with pytest.raises(N.VxbError) as e:
        sampling.verify_drafts(torch.zeros(2, dtype=torch.int32), counts, p, None, u[:2], u[:2])
    assert "n_drafts" in str(e.value)


def test_lengths_are_whole_numbers_of_64_bits():
    for bad in ([-2 ** 63, 1], [2 ** 63, 1], [1.5, 2]):
        with pytest.raises(N.VxbError):
            kv_cache._ids_counts("f", [1, 2], bad, np.dtype(np.int64))
    _, lens = kv_cache._ids_counts("f", [1, 2], [2 ** 40, 0], np.dtype(np.int64))
    assert lens.tolist() == [2 ** 40, 0]


def test_whole_numbers_of_any_kind_are_taken():
    for ids in ([-3, 2 ** 63 - 1], (-3, 2 ** 63 - 1), np.array([-3, 2 ** 63 - 1]), np.array([-3, 0, 2 ** 63 - 1])[::2], torch.tensor([-3, 2 ** 63 - 1])):
        for counts in ([0, 2 ** 31 - 1], np.array([0, 2 ** 31 - 1], np.uint32), np.array([0, 2 ** 31 - 1], np.int32), np.array([0, 9, 2 ** 31 - 1], np.int32)[::2]):
            i, c = kv_cache._ids_counts("f", ids, counts)
            assert i.dtype == np.int64 and i.tolist() == [-3, 2 ** 63 - 1] and i.flags.c_contiguous
            assert c.dtype == np.int32 and c.tolist() == [0, 2 ** 31 - 1] and c.flags.c_contiguous
    i, c = kv_cache._ids_counts("f", range(3), np.zeros(3, np.uint8))
    assert i.tolist() == [0, 1, 2] and c.tolist() == [0, 0, 0]
