"""What BlockManager.plan_compact takes for rows: whole numbers of any width, none of which wraps into a sequence; a
mask or fractions are refused."""
import numpy as np
import pytest

from atomflow_amd import AF_ERR_OUT_OF_RANGE, kv


def manager():
    bm = kv.BlockManager(8, 8)
    s = bm.seq_create()
    bm.seq_extend(s, 20)
    return bm, s


@pytest.mark.parametrize("keep", [
    np.array([3, 2 ** 32 + 5]), np.array([-2 ** 32 + 3, 5]), np.array([2 ** 31]), np.array([2 ** 40, 2 ** 41]),
    np.array([2 ** 64 - 1], np.uint64)])
def test_rows_past_32_bits(keep):
    bm, s = manager()
    assert bm.plan_compact([s], [keep]) == AF_ERR_OUT_OF_RANGE
    assert bm.seq_len(s) == 20
    bm.close()


@pytest.mark.parametrize("keep", [np.array([False, True]), [0.5, 1.5], np.array([1.0, 2.0])])
def test_not_whole_numbers(keep):
    bm, s = manager()
    with pytest.raises(ValueError):
        bm.plan_compact([s], [keep])
    assert bm.seq_len(s) == 20
    bm.close()


@pytest.mark.parametrize("dtype", [np.int8, np.uint8, np.int32, np.int64, np.uint64])
def test_whole_numbers(dtype):
    bm, s = manager()
    plan = bm.plan_compact([s], [np.array([1, 4, 19], dtype)])
    assert list(plan["keep"]) == [1, 4, 19] and bm.seq_len(s) == 3
    assert bm.plan_compact([s], [[]])["max_rows"] == 0 and bm.seq_len(s) == 0
    bm.close()
