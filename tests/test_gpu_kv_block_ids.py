"""kv_build_tables with block ids that no slot can name."""
import numpy as np
import pytest
from test_gpu_kv_cache import run_tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block,shift", [(16, 4), (32, 5), (64, 6), (128, 7)])
def test_ids_whose_slots_do_not_fit(jkb, block, shift):
    """Of the free list and of a held block: no slot of another block comes out, and it is reported;
    the largest id that fits is as good as any."""
    most = 2**31 // block - 1
    table = np.full((2, 4), -1)
    table[1, 0] = 2 ** (32 - shift) + 5  # shifted, it would be block 5's
    new = [3 * block, 2]
    got = run_tables(jkb, table, [0, 3], new, [2 ** (32 - shift) + 3, most, 2], sum(new), block)
    with pytest.raises(jkb.TensorBoundsError):
        jkb.device_status()
    assert jkb.device_status() == 0
    off = np.arange(block, dtype=np.int64)
    want = np.concatenate([-np.ones(block), most * block + off, 2 * block + off, [-1, -1]])
    pos = np.concatenate([-np.ones(block), np.arange(block, 3 * block), [-1, -1]])
    assert np.array_equal(got[1], want) and np.array_equal(got[2], pos)
    assert got[5].tolist() == [sum(new), 3, 0]
    assert got[0][0, :3].tolist() == [2 ** (32 - shift) + 3, most, 2]


def test_ids_that_fit_are_not_reported(jkb):
    run_tables(jkb, np.full((1, 2), -1), [0], [20], [2**27 - 1, 0], 20, 16)
    assert jkb.device_status() == 0
