"""kv_build_tables reads its inputs while it writes its outputs: outputs that share memory with an
input or another output are refused before anything runs."""
import numpy as np
import pytest
import torch
from test_gpu_kv_cache import check_tables, i32

pytestmark = pytest.mark.gpu

NAMES = ("block_table", "slots", "positions", "q_starts", "kv_lens", "counts", "ctx_lens",
         "new_lens", "free_blocks")
SIZES = (8, 6, 6, 5, 4, 3, 4, 4, 7)


def tensors():
    """Each in a part of one buffer, with room between them."""
    flat = torch.zeros(16 * len(NAMES), dtype=torch.int32, device="cuda")
    at = {name: 16 * i for i, name in enumerate(NAMES)}
    t = {name: flat[at[name]:at[name] + n] for name, n in zip(NAMES, SIZES)}
    t["free_blocks"].copy_(i32(np.arange(7)))
    t["new_lens"].fill_(1)
    return flat, at, t


def call(jkb, t):
    jkb.kv_build_tables(t["block_table"].view(4, 2), *(t[n] for n in NAMES[1:]), 16)


def test_neighbours_are_apart(jkb):
    flat, _, t = tensors()
    call(jkb, t)
    assert t["kv_lens"].tolist() == [1] * 4 and t["slots"].tolist() == [0, 16, 32, 48, -1, -1]
    parts, at = {}, 0
    for name, n in zip(NAMES, SIZES):  # without room between them
        parts[name] = flat[at:at + n]
        at += n
    flat.zero_()
    parts["free_blocks"].copy_(i32(np.arange(7)))
    parts["new_lens"].fill_(1)
    call(jkb, parts)
    assert parts["kv_lens"].tolist() == [1] * 4 and parts["counts"].tolist() == [4, 4, 0]


@pytest.mark.parametrize("a", range(6))  # the outputs
@pytest.mark.parametrize("b", range(9))
def test_overlaps_are_refused(jkb, a, b):
    if a == b:
        return
    for shift in (0, SIZES[a] - 1, 1 - SIZES[b]):  # from the start, the last and the first element
        flat, at, t = tensors()
        start = max(at[NAMES[a]] + shift, 0)
        t[NAMES[b]] = flat[start:start + SIZES[b]]
        before = flat.clone()
        with pytest.raises(jkb.TensorBoundsError, match="overlaps"):
            call(jkb, t)
        assert torch.equal(flat, before)


def test_inputs_may_be_one_tensor_and_rows_may_have_gaps(jkb):
    same = i32([3, 4])
    table, slots, pos = i32(np.full((2, 2), -1)), i32(np.zeros(8)), i32(np.zeros(8))
    table[0, 0], table[1, 0] = 5, 6
    starts, lens, counts = i32([0] * 3), i32([0] * 2), i32([0] * 3)
    jkb.kv_build_tables(table, slots, pos, starts, lens, counts, same, same, i32([1]), 16)
    assert lens.tolist() == [6, 8] and slots.tolist() == [83, 84, 85, 100, 101, 102, 103, -1]
    wide = i32(np.full((3, 7), 55))  # rows of two, lengths and counts between them
    flat = wide.view(-1)
    args = [i32(np.zeros(8)), i32(np.zeros(8)), i32(np.zeros(4)), flat[2:5], flat[9:12],
            i32([0, 0, 0]), i32([2, 3, 1]), i32([4, 2, 9]), 16]
    jkb.kv_build_tables(wide[:, :2], *args)
    assert wide[:, 0].tolist() == [4, 2, 9] and flat[2:5].tolist() == [2, 3, 1]
    assert flat[9:12].tolist() == [6, 3, 0] and flat[5:7].tolist() == [55, 55]
    args[3] = flat[5:8]  # its last element is the second row's first
    with pytest.raises(jkb.TensorBoundsError, match="overlaps block_table"):
        jkb.kv_build_tables(wide[:, :2], *args)


def test_lengths_in_place_are_refused(jkb):
    ctx = i32(np.arange(3000))
    n = 3000
    with pytest.raises(jkb.TensorBoundsError, match="ctx_lens overlaps kv_lens"):
        jkb.kv_build_tables(i32(np.zeros((n, 200))), i32(np.zeros(n)), i32(np.zeros(n)),
                            i32(np.zeros(n + 1)), ctx, i32(np.zeros(3)), ctx, i32(np.ones(n)),
                            i32(np.arange(n)), 16)
    check_tables(jkb, np.full((2, 2), -1), [0, 0], [3, 4], np.arange(4), 9, 16)
