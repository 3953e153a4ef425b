"""attention_kv8 where a long context is split into many pieces that are joined in several levels,
and where masks meet blocks of scale zero or queries that are not finite. Against softmax
attention in 64 bits; the bounds are kvref's."""
import math

import kvref
import numpy as np
import pytest
import torch
from test_gpu_kv_attention import check, i32, run, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,new", [([1100], [1]), ([9000], [2]), ([40_000], [1]),
                                      ([30_000, 200, 8000], [2, 1, 1]),
                                      ([1500], [4]), ([9000], [20]), ([20_000], [4]),
                                      ([12_000, 1, 19_000], [5, 1, 30])])
def test_one_kv_head(jkb, lens, new, kind):
    """Up to 300 pieces of one row tile, of 1 to 240 query rows."""
    check(jkb, lens, new, 8, 1, 128, 64, kind, seed=sum(lens))


@pytest.mark.parametrize("dim", [40, 64, 96, 256])
def test_one_kv_head_other_sizes(jkb, dim):
    check(jkb, [15_000], [3], 5, 1, dim, 32, seed=dim)
    check(jkb, [9000], [25], 5, 1, dim, 32, seed=dim)


def test_joined_rows_that_are_not_aligned(jkb):
    """Pieces of a prompt's tile and rows that cannot be stored 16 bytes at a time."""
    lens, heads, dim = [9000], 3, 72
    for new in (2, 50):
        c, cache, q, table, starts = setup(jkb, lens, [new], heads, 1, dim, 64, "bf16", seed=new)
        wide = torch.zeros(new, heads, dim + 1, dtype=q.dtype, device="cuda")
        out, lse = wide[..., 1:], torch.zeros(new, heads, device="cuda")
        jkb.attention_kv8(out, q, cache, jkb.AttentionWorkspace(cache), i32(table), i32(lens),
                          i32(starts), new, 0.1, lse=lse)
        ref = kvref.attention(c, q, table, lens, starts, 0.1, True, 0)
        kvref.check_attention(out, lse, ref, lens[0])
        assert not wide[..., 0].any()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [2, 150])
def test_masks_over_blocks_of_scale_zero(jkb, kind, new):
    """Keys of scale zero all score 0, but those behind a mask count for nothing."""
    c, cache, q, table, starts = setup(jkb, [300], [new], 4, 2, 64, 16, kind, seed=new)
    for blocks in (slice(None), slice(0, None, 2)):
        c.ks[blocks] = 0.0
        cache = kvref.to_device(jkb, c)
        for causal, window in ((True, 0), (True, 21), (False, 37)):
            out, lse = run(jkb, cache, q, table, [300], starts, 0.125, causal, window)
            ref = kvref.attention(c, q, table, [300], starts, 0.125, causal, window)
            kvref.check_attention(out, lse, ref, 300)
        c.ks[:] = np.float32(0.02)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [3, 150])
def test_queries_that_are_not_finite_and_see_nothing(jkb, kind, new):
    """More new tokens than cached ones: the first queries see nothing, whatever they hold."""
    n = new - 2
    c, cache, q, table, starts = setup(jkb, [n], [new], 4, 2, 64, 16, kind, seed=new)
    q[0, 1, 3], q[1, 2, 0] = math.nan, math.inf
    out, lse = run(jkb, cache, q, table, [n], starts, 0.125)
    assert not out[:2].any() and torch.isneginf(lse[:2]).all()
    q[:2] = 0.0
    ref = kvref.attention(c, q, table, [n], starts, 0.125, True, 0)
    kvref.check_attention(out, lse, ref, n)
