"""attention_kv8 where one block's values are far larger than the others': a block that a row does
not see, or that has no weight in it, takes no digits from the row's other tokens. Against softmax
attention in 64 bits; the bounds are kvref's."""
import kvref
import numpy as np
import pytest
import torch
from test_gpu_kv_attention import run, setup

pytestmark = pytest.mark.gpu


def check(jkb, c, q, table, lens, starts, scale, window=0):
    out, lse = run(jkb, kvref.to_device(jkb, c), q, table, lens, starts, scale, window=window)
    ref = kvref.attention(c, q, table, lens, starts, scale, True, window)
    kvref.check_attention(out, lse, ref, max(lens))
    assert jkb.device_status() == 0


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,dim,new", [(4, 64, 1), (6, 128, 4), (4, 256, 3), (4, 64, 50),
                                           (4, 128, 200)])
@pytest.mark.parametrize("at", [0, 5])
def test_a_block_without_weight(jkb, kind, heads, dim, new, at):
    """Values of 2^60 whose weights are about 2^-80, or far below f32's range."""
    c, _, q, table, starts = setup(jkb, [400], [new], heads, 2, dim, 16, kind, seed=new)
    q = q.abs() + 0.5
    c.k[:], c.ks[:], c.vs[:] = np.abs(c.k) // 2, 0.001, 2.0 ** -6
    c.k[table[0, at]], c.vs[table[0, at]] = -100, 2.0 ** 60
    for k_scale in (0.02, 0.5):
        c.ks[table[0, at]] = k_scale
        check(jkb, c, q, table, [400], starts, 16 / dim)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new,first", [(4, 95), (3, 94), (200, 80)])
def test_a_block_that_the_window_hides(jkb, kind, dim, new, first):
    """Tokens 80 .. 95 have values of 2^60. The first query sees from token `first` on, the later
    ones from one token more each."""
    c, _, q, table, starts = setup(jkb, [400], [new], 4, 2, dim, 16, kind, seed=dim)
    c.vs[:] = 2.0 ** -6
    c.vs[table[0, 5]] = 2.0 ** 60
    c.v[table[0, 5]] |= 1  # no code 0: each has more than 2^37 times the others' products
    check(jkb, c, q, table, [400], starts, dim ** -0.5, window=400 - new - first + 1)


@pytest.mark.parametrize("new", [1, 100])
def test_value_scales_against_weights(jkb, new):
    """Scales that grow as fast as the weights fall, so that every block counts as much, and scales
    that fall faster than the weights grow."""
    for slope in (1.0, 2.0, 0.5):
        c, _, q, table, starts = setup(jkb, [640], [new], 2, 1, 64, 16, "f32", seed=3)
        q[:] = 1.0
        n = 40
        c.k[:] = 64
        c.ks[table[0, :n], 0] = np.linspace(0.0, 0.5, n)  # scores of 0 to 60 in powers of e
        c.vs[table[0, :n], 0] = np.exp(-slope * np.linspace(0.0, 60.0, n))
        scale = 60.0 / (64 * 64 * 0.5)
        check(jkb, c, q, table, [640], starts, scale)
