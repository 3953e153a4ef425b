"""attention_kv8 at the ends of its arguments' ranges, against softmax attention in 64 bits; the
bounds are kvref's."""
import kvref
import numpy as np
import pytest
import torch
from test_gpu_kv_attention import TYPES, run, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new,dim", [(1, 64), (3, 128), (2, 256), (150, 64), (100, 128)])
@pytest.mark.parametrize("q_exp,k_exp,scale_exp", [(125, 0, -125), (125, -110, -15),
                                                   (-105, 105, 0), (-118, 118, 0)])
def test_queries_at_both_ends_of_the_range(jkb, kind, new, dim, q_exp, k_exp, scale_exp):
    """The scores of an ordinary call, whose query rows are 2^125 times as large, or 2^-118, and
    whose keys' scales or softmax scale make up for it. Rows of ordinary size stand beside the large
    ones in a tile."""
    lens = [300]
    c, _, q, table, starts = setup(jkb, lens, [new], 6, 2, dim, 32, "f32", seed=dim)
    c.ks *= np.float32(2.0 ** k_exp)
    q = q.clamp(-6, 6)
    q[:, :: 2 if q_exp > 0 else 1] *= 2.0 ** q_exp
    q = q.to(TYPES[kind])
    assert torch.isfinite(q).all() and np.isfinite(c.ks * np.float32(127)).all()
    scale = dim ** -0.5 * 2.0 ** scale_exp
    out, lse = run(jkb, kvref.to_device(jkb, c), q, table, lens, starts, scale)
    ref = kvref.attention(c, q, table, lens, starts, scale, True, 0)
    kvref.check_attention(out, lse, ref, 300)
    assert jkb.device_status() == 0


@pytest.mark.parametrize("window", [300, 301, 2**30, 2**31 - 200, 2**31 - 1, 2**31, 2**40])
@pytest.mark.parametrize("lens,new", [([120], [3]), ([3], [5]), ([40], [200]), ([250, 90], [70, 130])])
def test_windows_beyond_every_context(jkb, window, lens, new):
    """As no window, for queries before the first cached token too (more new tokens than cached
    ones): without a causal mask they see every token."""
    c, cache, q, table, starts = setup(jkb, lens, new, 4, 2, 64, 16, "f32", seed=5)
    for causal in (True, False):
        out, lse = run(jkb, cache, q, table, lens, starts, 0.1, causal, window)
        ref = kvref.attention(c, q, table, lens, starts, 0.1, causal, 0)
        kvref.check_attention(out, lse, ref, max(lens))
