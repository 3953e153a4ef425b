"""Where attention_kv8 rounds the weights of 16-bit rows: bounds that do not hide a weight of few
bits, against softmax attention in 64 bits."""
import math

import kvref
import numpy as np
import pytest
import torch
from test_gpu_kv_attention import run, setup

pytestmark = pytest.mark.gpu

LAST = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def check_tight(out, lse, ref, longest, prompt):
    """kvref's bound without its allowance of 2^-11 for 16-bit rows. A score's error, twice (in
    numerator and denominator), and the sums' are kvref's: 2 (slack + 2^-20 + (n / 16 + 64) 2^-23);
    2^-21 |lse| is the score's rounding in f32, 2^-20 the weights' split into 22 bits and ex2. None
    of the weights' 16-bit parts enter the lse. In prompts of 16-bit rows a weight is held in two
    bf16: the first cut to 8 bits (a rest below 2^-7), the second rounded to nearest (2^-9 of the
    rest): 2^-16. The output's own type rounds last; an f16 below 2^-14 by 2^-25."""
    want, want_lse, size, slack = ref
    rel = 2 * (slack + 2.0 ** -20 + (longest / 16 + 64) * 2.0 ** -23) + 2.0 ** -20
    rel = rel + 2.0 ** -21 * want_lse.abs().nan_to_num(posinf=0.0, neginf=0.0)
    both = rel + (2.0 ** -16 if prompt and out.dtype != torch.float32 else 0.0)
    tiny = 2.0 ** -25 if out.dtype == torch.float16 else 1e-37
    err = (out.double() - want).abs()
    bound = both[..., None] * size
    bound = bound + LAST[out.dtype] * (want.abs() + bound) + tiny
    assert torch.isfinite(out).all()
    assert bool((err <= bound).all()), float((err / bound).max())
    seen = ~torch.isinf(want_lse)
    err = (lse.double() - want_lse)[seen].abs()
    bound = (rel + 2.0 ** -21 * want_lse.abs())[seen]
    assert bool((err <= bound).all()), float((err / bound).max())


def check(jkb, c, q, table, lens, starts, scale, causal=True, window=0):
    out, lse = run(jkb, kvref.to_device(jkb, c), q, table, lens, starts, scale, causal, window)
    ref = kvref.attention(c, q, table, lens, starts, scale, causal, window)
    rows = int(np.diff(starts).max()) * q.shape[1] // c.k.shape[1]
    check_tight(out, lse, ref, max(lens), rows > 16 and q.shape[2] <= 128)
    assert jkb.device_status() == 0


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("new", [1, 4, 100])
def test_weights_of_two_tokens_that_cancel(jkb, kind, dim, new):
    """Two tokens have all the values, of opposite signs, so that in some elements of a row their
    weights' errors are all that is left: 11 bits of a weight would be off by up to 2^-12 of it."""
    n = 150
    c, _, q, table, starts = setup(jkb, [n], [new], 4, 2, dim, 16, kind, seed=dim + new, q_size=0.3)
    c.v[:] = 0
    c.v[table[0, 1], :, 3] = 127
    c.v[table[0, 2], :, 7] = -np.linspace(30, 127, dim).round().astype(np.int8)
    c.vs[:] = 2.0 ** -4
    check(jkb, c, q, table, [n], starts, dim ** -0.5)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,new,heads,dim", [([700, 41], [1, 1], 8, 128), ([333], [3], 6, 72),
                                                ([90], [2], 4, 256), ([600, 130], [200, 130], 4, 64),
                                                ([500], [61], 14, 80), ([1300], [150], 8, 128)])
def test_lse_of_every_row_type(jkb, kind, lens, new, heads, dim):
    """lse is f32 whatever the rows' type, so its bound does not widen with them."""
    c, _, q, table, starts = setup(jkb, lens, new, heads, 2, dim, 32, kind, seed=dim)
    check(jkb, c, q, table, lens, starts, dim ** -0.5)
    check(jkb, c, q, table, lens, starts, dim ** -0.5, causal=False, window=77)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(64, 8, 128), (96, 8, 96), (64, 32, 64), (32, 2, 128),
                                                (24, 8, 256)])
def test_few_row_scores_in_24_bits(jkb, kind, heads, kv_heads, dim):
    """With one cached token lse is the score itself. An element of q is off by half a unit of its
    row's 24 bits (the largest over 8355700, so 1.01 2^-24 of it) and by 2^-24 of itself; f32 steps
    (the unit and its inverse, the scales, the sum of the digits' products) by 2^-20 of the score;
    its weight, the logarithm and their sum by 2^-20. Digits of 16 bits would be 16 times that off or
    more (the same inputs rounded to 16 bits in numpy)."""
    for seed in range(4):
        lens = [1] * 6
        c, cache, q, table, starts = setup(jkb, lens, lens, heads, kv_heads, dim, 16, kind, seed=seed)
        scale = dim ** -0.5
        _, lse = run(jkb, cache, q, table, lens, starts, scale)
        k = torch.from_numpy(c.k[table[:, 0], :, 0]).cuda().double()
        k = k * torch.from_numpy(c.ks[table[:, 0]]).cuda().double()[..., None]
        k = k.repeat_interleave(heads // kv_heads, 1)
        x = q.double()
        s = scale * (x * k).sum(2)
        tol = scale * 2.0 ** -24 * (1.01 * x.abs().amax(2) * k.abs().sum(2) + (x * k).abs().sum(2))
        tol = tol + 2.0 ** -20 * (s.abs() + 1)
        err = (lse.double() - s).abs()
        assert bool((err <= tol).all()), float((err / tol).max())
