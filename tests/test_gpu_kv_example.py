"""The example attention layer: projections, tables, append and attention together, prompts and
decode steps, against plain attention in 64 bits over the cache's own values.

Tolerance, relative to the largest output: the queries' rounding to 22 bits or more moves a score
by at most 2^-22 of scale * |q| |k| (below 16 here, so 2^-18 of a weight), the weights carry 22
bits or more, the sums f32's with a truncation of 2^-23 a step of 16 tokens (below 2^-18 over the
320 tokens). Twice their sum, 2^-16, leaves room for outputs smaller than the largest value."""
import importlib.util
import os

import pytest

import conftest

pytestmark = pytest.mark.gpu


def example():
    path = os.path.join(conftest.PKG_PARENT, "examples", "attention_layer.py")
    spec = importlib.util.spec_from_file_location("attention_layer", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("heads,kv_heads,dim,block", [(16, 4, 64, 32), (8, 1, 128, 16),
                                                      (6, 6, 80, 64)])
def test_attention_layer(jkb, heads, kv_heads, dim, block):
    import torch

    outs, errors = example().run(hidden=512, heads=heads, kv_heads=kv_heads, dim=dim,
                                 prompts=(300, 17, 1, 128), steps=6, block_tokens=block)
    assert [tuple(o.shape) for o in outs] == [(446, 512)] + [(4, 512)] * 6
    assert all(torch.isfinite(o).all() for o in outs)
    assert max(errors) <= 2.0 ** -16, errors
