"""kv_append with skipped tokens and gaps: which tokens are written, and what is reported. Exact, as
in test_gpu_kv_cache."""
import kvref
import numpy as np
import pytest
import torch
from test_gpu_kv_cache import i32, rows

pytestmark = pytest.mark.gpu


def kept(slots, block, n_blocks):
    """(indexes of the tokens that are written, whether one is reported)."""
    keep, bad, last = [], False, None  # last: (index, slot, written) of the last token not skipped
    for t, s in enumerate(slots):
        if s >= n_blocks * block:
            bad = True
            s = -1
        if s < 0:
            continue
        ok = True
        if last and last[1] // block == s // block:
            ok = last[0] == t - 1 and last[1] == s - 1
            bad |= not ok
            ok = ok and last[2]
        if ok:
            keep.append(t)
        last = (t, s, ok)
    return keep, bad


def check(jkb, slots, block, n_blocks, heads, dim=64, kind="f32"):
    rng = np.random.default_rng(len(slots))
    c = kvref.filled(rng, n_blocks, heads, block, dim, 0.5, 0.5)
    cache = kvref.to_device(jkb, c)
    k, v = (rows(rng, len(slots), heads, dim, kind).cuda() for _ in range(2))
    jkb.kv_append(cache, k, v, i32(slots))
    keep, bad = kept(slots, block, n_blocks)
    if bad:
        with pytest.raises(jkb.TensorBoundsError):
            jkb.device_status()
    assert jkb.device_status() == 0
    c.append(k.float().cpu().numpy()[keep], v.float().cpu().numpy()[keep],
             [slots[t] for t in keep])
    got = kvref.exported(cache, list(range(n_blocks)))
    for name, a, b in zip(("k", "v", "k scales", "v scales"), got, (c.k, c.v, c.ks, c.vs)):
        assert np.array_equal(a, b), name


def test_the_rule():
    assert kept([5, -1, 6, 7], 16, 4) == ([0], True)
    assert kept([5, -1, 32, 33], 16, 4) == ([0, 2, 3], False)
    assert kept([3, 4, 7, 8, 20], 16, 4) == ([0, 1, 4], True)
    assert kept([5, 64, 6, -2, -3, 16], 16, 4) == ([0, 5], True)


@pytest.mark.parametrize("skipped", [1, 2, 3, 4, 5, 31, 32, 33, 64, 190, 700])
@pytest.mark.parametrize("lead", [0, 1, 2, 3])
def test_skipped_tokens_within_a_block(jkb, skipped, lead):
    """The token behind them is in the block of the last one before them, however far that is (the
    ranges of the CTAs begin anywhere in between), or in another one."""
    other = [16 * (2 + i) for i in range(lead)]
    check(jkb, other + [5] + [-1] * skipped + [6, 7, 96, 97], 16, 8, 1)
    check(jkb, other + [5] + [-1] * skipped + [3, 96], 16, 8, 1)
    check(jkb, other + [5] + [-1] * skipped + [96, 97, -1], 16, 8, 1)
    check(jkb, [-1] * skipped + other + [9], 16, 8, 1)


def test_slots_beyond_the_cache_within_a_block(jkb):
    check(jkb, [5, 128, 6, 40, 41, 2**31 - 1, 42, 64], 16, 8, 2)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_skipped_tokens_within_a_prompt(jkb, kind):
    """Enough tokens for the CTA-wide form: single ones, and long stretches that begin and end
    inside a block."""
    block, n = 32, 60
    slots = list(range(7, n * block))
    for a, b in ((100, 101), (130, 131), (200, 330), (640, 641), (703, 767), (1000, 1500)):
        slots[a:b] = [-1] * (b - a)
    check(jkb, slots, block, n, 8, 64, kind)
