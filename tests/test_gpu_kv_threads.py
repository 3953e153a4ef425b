"""Key/value cache and attention calls from several host threads: what one thread's calls need of
the process must not be taken away by another's."""
import threading

import kvref
import numpy as np
import pytest
import torch
from test_gpu_kv_attention import i32, run, setup

pytestmark = pytest.mark.gpu


def in_thread(f):
    out = []

    def body():
        try:
            out.append(f())
        except BaseException as e:  # noqa: BLE001
            out.append(e)

    t = threading.Thread(target=body)
    t.start()
    t.join()
    if isinstance(out[0], BaseException):
        raise out[0]
    return out[0]


@pytest.mark.parametrize("dim,heads", [(64, 2), (64, 12), (96, 2), (128, 2), (128, 16), (192, 2),
                                       (256, 2)])
def test_a_second_thread_with_fewer_sequences(jkb, dim, heads):
    """The few-row kernel's shared memory grows with the sequences of a call."""
    n = 500
    lens = np.random.default_rng(dim).integers(1, 40, n).tolist()
    c, cache, q, table, starts = setup(jkb, lens, [1] * n, heads, 1, dim, 16, "f32", seed=dim)
    few = 3
    first, _ = run(jkb, cache, q, table, lens, starts, 0.1)
    out, out_lse = in_thread(lambda: run(jkb, cache, q[:few], table[:few], lens[:few],
                                         starts[:few + 1], 0.1))
    again, lse = run(jkb, cache, q, table, lens, starts, 0.1)
    ref = kvref.attention(c, q, table, lens, starts, 0.1, True, 0)
    kvref.check_attention(again, lse, ref, 40)
    kvref.check_attention(out, out_lse, [x[:few] for x in ref], 40)
    assert torch.equal(first, again)
