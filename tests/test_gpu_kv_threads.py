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


def test_tables_of_two_threads_at_once(jkb):
    """More sequences than the default shared memory holds, of two sizes, in turn and at once."""

    def call(n):
        ctx, new = i32(np.zeros(n)), i32(np.ones(n))
        table, slots, pos = i32(np.full((n, 1), -1)), i32(np.zeros(n)), i32(np.zeros(n))
        starts, lens, counts = i32(np.zeros(n + 1)), i32(np.zeros(n)), i32(np.zeros(3))
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        free = i32(np.arange(n))
        torch.cuda.synchronize()
        for _ in range(200):
            jkb.kv_build_tables(table, slots, pos, starts, lens, counts, ctx, new, free, 16,
                                stream=st)
        st.synchronize()
        return counts.tolist()

    assert call(8192) == [8192, 8192, 0]
    results = {}
    threads = [threading.Thread(target=lambda n=n: results.update({n: call(n)}))
               for n in (8192, 6200)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert results == {n: [n, n, 0] for n in (8192, 6200)}
