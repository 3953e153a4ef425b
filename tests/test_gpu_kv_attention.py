"""attention_kv8 on the GPU against softmax attention in 64 bits over the same codes and scales,
at the lengths, masks and layouts where a kernel can go wrong. The bounds are kvref's."""
import math

import kvref
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def i32(a):
    return torch.tensor(np.asarray(a, np.int32), device="cuda")


def setup(jkb, lens, new, heads, kv_heads, dim, block, kind, seed=0, q_size=1.5, spare=2):
    rng = np.random.default_rng(seed)
    need = [-(-n // block) for n in lens]
    total = sum(need) + spare
    c = kvref.filled(rng, total, kv_heads, block, dim)
    ids = rng.permutation(total)
    table, at = np.full((len(lens), max(need) + 1), -1, np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = torch.from_numpy(rng.normal(0, q_size, (int(starts[-1]), heads, dim)).astype(np.float32))
    return c, kvref.to_device(jkb, c), q.to(TYPES[kind]).cuda(), table, starts


def run(jkb, cache, q, table, lens, starts, scale, causal=True, window=0, with_lse=True,
        most=None, ws=None):
    out = torch.full_like(q, 7.0)
    lse = torch.full(q.shape[:2], 7.0, device="cuda") if with_lse else None
    ws = ws or jkb.AttentionWorkspace(cache)
    most = int(np.diff(starts).max(initial=0)) if most is None else most
    jkb.attention_kv8(out, q, cache, ws, i32(table), i32(lens), i32(starts), most, scale,
                      causal=causal, window=window, lse=lse)
    return out, lse


def check(jkb, lens, new, heads, kv_heads, dim, block, kind="f32", causal=True, window=0, seed=0,
          **more):
    c, cache, q, table, starts = setup(jkb, lens, new, heads, kv_heads, dim, block, kind, seed)
    scale = 1 / math.sqrt(dim)
    out, lse = run(jkb, cache, q, table, lens, starts, scale, causal, window, **more)
    ref = kvref.attention(c, q, table, lens, starts, scale, causal, window)
    kvref.check_attention(out, lse, ref, max(lens))
    again, _ = run(jkb, cache, q, table, lens, starts, scale, causal, window, **more)
    assert torch.equal(out, again)
    assert jkb.device_status() == 0


# ------------------------------------------------------------------------------- single tokens

@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 1000, 5001])
@pytest.mark.parametrize("block", [16, 64])
def test_decode_lengths(jkb, n, block):
    check(jkb, [n], [1], 8, 2, 128, block, seed=n)


@pytest.mark.parametrize("dim", [8, 32, 40, 64, 72, 80, 96, 120, 128, 160, 192, 200, 256])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_decode_head_sizes_and_types(jkb, dim, kind):
    check(jkb, [333, 64, 1, 90], [1, 1, 1, 1], 6, 2, dim, 32, kind, seed=dim)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (7, 1), (8, 1), (9, 1), (16, 1),
                                            (17, 1), (40, 2), (32, 8), (20, 5)])
def test_decode_head_layouts(jkb, heads, kv_heads):
    check(jkb, [200, 47], [1, 1], heads, kv_heads, 64, 16, seed=heads)
    check(jkb, [200, 47], [1, 1], heads, kv_heads, 256, 16, seed=heads)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_decode_many_ragged_sequences(jkb, block):
    rng = np.random.default_rng(block)
    lens = rng.integers(0, 700, 97).tolist()
    lens[3], lens[40] = 0, 4000
    check(jkb, lens, [1] * 97, 8, 2, 64, block, seed=block)


def test_decode_one_long_sequence_beside_short_ones(jkb):
    check(jkb, [30_011, 5, 900], [1, 1, 1], 8, 1, 128, 64, seed=1)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 300, 100_000])
def test_decode_window(jkb, window):
    check(jkb, [1, 500, 64, 77, 1000], [1] * 5, 4, 2, 64, 16, window=window, seed=window)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 40])
def test_few_new_tokens(jkb, causal, window):
    """Several query tokens a sequence, none for some, more than cached tokens for one: the
    queries before the first cached token see nothing."""
    for dim in (64, 128, 256):
        check(jkb, [100, 3, 50, 1, 0, 260], [3, 5, 0, 1, 2, 4], 6, 2, dim, 16, causal=causal,
              window=window, seed=dim)


def test_thousands_of_sequences(jkb):
    rng = np.random.default_rng(2)
    check(jkb, rng.integers(1, 60, 3000).tolist(), [1] * 3000, 2, 1, 64, 16, seed=2)


# ------------------------------------------------------------------------------- prompts

@pytest.mark.parametrize("n", [17, 64, 127, 128, 129, 255, 257, 700])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_prompt_lengths(jkb, n, kind):
    check(jkb, [n], [n], 8, 2, 128, 64, kind, seed=n)


@pytest.mark.parametrize("dim", [8, 40, 64, 72, 80, 96, 128, 160, 256])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_prompt_head_sizes_and_types(jkb, dim, kind):
    check(jkb, [333, 130], [200, 130], 4, 2, dim, 32, kind, seed=dim)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (7, 1), (14, 2), (40, 2), (130, 1)])
def test_prompt_head_layouts(jkb, heads, kv_heads):
    check(jkb, [150, 290], [150, 61], heads, kv_heads, 64, 16, seed=heads)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_chunks_behind_context_and_decodes_together(jkb, block, kind):
    lens = [700, 1, 333, 64, 0, 2000, 129, 128, 5]
    new = [100, 1, 333, 0, 3, 1, 129, 17, 9]
    check(jkb, lens, new, 8, 2, 64, block, kind, seed=block)
    check(jkb, lens, new, 14, 2, 80, block, kind, causal=False, seed=block)


@pytest.mark.parametrize("window", [1, 30, 128, 129, 500])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_window(jkb, window, causal):
    check(jkb, [600, 300], [400, 300], 4, 1, 128, 32, causal=causal, window=window, seed=window)
    check(jkb, [600, 300], [400, 300], 4, 1, 64, 32, "bf16", causal=causal, window=window)


def test_prompt_of_more_tokens_than_are_cached(jkb):
    check(jkb, [40, 300], [200, 310], 4, 2, 128, 16, seed=3)
    check(jkb, [40, 300], [200, 310], 4, 2, 128, 16, "f16", window=20, seed=3)


def test_understated_max_new(jkb):
    check(jkb, [300, 40], [150, 1], 4, 2, 64, 16, most=1, seed=4)
    check(jkb, [300, 40], [2, 1], 4, 2, 64, 16, most=4000, seed=4)


# ------------------------------------------------------------------------------- values

def reference_and_run(jkb, c, cache, q, table, lens, starts, scale):
    out, lse = run(jkb, cache, q, table, lens, starts, scale)
    return out, lse, kvref.attention(c, q, table, lens, starts, scale, True, 0)


@pytest.mark.parametrize("new", [1, 200])
def test_scales_far_apart(jkb, new):
    """Value scales of 2^-100 to 2^60 and zero blocks, and keys so large that one token has all
    the weight: f16 parts must neither overflow nor lose the small blocks' share of the sum."""
    c, _, q, table, starts = setup(jkb, [400], [new], 4, 2, 64, 16, "f32", seed=5)
    rng = np.random.default_rng(5)
    c.vs[:] = 2.0 ** rng.uniform(-100, 60, c.vs.shape)
    c.vs[table[0, 3]] = 0
    out, lse, ref = reference_and_run(jkb, c, kvref.to_device(jkb, c), q, table, [400], starts, .1)
    kvref.check_attention(out, lse, ref, 400)
    c.vs[:] = 0.01
    c.ks[:] = 2.0 ** rng.uniform(-4, 8, c.ks.shape)
    c.ks[table[0, 5]] = 0
    out, lse, ref = reference_and_run(jkb, c, kvref.to_device(jkb, c), q, table, [400], starts, .1)
    kvref.check_attention(out, lse, ref, 400)


@pytest.mark.parametrize("new", [1, 150])
def test_rising_and_falling_scores(jkb, new):
    """Running maxima that grow at every step, and that never grow again after the first."""
    c, cache, q, table, starts = setup(jkb, [900], [new], 4, 2, 64, 16, "f32", seed=6, q_size=0.2)
    q[:] = q.abs() + 0.1
    for order in (1, -1):
        n = -(-900 // 16)
        c.k[:] = np.abs(c.k)
        c.ks[table[0, :n]] = np.linspace(0.01, 0.2, n).astype(np.float32)[::order, None]
        cache = kvref.to_device(jkb, c)
        out, lse, ref = reference_and_run(jkb, c, cache, q, table, [900], starts, 0.3)
        kvref.check_attention(out, lse, ref, 900)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [2, 140])
def test_queries_that_are_not_ordinary(jkb, kind, new):
    c, cache, q, table, starts = setup(jkb, [300], [new], 4, 2, 64, 32, kind, seed=7)
    bad = q.clone()
    bad[0, 0, 5], bad[new - 1, 3, 0], bad[new - 1, 2] = math.nan, math.inf, 0.0
    out, lse = run(jkb, cache, bad, table, [300], starts, 0.125)
    good = q.clone()
    good[0, 0], good[new - 1, 3], good[new - 1, 2] = 0.0, 0.0, 0.0
    ref = kvref.attention(c, good, table, [300], starts, 0.125, True, 0)
    for t, h in ((0, 0), (new - 1, 3)):
        assert torch.isnan(out[t, h]).all() and torch.isnan(lse[t, h])
        out[t, h], lse[t, h] = ref[0][t, h].to(out.dtype), ref[1][t, h].float()
    kvref.check_attention(out, lse, ref, 300)
    for size in (1e-20, 1e-36, 2e3):
        if kind == "f16" and size < 1:
            continue
        c2, cache2, q2, table2, starts2 = setup(jkb, [300], [new], 4, 2, 64, 32, kind, 8, size)
        out, lse, ref = reference_and_run(jkb, c2, cache2, q2, table2, [300], starts2, 0.125)
        kvref.check_attention(out, lse, ref, 300)


@pytest.mark.parametrize("new", [1, 100])
def test_scale_zero_and_negative(jkb, new):
    c, cache, q, table, starts = setup(jkb, [200], [new], 4, 2, 64, 32, "f32", seed=8)
    for scale in (0.0, -0.2):
        out, lse, ref = reference_and_run(jkb, c, cache, q, table, [200], starts, scale)
        kvref.check_attention(out, lse, ref, 200)


# ------------------------------------------------------------------------------- layouts

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [1, 70])
def test_strided_queries_and_outputs(jkb, kind, new):
    lens, news = [120, 77], [new, min(new, 60)]
    c, cache, q, table, starts = setup(jkb, lens, news, 6, 2, 40, 16, kind, seed=9)
    ref = kvref.attention(c, q, table, lens, starts, 0.2, True, 0)
    ws = jkb.AttentionWorkspace(cache)
    for off in (0, 1, 8):
        wide = torch.zeros(q.shape[0], 9, 40 + off, dtype=q.dtype, device="cuda")
        qv = wide[:, 2:8, off:]
        qv.copy_(q)
        room = torch.full((q.shape[0], 8, 48 + off), 3.0, dtype=q.dtype, device="cuda")
        out = room[:, 1:7, off:off + 40]
        jkb.attention_kv8(out, qv, cache, ws, i32(table), i32(lens), i32(starts), new, 0.2)
        kvref.check_attention(out, None, ref, 120)
        assert (room[:, 0] == 3).all() and (room[:, 7] == 3).all()
        assert (room[:, :, off + 40:] == 3).all() and (room[:, :, :off] == 3).all()


@pytest.mark.parametrize("new", [1, 100])
def test_ids_and_lengths_that_are_out_of_range(jkb, new):
    """A bad id's tokens are not seen, a length beyond its row is clamped, both are reported."""
    c, cache, q, table, starts = setup(jkb, [160], [new], 4, 2, 64, 16, "f32", seed=10)
    bad = table[:, :10].copy()
    bad[0, 4], bad[0, 6] = c.k.shape[0], -1
    out, _ = run(jkb, cache, q, bad, [160], starts, 0.1)
    with pytest.raises(jkb.TensorBoundsError):
        jkb.device_status()
    assert torch.isfinite(out).all()
    if new == 1:  # the reference without those tokens
        keep = [i for i in range(10) if i not in (4, 6)]
        ref = kvref.attention(c, q, table[:, keep], [128], starts, 0.1, False, 0)
        kvref.check_attention(out, None, ref, 160)
    out, lse = run(jkb, cache, q, table[:, :10], [5000], starts, 0.1)
    with pytest.raises(jkb.TensorBoundsError):
        jkb.device_status()
    ref = kvref.attention(c, q, table, [160], starts, 0.1, True, 0)
    kvref.check_attention(out, lse, ref, 160)
    out, lse = run(jkb, cache, q, table, [-3], starts, 0.1)
    with pytest.raises(jkb.TensorBoundsError):
        jkb.device_status()
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("new", [1, 90])
def test_unused_tokens_of_a_block_do_not_matter(jkb, new):
    c, cache, q, table, starts = setup(jkb, [100], [new], 4, 2, 64, 64, "f32", seed=11)
    out, lse = run(jkb, cache, q, table, [100], starts, 0.1)
    for x in (c.k, c.v):
        x[table[0, 1], :, 36:] = -127
    out2, lse2 = run(jkb, kvref.to_device(jkb, c), q, table, [100], starts, 0.1)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


def test_past_four_gigabytes(jkb):
    """Block ids whose codes lie beyond 32-bit offsets."""
    n = 34_000
    cache = jkb.KvCache(n, 64, 8, 128)
    assert cache.device_bytes > 2**32
    rng = np.random.default_rng(12)
    c = kvref.filled(rng, 4, 8, 64, 128)
    ids = np.array([n - 1, n - 3, 0, n - 2], np.int32)
    cache.import_blocks(i32(ids), *(torch.from_numpy(x).cuda() for x in (c.k, c.v, c.ks, c.vs)))
    for new in (1, 120):
        q = torch.from_numpy(rng.normal(0, 1, (new, 16, 128)).astype(np.float32)).cuda()
        out, lse = run(jkb, cache, q, ids[None], [250], [0, new], 0.1)
        ref = kvref.attention(c, q, np.arange(4)[None], [250], [0, new], 0.1, True, 0)
        kvref.check_attention(out, lse, ref, 250)


@pytest.mark.parametrize("new", [1, 130])
def test_other_stream_graph_and_workspace_reuse(jkb, new):
    """The call runs on the stream it is given, can be captured, and leaves its workspace ready."""
    lens, news = [1500, 700], [new, 1]
    c, cache, q, table, starts = setup(jkb, lens, news, 8, 2, 64, 32, "f32", seed=13)
    ref = kvref.attention(c, q, table, lens, starts, 0.1, True, 0)
    ws = jkb.AttentionWorkspace(cache)
    out = torch.zeros_like(q)
    args = (i32(table), i32(lens), i32(starts), new, 0.1)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    jkb.attention_kv8(out, q, cache, ws, *args, stream=st)
    st.synchronize()
    kvref.check_attention(out, None, ref, 1500)
    first = out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        jkb.attention_kv8(out, q, cache, ws, *args)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)


def test_step_of_all_three(jkb):
    """Tables, append and attention as a serving loop runs them: two prompts, then decode steps
    that fill and open blocks, against attention over the cache's own values."""
    rng = np.random.default_rng(14)
    heads, kv, dim, block = 4, 2, 64, 16
    cache = jkb.KvCache(40, block, kv, dim)
    ws = jkb.AttentionWorkspace(cache)
    free = rng.permutation(40)
    table = torch.full((2, 12), -1, dtype=torch.int32, device="cuda")
    ctx = np.array([0, 0])
    for new in ([37, 5], [1, 1], [1, 1], [1, 1], [20, 1], [1, 30]):
        new = np.array(new)
        n = int(new.sum())
        slots, pos = (torch.empty(n + 3, dtype=torch.int32, device="cuda") for _ in range(2))
        starts, lens, counts = i32([0] * 3), i32([0] * 2), i32([0] * 3)
        jkb.kv_build_tables(table, slots, pos, starts, lens, counts, i32(ctx), i32(new),
                            i32(free), block)
        k, v = (torch.from_numpy(rng.normal(0, 1, (n, kv, dim)).astype(np.float32)).cuda()
                for _ in range(2))
        jkb.kv_append(cache, k, v, slots[:n])
        q = torch.from_numpy(rng.normal(0, 1, (n, heads, dim)).astype(np.float32)).cuda()
        out, lse = torch.empty_like(q), torch.empty(n, heads, device="cuda")
        jkb.attention_kv8(out, q, cache, ws, table, lens, starts, int(new.max()), 0.125, lse=lse)
        assert counts.tolist()[0] == n and counts.tolist()[2] == 0
        free = free[counts.tolist()[1]:]
        ctx = ctx + new
        assert lens.tolist() == ctx.tolist()
        c = kvref.Cache(40, kv, block, dim)
        c.k, c.v, c.ks, c.vs = kvref.exported(cache, list(range(40)))
        ref = kvref.attention(c, q, table.cpu().numpy(), ctx.tolist(), starts.tolist(), 0.125,
                              True, 0)
        kvref.check_attention(out, lse, ref, int(ctx.max()))
    assert jkb.device_status() == 0


def test_attention_refusals(jkb):
    cache = jkb.KvCache(4, 16, 2, 64)
    ws = jkb.AttentionWorkspace(cache)
    q = torch.zeros(3, 4, 64, device="cuda")
    base = dict(out=torch.empty_like(q), q=q, cache=cache, workspace=ws,
                block_table=i32([[0, 1]]), kv_lens=i32([3]), q_starts=i32([0, 3]), max_new=3,
                scale=0.1)

    def call(**more):
        jkb.attention_kv8(**{**base, **more})

    call()
    with pytest.raises(jkb.TensorBoundsError):
        call(q=q[:, :3], out=torch.empty(3, 3, 64, device="cuda"))  # 3 heads over 2 kv heads
    with pytest.raises(jkb.CapabilityMismatch):
        call(out=torch.empty_like(q).half())
    with pytest.raises(jkb.TensorBoundsError):
        call(scale=math.inf)
    with pytest.raises(jkb.InvalidHandle):
        call(workspace=jkb.AttentionWorkspace(jkb.KvCache(1, 16, 1, 128)))
    for more in (dict(out=torch.empty(2, 4, 64, device="cuda")), dict(q_starts=i32([0])),
                 dict(kv_lens=i32([3, 3])), dict(window=-1), dict(max_new=-1),
                 dict(lse=torch.empty(3, 3, device="cuda")),
                 dict(q=torch.zeros(3, 4, 32, device="cuda"))):
        with pytest.raises(ValueError):
            call(**more)
    for more in (dict(q=q.double()), dict(block_table=torch.zeros(1, 2, device="cuda")),
                 dict(kv_lens=torch.zeros(1, device="cuda"))):
        with pytest.raises(TypeError):
            call(**more)
    call(q=q[:0], out=base["out"][:0], q_starts=i32([0, 0]))
    ws.destroy()
    with pytest.raises(jkb.InvalidHandle):
        call()
