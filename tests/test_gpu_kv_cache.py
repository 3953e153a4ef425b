"""The 8-bit key/value cache on the GPU: block tables and slot maps, append with its quantization,
copies in and out. Everything here is compared exactly: the tables are integers, and the codes
and scales follow f32 steps that numpy repeats."""
import kvref
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def i32(a):
    return torch.tensor(np.asarray(a, np.int32), device="cuda")


# ------------------------------------------------------------------------------- block tables

def run_tables(jkb, table, ctx, new, free, n_slots, block, shift=0):
    n = len(ctx)
    dt = i32(table)
    pad = torch.full((n_slots + shift,), 77, dtype=torch.int32, device="cuda")
    slots, pos = pad.clone()[shift:], pad.clone()[shift:]
    starts, lens, counts = i32(np.full(n + 1, 9)), i32(np.full(n, 9)), i32([9, 9, 9])
    jkb.kv_build_tables(dt, slots, pos, starts, lens, counts, i32(ctx), i32(new), i32(free), block)
    return [t.cpu().numpy() for t in (dt, slots, pos, starts, lens, counts)]


def check_tables(jkb, table, ctx, new, free, n_slots, block, shift=0):
    got = run_tables(jkb, table, ctx, new, free, n_slots, block, shift)
    ref = kvref.build_tables(np.asarray(table, np.int32), ctx, new, free, n_slots, block)
    for name, a, b in zip(("table", "slots", "positions", "starts", "lens", "counts"), got, ref):
        assert np.array_equal(a, b), name
    return got


def step(rng, n, block, ctx_to, new_to, spare=3):
    ctx, new = rng.integers(0, ctx_to + 1, n), rng.integers(0, new_to + 1, n)
    held = -(-ctx // block)
    need = -(-(ctx + new) // block)
    width = int(need.max(initial=0)) + 1
    ids = rng.permutation(int(need.sum()) + spare).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = ids[at:at + h]
        at += h
    return table, ctx, new, ids[at:]


@pytest.mark.parametrize("n", [1, 2, 31, 33, 511, 513, 1500])
@pytest.mark.parametrize("block", [16, 128])
def test_tables_match_the_loop(jkb, n, block):
    rng = np.random.default_rng(n + block)
    table, ctx, new, free = step(rng, n, block, 300, 90)
    total = int(new.sum())
    for n_slots in (total, total + 37):
        check_tables(jkb, table, ctx, new, free, n_slots, block)


@pytest.mark.parametrize("shift", [0, 1, 3])
def test_tables_decode_step_and_unaligned_maps(jkb, shift):
    rng = np.random.default_rng(shift)
    table, ctx, _, free = step(rng, 70, 64, 1000, 0, spare=70)
    table = np.concatenate([table, np.full((70, 1), -1, np.int32)], 1)
    check_tables(jkb, table, ctx, np.ones(70, int), free, 71, 64, shift)


def test_tables_most_sequences_and_large_prompt(jkb):
    rng = np.random.default_rng(5)
    table, ctx, new, free = step(rng, 8192, 32, 40, 6)
    check_tables(jkb, table, ctx, new, free, int(new.sum()) + 5, 32)
    table, ctx, new, free = np.full((1, 5000), -1), [0], [70_001], np.arange(5000)
    check_tables(jkb, table, ctx, new, free, 70_001, 16)


def test_tables_zero_lengths_and_no_sequences(jkb):
    free = np.arange(9)
    check_tables(jkb, np.full((5, 2), -1), [0, 16, 0, 3, 32], [0, 0, 0, 0, 0], free, 4, 16)
    check_tables(jkb, np.full((3, 2), -1), [0, 0, 0], [0, 5, 0], free, 5, 16)
    check_tables(jkb, np.full((2, 2), -1), [-4, -1], [3, -7], free, 6, 16)
    check_tables(jkb, np.full((2, 2), -1), [0, 0], [3, 4], free, 0, 16)
    got = run_tables(jkb, np.zeros((0, 3), np.int32), [], [], free, 6, 16)
    assert (got[1] == -1).all() and got[3].tolist() == [0] and got[5].tolist() == [0, 0, 0]


def test_tables_without_room(jkb):
    """A row that is too short refuses its sequence alone; an empty list refuses every later
    sequence that needs a block, and none that does not."""
    free = np.arange(100, 104)
    check_tables(jkb, np.full((4, 2), -1), [0, 0, 0, 0], [20, 33, 16, 5], free, 80, 16)
    table = np.full((5, 3), -1)
    table[3, 0] = 7
    check_tables(jkb, table, [0, 0, 0, 9, 0], [40, 17, 1, 6, 3], free, 70, 16)
    check_tables(jkb, table, [0, 0, 0, 9, 0], [40, 17, 1, 6, 3], np.zeros(0), 70, 16)
    check_tables(jkb, table, [0, 0, 0, 9, 0], [40, 17, 1, 6, 3], free, 20, 16)  # short maps
    big = 2**31 - 1
    check_tables(jkb, np.full((2, 2), -1), [big, 3], [0, 2], free, 4, 16)


def test_tables_strided_rows(jkb):
    wide = i32(np.full((3, 7), 55))
    view = wide[:, :2]
    slots, pos = i32(np.zeros(8)), i32(np.zeros(8))
    starts, lens, counts = i32(np.zeros(4)), i32(np.zeros(3)), i32(np.zeros(3))
    jkb.kv_build_tables(view, slots, pos, starts, lens, counts, i32([0, 0, 0]), i32([2, 3, 1]),
                        i32([4, 2, 9]), 16)
    assert wide[:, 0].tolist() == [4, 2, 9] and (wide[:, 1:] == 55).all()
    assert slots.tolist() == [64, 65, 32, 33, 34, 144, -1, -1]


def test_tables_refusals(jkb):
    a = i32(np.zeros(4))
    t = i32(np.zeros((4, 2)))

    def call(table=t, slots=a, positions=a, starts=i32(np.zeros(5)), lens=a, counts=a[:3], ctx=a,
             new=a, free=a, block=16):
        jkb.kv_build_tables(table, slots, positions, starts, lens, counts, ctx, new, free, block)

    for block in (0, 8, 24, 256):
        with pytest.raises(jkb.TensorBoundsError):
            call(block=block)
    with pytest.raises(ValueError):
        call(starts=a)
    with pytest.raises(ValueError):
        call(positions=a[:2])
    with pytest.raises(TypeError):
        call(free=a.float())
    n = 8193
    with pytest.raises(jkb.TensorBoundsError):
        z = i32(np.zeros(n))
        call(table=i32(np.zeros((n, 1))), starts=i32(np.zeros(n + 1)), lens=z, ctx=z, new=z)


# ------------------------------------------------------------------------------- copies

@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [8, 40, 64, 72, 96, 128, 200, 256])
def test_import_export_read(jkb, block, dim):
    rng = np.random.default_rng(block + dim)
    c = kvref.filled(rng, 5, 3, block, dim)
    cache = jkb.KvCache(7, block, 3, dim)
    ids = [6, 0, 3, 2, 5]
    cache.import_blocks(i32(ids), *(torch.from_numpy(x).cuda() for x in (c.k, c.v, c.ks, c.vs)))
    for a, b in zip(kvref.exported(cache, ids), (c.k, c.v, c.ks, c.vs)):
        assert np.array_equal(a, b)
    assert all((x == 0).all() for x in kvref.exported(cache, [1, 4]))  # fresh blocks
    out = [torch.empty(c.k.shape, device="cuda") for _ in range(2)]
    cache.read_blocks(i32(ids), *out)
    for got, codes, scales in zip(out, (c.k, c.v), (c.ks, c.vs)):
        want = codes.astype(np.float32) * scales[..., None, None]
        assert np.array_equal(got.cpu().numpy(), want)


def test_copies_skip_ids_that_are_out_of_range(jkb):
    rng = np.random.default_rng(1)
    c = kvref.filled(rng, 3, 2, 16, 64)
    cache = kvref.to_device(jkb, c)
    out = [torch.full((3, 2, 16, 64), 5.0, device="cuda") for _ in range(2)]
    cache.read_blocks(i32([1, 3, -1]), *out)
    with pytest.raises(jkb.TensorBoundsError):
        jkb.device_status()
    assert jkb.device_status() == 0
    assert (out[0][1:] == 5).all() and not (out[0][0] == 5).any()


# ------------------------------------------------------------------------------- append

def rows(rng, tokens, heads, dim, kind, size=1.0):
    x = torch.from_numpy(rng.normal(0, size, (tokens, heads, dim)).astype(np.float32))
    return x.to(TYPES[kind])


def check_append(jkb, cache, c, k, v, slots):
    jkb.kv_append(cache, k, v, i32(slots))
    c.append(k.float().cpu().numpy(), v.float().cpu().numpy(), slots)
    got = kvref.exported(cache, list(range(c.k.shape[0])))
    for name, a, b in zip(("k", "v", "k scales", "v scales"), got, (c.k, c.v, c.ks, c.vs)):
        assert np.array_equal(a, b), name
    assert jkb.device_status() == 0


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block,dim,heads", [(16, 128, 2), (32, 72, 3), (64, 80, 1), (128, 256, 1),
                                             (64, 8, 5)])
def test_append_prompts_then_single_tokens(jkb, kind, block, dim, heads):
    """A ragged prompt, then tokens one at a time, whose growing scales round old codes again."""
    rng = np.random.default_rng(dim + block)
    c = kvref.filled(rng, 9, heads, block, dim)
    cache = kvref.to_device(jkb, c)
    first = 2 * block + 3  # blocks 4, 7 and the start of 2
    slots = [4 * block + i for i in range(block)] + [7 * block + i for i in range(block)]
    slots += [2 * block + i for i in range(3)]
    slots[block + 5:block + 5] = []
    check_append(jkb, cache, c, rows(rng, first, heads, dim, kind).cuda(),
                 rows(rng, first, heads, dim, kind, 0.1).cuda(), slots)
    for i in range(3, 14):
        k, v = (rows(rng, 1, heads, dim, kind, 0.3 * i ** 0.7).cuda() for _ in range(2))
        check_append(jkb, cache, c, k, v, [2 * block + i])


def test_append_decode_step_of_many_sequences(jkb):
    rng = np.random.default_rng(3)
    c = kvref.filled(rng, 300, 2, 16, 64, 0.3, 3.0)
    cache = kvref.to_device(jkb, c)
    slots = rng.permutation(300) * 16 + rng.integers(0, 16, 300)
    slots[::17] = -1
    check_append(jkb, cache, c, rows(rng, 300, 2, 64, "f32").cuda(),
                 rows(rng, 300, 2, 64, "f32").cuda(), slots)


def test_append_long_and_ragged(jkb):
    """Enough tokens for the CTA-wide form, blocks that start and end anywhere in its ranges."""
    rng = np.random.default_rng(4)
    block, lens, slots, b = 32, [1, 700, 33, 5, 1900, 64, 31, 900], [], 0
    for n in lens:
        o = int(rng.integers(0, block))
        slots += [b * block + o + i for i in range(n)]
        b += -(-(o + n) // block)
    c = kvref.filled(rng, b, 4, block, 96)
    cache = kvref.to_device(jkb, c)
    check_append(jkb, cache, c, rows(rng, len(slots), 4, 96, "bf16").cuda(),
                 rows(rng, len(slots), 4, 96, "bf16").cuda(), slots)


def test_append_strided_and_unaligned_rows(jkb):
    rng = np.random.default_rng(6)
    heads, dim = 3, 40
    for kind, off in (("f32", 4), ("f32", 1), ("bf16", 4), ("f16", 3)):
        c = kvref.filled(rng, 4, heads, 16, dim)
        cache = kvref.to_device(jkb, c)
        fused = rows(rng, 20, 4 * heads, dim + off, kind).cuda()
        k, v = fused[:, :heads, off:], fused[:, heads::2, :dim][:, :heads]
        check_append(jkb, cache, c, k, v, list(range(3, 23)))


def test_append_values_that_are_not_ordinary(jkb):
    rng = np.random.default_rng(7)
    c = kvref.filled(rng, 6, 2, 16, 64)
    cache = kvref.to_device(jkb, c)
    k = rows(rng, 12, 2, 64, "f32")
    k[0, 0, 3], k[1, 1, 5], k[2, 0, :] = float("nan"), float("inf"), -float("inf")
    v = torch.zeros(12, 2, 64)
    v[4] = 1e-39        # absmax / 127 below the smallest normal: code 0, scale 0
    v[8, 0, 0] = 3e38
    v[8, 0, 1] = -1e30
    slots = [0, 1, 2, 3, 16, 17, 18, 19, 32, 33, 34, 35]
    check_append(jkb, cache, c, k.cuda(), v.cuda(), slots)
    check_append(jkb, cache, c, k[:1].cuda(), v[:1].cuda(), [20])  # after scale 0
    check_append(jkb, cache, c, k[3:5].cuda(), k[3:5].cuda(), [21, 22])


def test_append_skips_and_reports_bad_slots(jkb):
    rng = np.random.default_rng(8)
    c = kvref.filled(rng, 3, 2, 16, 64)
    cache = kvref.to_device(jkb, c)
    k = rows(rng, 6, 2, 64, "f32").cuda()
    before = kvref.exported(cache, [0, 1, 2])
    jkb.kv_append(cache, k, k, i32([48, 2**31 - 1, 50, -3, 99, 48]))
    with pytest.raises(jkb.TensorBoundsError):
        jkb.device_status()
    assert all(np.array_equal(a, b) for a, b in zip(before, kvref.exported(cache, [0, 1, 2])))
    jkb.kv_append(cache, k, k, i32([3, 4, 7, 8, 20, 21]))  # a gap inside block 0
    with pytest.raises(jkb.TensorBoundsError):
        jkb.device_status()
    kn = k.cpu().numpy()
    c.append(kn[:2], kn[:2], [3, 4])
    c.append(kn[4:], kn[4:], [20, 21])
    assert np.array_equal(kvref.exported(cache, [0, 1, 2])[0], c.k)


def test_append_past_four_gigabytes(jkb):
    """Code offsets that need more than 32 bits."""
    rng = np.random.default_rng(9)
    n = 34_000  # x 8 heads x 64 tokens x 256 bytes = 4.46e9
    cache = jkb.KvCache(n, 64, 8, 128)
    assert cache.device_bytes > 2**32
    k, v = (rows(rng, 70, 8, 128, "f32").cuda() for _ in range(2))
    slots = [(n - 1) * 64 + i for i in range(64)] + [(n - 7) * 64 + i for i in range(6)]
    jkb.kv_append(cache, k, v, i32(slots))
    c = kvref.Cache(2, 8, 64, 128)
    c.append(k.cpu().numpy(), v.cpu().numpy(), list(range(64)) + [64 + i for i in range(6)])
    for a, b in zip(kvref.exported(cache, [n - 1, n - 7]), (c.k, c.v, c.ks, c.vs)):
        assert np.array_equal(a, b)


def test_append_on_another_stream(jkb):
    rng = np.random.default_rng(10)
    c = kvref.filled(rng, 8, 2, 16, 64)
    cache = kvref.to_device(jkb, c)
    k, v = (rows(rng, 128, 2, 64, "f32").cuda() for _ in range(2))
    slots = i32(range(128))
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    jkb.kv_append(cache, k, v, slots, stream=st)
    st.synchronize()
    c.append(k.cpu().numpy(), v.cpu().numpy(), list(range(128)))
    assert np.array_equal(kvref.exported(cache, list(range(8)))[1], c.v)


def test_cache_refusals(jkb):
    for args in ((0, 16, 1, 64), (4, 24, 1, 64), (4, 16, 0, 64), (4, 16, 1, 0), (4, 16, 1, 257),
                 (4, 16, 1, 12), (2**31, 16, 1, 64), (4, 256, 1, 64)):
        with pytest.raises(jkb.TensorBoundsError):
            jkb.KvCache(*args)
    cache = jkb.KvCache(4, 16, 2, 64)
    k = torch.zeros(3, 2, 64, device="cuda")
    s = i32([0, 1, 2])
    with pytest.raises(ValueError):
        jkb.kv_append(cache, k, k[:2], s)
    with pytest.raises(ValueError):
        jkb.kv_append(cache, k[:, :1], k, s)
    with pytest.raises(jkb.CapabilityMismatch):
        jkb.kv_append(cache, k, k.half(), s)
    with pytest.raises(TypeError):
        jkb.kv_append(cache, k.double(), k.double(), s)
    with pytest.raises(TypeError):
        jkb.kv_append(cache, k, k, s.long())
    with pytest.raises(ValueError):
        jkb.kv_append(cache, k.transpose(1, 2).contiguous().transpose(1, 2), k, s)
    with pytest.raises(ValueError):
        cache.read_blocks(s, torch.empty(3, 2, 16, 32, device="cuda"),
                          torch.empty(3, 2, 16, 32, device="cuda"))
    jkb.kv_append(cache, k[:0], k[:0], s[:0])
    cache.destroy()
    with pytest.raises(jkb.InvalidHandle):
        jkb.kv_append(cache, k, k, s)
