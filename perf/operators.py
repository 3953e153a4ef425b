"""Cases of the 8-bit key/value cache operators, in plain torch and as the library's kernels.

Three operators that a serving step runs one after the other:

  tables     block tables and slot maps built on the GPU from request lengths
  append     new key/value rows written into a paged cache of int8 codes, with one f32 scale for
             each block of tokens and head; the values that the touched blocks then stand for
  attention  softmax(q k^T) v over that cache, for single tokens and for prompts and chunks

`run` takes what `prepare` made and returns the operator's whole outputs: in plain torch in 32
bits where `own` is false, through the jkb200 package where it is true.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _library():
    path = os.path.join(os.getcwd(), "jero-kernels-rvv_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import jkb200

    return jkb200


# ---------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one decode step of a small server: the launch is the cost
        {"name": "tables 24 decodes", "op": "tables", "requests": 24, "ctx": 200, "ctx_to": 3000,
         "new": 1, "new_to": 1, "block": 64, "lengths": 1},
        # a full scheduler: prompts, chunks and decodes of 1500 requests in short blocks
        {"name": "tables 1500 ragged", "op": "tables", "requests": 1500, "ctx": 0, "ctx_to": 2000,
         "new": 1, "new_to": 700, "block": 16, "lengths": 2},
        # the rows of one decode step, f32 from the GEMVs (32 query and 8 key/value heads of 128)
        {"name": "append 24 decodes f32", "op": "append", "requests": 24, "ctx": 200,
         "ctx_to": 3000, "new": 1, "new_to": 1, "block": 64, "kv_heads": 8, "dim": 128,
         "type": "f32", "fused": False, "lengths": 3},
        # several prompts and chunks behind earlier context, f32 from the GEMMs
        {"name": "append 6 prompts f32", "op": "append", "requests": 6, "ctx": 0, "ctx_to": 900,
         "new": 300, "new_to": 2500, "block": 32, "kv_heads": 8, "dim": 128, "type": "f32",
         "fused": False, "lengths": 4},
        # one long prompt, a strided part of a fused bf16 q/k/v projection
        {"name": "append long prompt bf16", "op": "append", "requests": 1, "ctx": 17,
         "ctx_to": 17, "new": 16411, "new_to": 16411, "block": 64, "kv_heads": 8, "dim": 128,
         "type": "bf16", "fused": True, "lengths": 5},
        # one user's decode step over a short chat: latency
        {"name": "decode 1 x 700 f32", "op": "attention", "requests": 1, "ctx": 700,
         "ctx_to": 700, "new": 1, "new_to": 1, "block": 64, "heads": 32, "kv_heads": 8,
         "dim": 128, "type": "f32", "causal": True, "window": 0, "lengths": 6},
        # a server's decode step over ragged contexts
        {"name": "decode 64 ragged f32", "op": "attention", "requests": 64, "ctx": 500,
         "ctx_to": 9000, "new": 1, "new_to": 1, "block": 64, "heads": 32, "kv_heads": 8,
         "dim": 128, "type": "f32", "causal": True, "window": 0, "lengths": 7},
        # one very long document, eight query heads to a key/value head
        {"name": "decode 1 x 131071 bf16", "op": "attention", "requests": 1, "ctx": 131070,
         "ctx_to": 131070, "new": 1, "new_to": 1, "block": 64, "heads": 64, "kv_heads": 8,
         "dim": 128, "type": "bf16", "causal": True, "window": 0, "lengths": 8},
        # sliding-window decodes in short blocks (20 query and 5 key/value heads)
        {"name": "decode 160 windowed f16", "op": "attention", "requests": 160, "ctx": 100,
         "ctx_to": 6000, "new": 1, "new_to": 1, "block": 16, "heads": 20, "kv_heads": 5,
         "dim": 128, "type": "f16", "causal": True, "window": 1024, "lengths": 9},
        # a prompt's second chunk in the framework's own f32
        {"name": "prompt 2048 f32", "op": "attention", "requests": 1, "ctx": 1111,
         "ctx_to": 1111, "new": 2048, "new_to": 2048, "block": 64, "heads": 32, "kv_heads": 8,
         "dim": 128, "type": "f32", "causal": True, "window": 0, "lengths": 10},
        # a long prompt at once
        {"name": "prompt 8192 bf16", "op": "attention", "requests": 1, "ctx": 0, "ctx_to": 0,
         "new": 8192, "new_to": 8192, "block": 64, "heads": 32, "kv_heads": 8, "dim": 128,
         "type": "bf16", "causal": True, "window": 0, "lengths": 11},
        # ragged chunks and decodes together, an odd head size
        {"name": "chunks 9 ragged f16", "op": "attention", "requests": 9, "ctx": 0,
         "ctx_to": 3000, "new": 1, "new_to": 900, "block": 32, "heads": 14, "kv_heads": 2,
         "dim": 80, "type": "f16", "causal": True, "window": 0, "lengths": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    block = rng.choice([16, 32, 64, 128])
    what = rng.choice(["tables", "append", "decode", "decode", "prompt", "prompt"])
    lengths = rng.randrange(1 << 30)
    if what == "tables":
        new = _log(rng, 1, 1500)
        n = _log(rng, 1, min(2000, 600_000 // new))
        return {"op": "tables", "requests": n, "ctx": 0, "ctx_to": _log(rng, 1, 4000), "new": 1,
                "new_to": new, "block": block, "lengths": lengths}
    heads, kv_heads = rng.choice([(32, 8), (64, 8), (20, 5), (8, 1), (16, 16), (14, 2)])
    dim = rng.choice([64, 80, 96, 128, 128])
    kind = rng.choice(["f32", "f32", "f16", "bf16"])
    if what == "append":
        new = rng.choice([1, _log(rng, 1, 4000)])
        n = _log(rng, 1, max(2, min(256, 16_000 // new)))
        return {"op": "append", "requests": n, "ctx": 0, "ctx_to": _log(rng, 1, 3000), "new": 1,
                "new_to": new, "block": block, "kv_heads": kv_heads, "dim": dim, "type": kind,
                "fused": rng.random() < 0.5, "lengths": lengths}
    c = {"op": "attention", "block": block, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "type": kind, "causal": rng.random() < 0.9,
         "window": rng.choice([0, 0, _log(rng, 16, 4000)]), "lengths": lengths}
    if what == "decode":
        ctx = _log(rng, 1, 60_000)
        c.update(requests=_log(rng, 1, max(2, min(256, 250_000 // ctx))), ctx=0, ctx_to=ctx,
                 new=1, new_to=rng.choice([1, 1, 1, 4]))
    else:
        new = _log(rng, 20, 4000)
        c.update(requests=_log(rng, 1, max(2, min(16, 6000 // new))), ctx=0,
                 ctx_to=_log(rng, 1, 4000), new=1, new_to=new)
    return c


def _lengths(c):
    """(tokens held before, new tokens) of each request: the case's own, not the seed's."""
    rng = random.Random(c["lengths"])
    ctx = [rng.randint(c["ctx"], c["ctx_to"]) for _ in range(c["requests"])]
    new = [rng.randint(c["new"], c["new_to"]) for _ in range(c["requests"])]
    return ctx, new


def _visible(c):
    """(keys read, query-key pairs) of the attention, over all requests, for one head."""
    keys = pairs = 0
    for ctx, new in zip(*_lengths(c)):
        n, w = ctx + new, c["window"]
        first = n
        for p in range(ctx, n):
            hi = p + 1 if c["causal"] else n
            lo = max(0, p - w + 1) if w else 0
            pairs += max(0, hi - lo)
            first = min(first, lo)
        keys += n - first
    return keys, pairs


def work(c):
    ctx, new = _lengths(c)
    b, tokens = c["block"], sum(new)
    if c["op"] == "tables":
        taken = sum(-(-(x + n) // b) - -(-x // b) for x, n in zip(ctx, new))
        held = sum(1 for x in ctx if x % b)
        return {"bytes": 16 * c["requests"] + 8 * _capacity(tokens) + 8 * taken + 4 * held,
                "flops": 0}
    hk, d = c["kv_heads"], c["dim"]
    if c["op"] == "append":
        blocks = sum(-(-(x + n) // b) - x // b for x, n in zip(ctx, new))
        rows, values = tokens * hk * d, blocks * hk * b * d
        return {"bytes": 2 * (rows * BYTES[c["type"]] + rows + 4 * values) + 4 * tokens
                + 8 * blocks * hk, "flops": 4 * rows}
    keys, pairs = _visible(c)
    rows = tokens * c["heads"] * d
    return {"bytes": 2 * keys * hk * d + 8 * hk * (keys // b + len(ctx))
            + 2 * rows * BYTES[c["type"]] + 4 * tokens * c["heads"],
            "flops": 4 * pairs * c["heads"] * d}


def _capacity(tokens):
    """Slots of a step's map: a server pads it so that one captured graph serves many steps."""
    return -(-tokens // 32) * 32


# ---------------------------------------------------------------------------------- the inputs

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _quantized(x):
    """int8 codes [n][heads][block][dim] and scales [n][heads] of values of that shape."""
    s = x.abs().amax((2, 3)) / 127
    return (x / s[:, :, None, None]).round().clamp(-127, 127).to(torch.int8), s


def _blocks_of_codes(n, c, g):
    """A filled cache: keys whose channels differ in size, as projections give them."""
    shape = (n, c["kv_heads"], c["block"], c["dim"])
    ks, vs = [], []
    for at in range(0, n, 2048):
        part = (min(2048, n - at),) + shape[1:]
        for into, spread in ((ks, 0.6), (vs, 0.3)):
            gain = torch.empty((1, shape[1], 1, shape[3]), device="cuda")
            gain.normal_(0, spread, generator=torch.Generator("cuda").manual_seed(
                g.initial_seed() + (7 if into is ks else 8)))
            x = torch.empty(part, device="cuda").normal_(0, 1, generator=g)
            into.append(_quantized(x * gain.exp()))
    (kc, ksc), (vc, vsc) = (tuple(torch.cat(t) for t in zip(*p)) for p in (ks, vs))
    return kc, vc, ksc, vsc


def prepare(c, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    ctx, new = _lengths(c)
    b, n = c["block"], c["requests"]
    tokens = sum(new)
    held = [-(-x // b) for x in ctx]
    need = [-(-(x + m) // b) for x, m in zip(ctx, new)]
    width = max(need) + 1
    s = {"case": c}
    if c["op"] == "tables":
        ids = torch.randperm(sum(need) + 16, generator=g, device="cuda").to(torch.int32)
        at, table = 0, torch.full((n, width), -1, dtype=torch.int32)
        ids_host = ids.cpu()
        for i, h in enumerate(held):
            table[i, :h] = ids_host[at:at + h]
            at += h
        cap = _capacity(tokens)
        s.update(table=table.cuda(), free=ids[at:].contiguous(), ctx=_ints(ctx), new=_ints(new),
                 slots=torch.empty(cap, dtype=torch.int32, device="cuda"),
                 positions=torch.empty(cap, dtype=torch.int32, device="cuda"),
                 starts=torch.empty(n + 1, dtype=torch.int32, device="cuda"),
                 lens=torch.empty(n, dtype=torch.int32, device="cuda"),
                 counts=torch.empty(3, dtype=torch.int32, device="cuda"))
        if own:
            s["lib"] = _library()
        return s

    hk, d, dtype = c["kv_heads"], c["dim"], TYPES[c["type"]]
    first = [x // b for x in ctx] if c["op"] == "append" else [0] * n
    blocks = sum(m - f for m, f in zip(need, first)) + 3
    ids = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    kc, vc, ksc, vsc = _blocks_of_codes(blocks, c, g)
    if c["op"] == "append":
        # the pool here holds the blocks that the step touches; slots as the tables give them
        start, slots = 0, []
        ids_host = ids.tolist()
        for x, m, f, h in zip(ctx, new, first, need):
            own_ids = ids_host[start:start + h - f]
            slots += [own_ids[p // b - f] * b + p % b for p in range(x, x + m)]
            start += h - f
        width = hk * d
        if c["fused"]:
            qkv = torch.empty((tokens, 4 * width), device="cuda").normal_(0, 1, generator=g)
            qkv = qkv.to(dtype)
            k, v = qkv[:, 2 * width:3 * width], qkv[:, 3 * width:]
        else:
            k, v = (torch.empty((tokens, width), device="cuda").normal_(0, 1, generator=g)
                    .to(dtype) for _ in range(2))
        s.update(k=k.unflatten(1, (hk, d)), v=v.unflatten(1, (hk, d)), slots=_ints(slots),
                 touched=torch.sort(ids[:start]).values)
        s["k_out"], s["v_out"] = (torch.empty((start, hk, b, d), device="cuda")
                                  for _ in range(2))
    else:
        table = torch.full((n, width), -1, dtype=torch.int32)
        ids_host, at = ids.cpu(), 0
        for i, m in enumerate(need):
            table[i, :m] = ids_host[at:at + m]
            at += m
        starts = [0]
        for m in new:
            starts.append(starts[-1] + m)
        q = torch.empty((tokens, c["heads"], d), device="cuda").normal_(0, 2, generator=g)
        s.update(q=q.to(dtype), table=table.cuda(), lens=_ints([x + m for x, m in zip(ctx, new)]),
                 starts=_ints(starts), most=max(new), scale=1 / math.sqrt(d))
    if own:
        lib = s["lib"] = _library()
        s["cache"] = lib.KvCache(blocks, b, hk, d)
        s["cache"].import_blocks(torch.arange(blocks, dtype=torch.int32, device="cuda"), kc, vc,
                                 ksc, vsc)
        if c["op"] == "attention":
            s["space"] = lib.AttentionWorkspace(s["cache"])
            s["out"] = torch.empty_like(s["q"])
            s["lse"] = torch.empty((tokens, c["heads"]), device="cuda")
    else:
        s.update(kc=kc, vc=vc, ksc=ksc, vsc=vsc)
    return s


# ---------------------------------------------------------------------------------- the passes

def run(s):
    op = s["case"]["op"]
    if own:
        return {"tables": _own_tables, "append": _own_append,
                "attention": _own_attention}[op](s)
    return {"tables": _plain_tables, "append": _plain_append,
            "attention": _plain_attention}[op](s)


def _own_tables(s):
    s["lib"].kv_build_tables(s["table"], s["slots"], s["positions"], s["starts"], s["lens"],
                             s["counts"], s["ctx"], s["new"], s["free"], s["case"]["block"])
    return {k: s[k] for k in ("table", "slots", "positions", "starts", "lens", "counts")}


def _own_append(s):
    s["lib"].kv_append(s["cache"], s["k"], s["v"], s["slots"])
    s["cache"].read_blocks(s["touched"], s["k_out"], s["v_out"])
    return {"k": s["k_out"], "v": s["v_out"]}


def _own_attention(s):
    c = s["case"]
    s["lib"].attention_kv8(s["out"], s["q"], s["cache"], s["space"], s["table"], s["lens"],
                           s["starts"], s["most"], s["scale"], causal=c["causal"],
                           window=c["window"], lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def _plain_tables(s):
    """Whole blocks are taken from the free list in the requests' order; a request that finds no
    room in its table's row or in the list gets none, and -1 in the slot map."""
    b, table, free, ctx, new = s["case"]["block"], s["table"], s["free"], s["ctx"], s["new"]
    width, cap = table.shape[1], s["slots"].shape[0]
    first = (ctx + b - 1) // b
    room = ctx + new <= width * b
    need = torch.where(room, (ctx + new + b - 1) // b - first, 0)
    upto = torch.cumsum(need, 0, dtype=torch.int32)
    fits = room & ((upto <= free.shape[0]) | (need == 0))
    j = torch.arange(width, device="cuda")
    fresh = fits[:, None] & (j >= first[:, None]) & (j < (first + need)[:, None])
    at = ((upto - need)[:, None] + j - first[:, None]).clamp(0, free.shape[0] - 1)
    table.copy_(torch.where(fresh, free[at], table))
    ends = torch.cumsum(new, 0, dtype=torch.int32)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    t = torch.arange(cap, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(ends, t, right=True).clamp(max=ends.shape[0] - 1)
    pos = ctx[seq] + t - starts[seq]
    held = (t < ends[-1]) & fits[seq]
    slot = table[seq, (pos // b).clamp(max=width - 1)] * b + pos % b
    return {"table": table, "slots": torch.where(held, slot, -1),
            "positions": torch.where(held, pos, -1), "starts": starts,
            "lens": ctx + torch.where(fits, new, 0),
            "counts": torch.stack([ends[-1], torch.where(fits, upto, 0).amax(),
                                   (~fits).sum().to(torch.int32)])}


def _plain_append(s):
    """A block and head's scale is its absmax / 127: a block that starts with this call takes the
    new rows' alone, one that goes on keeps the larger of its own and theirs, and its earlier
    codes are rounded again where it grew. Rounding is to nearest, ties to even."""
    touched, slots, b = s["touched"].long(), s["slots"].long(), s["case"]["block"]
    at = torch.searchsorted(touched, slots // b)
    off = slots % b
    first = torch.full((touched.shape[0],), b, device="cuda").scatter_reduce(
        0, at, off, "amin")
    out = {}
    for name, codes, scales in (("k", s["kc"], s["ksc"]), ("v", s["vc"], s["vsc"])):
        x = s[name].float()
        most = torch.zeros((touched.shape[0], x.shape[1]), device="cuda").index_reduce(
            0, at, x.abs().amax(2), "amax")
        old = torch.where(first[:, None] == 0, 0.0, scales[touched])
        new = torch.maximum(old, most / 127.0)
        ratio = torch.where(new > 0, old / new, 0.0)
        inv = torch.where(new > 0, 1.0 / new, 0.0)
        was = codes[touched]
        again = (was.float() * ratio[:, :, None, None]).round().to(torch.int8)
        earlier = (torch.arange(b, device="cuda") < first[:, None])[:, None, :, None]
        now = torch.where(earlier, again, was)
        now[at, :, off] = (x * inv[at][:, :, None]).round().clamp(-127, 127).to(torch.int8)
        codes[touched], scales[touched] = now, new
        out[name] = now.float() * new[:, :, None, None]
    return out


def _plain_attention(s):
    c, table, lens, starts = s["case"], s["table"].clamp(min=0).long(), s["lens"], s["starts"]
    n, width = table.shape
    hk, b, d, most = c["kv_heads"], c["block"], c["dim"], s["most"]
    g, length = c["heads"] // hk, width * b

    def dense(codes, scales):
        x = codes[table].float() * scales[table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(n, hk, length, d)

    q = s["q"]
    count = starts[1:] - starts[:-1]
    i = torch.arange(most, device="cuda")
    rows = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1).long()
    padded = q[rows].float().reshape(n, most, hk, g, d).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(padded.reshape(n, hk, g * most, d),
                          dense(s["kc"], s["ksc"]).transpose(2, 3)).mul_(s["scale"])
    j = torch.arange(length, device="cuda")
    pos = (lens - count)[:, None] + i
    seen = (j < lens[:, None])[:, None, :] & (i < count[:, None])[:, :, None]
    if c["causal"]:
        seen = seen & (j <= pos[:, :, None])
    if c["window"]:
        seen = seen & (j > pos[:, :, None] - c["window"])
    scores = scores.view(n, hk, g, most, length)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    p = scores.sub_(top).exp_()
    total = p.sum(-1)
    o = torch.matmul(p.view(n, hk, g * most, length), dense(s["vc"], s["vsc"]))
    o = o.view(n, hk, g, most, d)
    o = torch.where(total[..., None] > 0, o / total[..., None], 0.0)
    lse = top[..., 0] + total.log()
    t = torch.arange(q.shape[0], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    at = (t - starts[seq]).long()
    o = o.permute(0, 3, 1, 2, 4)[seq, at].reshape(q.shape)
    return {"out": o.to(q.dtype),
            "lse": lse.permute(0, 3, 1, 2)[seq, at].reshape(q.shape[0], c["heads"])}


# ---------------------------------------------------------------------------------- in 64 bits

def exact(c, seed):
    """What `run` returns, from the definitions, request by request in 64 bits."""
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    return {"tables": _exact_tables, "append": _exact_append,
            "attention": _exact_attention}[c["op"]](c, s)


def _exact_tables(c, s):
    b = c["block"]
    table, free = s["table"].tolist(), s["free"].tolist()
    slots, positions, starts, lens, taken, refused = [], [], [0], [], 0, 0
    for row, x, m in zip(table, s["ctx"].tolist(), s["new"].tolist()):
        first, last = -(-x // b), -(-(x + m) // b)
        if x + m > len(row) * b or taken + last - first > len(free):
            raise ValueError("the cases give every request its room")
        row[first:last] = free[taken:taken + last - first]
        taken += last - first
        slots += [row[p // b] * b + p % b for p in range(x, x + m)]
        positions += range(x, x + m)
        starts.append(starts[-1] + m)
        lens.append(x + m)
    pad = [-1] * (_capacity(starts[-1]) - starts[-1])
    return {"table": _ints(table), "slots": _ints(slots + pad),
            "positions": _ints(positions + pad), "starts": _ints(starts), "lens": _ints(lens),
            "counts": _ints([starts[-1], taken, refused])}


def _exact_append(c, s):
    b = c["block"]
    runs = {}
    for t, slot in enumerate(s["slots"].tolist()):
        runs.setdefault(slot // b, []).append(t)
    out = {}
    for name, codes, scales in (("k", s["kc"], s["ksc"]), ("v", s["vc"], s["vsc"])):
        rows, parts = s[name], []
        for block in s["touched"].tolist():
            at = runs[block]
            x = rows[at[0]:at[-1] + 1].double().transpose(0, 1)
            o = int(s["slots"][at[0]]) % b
            new = x.abs().amax((1, 2)) / 127
            if o:
                new = torch.maximum(new, scales[block].double())
            now = codes[block].double()
            now[:, :o] = (now[:, :o] * (scales[block].double() / new)[:, None, None]).round()
            now[:, o:o + len(at)] = (x / new[:, None, None]).round()
            parts.append(now * new[:, None, None])
        out[name] = torch.stack(parts)
    return out


def _exact_attention(c, s):
    keys, pairs = _visible(c)
    if pairs * c["heads"] * c["dim"] > 1 << 40:
        return None
    b, d, g = c["block"], c["dim"], c["heads"] // c["kv_heads"]
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(out.shape[:2], dtype=torch.float64, device="cuda")
    for r, n in enumerate(lens):
        lo, hi = starts[r], starts[r + 1]
        ids = s["table"][r, :-(-n // b)].long()
        j = torch.arange(n, device="cuda")
        pos = n - (hi - lo) + torch.arange(hi - lo, device="cuda")
        hide = (j > pos[:, None]) if c["causal"] else torch.zeros((hi - lo, n), dtype=torch.bool,
                                                                  device="cuda")
        if c["window"]:
            hide = hide | (j <= pos[:, None] - c["window"])
        for h in range(c["kv_heads"]):
            k, v = ((codes[ids, h].double() * scales[ids, h].double()[:, None, None])
                    .reshape(-1, d)[:n] for codes, scales in ((s["kc"], s["ksc"]),
                                                              (s["vc"], s["vsc"])))
            for e in range(h * g, h * g + g):
                x = (s["q"][lo:hi, e].double() * s["scale"]) @ k.T
                x = x.masked_fill(hide, -math.inf)
                total = torch.logsumexp(x, 1)
                lse[lo:hi, e] = total
                w = torch.exp(x - torch.where(total > -math.inf, total, 0.0)[:, None])
                out[lo:hi, e] = w @ v
    return {"out": out, "lse": lse}
