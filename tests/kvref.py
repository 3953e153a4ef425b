"""Plain forms of the 8-bit key/value cache operators for the tests: numpy and 64-bit torch, one
token, block or sequence at a time, written from the definitions in include/jkb200.h."""
import math

import numpy as np
import torch

F = np.float32


def build_tables(table, ctx, new, free, n_slots, block):
    """(table, slots, positions, q_starts, kv_lens, counts) of kv_build_tables."""
    table = table.copy()
    slots, pos, starts, lens = [], [], [0], []
    taken, refused, over = 0, 0, False
    asked = 0
    for i, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(int(c), 0), max(int(n), 0)
        room = c + n <= table.shape[1] * block
        first = -(-c // block)
        need = -(-(c + n) // block) - first if room else 0
        asked += need
        fits = room and (need == 0 or asked <= len(free))
        if fits and need:
            table[i, first:first + need] = free[asked - need:asked]
            taken = asked
        refused += not fits
        for p in range(c, c + n):
            fits_here = fits and table[i, p // block] >= 0  # a held block that the row lacks
            slots.append(table[i, p // block] * block + p % block if fits_here else -1)
            pos.append(p if fits_here else -1)
        starts.append(starts[-1] + n)
        lens.append(c + n if fits else c)
    total = len(slots)
    slots = (slots + [-1] * n_slots)[:n_slots]
    pos = (pos + [-1] * n_slots)[:n_slots]
    return (table, np.array(slots, np.int32), np.array(pos, np.int32),
            np.array(starts, np.int32), np.array(lens, np.int32),
            np.array([total, taken, refused], np.int32))


class Cache:
    """A cache as plain arrays: codes [blocks][heads][block][dim], scales [blocks][heads]."""

    def __init__(self, n, heads, block, dim):
        self.block = block
        self.k, self.v = (np.zeros((n, heads, block, dim), np.int8) for _ in range(2))
        self.ks, self.vs = (np.zeros((n, heads), F) for _ in range(2))

    def append(self, k, v, slots):
        """The f32 steps of kv_append, block by block (k, v: float32 [tokens][heads][dim])."""
        runs = []
        for t, s in enumerate(slots):
            if s < 0:
                continue
            if runs and runs[-1][-1][0] == t - 1 and runs[-1][-1][1] // self.block == s // self.block:
                runs[-1].append((t, s))
            else:
                runs.append([(t, s)])
        for run in runs:
            b, o = run[0][1] // self.block, run[0][1] % self.block
            ts = [t for t, _ in run]
            for rows, codes, scales in ((k, self.k, self.ks), (v, self.v, self.vs)):
                x = np.where(np.isfinite(rows[ts]), rows[ts], F(0)).astype(F)
                for h in range(codes.shape[1]):
                    old = scales[b, h] if o else F(0)
                    s = max(old, F(np.abs(x[:, h]).max() * F(1 / 127)))
                    if s < np.finfo(F).tiny:
                        s = F(0)
                    inv = F(1) / s if s > 0 else F(0)
                    if o and s > old:
                        codes[b, h, :o] = np.rint(codes[b, h, :o].astype(F) * F(old / s))
                    codes[b, h, o:o + len(run)] = np.clip(np.rint(x[:, h] * inv), -127, 127)
                    scales[b, h] = s


def filled(rng, n, heads, block, dim, k_size=1.0, v_size=1.0):
    """A Cache of random codes and scales (scales spread over a factor of 8)."""
    c = Cache(n, heads, block, dim)
    for codes in (c.k, c.v):
        codes[:] = np.clip(np.rint(rng.normal(0, 40, codes.shape)), -127, 127)
    c.ks[:] = k_size / 40 * 2.0 ** rng.uniform(-1.5, 1.5, c.ks.shape)
    c.vs[:] = v_size / 40 * 2.0 ** rng.uniform(-1.5, 1.5, c.vs.shape)
    return c


def to_device(jkb, c, n_blocks=None):
    """A KvCache with the contents of `c` in its first blocks."""
    n, heads, block, dim = c.k.shape
    cache = jkb.KvCache(n_blocks or n, block, heads, dim)
    ids = torch.arange(n, dtype=torch.int32, device="cuda")
    cache.import_blocks(ids, *(torch.from_numpy(x).cuda() for x in (c.k, c.v, c.ks, c.vs)))
    return cache


def exported(cache, ids):
    """(k codes, v codes, k scales, v scales) of the blocks, as numpy arrays."""
    shape = (len(ids), cache.n_kv_heads, cache.block_tokens, cache.head_dim)
    out = [torch.empty(shape, dtype=torch.int8, device="cuda") for _ in range(2)]
    out += [torch.empty(shape[:2], device="cuda") for _ in range(2)]
    cache.export_blocks(torch.tensor(ids, dtype=torch.int32, device="cuda"), *out)
    return [t.cpu().numpy() for t in out]


def attention(c, q, table, lens, starts, scale, causal, window):
    """Per query the output and lse in 64 bits, and two sums for the error bounds (below):
    `size` = sum_j w_j |v_j| per output element, `slack` = the largest over the visible keys of
    scale (max_d |q_d| sum_d |k_d| 2^-24 + 2^-19 sum_d |q_d k_d|)."""
    q = q.double().cuda()
    tokens, heads, dim = q.shape
    g = heads // c.k.shape[1]
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64, device="cuda")
    slack = torch.zeros_like(lse)
    kv = [torch.from_numpy(x).cuda().double() * torch.from_numpy(s).cuda().double()[..., None, None]
          for x, s in ((c.k, c.ks), (c.v, c.vs))]
    for i, n in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        if a == b or n == 0:
            continue
        ids = torch.as_tensor(table[i][:-(-n // c.block)]).long().cuda()
        j = torch.arange(n, device="cuda")
        p = n - (b - a) + torch.arange(b - a, device="cuda")
        seen = torch.ones((b - a, n), dtype=torch.bool, device="cuda")
        if causal:
            seen &= j <= p[:, None]
        if window:
            seen &= j > p[:, None] - window
        for h in range(heads):
            k, v = (x[ids, h // g].reshape(-1, dim)[:n] for x in kv)
            x = q[a:b, h]
            s = (scale * (x @ k.T)).masked_fill(~seen, -math.inf)
            lse[a:b, h] = torch.logsumexp(s, 1)
            w = torch.exp(s - lse[a:b, h].nan_to_num(neginf=0.0)[:, None])
            out[a:b, h], size[a:b, h] = w @ v, w @ v.abs()
            e = abs(scale) * (x.abs().amax(1, keepdim=True) * k.abs().sum(1) * 2.0 ** -24
                              + 2.0 ** -19 * (x.abs() @ k.abs().T))
            slack[a:b, h] = (e * seen).amax(1)
    return out, lse, size, slack


def check_attention(got, got_lse, ref, longest):
    """Asserts the outputs within what the kernels' roundings can amount to.

    A score is off by at most `slack` (the row's 24-bit digits or the two f16 parts of q, and a
    truncated f32 sum of up to 16 tensor-core steps) plus 2^-21 of its own size; ex2 adds 2^-22;
    the weights' sums over n keys at most (n / 16 + 64) roundings of 2^-23; p's split into two f16
    2^-21, its single f16 (16-bit outputs of prompts) 2^-11. Both numerator and denominator have
    these. The output's own type rounds last."""
    out, lse, size, slack = ref
    rel = 2 * (slack + 2.0 ** -20 + (longest / 16 + 64) * 2.0 ** -23)
    rel = rel + 2.0 ** -21 * lse.abs().nan_to_num(posinf=0.0, neginf=0.0) + 2.0 ** -20
    last = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
    if got.dtype != torch.float32:
        rel = rel + 2.0 ** -11
    err = (got.double() - out).abs()
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 1e-37
    bound = rel[..., None] * size + last[got.dtype] * out.abs() + tiny
    assert torch.isfinite(got).all()
    assert bool((err <= bound).all()), float((err / bound).max())
    if got_lse is not None:
        empty = torch.isinf(lse)
        assert torch.equal(empty, torch.isinf(got_lse)) and not torch.isnan(got_lse).any()
        assert bool((got_lse[empty] < 0).all())
        e = (got_lse.double() - lse)[~empty].abs()
        assert bool((e <= (rel + 2.0 ** -21 * lse.abs())[~empty]).all()), float(e.max())
