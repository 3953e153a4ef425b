"""The attention half of a decoder layer over the 8-bit paged key/value cache: Q8_0 projections,
block tables, append and attention, for prompts and for decode steps.

    python jero-kernels-rvv_b200/examples/attention_layer.py

Three requests are prefilled in one ragged batch and then decoded a token at a time. The last
step's output is compared with plain attention in 64 bits over the cache's own values.
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import jkb200 as jkb  # noqa: E402


def q8_0_bytes(rows: int, cols: int, sigma: float, rng) -> np.ndarray:
    """GGUF Q8_0 bytes of a random matrix: per 32 elements an f16 scale and 32 int8."""
    blocks = np.zeros((rows * cols // 32, 34), np.uint8)
    x = rng.standard_normal((blocks.shape[0], 32), dtype=np.float32) * np.float32(sigma)
    d = (np.abs(x).max(1) / 127).astype(np.float16)
    blocks[:, :2] = d.view(np.uint8).reshape(-1, 2)
    blocks[:, 2:] = np.rint(x / d.astype(np.float32)[:, None]).astype(np.int8).view(np.uint8)
    return blocks.reshape(-1)


class AttentionLayer:
    """q/k/v projection (one fused weight), cache, attention and output projection. All buffers
    are made here, none during a step."""

    def __init__(self, hidden, heads, kv_heads, dim, n_blocks, block_tokens, max_seqs, row_blocks,
                 max_tokens, seed=0):
        rng = np.random.default_rng(seed)
        self.heads, self.kv_heads, self.dim, self.hidden = heads, kv_heads, dim, hidden
        width = (heads + 2 * kv_heads) * dim

        def weight(name, rows, cols):
            raw = q8_0_bytes(rows, cols, cols ** -0.5, rng)
            view = jkb.TensorView(name, jkb.QuantType.Q8_0, [rows, cols], raw)
            return jkb.RepackedWeight.from_tensor(view, rows, cols)

        self.w_qkv, self.w_out = weight("qkv", width, hidden), weight("out", hidden, heads * dim)
        self.act_in = jkb.QuantizedActQ8(max_tokens, hidden)
        self.act_out = jkb.QuantizedActQ8(max_tokens, heads * dim)
        self.cache = jkb.KvCache(n_blocks, block_tokens, kv_heads, dim)
        self.workspace = jkb.AttentionWorkspace(self.cache)

        def ints(*shape):
            return torch.zeros(shape, dtype=torch.int32, device="cuda")

        self.table = ints(max_seqs, row_blocks)
        self.slots, self.positions = ints(max_tokens), ints(max_tokens)
        self.q_starts, self.kv_lens, self.counts = ints(max_seqs + 1), ints(max_seqs), ints(3)
        self.free = torch.randperm(n_blocks, generator=torch.Generator().manual_seed(seed))
        self.free = self.free.to(torch.int32).cuda()
        self.qkv = torch.empty(max_tokens, heads + 2 * kv_heads, dim, device="cuda")
        self.attn = torch.empty(max_tokens, heads, dim, device="cuda")
        self.out = torch.empty(max_tokens, hidden, device="cuda")

    def step(self, x, ctx_lens, new_lens, max_new: int):
        """x [tokens, hidden]: the new tokens of all sequences, in order; ctx_lens, new_lens int32
        [sequences]. Returns the layer's output [tokens, hidden]."""
        n, seqs = x.shape[0], ctx_lens.numel()
        qkv, attn, out = self.qkv[:n], self.attn[:n], self.out[:n]
        table, kv_lens = self.table[:seqs], self.kv_lens[:seqs]
        q_starts, slots = self.q_starts[:seqs + 1], self.slots[:n]
        jkb.gemm_repacked_f32(qkv, self.w_qkv, x, n, self.act_in)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)  # strided views
        jkb.kv_build_tables(table, slots, self.positions[:n], q_starts, kv_lens, self.counts,
                            ctx_lens, new_lens, self.free, self.cache.block_tokens)
        jkb.kv_append(self.cache, k, v, slots)
        jkb.attention_kv8(attn, q, self.cache, self.workspace, table, kv_lens, q_starts, max_new,
                          self.dim ** -0.5)
        jkb.gemm_repacked_f32(out, self.w_out, attn, n, self.act_out)
        self.free = self.free[int(self.counts[1]):]  # the scheduler's part: blocks taken
        return out

    def plain_attention(self, n, ctx_lens, new_lens):
        """The last step's attention in 64 bits, over the cache's values."""
        heads, kv_heads, dim, bt = self.heads, self.kv_heads, self.dim, self.cache.block_tokens
        q = self.qkv[:n, :heads].double()
        out, at = torch.empty_like(q), 0
        for i, (c, m) in enumerate(zip(ctx_lens.tolist(), new_lens.tolist())):
            blocks = self.table[i, :-(-(c + m) // bt)].contiguous()
            k = torch.empty(blocks.numel(), kv_heads, bt, dim, device="cuda")
            v = torch.empty_like(k)
            self.cache.read_blocks(blocks, k, v)
            k, v = (t.transpose(0, 1).reshape(kv_heads, -1, dim)[:, :c + m].double()
                    .repeat_interleave(heads // kv_heads, 0) for t in (k, v))
            s = torch.einsum("thd,hjd->htj", q[at:at + m], k) * dim ** -0.5
            pos = torch.arange(c, c + m, device="cuda")
            s.masked_fill_(torch.arange(c + m, device="cuda") > pos[:, None], -torch.inf)
            out[at:at + m] = torch.einsum("htj,hjd->thd", s.softmax(-1), v)
            at += m
        return out


def run(hidden=1024, heads=16, kv_heads=4, dim=64, prompts=(300, 17, 128), steps=20,
        block_tokens=32, seed=0):
    """Prefill and decode; (outputs of all steps, largest attention error of a prefill and of a
    decode step relative to the largest output)."""
    total = sum(prompts) + steps * len(prompts)
    row_blocks = -(-(max(prompts) + steps) // block_tokens)
    layer = AttentionLayer(hidden, heads, kv_heads, dim, total // block_tokens + len(prompts) + 1,
                           block_tokens, len(prompts), row_blocks, max(sum(prompts), 1), seed)
    gen = torch.Generator().manual_seed(seed)

    def error(n, ctx, new):
        want = layer.plain_attention(n, ctx, new)
        return float((layer.attn[:n].double() - want).abs().max() / want.abs().max())

    new = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    ctx = torch.zeros_like(new)
    x = torch.randn(sum(prompts), hidden, generator=gen).cuda()
    outs = [layer.step(x, ctx, new, max(prompts)).clone()]
    errors = [error(x.shape[0], ctx, new)]
    for _ in range(steps):
        ctx = ctx + new
        new = torch.ones_like(ctx)
        x = torch.randn(len(prompts), hidden, generator=gen).cuda()
        outs.append(layer.step(x, ctx, new, 1).clone())
    errors.append(error(len(prompts), ctx, new))
    status = jkb.device_status()
    assert status == 0, f"device status {status}"
    return outs, errors


if __name__ == "__main__":
    outs, errors = run()
    print(f"prefill {tuple(outs[0].shape)}, {len(outs) - 1} decode steps of "
          f"{tuple(outs[-1].shape)}; attention against 64 bits: prefill {errors[0]:.1e}, "
          f"decode {errors[1]:.1e}")
