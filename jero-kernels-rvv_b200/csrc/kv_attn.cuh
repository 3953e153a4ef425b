// What the two attention kernels share (kv_attn.cu: few query rows; kv_attn_tc.cu: prompts).
#pragma once

#include "kv_cache.cuh"
#include "ptx.cuh"

namespace jkb {

struct AttnParams {
    const uint8_t *codes;
    const float2 *scales;
    int n_blocks, kv_heads, log_block, dim;
    int group;  // query heads of a kv head
    const void *q;
    void *out;
    size_t q_token, q_head, out_token, out_head;
    int q_vec, out_vec;  // rows may be read / written 16 bytes at a time
    float *lse;
    int n_tokens;
    const int32_t *table, *kv_lens, *q_starts;
    size_t table_stride;
    int n_seqs, row_blocks;
    int window, causal;
    float scale2;        // scale * log2(e): the softmax works in powers of two
    int min_rows, max_rows;  // query rows (tokens * group) of the sequences this launch takes
    float *partial;       // the workspace's (kv_cache.cuh)
    int *counters;
    float *tile_partial;
    int *tile_counters;
    int *err;
};

// Pieces of a row tile that are joined at a time, in a tree whose shape only the line decides. (One
// CTA that joins all 38 pieces of a kv head takes 7.6 us, 4.1 with the tree; a call over one kv
// head with 47 and 79 pieces 44 and 27 us.)
constexpr int JOIN = 8, JOIN_LEVELS = 3;

// One sequence of a launch: query tokens q0 .. q0 + nq, cached tokens len, the visible ones
// lo .. len. nq = 0 where the launch does not take it.
struct AttnSeq {
    int q0, nq, len, lo;
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnParams &p, int i) {
    AttnSeq s;
    s.q0 = min(max(__ldg(p.q_starts + i), 0), p.n_tokens);
    const int q1 = min(max(__ldg(p.q_starts + i + 1), s.q0), p.n_tokens);
    s.nq = q1 - s.q0;
    const long long rows = (long long)s.nq * p.group;
    if (rows < p.min_rows || rows > p.max_rows) s.nq = 0;
    const int room = p.row_blocks << p.log_block, len = __ldg(p.kv_lens + i);
    if (s.nq && (len < 0 || len > room)) atomicOr(p.err, ERR_KV_RANGE);
    s.len = min(max(len, 0), room);
    s.lo = 0;
    if (p.window) s.lo = min(max((long long)s.len - s.nq + 1 - p.window, 0ll), (long long)s.len);
    return s;
}

// The first token that a query at position pos sees (pos is negative for queries before the first
// cached token; the difference is only taken where it cannot overflow).
__device__ __forceinline__ int first_seen(const AttnParams &p, int pos) {
    return p.window && pos >= p.window ? pos - p.window + 1 : 0;
}

// A bounded wait in few instructions (the roles' loops hold many): at most 2^20 tries of about a
// microsecond.
__device__ __forceinline__ bool mbar_wait_short(uint64_t *b, uint32_t parity,
                                                volatile int *abort_flag, int *err) {
#pragma unroll 1
    for (uint32_t i = 0;; i++) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(b)), "r"(parity)
            : "memory");
        if (ok) return true;
        if (*abort_flag || i >> 20) break;
    }
    if (!*abort_flag) {
        *abort_flag = 1;
        atomicOr(err, ERR_ATTN_WAIT);
    }
    return false;
}

int attn_decode_launch(const AttnParams &p, int type, int dim_p, size_t max_rows,
                       cudaStream_t st);

// Sequences of at most `rows` query rows a kv head are few-row ones; head sizes up to 128.
int attn_prompt_launch(const AttnParams &p, int type, int dim_p, cudaStream_t st);

}  // namespace jkb
