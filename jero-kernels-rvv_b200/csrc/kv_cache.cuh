// The 8-bit paged key/value cache: handle and code layout (kv_cache.cu writes it, the attention
// kernels read it).
//
// A block and kv head hold block_tokens / 16 groups of 16 tokens; a group is one contiguous run
// of 32 * dim_p bytes (dim_p: head_dim rounded up to 64, 96, 128, 192 or 256; elements past
// head_dim are code 0), so that one bulk copy brings the keys and values of 16 tokens:
//   keys   [2][dim_p / 32][8 tokens][32 dims]: eight tokens' 32 dims are 256 bytes, of which lane
//          4 g + t of a warp takes bytes 8 t .. 8 t + 8 of token g -- the B operand of
//          mma.m16n8k32 with dims in the order 8 t + {0..3}, 8 t + {4..7}. Codes are int8.
//   values [dim_p / 32][8 (g)][4 (t)][4 (j)][4 tokens]: lane 4 g + t takes 16 bytes: dims 4 g + j
//          of the 32, tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 -- the B operands of four
//          mma.m16n8k16 over 16 tokens. Bytes are code + 128, which two byte permutes and a
//          packed subtraction turn into f16.
// Both reads are contiguous 256- and 512-byte runs of a warp: free of bank conflicts.
#pragma once

#include "jkb_internal.h"

struct jkb_kv_cache {
    uint32_t magic;
    int device;
    size_t n_blocks, n_heads, device_bytes;
    int block_tokens, dim, dim_p;
    uint8_t *codes;  // [n_blocks][n_heads][block_tokens / 16] groups of 32 * dim_p bytes
    float2 *scales;  // [n_blocks][n_heads]: (key scale, value scale)
};

// Partial results of attention pieces, and the counters by which a piece knows that it is its
// row tile's last (zero between calls).
struct jkb_attn_workspace {
    uint32_t magic;
    int device;
    int dim_p;
    int ctas;          // pieces' slots: 2 per CTA
    float *partial;    // [2 * ctas][ATTN_ROWS][dim_p + 2]
    int *counters;     // [ctas]
};

namespace jkb {

constexpr uint32_t KV_MAGIC = 0x4A4B4331u;       // "JKC1"
constexpr uint32_t ATTN_WS_MAGIC = 0x4A4B5331u;  // "JKS1"
// bits of the device error word
constexpr int ERR_KV_RANGE = 4, ERR_ATTN_WAIT = 8;
constexpr int KV_GROUP = 16;   // tokens of a group
constexpr int ATTN_ROWS = 16;  // most query rows of a decode row tile

int check_kv_cache(const jkb_kv_cache *c, const char *fn);

// Byte of the key code of (token, dim) in its group, and of the value code.
__host__ __device__ inline int kv_key_at(int token, int dim, int dim_p) {
    return (token >> 3) * 8 * dim_p + (dim >> 5) * 256 + (token & 7) * 32 + (dim & 31);
}
__host__ __device__ inline int kv_value_at(int token, int dim, int dim_p) {
    const int d = dim & 31;
    return 16 * dim_p + (dim >> 5) * 512 + ((d >> 2) * 4 + ((token & 7) >> 1)) * 16 +
           (d & 3) * 4 + (token & 1) + 2 * (token >> 3);
}

}  // namespace jkb
