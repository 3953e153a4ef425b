// The 8-bit paged key/value cache: handle and code layout (kv_cache.cu writes it, the attention
// kernels read it).
//
// A block and kv head hold block_tokens / 16 groups of 16 tokens; a group is one contiguous run
// of 32 * dim_p bytes (dim_p: head_dim rounded up to 64, 96, 128, 192 or 256; elements past
// head_dim are code 0), so that one bulk copy brings the keys and values of 16 tokens:
//   keys   [2][dim_p / 32][8 tokens][32 dims]: eight tokens' 32 dims are 256 bytes, of which lane
//          4 g + t of a warp takes bytes 8 t .. 8 t + 8 of token g -- the B operand of
//          mma.m16n8k32 with dims in the order 8 t + {0..3}, 8 t + {4..7}. Codes are int8.
//   values [dim_p / 32][4 (t)][8][4 (j)][4 tokens]: 16-byte piece (g, t) stands at g ^ 2t of row t
//          and holds dims 4 g + j of the 32, tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9. Lane 4 g + t
//          takes piece (g, t), the B operands of four mma.m16n8k16 over 16 tokens; a converter
//          thread takes pieces (g, 0..3), the 16 tokens of four dims. Bytes are code + 128, which
//          two byte permutes and a packed subtraction turn into f16.
// Each of these reads is free of bank conflicts (hence the exclusive or).
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

// Partial results of attention pieces (two slots a CTA), and the counters by which a piece knows
// that it is its row tile's last to finish (zero between calls).
struct jkb_attn_workspace {
    uint32_t magic;
    int device;
    int dim_p;
    int ctas;             // most CTAs of the few-row kernel; the prompt kernel has one an SM
    uint8_t *base;
    float *partial;       // [2 * ctas][ATTN_ROWS][dim_p + 2]
    float *tile_partial;  // [2 * SMs][dim_p + 2][128]; nullptr above 128 dims
    int *counters;        // [3][ctas]
    int *tile_counters;   // [3][SMs]
};

namespace jkb {

constexpr uint32_t KV_MAGIC = 0x4A4B4331u;       // "JKC1"
constexpr uint32_t ATTN_WS_MAGIC = 0x4A4B5331u;  // "JKS1"
// bits of the device error word
constexpr int ERR_KV_RANGE = 4, ERR_ATTN_WAIT = 8;
constexpr int KV_GROUP = 16;   // tokens of a group
constexpr int ATTN_ROWS = 16;  // most query rows of a decode row tile

int check_kv_cache(const jkb_kv_cache *c, const char *fn);

// Byte of the key code of (token, dim) in its group.
__host__ __device__ inline int kv_key_at(int token, int dim, int dim_p) {
    return (token >> 3) * 8 * dim_p + (dim >> 5) * 256 + (token & 7) * 32 + (dim & 31);
}
}  // namespace jkb
