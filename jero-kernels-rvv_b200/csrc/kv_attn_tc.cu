// Attention over the 8-bit key/value cache for many query rows a kv head (prompts and chunks), on
// the fifth-generation tensor cores.
//
// A tile is 128 query rows (tokens x the query heads of one kv head, heads fastest, so that the
// rows stand close together and a causal tile wastes little); its cached tokens go by in units of
// 128. Per unit, with the unit's blocks' scales ks and vs and c = scale log2(e):
//   S = Q K^T           Q in f16 with a power of two of its own per row (exact for 16-bit rows;
//                       f32 rows as two f16, 22 bits), K the codes, exact in f16
//   s = c ks S,  m = max s,  p = 2^(s - m),  l = sum p          (of the unit alone)
//   o = a o + b (p vs) V,  l' = a l' + b l,  m' = max(m', m),  a, b = 2^(old m' - m'), 2^(m - m')
//                       V the codes, exact in bf16; p vs in two bf16 (16-bit rows: 16 bits, five
//                       more than an f16 output has) or three (f32 rows: 24). bf16 has f32's
//                       range: a weight that is far below its row's largest keeps its digits, and
//                       so do the weights beside a block whose value scale is far above theirs.
// The tensor core truncates its f32 sums, about 2^-25 of the sum at every 16-element step. So S
// takes the small part of Q first, and each unit's P V starts from zero, small parts first, and
// is added to o in registers, rounded, with the rescale.
//
// Work: MMA time is (DIM / 16) NQ + 8 NP steps a unit against 16 for one plain product pair; the
// exponentials are 128 x 128 a unit on 16 lanes an SM and clock, about as long as two products;
// and the issue slots: about 850 (16-bit rows) to 1200 (f32) a softmax warp, 500 a conversion
// warp and 200 an accumulation warp a unit, on each of the SM's four sub-partitions (2250 to 2750 in
// all with the tiles' starts and ends).
// One CTA an SM, six warpgroups, every hand-over an mbarrier:
//   0, 1  the query rows of a new tile; softmax, every other unit each (a unit's needs nothing of
//         the one before): a thread a row; S from TMEM, p's parts back over it
//   2     accumulation: a thread a row; the unit's P V from TMEM, o in registers; the output
//   3, 4  conversion of keys (f16), of values (bf16): codes from the raw rings to operand tiles
//         (128-byte swizzle)
//   5     a warp that issues the MMAs, one that loads keys and one that loads values (a bulk copy
//         for 16 tokens each, kv_cache.cuh), and one that finds this CTA's pieces of tiles and
//         hands them to the others
// NB buffers of S: the order of the MMAs is S(i + NB - 1), P V(i), S(i + NB), .. so that they run
// under the softmax. One K operand tile is enough (K(i) is converted while other MMAs run), and
// for f32 rows, whose products take longer, one V tile (V(i + 1) during S(i + 2)).
//
// The code has to be small: beyond about 32 KB of loops, and 128 KB in all, instruction fetches
// take longer than the instructions (measured: 2 and 6 clocks each). So loops are rolled, what
// happens once a tile is there once, and the pieces are found by one warp.
//
// Tiles of all sequences and kv heads form one line of units (and of TILE_COST more a tile, for
// what its start and end take), cut into equal parts, one a CTA; a tile that spans CTAs is put
// together from the workspace by the last of them to finish, in the order of the line (as in
// kv_attn.cu).
//
// Measured, 32 query heads over 8 kv heads of 128 dims: a causal prompt of 2048 f32 tokens behind
// 1111 cached ones takes 212 us (337 TFLOP/s of its two products; the 5 f16 products that f32
// needs run at 840), one of 8192 bf16 tokens 1000 us (550 TFLOP/s; with p's second part 825); nine ragged f16 chunks, 5331 tokens of 14 query
// heads over 2 of 80 dims, 166 us (155 with p in one f16 part, 11 bits, whose error is as large as
// the output's rounding). A unit takes 3400 (16-bit rows) to 4600 clocks (f32), of which the issue
// slots fill 62 and 47 % and the MMAs 42 and 43 %: what bounds it is the latency of the roles' waits
// for tensor memory and for one another. A tile's start and end cost as much as 5 units.
#include "kv_attn.cuh"
#include "ptx.cuh"

#include <cuda_bf16.h>

#include <cfloat>

namespace jkb {

namespace {

constexpr int TM = 128;        // query rows of a tile
constexpr int TN = 128;        // cached tokens of a unit
constexpr int GROUPS = TN / KV_GROUP;
constexpr int THREADS = 768;
constexpr int TILE_COST = 5;   // of a tile's start and end, in units (measured: 5 best of 3, 5, 7)
constexpr int RAW = 2;         // raw rings of codes, units
constexpr int SC = 8;          // ring of block scales, units
constexpr int REGS_SOFT = 88, REGS_SUM = 184, REGS_CONV = 40, REGS_REST = 40;  // of a warpgroup
constexpr int REGS_LAUNCH = 80;  // what the launch gives each
static_assert(2 * REGS_SOFT + REGS_SUM + 2 * REGS_CONV + REGS_REST <= 6 * REGS_LAUNCH &&
                  6 * 128 * REGS_LAUNCH <= 65536,
              "the shares come from what the launch holds");
static_assert(REGS_SOFT >= REGS_LAUNCH && REGS_SUM >= REGS_LAUNCH && REGS_CONV <= REGS_LAUNCH &&
                  REGS_REST <= REGS_LAUNCH,
              "an increase must not go down, nor a decrease up: either is an illegal instruction");

// TYPE: the rows'. NQ: f16 parts of a query element; NP: bf16 parts of p.
template <int DT_, int TYPE_>
struct PreCfg {
    static constexpr int DT = DT_, TYPE = TYPE_;
    static constexpr int NQ = TYPE == JKB_F32 ? 2 : 1;
    static constexpr int NP = TYPE == JKB_F32 ? 3 : 2;
    static constexpr int DIM = 32 * DT;
    static constexpr int KA = (DIM + 63) / 64;       // 64-element swizzle atoms of a head
    static constexpr int NV = NQ == 2 ? 1 : 2;       // V buffers
    static constexpr int SIDE_BYTES = 16 * DIM;      // a group's keys, or its values
    // TMEM: NB buffers of S, then of p's parts (a third part stands behind the 128 columns of S)
    static constexpr int S_COLS = NP == 3 ? 192 : 128;
    static constexpr int NB = NP == 3 ? 2 : 3;
    static constexpr int O_COL = NB * S_COLS;
    static_assert(DIM <= 128 && O_COL + 128 <= 512, "TMEM");
};

// Units key0 / TN .. + n of one tile (n = 0: no more pieces).
struct Piece {
    int n, key0;
    int row0, head, q0, nq;      // the tile's first row; the sequence's query tokens
    int pos0, len;               // position of query token 0; cached tokens
    int lo, hi;                  // tokens that some row of the tile sees
    int all_lo, all_hi;          // tokens that every row sees
    int seq, cta0, cta1;         // the CTAs that have units of the tile
};

template <class C>
struct PreSmem {
    alignas(1024) uint8_t q[C::NQ][C::KA][TM * 128];
    alignas(1024) uint8_t k[C::KA][TN * 128];
    alignas(1024) uint8_t v[C::NV][2][C::DIM * 128];
    alignas(128) uint8_t raw_k[RAW][GROUPS * C::SIDE_BYTES];
    alignas(128) uint8_t raw_v[RAW][GROUPS * C::SIDE_BYTES];
    float2 sc[SC][GROUPS];   // (ks, vs)
    uint32_t valid[SC];      // bit: this group of the unit is there
    float2 stats[4][TM];     // (m, l) of a unit's rows
    float row_scale[TM];
    uint64_t rk_full[RAW], rk_empty[RAW], rv_full[RAW], rv_empty[RAW], k_full, k_empty,
        v_empty[C::NV], q_full, q_empty, s_full[C::NB], pv_ready[4], o_full, merge, done;
    Piece pieces[2];
    uint64_t piece_full[2], piece_empty[2];
    uint32_t tmem;
    int abort_flag, is_last;
};

// ---------------------------------------------------------------- PTX

// The upper half of an operand descriptor is a constant (smem_desc); the lower holds the address.
constexpr uint32_t DESC_HI = (uint32_t)(((uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61) >> 32);
__device__ __forceinline__ uint32_t desc_lo(const void *p) {
    return ((smem_u32(p) >> 4) & 0x3FFFu) | 1u << 16;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                       bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "n"(DESC_HI)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                       bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 y, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "n"(DESC_HI)
        : "memory");
}
// kind::f16 instruction descriptor: D f32, A and B f16 or bf16, both K-major, M = 128.
constexpr uint32_t idesc_f16(int n, bool bf16) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(TM >> 4) << 24);
}
// 32 lanes x 32 columns: thread = lane
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                 "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// One lane of the warp, which the compiler knows to be one: what the MMAs take from uniform
// registers then stays in them.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(~0u, x, 0); }
__device__ __forceinline__ void proxy_fence() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t pkf(float a, float b) {
    return pk2(__float_as_uint(a), __float_as_uint(b));
}
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes,
                                          uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
        : "memory");
}

// Two bytes (byte 0 and 1, or 2 and 3, of code + 128) as f16: 0x6400 | byte is 1024 + byte.
__device__ __forceinline__ uint32_t pair_f16(uint32_t w, uint32_t sel) {
    uint32_t a = __byte_perm(w, 0x64646464u, sel);
    const __half2 x = __hsub2(*reinterpret_cast<__half2 *>(&a), __float2half2_rn(1152.0f));
    return *reinterpret_cast<const uint32_t *>(&x);
}
// The same as bf16: 0x4B000000 | byte is the f32 2^23 + byte; a code fits bf16's 8 bits.
__device__ __forceinline__ uint32_t pair_bf16(uint32_t w, int first) {
    const uint32_t a = __byte_perm(w, 0x4B000000u, first ? 0x7442 : 0x7440);
    const uint32_t b = __byte_perm(w, 0x4B000000u, first ? 0x7443 : 0x7441);
    uint64_t s = add2(pk2(a, b), pkf(-8388736.0f, -8388736.0f));
    float x, y;
    upk2(s, x, y);
    return __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
}

// ---------------------------------------------------------------- the line of units

// One tile: rows row0 .. of the sequence; units first .. first + units of 128 tokens.
struct Tile {
    int row0, first, units, pos0, lo, hi;
};
__device__ __forceinline__ Tile tile_of(const AttnParams &p, const AttnSeq &s, int tile) {
    Tile t;
    t.row0 = tile * TM;
    t.pos0 = s.len - s.nq;
    const int last = (int)min((long long)t.row0 + TM - 1, (long long)s.nq * p.group - 1) / p.group;
    t.hi = p.causal ? max(0, min(s.len, t.pos0 + last + 1)) : s.len;
    t.lo = 0;
    if (p.window)
        t.lo = (int)min(max((long long)t.pos0 + t.row0 / p.group - p.window + 1, 0ll),
                        (long long)t.hi);
    t.first = t.lo / TN;
    t.units = max(1, (t.hi + TN - 1) / TN - t.first);
    return t;
}
__device__ __forceinline__ int tiles_of(const AttnParams &p, const AttnSeq &s) {
    return (int)(((long long)s.nq * p.group + TM - 1) / TM);
}
// A warp: the line's length up to tile `from` (counted from the last: tile tiles - 1 first) of
// one sequence and kv head.
__device__ __forceinline__ long long line_of(const AttnParams &p, const AttnSeq &s, int from,
                                             int lane) {
    long long x = 0;
    for (int r = from + lane; r < tiles_of(p, s); r += 32) x += tile_of(p, s, r).units + TILE_COST;
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(~0u, x, d);
    return x;
}

// Query rows in, output rows out.
// Elements i .. i + 15 as they are; those from n on are 0 (n a multiple of 8). The loads alone, so
// that nothing waits between them; as f32 bits: widen16.
template <int TYPE>
struct Raw16 {
    static constexpr int N = TYPE == JKB_F32 ? 16 : 8;
    uint32_t w[N];
};
template <int TYPE>
__device__ __forceinline__ void load16(const AttnParams &p, size_t i, int n, Raw16<TYPE> &x) {
    constexpr int N = Raw16<TYPE>::N, PER = 16 / N;  // elements of a word
#pragma unroll
    for (int k = 0; k < N; k++) x.w[k] = 0;
    if (p.q_vec) {
        const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const uint32_t *>(p.q) +
                                                         i / PER);
#pragma unroll
        for (int k = 0; k < N / 4; k++)
            if (4 * PER * k < n) {
                const uint4 a = __ldg(q + k);
                x.w[4 * k] = a.x, x.w[4 * k + 1] = a.y;
                x.w[4 * k + 2] = a.z, x.w[4 * k + 3] = a.w;
            }
        return;
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
        if (PER * k >= n) continue;
        if constexpr (TYPE == JKB_F32) {
            x.w[k] = __ldg(static_cast<const uint32_t *>(p.q) + i + k);
        } else {
            const uint16_t *q = static_cast<const uint16_t *>(p.q) + i + 2 * k;
            x.w[k] = __ldg(q) | (uint32_t)__ldg(q + 1) << 16;
        }
    }
}
template <int TYPE>
__device__ __forceinline__ void widen16(const Raw16<TYPE> &raw, uint32_t (&x)[16]) {
#pragma unroll
    for (int k = 0; k < Raw16<TYPE>::N; k++) {
        const uint32_t w = raw.w[k];
        if constexpr (TYPE == JKB_F32) {
            x[k] = w;
        } else if constexpr (TYPE == JKB_F16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
            x[2 * k] = __float_as_uint(f.x), x[2 * k + 1] = __float_as_uint(f.y);
        } else {
            x[2 * k] = w << 16, x[2 * k + 1] = w & 0xFFFF0000u;
        }
    }
}
template <int TYPE>
__device__ __forceinline__ void store8(const AttnParams &p, size_t i, const float (&x)[8],
                                       bool vec) {
    if constexpr (TYPE == JKB_F32) {
        float *o = static_cast<float *>(p.out) + i;
        if (vec) {
            *reinterpret_cast<float4 *>(o) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4 *>(o + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) o[k] = x[k];
        }
    } else {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if constexpr (TYPE == JKB_F16) {
                const __half2 y = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
                w[k] = *reinterpret_cast<const uint32_t *>(&y);
            } else {
                const __nv_bfloat162 y = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
                w[k] = *reinterpret_cast<const uint32_t *>(&y);
            }
        }
        uint16_t *o = static_cast<uint16_t *>(p.out) + i;
        if (vec) {
            *reinterpret_cast<uint4 *>(o) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                o[2 * k] = (uint16_t)w[k];
                o[2 * k + 1] = (uint16_t)(w[k] >> 16);
            }
        }
    }
}

// Tokens outside lo .. hi of the unit, and of groups that are not there, get S = -inf, before
// softmax_unit, which so needs no test for them: beside a second form of it with the tests, which
// a tile's last units ran from a cold instruction cache, this took 5 to 9 us less a tile.
__device__ __forceinline__ void mask_unit(uint32_t ts, uint32_t valid, int lo, int hi) {
#pragma unroll 1
    for (int h = 0; h < 4; h++) {
        const int a = min(max(lo - 32 * h, 0), 32), b = min(max(hi - 32 * h, 0), 32);
        uint32_t m = (uint32_t)((1ull << b) - 1) & ~(uint32_t)((1ull << a) - 1);
        if (!((valid >> (2 * h)) & 1)) m &= 0xFFFF0000u;
        if (!((valid >> (2 * h + 1)) & 1)) m &= 0x0000FFFFu;
        if (__all_sync(~0u, m == ~0u)) continue;
        uint32_t r[32];
        tmem_ld32(ts + 32 * h, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t x[8];
#pragma unroll
            for (int i = 0; i < 8; i++)
                x[i] = m & (1u << (8 * j + i)) ? r[8 * j + i] : 0xFF800000u;
            tmem_st8(ts + 32 * h + 8 * j, x);
        }
    }
    tmem_st_wait();
}

// One unit of one row (thread): S from TMEM at ts, scaled by rs ks; returns (m, l). p's parts go
// back to TMEM over S: of the 16 columns of a group of tokens, the first 8 take part 0, the last
// 8 part 1; part 2 stands behind S.
// S is read twice (maximum, then weights), 32 columns at a time: loops stay rolled where they
// can: with more unrolling the roles' code outgrows the SM's instruction cache, and every unit
// fetches it anew (unrolled over 128 columns, four times slower).
// rs and ks are not negative (a negative softmax scale's sign is in Q); where they give 0, the
// smallest normal number in its place keeps a masked token's -inf.
template <class C>
__device__ __forceinline__ float2 softmax_unit(uint32_t ts, const float2 *sc, float rs) {
    constexpr int NP = C::NP;
    float top = -INFINITY, most = -INFINITY;  // of s; of S
    uint32_t r[32];
    tmem_ld32(ts, r);
#pragma unroll 1
    for (int h = 0; h < 4; h++) {
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 2; k++) {
            float t2[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float u = __uint_as_float(r[16 * k + 2 * i]);
                const float w = __uint_as_float(r[16 * k + 2 * i + 1]);
                t2[i & 1] = fmaxf(t2[i & 1], fmaxf(u, w));
            }
            const float raw = fmaxf(t2[0], t2[1]);
            most = fmaxf(most, raw);
            top = fmaxf(top, raw == -INFINITY ? raw : raw * (rs * sc[2 * h + k].x));
        }
        tmem_ld32(ts + 32 * ((h + 1) & 3), r);
    }
    const float ref = top == -INFINITY ? 0.0f : top;
    if (most == -INFINITY) rs = 0.0f;  // sees nothing here: no NaN from its scale either
    const uint64_t nref = pkf(-ref, -ref), minus = pkf(-1.0f, -1.0f);
    uint64_t sum = 0;
#pragma unroll 1
    for (int h = 0; h < 4; h++) {
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int g = 2 * h + k;
            float f = rs * sc[g].x;
            f = f < FLT_MIN ? FLT_MIN : f;
            const float vs = sc[g].y;
            uint32_t part[NP][8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float u, w;
                upk2(fma2(pk2(r[16 * k + 2 * i], r[16 * k + 2 * i + 1]), pkf(f, f), nref), u, w);
                uint64_t e = pkf(ex2(u), ex2(w));
                sum = add2(sum, e);
                e = mul2(e, pkf(vs, vs));
                upk2(e, u, w);
                // all parts but the last are cut off, not rounded: the upper halves
#pragma unroll
                for (int j = 0; j < NP - 1; j++) {
                    const uint32_t a = __float_as_uint(u), b = __float_as_uint(w);
                    part[j][i] = __byte_perm(a, b, 0x7632);
                    e = fma2(pk2(a & 0xFFFF0000u, b & 0xFFFF0000u), minus, e);
                    upk2(e, u, w);
                }
                const __nv_bfloat162 y = __floats2bfloat162_rn(u, w);
                part[NP - 1][i] = *reinterpret_cast<const uint32_t *>(&y);
            }
            tmem_st8(ts + 16 * g, part[0]);
            tmem_st8(ts + 16 * g + 8, part[1]);
            if (NP > 2) tmem_st8(ts + TN + 8 * g, part[NP - 1]);
        }
        if (h < 3) tmem_ld32(ts + 32 * (h + 1), r);
    }
    float su, sw;
    upk2(sum, su, sw);
    return make_float2(top, su + sw);
}

template <class C>
__global__ void __launch_bounds__(THREADS, 1)
    attn_prompt_kernel(const __grid_constant__ AttnParams p) {
    constexpr int DIM = C::DIM, DT = C::DT, NP = C::NP, NQ = C::NQ, NV = C::NV;
    extern __shared__ uint8_t smem_raw[];
    PreSmem<C> &sm =
        *reinterpret_cast<PreSmem<C> *>((((uintptr_t)smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wg = warp >> 2;
    volatile int *abort_flag = &sm.abort_flag;

    if (tid == 0) {
        sm.abort_flag = 0;
        for (int i = 0; i < RAW; i++) {
            mbar_init(&sm.rk_full[i], 1);
            mbar_init(&sm.rk_empty[i], 4);
            mbar_init(&sm.rv_full[i], 1);
            mbar_init(&sm.rv_empty[i], 4);
        }
        mbar_init(&sm.k_full, 4);
        mbar_init(&sm.k_empty, 1);
        for (int i = 0; i < C::NB; i++) mbar_init(&sm.s_full[i], 1);
        for (int i = 0; i < NV; i++) mbar_init(&sm.v_empty[i], 1);
        for (int i = 0; i < 4; i++) mbar_init(&sm.pv_ready[i], 12);
        mbar_init(&sm.q_full, 8);
        mbar_init(&sm.q_empty, 9);
        mbar_init(&sm.o_full, 1);
        mbar_init(&sm.merge, 4);
        mbar_init(&sm.done, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&sm.piece_full[i], 1);
            mbar_init(&sm.piece_empty[i], 23);  // every other warp
        }
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (warp == 20) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&sm.tmem)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" :::);
    __syncthreads();
    tc_fence_after();

    const uint32_t tmem = sm.tmem;
    // a warp's wait: all of its lanes go on, or (after the limit, or an abort) none
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        return __all_sync(~0u, mbar_wait_short(bar, parity & 1, abort_flag, p.err)) != 0;
    };

    // two barriers at once
    auto wait2 = [&](uint64_t *bar0, uint32_t parity0, uint64_t *bar1, uint32_t parity1) {
        const bool a = mbar_try(bar0, parity0 & 1), b = mbar_try(bar1, parity1 & 1);
        return __all_sync(~0u, a && b) || (wait(bar0, parity0) && wait(bar1, parity1));
    };
    // the next piece: waits for it, copies it and gives its slot back; false at the end
    uint32_t pieces = 0;
    Piece cur;
    auto next_piece = [&](bool &ok) {
        const uint32_t i = pieces & 1;
        ok = wait(&sm.piece_full[i], pieces >> 1);
        cur = sm.pieces[i];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.piece_empty[i]);
        pieces++;
        return ok && cur.n > 0;
    };
    bool ok = true;

    // (one instruction for all warps of a group; what is taken was given back first)
    if (wg < 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFT));
    else if (wg == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SUM));
    else if (wg < 5) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CONV));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_REST));

    if (wg < 2) {
        // ------------------------------------------------------------ softmax
        const int row = tid & 127;  // of the tile
        constexpr int QROUNDS = NQ == 2 ? 1 : 2;
        const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        uint32_t it = 0;
        while (next_piece(ok)) {
            // ---- the query rows, 16 a warp: f16 parts of x times a power of two of the row ----
            // eight lanes a row, 16 dims a lane; a round's rows are loaded before the one before
            // is converted, the first before the tile before gives its place up
            {
                const int d0 = 16 * (lane & 7);
                int rr = cur.row0 + warp * 16 + (lane >> 3), tok = rr / p.group;
                int h = rr - tok * p.group;
                const size_t head0 = (size_t)(cur.head * p.group);
                auto load_round = [&](Raw16<C::TYPE>(&x)[QROUNDS]) {
#pragma unroll
                    for (int j = 0; j < QROUNDS; j++) {
                        const size_t at = (size_t)(cur.q0 + tok) * p.q_token +
                                          (head0 + h) * p.q_head + d0;
                        load16<C::TYPE>(p, at, tok < cur.nq ? p.dim - d0 : 0, x[j]);
                        h += 4;
                        while (h >= p.group) {
                            h -= p.group;
                            tok++;
                        }
                    }
                };
                Raw16<C::TYPE> next[QROUNDS];
                load_round(next);
                if (!wait(&sm.q_empty, pieces)) goto out;
#pragma unroll 1
                for (int r0 = 0; r0 < 16; r0 += 4 * QROUNDS) {
                    uint32_t x[QROUNDS][16];
#pragma unroll
                    for (int j = 0; j < QROUNDS; j++) widen16<C::TYPE>(next[j], x[j]);
                    if (r0 + 4 * QROUNDS < 16) load_round(next);
#pragma unroll
                    for (int j = 0; j < QROUNDS; j++) {
                        const int r = warp * 16 + r0 + 4 * j + (lane >> 3);
                        // the largest magnitude's bits; infinities and NaN are above all others
                        uint32_t top = 0;
#pragma unroll
                        for (int k = 0; k < 16; k++) top = max(top, x[j][k] & 0x7FFFFFFFu);
                        for (int d = 4; d; d >>= 1) top = max(top, __shfl_xor_sync(~0u, top, d));
                        const bool fine = top < 0x7F800000u;
                        // 2^e brings the largest element into [2^14, 2^15)
                        const int e = min(14 + 127 - (int)(top >> 23), 126);
                        float up = fine ? __uint_as_float((uint32_t)(127 + e) << 23) : 0.0f;
                        if ((lane & 7) == 0)
                            sm.row_scale[r] = !fine ? __int_as_float(0x7FC00000)
                                              : top == 0 ? 0.0f : fabsf(p.scale2) / up;
                        up = copysignf(up, p.scale2);
                        if (64 * C::KA <= d0) continue;
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            float v[8];
#pragma unroll
                            for (int k = 0; k < 8; k++)
                                v[k] = fine ? __uint_as_float(x[j][8 * i + k]) * up : 0.0f;
                            const int ch = (2 * (lane & 7) + i) & 7;
                            uint8_t *dst = &sm.q[0][d0 >> 6][r * 128 + ((ch ^ (r & 7)) << 4)];
#pragma unroll
                            for (int k = 0; k < NQ; k++) {
                                uint32_t w[4];
#pragma unroll
                                for (int t = 0; t < 4; t++) {
                                    const __half2 y = __floats2half2_rn(v[2 * t], v[2 * t + 1]);
                                    const float2 f = __half22float2(y);
                                    w[t] = *reinterpret_cast<const uint32_t *>(&y);
                                    v[2 * t] -= f.x;
                                    v[2 * t + 1] -= f.y;
                                }
                                *reinterpret_cast<uint4 *>(dst + k * sizeof(sm.q[0])) =
                                    make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }
                }
            }
            proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.q_full);
            if (!wait(&sm.q_full, pieces - 1)) goto out;
            const float rs = sm.row_scale[row];
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.q_empty);
            const int pos = cur.pos0 + (cur.row0 + row) / p.group;
            const int hi = p.causal ? min(cur.len, pos + 1) : cur.len;
            const int lo = first_seen(p, pos);
            const uint32_t end = it + cur.n;
            uint32_t i = it + ((it ^ wg) & 1);
            int key0 = cur.key0 + (int)(i - it) * TN;
            it = end;
            for (; i < end; i += 2, key0 += 2 * TN) {
                const uint32_t b = i % C::NB;
                if (!wait(&sm.s_full[b], i / C::NB)) goto out;
                tc_fence_after();
                const uint32_t valid = sm.valid[i % SC];
                const float2 *sc = sm.sc[i % SC];
                const uint32_t ts = tl + b * C::S_COLS;
                if (key0 < cur.all_lo || key0 + TN > cur.all_hi || valid != 0xFFu)
                    mask_unit(ts, valid, lo - key0, hi - key0);
                const float2 st = softmax_unit<C>(ts, sc, rs);
                sm.stats[i & 3][row] = st;
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.pv_ready[i & 3]);
            }
        }
    } else if (wg == 2) {
        // ------------------------------------------------------------ accumulation and output
        const int row = tid & 127;
        const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16) + C::O_COL;
        uint32_t it = 0, merges = 0;
        if (lane == 0) mbar_arrive(&sm.pv_ready[0]);  // o is free for the first unit
        while (next_piece(ok)) {
            uint64_t o[DIM / 2];  // pairs of columns
#pragma unroll
            for (int i = 0; i < DIM / 2; i++) o[i] = 0;
            float m = -INFINITY, l = 0.0f;
            for (int c = 0; c < cur.n; c++, it++) {
                if (!wait(&sm.o_full, it)) goto out;
                tc_fence_after();
                const float2 st = sm.stats[it & 3][row];
                const float mn = fmaxf(m, st.x), ref = mn == -INFINITY ? 0.0f : mn;
                const float a = ex2(m - ref), b = ex2(st.x - ref);
                l = fmaf(l, a, b * st.y);
                m = mn;
                const uint64_t a2 = pkf(a, a);
                const uint64_t b2 = pkf(b, b);
#pragma unroll
                for (int q = 0; q < DT; q++) {
                    uint32_t r[32];
                    tmem_ld32(tl + 32 * q, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        o[16 * q + i] =
                            fma2(o[16 * q + i], a2, mul2(pk2(r[2 * i], r[2 * i + 1]), b2));
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.pv_ready[(it + 1) & 3]);
            }

            const int rr = cur.row0 + row, tok = rr / p.group, h = cur.head * p.group + rr - tok * p.group;
            const size_t at = (size_t)(cur.q0 + tok) * p.out_token + (size_t)h * p.out_head;
            const bool on = tok < cur.nq;
            // A tile of several CTAs: each leaves its (m, l, o) in a slot of the workspace (two
            // slots where a CTA starts within one such tile and ends within another)
            auto slot_of = [&](int cta) {
                const int slot = 2 * cta + (cta == cur.cta0 ? 1 : 0);
                return p.tile_partial + (size_t)slot * TM * (DIM + 2) + row;
            };
            auto put = [&](float *slot) {
                if (!on) return;
#pragma unroll
                for (int i = 0; i < DIM / 2; i++) {
                    float u, w;
                    upk2(o[i], u, w);
                    slot[2 * i * TM] = u;
                    slot[(2 * i + 1) * TM] = w;
                }
                slot[DIM * TM] = m;
                slot[(DIM + 1) * TM] = l;
            };
            const int n = cur.cta1 - cur.cta0 + 1;
            int at_cta = (int)blockIdx.x - cur.cta0;  // has the sum of pieces at_cta .. + span - 1
            bool mine = true;
            for (int span = 1, level = 0; span < n; span *= JOIN, level++) {
                const int base = at_cta - at_cta % (span * JOIN);
                const int cnt = min(JOIN, (n - base + span - 1) / span);
                if (cnt > 1) put(slot_of(cur.cta0 + at_cta));
                at_cta = base;
                if (cnt == 1) continue;
                __threadfence();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.merge);
                if (!wait(&sm.merge, merges++)) goto out;
                if (row == 0) {
                    int *counter = p.tile_counters + level * gridDim.x + cur.cta0 + base;
                    sm.is_last = atomicAdd(counter, 1) == cnt - 1;
                    if (sm.is_last) *counter = 0;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.merge);
                if (!wait(&sm.merge, merges++)) goto out;
                mine = *(volatile int *)&sm.is_last;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.merge);  // is_last may be written again
                if (!wait(&sm.merge, merges++)) goto out;
                if (!mine) break;
                __threadfence();
                m = -INFINITY;
                l = 0.0f;
#pragma unroll
                for (int i = 0; i < DIM / 2; i++) o[i] = 0;
                if (!on) continue;
#pragma unroll 1
                for (int k = 0; k < cnt; k++)
                    m = fmaxf(m, __ldcg(slot_of(cur.cta0 + base + k * span) + DIM * TM));
                const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll 1
                for (int k = 0; k < cnt; k++) {
                    const float *slot = slot_of(cur.cta0 + base + k * span);
                    const float w = ex2(__ldcg(slot + DIM * TM) - ref);
                    l = fmaf(w, __ldcg(slot + (DIM + 1) * TM), l);
                    const uint64_t w2 = pkf(w, w);
#pragma unroll
                    for (int q = 0; q < DT; q++) {
                        float x[32];
#pragma unroll
                        for (int i = 0; i < 32; i++) x[i] = __ldcg(slot + (32 * q + i) * TM);
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            o[16 * q + i] =
                                fma2(w2, pkf(x[2 * i], x[2 * i + 1]), o[16 * q + i]);
                    }
                }
            }
            __syncwarp();
            if (!mine) continue;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            if (on && p.lse)
                p.lse[(size_t)(cur.q0 + tok) * p.group * p.kv_heads + h] =
                    (m + log2f(l)) * 0.69314718055994531f;
            // column 32 c + 8 j + g of o is dim 32 c + 4 g + j
            if (on && p.out_vec) {
#pragma unroll
                for (int c = 0; c < DT; c++)
#pragma unroll
                    for (int g = 0; g < 8; g += 2) {
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 4; i++) {  // columns 8 i + g and 8 i + g + 1
                            upk2(o[16 * c + 4 * i + g / 2], x[i], x[4 + i]);
                            x[i] *= inv;
                            x[4 + i] *= inv;
                        }
                        if (32 * c + 4 * g < p.dim)
                            store8<C::TYPE>(p, at + 32 * c + 4 * g, x, true);
                    }
            } else if (on) {  // rows not aligned for wide stores: by way of the CTA's slot
                float *slot = slot_of((int)blockIdx.x);
                put(slot);
#pragma unroll 1
                for (int d = 0; d < p.dim; d += 8) {
                    const float *col = slot + ((d & ~31) + ((d & 31) >> 2)) * TM;
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        x[i] = __ldcg(col + (8 * (i & 3) + (i >> 2)) * TM) * inv;
                    store8<C::TYPE>(p, at + d, x, false);
                }
            }
            __syncwarp();
        }
    } else if (wg == 3) {
        // ------------------------------------------------------------ conversion of keys
        const int cw = warp & 3;
        uint32_t it = 0;
        while (next_piece(ok)) {
            for (int c = 0; c < cur.n; c++, it++) {
                if (!wait2(&sm.rk_full[it % RAW], it / RAW, &sm.k_empty, it + 1)) goto out;
                const uint8_t *raw = sm.raw_k[it % RAW];
                // a lane takes a token's 32 dims, their halves in the order that keeps eight
                // lanes (eight tokens) on eight bank groups; a warp 8 tokens, or 16 of 64 dims
                constexpr int PER = DT == 2 ? 2 : 1;  // eights of tokens a warp and round
                const int tk = lane & 7, sub = lane >> 3;
                const int chunk = DT == 2 ? sub & 1 : sub, eighth = DT == 2 ? sub >> 1 : 0;
                const int swap = tk >> 2;
                const int hg0 = cw * PER + eighth;
                const uint8_t *src = raw + hg0 * 8 * DIM + chunk * 256 + tk * 32 + 16 * swap;
                uint8_t *dst = &sm.k[0][0] + (chunk >> 1) * (TN * 128) + (hg0 * 8 + tk) * 128;
                const int ch = (chunk & 1) * 4 + 2 * swap;
                const int d00 = (ch ^ tk) << 4, d01 = ((ch + 1) ^ tk) << 4;
#pragma unroll 2
                for (int i = 0; i < TN / 8 / (4 * PER); i++) {
                    if (chunk < DT) {
#pragma unroll
                        for (int h = 0; h < 2; h++) {  // the second half: 32 bytes of dst away
                            const uint4 x = *reinterpret_cast<const uint4 *>(
                                h ? src + 16 - 32 * swap : src);
                            const uint32_t w[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u,
                                                   x.z ^ 0x80808080u, x.w ^ 0x80808080u};
                            *reinterpret_cast<uint4 *>(dst + (d00 ^ (32 * h))) =
                                make_uint4(pair_f16(w[0], 0x4140), pair_f16(w[0], 0x4342),
                                           pair_f16(w[1], 0x4140), pair_f16(w[1], 0x4342));
                            *reinterpret_cast<uint4 *>(dst + (d01 ^ (32 * h))) =
                                make_uint4(pair_f16(w[2], 0x4140), pair_f16(w[2], 0x4342),
                                           pair_f16(w[3], 0x4140), pair_f16(w[3], 0x4342));
                        }
                    }
                    src += 4 * PER * 8 * DIM;
                    dst += 4 * PER * 8 * 128;
                }
                proxy_fence();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sm.rk_empty[it % RAW]);
                    mbar_arrive(&sm.k_full);
                }
            }
        }
    } else if (wg == 4) {
        // ------------------------------------------------------------ conversion of values
        const int cw = warp & 3;
        uint32_t it = 0;
        while (next_piece(ok)) {
            for (int c = 0; c < cur.n; c++, it++) {
                const int vb = it % NV;
                if (!wait2(&sm.rv_full[it % RAW], it / RAW, &sm.v_empty[vb], it / NV + 1))
                    goto out;
                const uint8_t *raw = sm.raw_v[it % RAW];
                // a lane takes 16 tokens of four dims (4 g + j), to rows 8 j + g; a warp a group
                // of tokens, or two of 64 dims
                constexpr int PER = DT == 2 ? 2 : 1;
                const int g = lane & 7, sub = lane >> 3;
                const int chunk = DT == 2 ? sub & 1 : sub, other = DT == 2 ? sub >> 1 : 0;
#pragma unroll 1
                for (int grp = cw * PER + other; grp < GROUPS; grp += 4 * PER) {
                    if (chunk >= DT) continue;
                    const uint8_t *src = raw + grp * C::SIDE_BYTES + chunk * 512;
                    uint32_t w[4][4];  // [t][j]
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(
                            src + (t * 8 + (g ^ (2 * t))) * 16);
                        w[t][0] = x.x, w[t][1] = x.y, w[t][2] = x.z, w[t][3] = x.w;
                    }
                    uint8_t *dst = &sm.v[vb][grp >> 2][(32 * chunk + g) * 128];
                    const int d0 = (((grp & 3) * 2) ^ g) << 4;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
#pragma unroll
                        for (int i = 0; i < 2; i++) {  // tokens 8 i .. 8 i + 7
                            uint32_t y[4];
#pragma unroll
                            for (int t = 0; t < 4; t++)
                                y[t] = pair_bf16(w[t][j], i);
                            *reinterpret_cast<uint4 *>(dst + j * 8 * 128 + (d0 ^ (16 * i))) =
                                make_uint4(y[0], y[1], y[2], y[3]);
                        }
                    }
                }
                proxy_fence();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sm.rv_empty[it % RAW]);
                    mbar_arrive(&sm.pv_ready[it & 3]);
                }
            }
        }
    } else if (warp == 20) {
        // ------------------------------------------------------------ MMA
        constexpr uint32_t ID_S = idesc_f16(TN, false), ID_O = idesc_f16(DIM, true);
        uint32_t it = 0, pv = 0;  // S and P V issued so far
        const uint32_t ut = uniform(tmem), vd0 = uniform(desc_lo(&sm.v[0][0][0]));
        const uint32_t kd = uniform(desc_lo(&sm.k[0][0])), qd = uniform(desc_lo(&sm.q[0][0][0]));
        auto issue_pv = [&]() {
            const uint32_t b = pv % C::NB, vb = pv % NV;
            // its p, its V, and o free of the unit before
            if (!wait(&sm.pv_ready[pv & 3], pv >> 2)) return false;
            tc_fence_after();
            const uint32_t vd = uniform(vd0 + vb * (uint32_t)(sizeof(sm.v[0]) / 16));
            const uint32_t pt = uniform(ut + b * C::S_COLS), od = ut + C::O_COL;
            if (elect_one()) {
                // parts of p from the last; their columns as softmax_unit leaves them. V of step
                // s: atom s / 4, 32 bytes a step
                bool acc = false;
#pragma unroll 1
                for (int k = NP - 1; k >= 0; k--) {
                    uint32_t a = pt + (k == 2 ? TN : 8 * k), v = vd;
                    const uint32_t step = k == 2 ? 8 : 16;
#pragma unroll 1
                    for (int s = 0; s < TN / 32; s++) {
                        mma_ts(od, a, v, ID_O, acc);
                        mma_ts(od, a + step, v + 2, ID_O, true);
                        acc = true;
                        a += 2 * step;
                        v += s == 1 ? DIM * 128 / 16 - 4 : 4;
                    }
                }
                tc_commit(&sm.v_empty[vb]);
                tc_commit(&sm.o_full);
            }
            __syncwarp();
            pv++;
            return true;
        };
        // one loop over S's units and the P V that are left at the end, so that the code of each
        // is there once
        int c = 0;
        bool more = true, fetched = false;
        while (more || pv < it) {
            bool s_next = more;
            // a new tile and its query rows may be long in coming: finish what is left before them
            if (more && c == 0) {
                if (!fetched && (pv == it || __any_sync(~0u, mbar_try(&sm.piece_full[pieces & 1],
                                                                      (pieces >> 1) & 1)))) {
                    more = next_piece(ok);
                    if (!ok) goto out;
                    fetched = true;
                    if (!more) continue;
                }
                s_next = fetched && (pv == it || __any_sync(~0u, mbar_try(&sm.q_full,
                                                                          (pieces - 1) & 1)));
                if (!s_next && pv == it) continue;
            }
            if (s_next) {
                if ((c == 0 && !wait(&sm.q_full, pieces - 1)) || !wait(&sm.k_full, it)) goto out;
                tc_fence_after();
                const uint32_t sd = uniform(ut + it % C::NB * C::S_COLS);
                const bool last_unit = c == cur.n - 1;
                if (elect_one()) {
                    bool acc = false;
#pragma unroll 1
                    for (int k = NQ - 1; k >= 0; k--) {
                        uint32_t a = qd + k * (C::KA * TM * 128 / 16), b = kd;
#pragma unroll 1
                        for (int s = 0; s < DIM / 32; s++) {
                            mma_ss(sd, a, b, ID_S, acc);
                            mma_ss(sd, a + 2, b + 2, ID_S, true);
                            acc = true;
                            const uint32_t d = s == 1 ? TM * 128 / 16 - 4 : 4;
                            a += d;
                            b += d;
                        }
                    }
                    tc_commit(&sm.k_empty);
                    if (last_unit) tc_commit(&sm.q_empty);
                    tc_commit(&sm.s_full[it % C::NB]);
                }
                __syncwarp();
                it++;
                if (++c == cur.n) {
                    c = 0;
                    fetched = false;
                }
                if (it - pv < C::NB) continue;
            }
            if (!issue_pv()) goto out;
        }
    } else if (warp == 21 || warp == 22) {
        // ------------------------------------------------------------ loads
        const bool keys = warp == 21;
        uint64_t *full = keys ? sm.rk_full : sm.rv_full, *empty = keys ? sm.rk_empty : sm.rv_empty;
        uint8_t *ring = keys ? sm.raw_k[0] : sm.raw_v[0];
        const uint8_t *codes = p.codes + (keys ? 0 : C::SIDE_BYTES);
        uint32_t it = 0;
        while (next_piece(ok)) {
            const int32_t *ids = p.table + (size_t)cur.seq * p.table_stride;
            const int hi = cur.hi, lo = cur.lo;
            // the lookups of 32 groups (four units) at a time, the next ones ahead of their use
            int id;
            float2 sc;
            auto look = [&](int c) {
                id = -1;
                sc = make_float2(0.f, 0.f);
                const int t0 = cur.key0 + c * TN + lane * KV_GROUP;
                if (c + lane / GROUPS < cur.n && t0 < hi && t0 + KV_GROUP > lo) {
                    id = __ldg(ids + (t0 >> p.log_block));
                    if (id < 0 || id >= p.n_blocks) {
                        atomicOr(p.err, ERR_KV_RANGE);
                        id = -1;
                    } else if (keys) {
                        sc = __ldg(p.scales + (size_t)id * p.kv_heads + cur.head);
                    }
                }
            };
            look(0);
            int id_now = id;
            float2 sc_now = sc;
            for (int c = 0; c < cur.n; c++, it++) {
                if (c % 4 == 0) {
                    id_now = id;
                    sc_now = sc;
                    if (c + 4 < cur.n) look(c + 4);
                }
                const int slot = it % RAW;
                // lanes 8 (c % 4) .. + 8 hold this unit's groups; lane i < 8 takes group i
                const int from = (c % 4) * GROUPS + (lane & 7);
                const int gid = __shfl_sync(~0u, id_now, from);
                const float2 gs = make_float2(__shfl_sync(~0u, sc_now.x, from),
                                              __shfl_sync(~0u, sc_now.y, from));
                const unsigned there = __ballot_sync(~0u, gid >= 0) & 0xFFu;
                if (!wait(&empty[slot], it / RAW + 1)) goto out;
                if (keys) {  // whoever sees the keys (and what follows from them) sees these
                    if (lane < GROUPS) sm.sc[it % SC][lane] = gs;
                    if (lane == 0) sm.valid[it % SC] = there;
                    __syncwarp();
                }
                if (lane == 0)
                    mbar_arrive_tx(&full[slot], __popc(there) * C::SIDE_BYTES);
                __syncwarp();
                if (lane < GROUPS && gid >= 0) {
                    const int t0 = cur.key0 + c * TN + lane * KV_GROUP;
                    const int grp = (t0 & ((1 << p.log_block) - 1)) / KV_GROUP;
                    const size_t bh = (size_t)gid * p.kv_heads + cur.head;
                    bulk_load(ring + (size_t)(slot * GROUPS + lane) * C::SIDE_BYTES,
                              codes + ((bh << p.log_block) / KV_GROUP + grp) *
                                          (size_t)(2 * C::SIDE_BYTES),
                              C::SIDE_BYTES, &full[slot]);
                }
            }
        }
    } else if (warp == 23) {
        // ------------------------------------------------------------ this CTA's pieces
        // twice over the sequences, 32 at a time: the line's length; then where the part starts
        long long total = 0, per = 0, u0 = 0, u1 = 0, at = 0, in = 0;
        int seq = -1;
#pragma unroll 1
        for (int round = 0; round < 2 && seq < 0; round++) {
            at = 0;
#pragma unroll 1
            for (int base = 0; base < p.n_seqs && seq < 0; base += 32) {
                long long x = 0;
                bool big = false;
                if (base + lane < p.n_seqs) {
                    const AttnSeq s = attn_seq(p, base + lane);
                    const int tiles = tiles_of(p, s);
                    big = tiles > 2;
#pragma unroll 1
                    for (int r = 0; r < tiles && !big; r++)
                        x += tile_of(p, s, r).units + TILE_COST;
                }
                unsigned left = __ballot_sync(~0u, big);
#pragma unroll 1
                for (; left; left &= left - 1) {  // a long one: all lanes over its tiles
                    const int i = __ffs(left) - 1;
                    const long long y = line_of(p, attn_seq(p, base + i), 0, lane);
                    if (lane == i) x = y;
                }
                x *= p.kv_heads;
                long long upto = x;
                for (int d = 1; d < 32; d <<= 1) {
                    const long long y = __shfl_up_sync(~0u, upto, d);
                    if (lane >= d) upto += y;
                }
                if (round == 1) {
                    const unsigned hit = __ballot_sync(~0u, u0 < at + upto);
                    if (hit) {
                        const int i = __ffs(hit) - 1;
                        seq = base + i;
                        in = u0 - (at + __shfl_sync(~0u, upto - x, i));
                        at = u0 - in;
                    }
                }
                if (seq < 0) at += __shfl_sync(~0u, upto, 31);
            }
            if (round == 0) {
                total = at;
                per = (total + gridDim.x - 1) / gridDim.x;
                u0 = min(per * blockIdx.x, total);
                u1 = min(u0 + per, total);
                if (u0 >= u1) break;
            }
        }
        // the tile within the sequence: tiles from the last, kv heads of each together
        AttnSeq s{};
        Tile t{};
        int tile = 0, head = 0;
        long long start = at;  // the line's unit where the tile (and head) starts
        if (seq >= 0) {
            s = attn_seq(p, seq);
            int lo = 0, hi = tiles_of(p, s) - 1;  // the last tile whose line includes `in`
#pragma unroll 1
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (line_of(p, s, mid, lane) * p.kv_heads > in) lo = mid;
                else hi = mid - 1;
            }
            tile = lo;
            t = tile_of(p, s, tile);
            const int len = t.units + TILE_COST;
            const long long before = line_of(p, s, tile + 1, lane) * p.kv_heads;
            head = (int)((in - before) / len);
            start = at + before + (long long)head * len;
        }
        for (uint32_t i = 0;;) {
            const bool end = seq < 0 || start >= u1;
            const long long base = start + TILE_COST;
            const int c0 = (int)max(u0 - base, 0ll);
            const int n = end ? 0 : (int)max(min(base + t.units, u1) - (base + c0), 0ll);
            if (end || n) {
                if (!wait(&sm.piece_empty[i & 1], (i >> 1) + 1)) goto out;
                if (lane == 0) {
                    Piece q{};
                    if (!end) {
                        const int first = t.pos0 + t.row0 / p.group;
                        const int last = t.pos0 + (t.row0 + TM - 1) / p.group;
                        q.n = n;
                        q.key0 = (t.first + c0) * TN;
                        q.row0 = t.row0, q.head = head, q.q0 = s.q0, q.nq = s.nq;
                        q.pos0 = t.pos0, q.len = s.len, q.lo = t.lo, q.hi = t.hi;
                        q.all_hi = p.causal ? min(s.len, first + 1) : s.len;
                        q.all_lo = first_seen(p, last);
                        q.seq = seq;
                        q.cta0 = (int)(base / per);
                        q.cta1 = (int)((base + t.units - 1) / per);
                    }
                    sm.pieces[i & 1] = q;
                    mbar_arrive(&sm.piece_full[i & 1]);
                }
                __syncwarp();
                i++;
                // its query rows, on their way to the L2 while the piece before it runs
                constexpr int SIZE = C::TYPE == JKB_F32 ? 4 : 2;
                for (int r = lane; r < TM && !end; r += 32) {
                    const int tok = (t.row0 + r) / p.group;
                    if (tok >= s.nq) break;
                    const char *q = static_cast<const char *>(p.q) +
                                    ((size_t)(s.q0 + tok) * p.q_token +
                                     (size_t)(head * p.group + t.row0 + r - tok * p.group) *
                                         p.q_head) * SIZE;
                    for (int d = 0; d < p.dim * SIZE; d += 128)
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(q + d));
                }
                __syncwarp();
            }
            if (end) break;
            start += TILE_COST + t.units;
            if (++head == p.kv_heads) {
                head = 0;
                if (--tile < 0) {
                    do {
                        if (++seq == p.n_seqs) break;
                        s = attn_seq(p, seq);
                    } while (s.nq == 0);
                    tile = tiles_of(p, s) - 1;
                }
                t = tile_of(p, s, tile);
            }
        }
    }
out:
    // On expiry of a wait: the loads and MMAs in flight end (bounded) before the memory goes. (A
    // commit follows its own thread's MMAs: the elected one's.)
    __syncwarp();
    if (warp == 20 && elect_one()) {
        tc_commit(&sm.done);
        const unsigned long long t0 = globaltimer();
        while (!mbar_try(&sm.done, 0) && globaltimer() - t0 < WAIT_NS) {
        }
    }
    __syncwarp();
    if ((warp == 21 || warp == 22) && *abort_flag) {
        const unsigned long long t0 = globaltimer();
        while (globaltimer() - t0 < 50000000ull) __nanosleep(1000);  // 50 ms: any copy has landed
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 20)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(512));
}

template <class C>
int launch_cfg(const AttnParams &p, cudaStream_t st) {
    static const char *fn = "attention_kv8";
    constexpr size_t smem = sizeof(PreSmem<C>) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory");
    static thread_local int allowed_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev != allowed_dev) {
        cudaError_t e = cudaFuncSetAttribute(
            attn_prompt_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return fail_cuda(e, fn);
        allowed_dev = dev;
    }
    cudaError_t e = launch_pdl(attn_prompt_kernel<C>, dim3((unsigned)num_sms()), dim3(THREADS),
                               smem, st, p);
    return e == cudaSuccess ? JKB_OK : fail_cuda(e, fn);
}

template <int DT>
int launch_dim(const AttnParams &p, int type, cudaStream_t st) {
    if (type == JKB_F32) return launch_cfg<PreCfg<DT, JKB_F32>>(p, st);
    if (type == JKB_F16) return launch_cfg<PreCfg<DT, JKB_F16>>(p, st);
    return launch_cfg<PreCfg<DT, JKB_BF16>>(p, st);
}

}  // namespace

int attn_prompt_launch(const AttnParams &p, int type, int dim_p, cudaStream_t st) {
    switch (dim_p) {
    case 64: return launch_dim<2>(p, type, st);
    case 96: return launch_dim<3>(p, type, st);
    default: return launch_dim<4>(p, type, st);
    }
}

}  // namespace jkb
