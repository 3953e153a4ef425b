// Attention over the 8-bit key/value cache for many query rows a kv head (prompts and chunks), on
// the fifth-generation tensor cores.
//
// A tile is 128 query rows (tokens x the query heads of one kv head, heads fastest, so that the
// rows stand close together and a causal tile wastes little); its cached tokens go by in units of
// 128. Per unit, with the unit's blocks' scales ks and vs and c = scale log2(e):
//   S = Q K^T           Q in f16 with a power of two of its own per row (exact for 16-bit rows;
//                       f32 rows as two f16, 22 bits), K the codes, exact in f16
//   s = c ks S,  m' = max(m, max s),  a = 2^(m - m'),  p = 2^(s - m'),  l = a l + sum p
//   o = a o + (p vs) V  V the codes, exact in f16 and bf16; p vs in f16 (f16 rows), in two bf16
//                       (bf16 rows) or three (f32 rows). bf16 has f32's range: a weight that is
//                       far below its row's largest keeps its digits.
// The tensor core truncates its f32 sums, about 2^-25 of the sum at every 16-element step. So S
// takes the small part of Q first, and each unit's P V starts from zero, small parts first, and
// is added to o in registers, rounded, with the rescale.
//
// Work: MMA time is (DIM / 16) NQ + 8 NP steps a unit against 16 for one plain product pair; the
// exponentials are 128 x 128 a unit on 16 lanes an SM and clock, about as long as two products.
// One CTA an SM, four warpgroups, every hand-over an mbarrier:
//   0  softmax: a thread a row; S from TMEM to registers, p's parts back over S
//   1  accumulation: a thread a row; the unit's P V from TMEM, o in registers; writes the output
//   2  conversion: codes from the raw rings to f16 / bf16 operand tiles (128-byte swizzle), and
//      the query rows of a new tile
//   3  a warp that issues the MMAs, one that loads keys and one that loads values (a bulk copy
//      for 16 tokens each, kv_cache.cuh)
// S is double-buffered: the order of the MMAs is S(i + 1), P V(i), S(i + 2), .. so that they run
// under the softmax. One K operand tile is enough (K(i + 2) is converted during P V(i)), and for
// f32 rows, whose products take longer, one V tile (V(i + 1) during S(i + 2)).
//
// Tiles of all sequences and kv heads form one line of units, cut into equal parts, one a CTA; a
// tile that spans CTAs is put together from the workspace by the last of them to finish, in the
// order of the line (as in kv_attn.cu).
#include "kv_attn.cuh"
#include "ptx.cuh"

#include <cuda_bf16.h>

namespace jkb {

namespace {

constexpr int TM = 128;        // query rows of a tile
constexpr int TN = 128;        // cached tokens of a unit
constexpr int GROUPS = TN / KV_GROUP;
constexpr int THREADS = 512;
constexpr int RAW = 2;         // raw rings of codes, units
constexpr int SC = 8;          // ring of block scales, units
constexpr int REGS_SOFT = 136, REGS_SUM = 208, REGS_CONV = 96, REGS_REST = 72;  // of a warpgroup
static_assert(REGS_SOFT + REGS_SUM + REGS_CONV + REGS_REST <= 4 * 128, "what the launch holds");

// TYPE: the rows'. NQ: f16 parts of a query element; NP: parts of p; F16: p and V are f16 (else
// bf16).
template <int DT_, int TYPE_>
struct PreCfg {
    static constexpr int DT = DT_, TYPE = TYPE_;
    static constexpr bool F16 = TYPE == JKB_F16;
    static constexpr int NQ = TYPE == JKB_F32 ? 2 : 1;
    static constexpr int NP = TYPE == JKB_F32 ? 3 : TYPE == JKB_BF16 ? 2 : 1;
    static constexpr int DIM = 32 * DT;
    static constexpr int KA = (DIM + 63) / 64;       // 64-element swizzle atoms of a head
    static constexpr int NV = NQ == 2 ? 1 : 2;       // V buffers
    static constexpr int SIDE_BYTES = 16 * DIM;      // a group's keys, or its values
    static constexpr int S_COLS = 192;               // TMEM columns of an S / P buffer
    static constexpr int O_COL = 2 * S_COLS;
    static_assert(DIM <= 128 && NP * TN / 2 <= S_COLS, "TMEM: two S / P buffers and one o");
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
    float alpha[4][TM];
    float row_scale[TM], fin_m[TM], fin_l[TM];
    uint64_t rk_full[RAW], rk_empty[RAW], rv_full[RAW], rv_empty[RAW], sc_full[SC], k_full,
        k_empty, v_full[C::NV], v_empty[C::NV], q_full, q_empty, s_full[2], p_full[2], o_full, o_empty, a_full[4],
        fin_full, fin_empty, merge, done;
    long long warp_sum[THREADS / 32];
    long long line_total, first_start;
    int first_seq, first_tile, first_head;
    uint32_t tmem;
    int abort_flag, is_last, n_big;
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
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
        "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
        "%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
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
    int row0, first, units, pos0;  // pos0: position of query token 0
};
__device__ __forceinline__ Tile tile_of(const AttnParams &p, const AttnSeq &s, int tile) {
    Tile t;
    t.row0 = tile * TM;
    t.pos0 = s.len - s.nq;
    const int last = (int)min((long long)t.row0 + TM - 1, (long long)s.nq * p.group - 1) / p.group;
    const int hi = p.causal ? max(0, min(s.len, t.pos0 + last + 1)) : s.len;
    int lo = 0;
    if (p.window)
        lo = (int)min(max((long long)t.pos0 + t.row0 / p.group - p.window + 1, 0ll),
                      (long long)hi);
    t.first = lo / TN;
    t.units = max(1, (hi + TN - 1) / TN - t.first);
    return t;
}
__device__ __forceinline__ int tiles_of(const AttnParams &p, const AttnSeq &s) {
    return (int)(((long long)s.nq * p.group + TM - 1) / TM);
}

// A CTA's part of the line: pieces of tiles. Order: sequence, tile from the last (the longest of
// a causal prompt) to the first, kv head.
struct Cursor {
    long long u, end, start;  // this CTA's units left; the line's unit where the tile starts
    int seq, tile, head;
    AttnSeq s;
    Tile t;
    int c0, n;  // the piece: units c0 .. c0 + n of the tile
};
template <class C>
__device__ __forceinline__ bool cursor_first(const AttnParams &p, const PreSmem<C> &sm,
                                             long long u0, long long u1, Cursor &k) {
    k.u = u0;
    k.end = u1;
    k.start = sm.first_start;
    k.seq = sm.first_seq;
    k.tile = sm.first_tile;
    k.head = sm.first_head;
    k.s = attn_seq(p, k.seq);
    k.t = tile_of(p, k.s, k.tile);
    k.c0 = (int)(u0 - k.start);
    k.n = (int)min((long long)(k.t.units - k.c0), u1 - u0);
    return true;
}
__device__ __forceinline__ bool cursor_next(const AttnParams &p, Cursor &k) {
    k.u += k.n;
    if (k.u >= k.end) return false;
    k.start += k.t.units;
    if (++k.head == p.kv_heads) {
        k.head = 0;
        if (--k.tile < 0) {
            do {
                k.seq++;
                k.s = attn_seq(p, k.seq);
            } while (k.s.nq == 0);
            k.tile = tiles_of(p, k.s) - 1;
        }
        k.t = tile_of(p, k.s, k.tile);
    }
    k.c0 = 0;
    k.n = (int)min((long long)k.t.units, k.end - k.u);
    return true;
}

// Query rows in, output rows out.
template <int TYPE>
__device__ __forceinline__ float load1(const void *q, size_t i) {
    if constexpr (TYPE == JKB_F32) return __ldg(static_cast<const float *>(q) + i);
    else if constexpr (TYPE == JKB_F16)
        return __half2float(__ldg(static_cast<const __half *>(q) + i));
    else return __bfloat162float(__ldg(static_cast<const __nv_bfloat16 *>(q) + i));
}
template <int TYPE>
__device__ __forceinline__ float4 load4(const AttnParams &p, size_t i) {
    if (!p.q_vec)
        return make_float4(load1<TYPE>(p.q, i), load1<TYPE>(p.q, i + 1), load1<TYPE>(p.q, i + 2),
                           load1<TYPE>(p.q, i + 3));
    if constexpr (TYPE == JKB_F32) {
        return __ldg(reinterpret_cast<const float4 *>((const float *)p.q + i));
    } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>((const uint16_t *)p.q + i));
        if constexpr (TYPE == JKB_F16) {
            const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x));
            const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
            return make_float4(a.x, a.y, b.x, b.y);
        } else {
            return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u),
                               __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u));
        }
    }
}
template <int TYPE>
__device__ __forceinline__ void store8(const AttnParams &p, size_t i, const float (&x)[8]) {
    if constexpr (TYPE == JKB_F32) {
        float *o = static_cast<float *>(p.out) + i;
        if (p.out_vec) {
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
        if (p.out_vec) {
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

// f16 p: the unit's largest value scale is below 2^vexp, and vs enters as vs 2^(14 - vexp).
__device__ __forceinline__ int unit_vexp(const float2 *sc, uint32_t valid) {
    int e = -126;
#pragma unroll
    for (int g = 0; g < GROUPS; g++)
        if ((valid >> g) & 1)
            e = max(e, (int)((__float_as_uint(sc[g].y) >> 23) & 255) - 126);
    return e;
}
__device__ __forceinline__ float scale_f16(float vs, int vexp) {
    const uint32_t b = __float_as_uint(vs);
    return (b & 0x7F800000u) ? __uint_as_float((b & 0x807FFFFFu) | 0x3F000000u) *
                                   ex2((float)((int)((b >> 23) & 255) - 126 - vexp + 14))
                             : 0.0f;
}

// One unit of one row (thread): S from TMEM at ts, scaled by rs ks and masked to tokens lo .. hi
// of the unit, into the row's running m and l; alpha, the factor of what was summed before, goes
// to shared memory as soon as it is known. p's parts go back to TMEM over S: of the 16 columns of
// a group of tokens, the first 8 take part 0, the last 8 part 1; part 2 stands behind S.
// S is read twice (maximum, then weights), a group at a time, so that the loops stay rolled: with
// more unrolling the roles' loops together outgrow the SM's instruction cache, and every unit
// fetches them anew (unrolled over 128 columns, four times slower).
template <class C, bool MASKED>
__device__ __forceinline__ void softmax_unit(uint32_t ts, const float2 *sc, uint32_t valid,
                                             float rs, int lo, int hi, float &m, float &l,
                                             float *alpha_out, uint64_t *alpha_bar) {
    constexpr int NP = C::NP;
    uint32_t r[16];
    tmem_ld16(ts, r);
    float top[2] = {m, -INFINITY};
#pragma unroll 1
    for (int g = 0; g < GROUPS; g++) {
        const float f = rs * sc[g].x;
        uint64_t x[8];
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = mul2(pk2(r[2 * i], r[2 * i + 1]), pkf(f, f));
        tmem_ld16(ts + 16 * ((g + 1) % GROUPS), r);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float u, w;
            upk2(x[i], u, w);
            if (MASKED) {
                const int t = 16 * g + 2 * i;
                const bool on = (valid >> g) & 1;
                u = on && t >= lo && t < hi ? u : -INFINITY;
                w = on && t + 1 >= lo && t + 1 < hi ? w : -INFINITY;
            }
            top[i & 1] = fmaxf(top[i & 1], fmaxf(u, w));
        }
    }
    const float mn = fmaxf(top[0], top[1]);
    const float ref = mn == -INFINITY ? 0.0f : mn;
    const float alpha = ex2(m - ref);
    m = mn;
    *alpha_out = alpha;
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(alpha_bar);
    int vexp = 0;
    if (C::F16) vexp = unit_vexp(sc, valid);
    const uint64_t nref = pkf(-ref, -ref);
    uint64_t sum = 0;
#pragma unroll 1
    for (int g = 0; g < GROUPS; g++) {
        const float f = rs * sc[g].x, vs = C::F16 ? scale_f16(sc[g].y, vexp) : sc[g].y;
        uint64_t x[8];
        tmem_ld_wait();
        // (a product and a sum, rounded as in the first pass: the largest is 2^0 exactly)
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = mul2(pk2(r[2 * i], r[2 * i + 1]), pkf(f, f));
        if (g + 1 < GROUPS) tmem_ld16(ts + 16 * (g + 1), r);
        uint32_t part[NP][8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float u, w;
            upk2(add2(x[i], nref), u, w);
            if (MASKED) {
                const int t = 16 * g + 2 * i;
                const bool on = (valid >> g) & 1;
                u = on && t >= lo && t < hi ? u : -INFINITY;
                w = on && t + 1 >= lo && t + 1 < hi ? w : -INFINITY;
            }
            uint64_t e = pkf(ex2(u), ex2(w));
            sum = add2(sum, e);
            e = mul2(e, pkf(vs, vs));
#pragma unroll
            for (int k = 0; k < NP; k++) {
                upk2(e, u, w);
                if (C::F16) {
                    const __half2 y = __floats2half2_rn(u, w);
                    part[k][i] = *reinterpret_cast<const uint32_t *>(&y);
                } else {
                    const __nv_bfloat162 y = __floats2bfloat162_rn(u, w);
                    part[k][i] = *reinterpret_cast<const uint32_t *>(&y);
                    if (k < NP - 1)
                        e = add2(e, pk2((part[k][i] << 16) ^ 0x80000000u,
                                        (part[k][i] & 0xFFFF0000u) ^ 0x80000000u));
                }
            }
        }
        tmem_st8(ts + 16 * g, part[0]);
        if (NP > 1) tmem_st8(ts + 16 * g + 8, part[NP > 1 ? 1 : 0]);
        if (NP > 2) tmem_st8(ts + TN + 8 * g, part[NP - 1]);
    }
    float su, sw;
    upk2(sum, su, sw);
    l = fmaf(l, alpha, su + sw);
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
        sm.n_big = 0;
        for (int i = 0; i < RAW; i++) {
            mbar_init(&sm.rk_full[i], 1);
            mbar_init(&sm.rk_empty[i], 4);
            mbar_init(&sm.rv_full[i], 1);
            mbar_init(&sm.rv_empty[i], 4);
        }
        for (int i = 0; i < SC; i++) mbar_init(&sm.sc_full[i], 1);
        mbar_init(&sm.k_full, 4);
        mbar_init(&sm.k_empty, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.p_full[i], 4);
        }
        for (int i = 0; i < NV; i++) {
            mbar_init(&sm.v_full[i], 4);
            mbar_init(&sm.v_empty[i], 1);
        }
        for (int i = 0; i < 4; i++) mbar_init(&sm.a_full[i], 4);
        mbar_init(&sm.q_full, 4);
        mbar_init(&sm.q_empty, 5);
        mbar_init(&sm.o_full, 1);
        mbar_init(&sm.o_empty, 4);
        mbar_init(&sm.fin_full, 4);
        mbar_init(&sm.fin_empty, 4);
        mbar_init(&sm.merge, 4);
        mbar_init(&sm.done, 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (warp == 12) {
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

    // ---- this CTA's part of the line (the operand buffers are scratch until the roles start):
    // units a sequence, by its thread or, where it has many tiles, by a warp; then a block scan
    {
        long long *sum = reinterpret_cast<long long *>(&sm.q[0][0][0]);  // [n_seqs]
        int *big = reinterpret_cast<int *>(sum + p.n_seqs);              // [n_seqs]
        static_assert(offsetof(PreSmem<C>, sc) >= 12 * JKB_KV_MAX_SEQS, "scratch");
        const int per_t = (p.n_seqs + THREADS - 1) / THREADS;
        const int a = min(tid * per_t, p.n_seqs), b = min(a + per_t, p.n_seqs);
        for (int i = a; i < b; i++) {
            const AttnSeq s = attn_seq(p, i);
            const int tiles = tiles_of(p, s);
            long long x = 0;
            if (tiles <= 4)
                for (int r = 0; r < tiles; r++) x += tile_of(p, s, r).units;
            else
                big[atomicAdd(&sm.n_big, 1)] = i;
            sum[i] = x * p.kv_heads;
        }
        __syncthreads();
        for (int j = warp; j < sm.n_big; j += THREADS / 32) {
            const AttnSeq s = attn_seq(p, big[j]);
            const int tiles = tiles_of(p, s);
            long long x = 0;
            for (int r = lane; r < tiles; r += 32) x += tile_of(p, s, r).units;
            for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(~0u, x, d);
            if (lane == 0) sum[big[j]] = x * p.kv_heads;
        }
        __syncthreads();
        long long mine = 0;
        for (int i = a; i < b; i++) mine += sum[i];
        long long inc = mine;
        for (int d = 1; d < 32; d <<= 1) {
            const long long x = __shfl_up_sync(~0u, inc, d);
            if (lane >= d) inc += x;
        }
        if (lane == 31) sm.warp_sum[warp] = inc;
        __syncthreads();
        long long at = inc - mine, total = 0;
        for (int w = 0; w < THREADS / 32; w++) {
            if (w < warp) at += sm.warp_sum[w];
            total += sm.warp_sum[w];
        }
        if (tid == 0) sm.line_total = total;
        const long long per = (total + gridDim.x - 1) / gridDim.x;
        const long long u0 = min(per * blockIdx.x, total);
        for (int i = a; i < b; i++) {
            if (sum[i] && u0 >= at && u0 < at + sum[i]) {
                sm.first_seq = i;
                sm.first_start = at;  // of the sequence, until the tile is found
            }
            at += sum[i];
        }
        __syncthreads();
        if (warp == 0 && u0 < total) {
            const int seq = sm.first_seq;
            const AttnSeq s = attn_seq(p, seq);
            long long left = u0 - sm.first_start, start = sm.first_start;
            for (int r = tiles_of(p, s) - 1;; r -= 32) {
                const int units = r - lane >= 0 ? tile_of(p, s, r - lane).units : 0;
                long long x = (long long)units * p.kv_heads, upto = x;
                for (int d = 1; d < 32; d <<= 1) {
                    const long long y = __shfl_up_sync(~0u, upto, d);
                    if (lane >= d) upto += y;
                }
                const unsigned hit = __ballot_sync(~0u, left < upto);
                if (hit) {
                    if (lane == __ffs(hit) - 1) {
                        const long long in = left - (upto - x);
                        sm.first_tile = r - lane;
                        sm.first_head = (int)(in / units);
                        sm.first_start = start + (upto - x) + in / units * units;
                    }
                    break;
                }
                const long long all = __shfl_sync(~0u, upto, 31);
                left -= all;
                start += all;
            }
        }
        proxy_fence();  // the scratch becomes the target of bulk copies
        __syncthreads();
    }
    const long long total = sm.line_total, per = (total + gridDim.x - 1) / gridDim.x;
    const long long u0 = min(per * blockIdx.x, total), u1 = min(u0 + per, total);
    const uint32_t tmem = sm.tmem;
    Cursor cur;
    bool more = u0 < u1;
    if (more) cursor_first<C>(p, sm, u0, u1, cur);
    // a warp's wait: all of its lanes go on, or (after the limit, or an abort) none
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        return __all_sync(~0u, mbar_wait_short(bar, parity & 1, abort_flag, p.err)) != 0;
    };

    if (wg == 0) {
        // ------------------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFT));
        const uint32_t tl = tmem + ((uint32_t)(warp * 32) << 16);
        const int row = tid;  // of the tile
        uint32_t it = 0, piece = 0;
        for (; more; more = cursor_next(p, cur), piece++) {
            if (!wait(&sm.q_full, piece)) goto out;
            const float rs = sm.row_scale[row];
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.q_empty);
            const int tok = (cur.t.row0 + row) / p.group, pos = cur.t.pos0 + tok;
            const int hi = p.causal ? min(cur.s.len, pos + 1) : cur.s.len;
            const int lo = p.window ? max(0, pos - p.window + 1) : 0;
            // tokens that every row of the tile sees
            const int pos_a = cur.t.pos0 + cur.t.row0 / p.group;
            const int pos_b = cur.t.pos0 + (cur.t.row0 + TM - 1) / p.group;
            const int all_hi = p.causal ? min(cur.s.len, pos_a + 1) : cur.s.len;
            const int all_lo = p.window ? pos_b - p.window + 1 : 0;
            float m = -INFINITY, l = 0.0f;
            for (int c = 0; c < cur.n; c++, it++) {
                const int b = it & 1;
                if (!wait(&sm.sc_full[it % SC], it / SC) || !wait(&sm.s_full[b], it >> 1))
                    goto out;
                tc_fence_after();
                const int key0 = (cur.t.first + cur.c0 + c) * TN;
                const uint32_t valid = sm.valid[it % SC];
                const bool masked = key0 < all_lo || key0 + TN > all_hi || valid != 0xFFu;
                const float2 *sc = sm.sc[it % SC];
                const uint32_t ts = tl + b * C::S_COLS;
                if (masked)
                    softmax_unit<C, true>(ts, sc, valid, rs, lo - key0, hi - key0, m, l,
                                          &sm.alpha[it & 3][row], &sm.a_full[it & 3]);
                else
                    softmax_unit<C, false>(ts, sc, valid, rs, 0, TN, m, l,
                                           &sm.alpha[it & 3][row], &sm.a_full[it & 3]);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.p_full[b]);
            }
            if (!wait(&sm.fin_empty, piece + 1)) goto out;
            sm.fin_m[row] = m;
            sm.fin_l[row] = l;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.fin_full);
        }
    } else if (wg == 1) {
        // ------------------------------------------------------------ accumulation and output
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SUM));
        const int row = tid - 128;
        const uint32_t tl = tmem + ((uint32_t)((warp - 4) * 32) << 16) + C::O_COL;
        uint32_t it = 0, piece = 0, merges = 0;
        for (; more; more = cursor_next(p, cur), piece++) {
            uint64_t o[DIM / 2];  // pairs of columns
#pragma unroll
            for (int i = 0; i < DIM / 2; i++) o[i] = 0;
            for (int c = 0; c < cur.n; c++, it++) {
                if (!wait(&sm.a_full[it & 3], it >> 2)) goto out;
                const float alpha = sm.alpha[it & 3][row];
                const uint64_t al = pkf(alpha, alpha);
                float up = 1.0f;  // (a power of two that flushes to 0 is below f16's smallest)
                if (C::F16) up = ex2((float)(unit_vexp(sm.sc[it % SC], sm.valid[it % SC]) - 14));
                if (!wait(&sm.o_full, it)) goto out;
                tc_fence_after();
                uint32_t r[2][32];
                tmem_ld32(tl, r[0]);
#pragma unroll
                for (int q = 0; q < DT; q++) {
                    tmem_ld_wait();
                    if (q + 1 < DT) tmem_ld32(tl + 32 * (q + 1), r[(q + 1) & 1]);
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        uint64_t x = pk2(r[q & 1][2 * i], r[q & 1][2 * i + 1]);
                        if (C::F16) x = mul2(x, pkf(up, up));
                        o[16 * q + i] = fma2(o[16 * q + i], al, x);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.o_empty);
            }
            if (!wait(&sm.fin_full, piece)) goto out;
            float m = sm.fin_m[row], l = sm.fin_l[row];
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.fin_empty);

            const int cta0 = (int)(cur.start / per);
            const int cta1 = (int)((cur.start + cur.t.units - 1) / per);
            if (cta0 != cta1) {
                auto slot_of = [&](int cta) {
                    const int slot = 2 * cta + (cta == cta0 && cur.start != per * cta0 ? 1 : 0);
                    return p.tile_partial + (size_t)slot * TM * (DIM + 2);
                };
                float *mine = slot_of((int)blockIdx.x);
#pragma unroll
                for (int i = 0; i < DIM / 2; i++) {
                    float u, w;
                    upk2(o[i], u, w);
                    mine[2 * i * TM + row] = u;
                    mine[(2 * i + 1) * TM + row] = w;
                }
                mine[DIM * TM + row] = m;
                mine[(DIM + 1) * TM + row] = l;
                __threadfence();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.merge);
                if (!wait(&sm.merge, merges++)) goto out;
                if (tid == 128) {
                    const int before = atomicAdd(&p.tile_counters[cta0], 1);
                    sm.is_last = before == cta1 - cta0;
                    if (sm.is_last) p.tile_counters[cta0] = 0;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.merge);
                if (!wait(&sm.merge, merges++)) goto out;
                const bool last = *(volatile int *)&sm.is_last;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.merge);  // is_last may be written again
                if (!wait(&sm.merge, merges++)) goto out;
                if (!last) continue;
                __threadfence();
                m = -INFINITY;
                for (int k = cta0; k <= cta1; k++)
                    m = fmaxf(m, __ldcg(slot_of(k) + DIM * TM + row));
                const float ref = m == -INFINITY ? 0.0f : m;
                l = 0.0f;
#pragma unroll
                for (int i = 0; i < DIM / 2; i++) o[i] = 0;
                for (int k = cta0; k <= cta1; k++) {
                    const float *x = slot_of(k) + row;
                    const float w = ex2(__ldcg(x + DIM * TM) - ref);
                    l = fmaf(w, __ldcg(x + (DIM + 1) * TM), l);
#pragma unroll
                    for (int i = 0; i < DIM / 2; i++)
                        o[i] = fma2(pkf(w, w), pkf(__ldcg(x + 2 * i * TM),
                                                   __ldcg(x + (2 * i + 1) * TM)), o[i]);
                }
            }
            const int rr = cur.t.row0 + row, tok = rr / p.group;
            const int h = cur.head * p.group + rr - tok * p.group;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            if (tok < cur.s.nq) {
                if (p.lse)
                    p.lse[(size_t)(cur.s.q0 + tok) * p.group * p.kv_heads + h] =
                        (m + log2f(l)) * 0.69314718055994531f;
                const size_t at = (size_t)(cur.s.q0 + tok) * p.out_token + (size_t)h * p.out_head;
                // column 32 c + 8 j + g of o is dim 32 c + 4 g + j
#pragma unroll
                for (int c = 0; c < DT; c++)
#pragma unroll
                    for (int g = 0; g < 8; g += 2) {
                        const int d = 32 * c + 4 * g;
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 4; i++) {  // columns 8 i + g and 8 i + g + 1
                            upk2(o[16 * c + 4 * i + g / 2], x[i], x[4 + i]);
                            x[i] *= inv;
                            x[4 + i] *= inv;
                        }
                        if (d < p.dim) store8<C::TYPE>(p, at + d, x);
                    }
            }
            __syncwarp();
        }
    } else if (wg == 2) {
        // ------------------------------------------------------------ conversion
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CONV));
        const int ct = tid - 256, cw = warp - 8;
        uint32_t it = 0, piece = 0;
        for (; more; more = cursor_next(p, cur), piece++) {
            // ---- the query rows: f16 parts of x times a power of two of the row ----
            if (!wait(&sm.q_empty, piece + 1)) goto out;
            // eight lanes a row, 16 dims a lane
#pragma unroll 2
            for (int r0 = 0; r0 < 32; r0 += 4) {
                const int r = cw * 32 + r0 + (lane >> 3), d0 = 16 * (lane & 7);
                const int rr = cur.t.row0 + r, tok = rr / p.group;
                const size_t at = (size_t)(cur.s.q0 + tok) * p.q_token +
                                  (size_t)(cur.head * p.group + rr - tok * p.group) * p.q_head;
                float4 x[4];
                float top = 0.0f;
                bool fine = true;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (tok < cur.s.nq && d0 + 4 * k < p.dim)
                        x[k] = load4<C::TYPE>(p, at + d0 + 4 * k);
                }
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float a = fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)),
                                          fmaxf(fabsf(x[k].z), fabsf(x[k].w)));
                    top = fmaxf(top, a);
                    // a non-finite element makes the sum of the element times 0 a NaN
                    fine &= x[k].x * 0.0f + x[k].y * 0.0f + x[k].z * 0.0f + x[k].w * 0.0f == 0.0f;
                }
                for (int d = 4; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
                const unsigned rows_fine = __ballot_sync(~0u, fine);
                fine = ((rows_fine >> (lane & 24)) & 0xFFu) == 0xFFu;
                // 2^e brings the largest element into [2^14, 2^15)
                const int e = min(14 + 127 - (int)((__float_as_uint(top) >> 23) & 255), 126);
                float up = __uint_as_float((uint32_t)(127 + e) << 23);
                if ((lane & 7) == 0)
                    sm.row_scale[r] = !fine ? __int_as_float(0x7FC00000)
                                      : top == 0.0f ? 0.0f : p.scale2 / up;
                if (64 * C::KA > d0) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float v[8] = {x[2 * h].x, x[2 * h].y, x[2 * h].z, x[2 * h].w,
                                      x[2 * h + 1].x, x[2 * h + 1].y, x[2 * h + 1].z,
                                      x[2 * h + 1].w};
#pragma unroll
                        for (int k = 0; k < 8; k++) v[k] = fine ? v[k] * up : 0.0f;
                        const int ch = (2 * (lane & 7) + h) & 7;
#pragma unroll
                        for (int k = 0; k < NQ; k++) {
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const __half2 y = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                                const float2 f = __half22float2(y);
                                w[i] = *reinterpret_cast<const uint32_t *>(&y);
                                v[2 * i] -= f.x;
                                v[2 * i + 1] -= f.y;
                            }
                            *reinterpret_cast<uint4 *>(
                                &sm.q[k][d0 >> 6][r * 128 + ((ch ^ (r & 7)) << 4)]) =
                                make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
            }
            proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.q_full);

            // K(n), then V(n - 1)
            for (int c = 0; c <= cur.n; c++) {
                if (c < cur.n) {
                    const uint32_t n = it + c;
                    if (!wait(&sm.rk_full[n % RAW], n / RAW) || !wait(&sm.k_empty, n + 1))
                        goto out;
                    const uint8_t *raw = sm.raw_k[n % RAW];
                    // unit: a token's 32 dims, its halves in the order that keeps eight lanes
                    // (eight tokens) on eight bank groups
#pragma unroll 1
                    for (int u = ct; u < TN * DT; u += 128) {
                        const int tk = u & 7, rest = u >> 3, chunk = rest % DT, hg = rest / DT;
                        const uint8_t *src = raw + hg * 8 * DIM + chunk * 256 + tk * 32;
                        uint8_t *dst = &sm.k[chunk >> 1][(hg * 8 + tk) * 128];
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const int hh = i ^ (tk >> 2);
                            const uint4 x = *reinterpret_cast<const uint4 *>(src + 16 * hh);
                            const uint32_t w[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u,
                                                   x.z ^ 0x80808080u, x.w ^ 0x80808080u};
                            const int ch = (chunk & 1) * 4 + 2 * hh;
                            *reinterpret_cast<uint4 *>(dst + ((ch ^ tk) << 4)) =
                                make_uint4(pair_f16(w[0], 0x4140), pair_f16(w[0], 0x4342),
                                           pair_f16(w[1], 0x4140), pair_f16(w[1], 0x4342));
                            *reinterpret_cast<uint4 *>(dst + (((ch + 1) ^ tk) << 4)) =
                                make_uint4(pair_f16(w[2], 0x4140), pair_f16(w[2], 0x4342),
                                           pair_f16(w[3], 0x4140), pair_f16(w[3], 0x4342));
                        }
                    }
                    proxy_fence();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&sm.rk_empty[n % RAW]);
                        mbar_arrive(&sm.k_full);
                    }
                }
                if (c > 0) {
                    const uint32_t n = it + c - 1;
                    const int vb = n % NV;
                    if (!wait(&sm.rv_full[n % RAW], n / RAW) ||
                        !wait(&sm.v_empty[vb], n / NV + 1))
                        goto out;
                    const uint8_t *raw = sm.raw_v[n % RAW];
                    // unit: 16 tokens of four dims (4 g + j), to rows 8 j + g
#pragma unroll 1
                    for (int u = ct; u < GROUPS * DT * 8; u += 128) {
                        const int g = u & 7, rest = u >> 3, chunk = rest % DT, grp = rest / DT;
                        const uint8_t *src = raw + grp * C::SIDE_BYTES + chunk * 512;
                        uint32_t w[4][4];  // [t][j]
#pragma unroll
                        for (int t = 0; t < 4; t++) {
                            const uint4 x = *reinterpret_cast<const uint4 *>(
                                src + (t * 8 + (g ^ (2 * t))) * 16);
                            w[t][0] = x.x, w[t][1] = x.y, w[t][2] = x.z, w[t][3] = x.w;
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            uint8_t *dst = &sm.v[vb][grp >> 2][(32 * chunk + 8 * j + g) * 128];
#pragma unroll
                            for (int i = 0; i < 2; i++) {  // tokens 8 i .. 8 i + 7
                                uint32_t y[4];
#pragma unroll
                                for (int t = 0; t < 4; t++)
                                    y[t] = C::F16 ? pair_f16(w[t][j], i ? 0x4342 : 0x4140)
                                                  : pair_bf16(w[t][j], i);
                                *reinterpret_cast<uint4 *>(
                                    dst + ((((grp & 3) * 2 + i) ^ g) << 4)) =
                                    make_uint4(y[0], y[1], y[2], y[3]);
                            }
                        }
                    }
                    proxy_fence();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&sm.rv_empty[n % RAW]);
                        mbar_arrive(&sm.v_full[vb]);
                    }
                }
            }
            it += cur.n;
        }
    } else if (warp == 12) {
        // ------------------------------------------------------------ MMA
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_REST));
        constexpr uint32_t ID_S = idesc_f16(TN, false), ID_O = idesc_f16(DIM, !C::F16);
        uint32_t it = 0, piece = 0;
        auto issue_pv = [&](uint32_t i) {
            const int b = i & 1, vb = i % NV;
            if (!wait(&sm.p_full[b], i >> 1) || !wait(&sm.v_full[vb], i / NV) ||
                !wait(&sm.o_empty, i + 1))
                return false;
            tc_fence_after();
            if (lane == 0) {
                const uint32_t vd = desc_lo(&sm.v[vb][0][0]), pt = tmem + b * C::S_COLS;
                const uint32_t od = tmem + C::O_COL;
                // parts of p from the last; their columns as softmax_unit leaves them. V of step
                // s: atom s / 4, 32 bytes a step
#pragma unroll 1
                for (int k = NP - 1; k >= 0; k--) {
                    const uint32_t a = pt + (k == 2 ? TN : 8 * k), step = k == 2 ? 8 : 16;
#pragma unroll
                    for (int s = 0; s < TN / 16; s++)
                        mma_ts(od, a + s * step, vd + (s >> 2) * (DIM * 128 / 16) + (s & 3) * 2,
                               ID_O, s || k < NP - 1);
                }
                tc_commit(&sm.v_empty[vb]);
                tc_commit(&sm.o_full);
            }
            __syncwarp();
            return true;
        };
        for (; more; more = cursor_next(p, cur), piece++) {
            if (!wait(&sm.q_full, piece)) goto out;
            for (int c = 0; c < cur.n; c++, it++) {
                const int b = it & 1;
                if (!wait(&sm.k_full, it)) goto out;
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t kd = desc_lo(&sm.k[0][0]), qd = desc_lo(&sm.q[0][0][0]);
                    const uint32_t sd = tmem + b * C::S_COLS;
#pragma unroll 1
                    for (int k = NQ - 1; k >= 0; k--) {
                        const uint32_t ad = qd + k * (C::KA * TM * 128 / 16);
#pragma unroll
                        for (int s = 0; s < DIM / 16; s++) {
                            const uint32_t at = (s >> 2) * (TM * 128 / 16) + (s & 3) * 2;
                            mma_ss(sd, ad + at, kd + at, ID_S, s || k < NQ - 1);
                        }
                    }
                    tc_commit(&sm.k_empty);
                    if (c == cur.n - 1) tc_commit(&sm.q_empty);
                    tc_commit(&sm.s_full[b]);
                }
                __syncwarp();
                if (c > 0 && !issue_pv(it - 1)) goto out;
            }
            if (!issue_pv(it - 1)) goto out;
        }
    } else if (warp < 15) {
        // ------------------------------------------------------------ loads
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_REST));
        const bool keys = warp == 13;
        uint64_t *full = keys ? sm.rk_full : sm.rv_full, *empty = keys ? sm.rk_empty : sm.rv_empty;
        uint8_t *ring = keys ? sm.raw_k[0] : sm.raw_v[0];
        const uint8_t *codes = p.codes + (keys ? 0 : C::SIDE_BYTES);
        uint32_t it = 0;
        for (; more; more = cursor_next(p, cur)) {
            const int32_t *ids = p.table + (size_t)cur.seq * p.table_stride;
            const int last = (int)min((long long)cur.t.row0 + TM - 1,
                                      (long long)cur.s.nq * p.group - 1) / p.group;
            const int hi = p.causal ? min(cur.s.len, cur.t.pos0 + last + 1) : cur.s.len;
            const int lo = p.window
                               ? max(0, cur.t.pos0 + cur.t.row0 / p.group - p.window + 1) : 0;
            // the lookups of 32 groups (four units) at a time, the next ones ahead of their use
            int id;
            float2 sc;
            auto look = [&](int c) {
                id = -1;
                sc = make_float2(0.f, 0.f);
                const int t0 = (cur.t.first + cur.c0 + c) * TN + lane * KV_GROUP;
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
                if (lane == 0)
                    mbar_arrive_tx(&full[slot], __popc(there) * C::SIDE_BYTES);
                __syncwarp();
                if (lane < GROUPS && gid >= 0) {
                    const int t0 = (cur.t.first + cur.c0 + c) * TN + lane * KV_GROUP;
                    const int grp = (t0 & ((1 << p.log_block) - 1)) / KV_GROUP;
                    const size_t bh = (size_t)gid * p.kv_heads + cur.head;
                    bulk_load(ring + (size_t)(slot * GROUPS + lane) * C::SIDE_BYTES,
                              codes + ((bh << p.log_block) / KV_GROUP + grp) *
                                          (size_t)(2 * C::SIDE_BYTES),
                              C::SIDE_BYTES, &full[slot]);
                }
                if (keys) {
                    if (lane < GROUPS) sm.sc[it % SC][lane] = gs;
                    if (lane == 0) sm.valid[it % SC] = there;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.sc_full[it % SC]);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_REST));
    }
out:
    // On expiry of a wait: the loads and MMAs in flight end (bounded) before the memory goes.
    if (warp == 12 && lane == 0) {
        tc_commit(&sm.done);
        const unsigned long long t0 = globaltimer();
        while (!mbar_try(&sm.done, 0) && globaltimer() - t0 < WAIT_NS) {
        }
    }
    __syncwarp();
    if ((warp == 13 || warp == 14) && *abort_flag) {
        const unsigned long long t0 = globaltimer();
        while (globaltimer() - t0 < 50000000ull) __nanosleep(1000);  // 50 ms: any copy has landed
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12)
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
