// Attention over the 8-bit key/value cache for few query rows a kv head (decode steps), and the
// entry point.
//
// Per query row (a token and head) and cached token j, in powers of two with c = scale log2(e):
//   s_j = c q . k_j,  m = max s,  p_j = 2^(s_j - m),  out = sum p_j v_j / sum p_j,
// kept as a running (m, l = sum p, o = sum p v) that is rescaled when m grows.
//
// Every cached code is read once from DRAM and used by the group's few rows, so the codes' bytes
// bound the kernel: 2 dim a token and kv head. The arithmetic has to fit beside them, at f32's
// accuracy, since f32 is what the GEMVs hand over:
//   * q . k runs on the integer tensor core with no rounding at all: each query row is scaled to
//     integers of 24 bits and split into three signed base-256 digits, and mma.m16n8k32
//     multiplies digits and codes into int32. With up to 8 rows the lower half of the 16-row A
//     tile takes a row's second digit. (Two digits, 16 bits, would do for a 16-bit output but not
//     for its f32 lse: 1e-5 off.)
//   * p v runs as mma.m16n8k16 on f16: p, times the block's value scale relative to a power of
//     two of the row's, is split into two f16 (22 bits; the second in the A tile's lower half), the
//     codes are exact in f16. The tensor core truncates its sums, so each step starts from zero and
//     is added to o in f32 on the FMA pipe, together with the rescale. m is rounded up to a whole
//     number, and the row's power of two, 2^big, is that of the largest p vs among the tokens that
//     the row has seen, so both rescales are exact. (A p vs below 2^-37 of the row's largest falls
//     out of f16's range and counts as 0; a block that a row does not see, or gives no weight,
//     takes nothing from the others, whatever its scale.)
//
// A step of one warp is G groups of 16 tokens (kv_cache.cuh), each one bulk copy into the warp's
// ring, issued by the warp itself three steps ahead. Two groups share a step's softmax and its o
// update: 370 instructions for 16 tokens of 128 dims in place of 475 with one. The four warps of
// a CTA take consecutive steps and keep their own (m, l, o): they meet only when a row tile's
// tokens end. The tokens of all sequences and kv heads form one line of units of four steps, cut
// into equal parts, one a CTA, whatever the lengths (which only the device knows): a part that
// holds a piece of a row tile leaves (m, l, o) in the workspace, and of every JOIN pieces the one
// that arrives last adds all of them in the order of the line, so the result does not depend on
// which one that is.
//
// Measured, 8 kv heads of 128 dims: 64 sequences of 500 to 9000 tokens (32 query heads, f32, 0.59
// GB of codes) take 128 to 133 us, 4.4 to 4.6 TB/s of codes; one of 131,071 tokens (64 query heads,
// bf16, 0.27 GB) 64.5 us; one of 700 tokens (32, f32) 10 us. Long contexts are bound by the latency
// of a step's 736 instructions, which depend on one another and of which two warps a sub-partition
// issue 0.42 a clock (1.8 of an instruction's 4.2 clocks wait for the one before), short row tiles
// also by their starts and ends, where the warps meet at barriers.
#include "kv_attn.cuh"
#include "ptx.cuh"

#include <cuda_bf16.h>

#include <cstdlib>

namespace jkb {

namespace {

constexpr int NW = 4;        // warps of a CTA
// CTAs an SM: 8 warps of up to 255 registers. 12 warps of 168 were 3% faster over long ragged
// contexts and 15 to 30% slower where row tiles are short or split over many CTAs.
constexpr int DEC_CTAS = 2;

constexpr int ND = 3;                  // digits of a query element

template <int DT_, int ROWS_>
struct DecCfg {
    static constexpr int DT = DT_;      // 32-element chunks of a head
    static constexpr int ROWS = ROWS_;  // 8: two digits share an MMA; 16: one each
    static constexpr int DIM = 32 * DT;
    static constexpr int G = DT <= 4 ? 2 : 1;     // groups a step (registers and shared memory)
    static constexpr int STAGES = 3;
    static constexpr int STEP = G * KV_GROUP;     // tokens of a step
    static constexpr int UNIT = NW * STEP;        // of a unit
    static constexpr int BATCH = 32 / G;          // steps that are looked up together
    static constexpr int GROUP_BYTES = 32 * DIM;
    static constexpr int PASSES = ROWS * DIM > 1024 ? 4 : 2;
    static constexpr int PASS = DIM / PASSES;  // dims merged at a time
};

template <int G>
struct StepInfo {
    float2 sc[G];     // (ks, vs)
    uint32_t src[G];  // the groups' numbers in the cache, + 1; 0: no visible token in it
    int seq, item;    // item: kv head * row tiles + row tile
    int t0;           // first token (a multiple of 16), and the flags
};
// FIRST / LAST step of this CTA's piece of a row tile, the piece is the WHOLE tile
enum { STEP_FIRST = 1, STEP_LAST = 2, STEP_WHOLE = 4, STEP_FLAGS = 15 };

template <class C>
struct DecSmem {
    alignas(128) uint8_t ring[NW][C::STAGES][C::G * C::GROUP_BYTES];
    union {
        alignas(16) float merge[NW][C::ROWS][C::PASS + 4];  // while a piece ends
        alignas(16) uint8_t digits[C::ROWS][ND][C::DIM + 32];  // while one begins (+ 32: banks)
    };
    float row_m[NW][C::ROWS], row_l[NW][C::ROWS];
    float unit[C::ROWS];
    StepInfo<C::G> info[NW][2 * C::BATCH];
    uint64_t full[NW][C::STAGES];
    long long warp_sum[NW];
    int abort_flag, is_last;
};

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                       uint32_t a3, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// c = a b (FIRST) or c += a b
template <bool FIRST>
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
    if (FIRST)
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint64_t pkf(float a, float b) {
    return pk2(__float_as_uint(a), __float_as_uint(b));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Value bytes (code + 128) of tokens 2t, 2t + 1 (lo) and 2t + 8, 2t + 9 (hi) as f16 codes:
// 0x6400 | byte is 1024 + byte.
__device__ __forceinline__ void value_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const uint32_t magic = 0x64646464u;
    const __half2 off = __float2half2_rn(1152.0f);
    uint32_t a = __byte_perm(w, magic, 0x4140), b = __byte_perm(w, magic, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2 *>(&a), off);
    const __half2 y = __hsub2(*reinterpret_cast<__half2 *>(&b), off);
    lo = *reinterpret_cast<const uint32_t *>(&x);
    hi = *reinterpret_cast<const uint32_t *>(&y);
}
// (a, b) as f16 pairs hi + lo, hi = f16(x), lo = f16(x - hi)
__device__ __forceinline__ void split_f16(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// Elements i .. i + 3 of the query rows.
__device__ __forceinline__ float4 load4(const AttnParams &p, int type, size_t i) {
    if (type == JKB_F32) {
        const float *q = static_cast<const float *>(p.q) + i;
        if (p.q_vec) return __ldg(reinterpret_cast<const float4 *>(q));
        return make_float4(__ldg(q), __ldg(q + 1), __ldg(q + 2), __ldg(q + 3));
    }
    const uint16_t *q = static_cast<const uint16_t *>(p.q) + i;
    uint2 w;
    if (p.q_vec) {
        w = __ldg(reinterpret_cast<const uint2 *>(q));
    } else {
        w.x = __ldg(q) | (uint32_t)__ldg(q + 1) << 16;
        w.y = __ldg(q + 2) | (uint32_t)__ldg(q + 3) << 16;
    }
    if (type == JKB_F16) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u),
                       __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u));
}

// Four output elements.
__device__ __forceinline__ void store4(const AttnParams &p, int type, size_t i, float4 v) {
    if (type == JKB_F32) {
        float *o = static_cast<float *>(p.out) + i;
        if (p.out_vec) {
            *reinterpret_cast<float4 *>(o) = v;
        } else {
            o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
        }
        return;
    }
    uint32_t a, b;
    if (type == JKB_F16) {
        const __half2 x = __floats2half2_rn(v.x, v.y), y = __floats2half2_rn(v.z, v.w);
        a = *reinterpret_cast<const uint32_t *>(&x), b = *reinterpret_cast<const uint32_t *>(&y);
    } else {
        const __nv_bfloat162 x = __floats2bfloat162_rn(v.x, v.y);
        const __nv_bfloat162 y = __floats2bfloat162_rn(v.z, v.w);
        a = *reinterpret_cast<const uint32_t *>(&x), b = *reinterpret_cast<const uint32_t *>(&y);
    }
    uint16_t *o = static_cast<uint16_t *>(p.out) + i;
    if (p.out_vec) {
        *reinterpret_cast<uint2 *>(o) = make_uint2(a, b);
    } else {
        o[0] = (uint16_t)a, o[1] = (uint16_t)(a >> 16), o[2] = (uint16_t)b;
        o[3] = (uint16_t)(b >> 16);
    }
}

// A query row is held as integers |n| < 127 * (65536 + 256 + 1) in three signed base-256 digits,
// x = unit / 65536 * n: the bytes of (n + 0x808080) ^ 0x808080. MOST leaves room for the rounding of
// n. A power of two brings the row's largest element near 1 before MOST is divided by it, so that
// rows of any finite size have their 24 bits; the 65536, which the scores put back, keeps unit a
// normal number for rows down to 2^-119 / scale (below, it has fewer bits). A row with a non-finite
// element has unit NaN, so that its output is NaN.
constexpr float MOST = 8355700.0f;

// Units of one sequence and its row tiles.
template <class C>
__device__ __forceinline__ void seq_units(const AttnParams &p, const AttnSeq &s, int &tiles,
                                          int &first_unit, int &units) {
    tiles = (int)(((long long)s.nq * p.group + C::ROWS - 1) / C::ROWS);
    first_unit = s.lo / C::UNIT;
    units = max(1, (s.len + C::UNIT - 1) / C::UNIT - first_unit);
}

template <class C>
__global__ void __launch_bounds__(32 * NW, DEC_CTAS)
    attn_decode_kernel(const __grid_constant__ AttnParams p, const int type) {
    constexpr int ROWS = C::ROWS, DT = C::DT, DIM = C::DIM, STAGES = C::STAGES;
    constexpr int RH = ROWS / 8;  // rows of a thread
    constexpr int G = C::G, BATCH = C::BATCH;
    extern __shared__ uint8_t smem_raw[];
    DecSmem<C> &sm =
        *reinterpret_cast<DecSmem<C> *>((((uintptr_t)smem_raw) + 127) & ~(uintptr_t)127);
    long long *prefix = reinterpret_cast<long long *>(&sm + 1);  // [n_seqs + 1] first units
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tg = lane & 3;

    if (tid == 0) sm.abort_flag = 0;
    if (lane == 0)
        for (int s = 0; s < STAGES; s++) mbar_init(&sm.full[warp][s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" :::);

    // ---- the line of units: exclusive sums over the sequences ----
    {
        const int per = (p.n_seqs + 32 * NW - 1) / (32 * NW);
        const int a = min(tid * per, p.n_seqs), b = min(a + per, p.n_seqs);
        long long sum = 0;
        for (int i = a; i < b; i++) {
            int tiles, first, units;
            seq_units<C>(p, attn_seq(p, i), tiles, first, units);
            sum += (long long)p.kv_heads * tiles * units;
        }
        long long inc = sum;
        for (int d = 1; d < 32; d <<= 1) {
            const long long x = __shfl_up_sync(~0u, inc, d);
            if (lane >= d) inc += x;
        }
        if (lane == 31) sm.warp_sum[warp] = inc;
        __syncthreads();
        long long at = inc - sum;
        for (int w = 0; w < warp; w++) at += sm.warp_sum[w];
        for (int i = a; i < b; i++) {
            int tiles, first, units;
            seq_units<C>(p, attn_seq(p, i), tiles, first, units);
            prefix[i] = at;
            at += (long long)p.kv_heads * tiles * units;
        }
        if (tid == 32 * NW - 1) prefix[p.n_seqs] = at;
        __syncthreads();
    }
    const long long total = prefix[p.n_seqs];
    const long long per = (total + gridDim.x - 1) / gridDim.x;
    const long long u0 = min(per * blockIdx.x, total), u1 = min(u0 + per, total);
    const int steps = (int)min(u1 - u0, (long long)INT32_MAX);
    if (steps == 0) return;

    // Starts the copies of a step (lane 0, by predicate: a branch would cost the warp its turn)
    auto issue = [&](int s, const uint32_t (&src)[2]) {
        const int n = (src[0] != 0) + (G > 1 && src[1] != 0);
        const uint32_t bar = smem_u32(&sm.full[warp][s % STAGES]);
        const uint32_t dst = smem_u32(sm.ring[warp][s % STAGES]);
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t"
            "@p mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
            "r"(n * C::GROUP_BYTES), "r"((uint32_t)(lane == 0 && n))
            : "memory");
#pragma unroll
        for (int i = 0; i < G; i++)
            asm volatile(
                "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                "@p cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes "
                "[%0], [%1], %2, [%3];\n\t}" ::"r"(dst + i * C::GROUP_BYTES),
                "l"(p.codes + (size_t)(src[i] - 1) * C::GROUP_BYTES), "r"(C::GROUP_BYTES),
                "r"(bar), "r"((uint32_t)(lane == 0 && src[i]))
                : "memory");
    };
    // Lookups of BATCH steps at a time (lane i: group i % G of step base + i / G), each in three
    // stages several steps apart, since each waits for a load of the one before, microseconds
    // where the memory is busy: which token, and its table entry; its place and scales; the
    // step's entry in info[].
    struct Look {
        int id, at;      // block id, token
        int head;        // kv head; -1: no visible token
        int seq, item, t0;
    };
    auto find = [&](int base) {
        Look f;
        f.id = f.head = -1;
        f.at = f.seq = f.item = f.t0 = 0;
        const long long u = u0 + base + lane / G;
        if (u >= u1) return f;
        int a = 0, b = p.n_seqs - 1;  // the last sequence that starts at or before u
        while (a < b) {
            const int mid = (a + b + 1) >> 1;
            if (prefix[mid] <= u) a = mid;
            else b = mid - 1;
        }
        const AttnSeq s = attn_seq(p, a);
        int tiles, first, units;
        seq_units<C>(p, s, tiles, first, units);
        const long long local = u - prefix[a];
        f.seq = a;
        f.item = (int)(local / units);
        f.head = f.item / tiles;
        const int c = (int)(local - (long long)f.item * units);
        const long long start = u - c;
        f.t0 = (first + c) * C::UNIT + warp * C::STEP;
        f.at = f.t0 + lane % G * KV_GROUP;
        f.t0 |= (c == 0 || u == u0 ? STEP_FIRST : 0) |
                (c == units - 1 || u == u1 - 1 ? STEP_LAST : 0) |
                (start >= u0 && start + units <= u1 ? STEP_WHOLE : 0);
        // the query rows of a piece that starts here, on their way to the L1
        if (f.t0 & STEP_FIRST && warp == 0 && lane % G == 0) {
            const int rows = min(ROWS, s.nq * p.group - (f.item - f.head * tiles) * ROWS);
            for (int r = 0; r < rows; r++) {
                const int row = (f.item - f.head * tiles) * ROWS + r, tok = row / p.group;
                const size_t bytes = type == JKB_F32 ? 4 : 2;
                const char *q = (const char *)p.q +
                                ((size_t)(s.q0 + tok) * p.q_token +
                                 (size_t)(f.head * p.group + row - tok * p.group) * p.q_head) *
                                    bytes;
                for (size_t d = 0; d < p.dim * bytes; d += 128)
                    asm volatile("prefetch.global.L1 [%0];" ::"l"(q + d));
            }
        }
        if (f.at < s.len && f.at + KV_GROUP > s.lo)
            f.id = __ldg(p.table + (size_t)a * p.table_stride + (f.at >> p.log_block));
        else
            f.head = -1;
        return f;
    };
    auto place = [&](const Look &f, float2 &sc) {  // the group's number in the cache, + 1; 0: none
        sc = make_float2(0.f, 0.f);
        if (f.head < 0) return 0u;
        if (f.id < 0 || f.id >= p.n_blocks) {
            atomicOr(p.err, ERR_KV_RANGE);
            return 0u;
        }
        const size_t bh = (size_t)f.id * p.kv_heads + f.head;
        sc = __ldg(p.scales + bh);
        return (uint32_t)(((bh << p.log_block) | (f.at & ((1 << p.log_block) - 1))) / KV_GROUP) +
               1;
    };
    auto enter = [&](int base, const Look &f, uint32_t src, float2 sc) {
        __syncwarp();
        StepInfo<G> &i = sm.info[warp][(base + lane / G) % (2 * BATCH)];
        i.src[lane % G] = src;
        i.sc[lane % G] = sc;
        if (lane % G == 0) {
            i.seq = f.seq;
            i.item = f.item;
            i.t0 = f.t0;
        }
        __syncwarp();
    };

    // ---- running state of the current row tile ----
    uint32_t qa[ND][DT][2 * RH];  // A registers of each digit
    float m[RH], l[RH], unit[RH];
    float big[RH];  // o is in units of 2^(big - 14)
    int lo[RH], hi[RH], all_lo = 0, all_hi = 0;  // tokens that the rows see; that all see
    uint64_t o[RH][DT][4];  // pairs: dims 32 c + 8 tg + j and + 4 + j of row g (+ 8)
    bool dead = false;
    uint32_t phases = 0;

    Look look = find(0);
    float2 look_sc;
    uint32_t look_src = place(look, look_sc);
    {   // the first copies start before their scales are there
        uint32_t src[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < STAGES; k++) {
#pragma unroll
            for (int i = 0; i < G; i++) src[i] = __shfl_sync(~0u, look_src, G * k + i);
            if (k < steps) issue(k, src);
        }
    }
    enter(0, look, look_src, look_sc);
    for (int s = 0; s < steps; s++) {
        const int phase = s % BATCH;
        if (phase == 0) look = find(s + BATCH);
        if (phase == BATCH / 2 - 2) look_src = place(look, look_sc);
        if (phase == BATCH - STAGES - 1) enter(s - phase + BATCH, look, look_src, look_sc);
        StepInfo<G> f = sm.info[warp][s % (2 * BATCH)];
        const int flags = f.t0 & STEP_FLAGS;
        f.t0 &= ~STEP_FLAGS;
        const bool any = f.src[0] || (G > 1 && f.src[G - 1]);
        // (past the last step nothing is looked up, and nothing copied)
        const uint32_t next_src[2] = {sm.info[warp][(s + STAGES) % (2 * BATCH)].src[0],
                                      sm.info[warp][(s + STAGES) % (2 * BATCH)].src[G - 1]};

        if (flags & STEP_FIRST) {
            const AttnSeq q = attn_seq(p, f.seq);
            const int tiles = (int)(((long long)q.nq * p.group + ROWS - 1) / ROWS);
            const int head = f.item / tiles, tile = f.item - head * tiles;
            // each warp brings its share of the rows into digits, for all
            constexpr int DL = (DIM + 127) / 128;  // 4-element pieces of a lane
#pragma unroll 2
            for (int r = warp; r < ROWS; r += NW) {
                const int row = tile * ROWS + r, tok = row / p.group;
                const size_t at = (size_t)(q.q0 + tok) * p.q_token +
                                  (size_t)(head * p.group + row - tok * p.group) * p.q_head;
                float4 x[DL];
                uint32_t top = 0;  // as bits: a NaN is above an infinity is above the rest
#pragma unroll
                for (int k = 0; k < DL; k++) {
                    const int d = 128 * k + 4 * lane;
                    x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (tok < q.nq && d < p.dim) x[k] = load4(p, type, at + d);
                    const uint32_t a = max(__float_as_uint(x[k].x) & 0x7FFFFFFFu,
                                           __float_as_uint(x[k].y) & 0x7FFFFFFFu);
                    const uint32_t b = max(__float_as_uint(x[k].z) & 0x7FFFFFFFu,
                                           __float_as_uint(x[k].w) & 0x7FFFFFFFu);
                    top = max(top, max(a, b));
                }
                top = __reduce_max_sync(~0u, top);
                const bool finite = top < 0x7F800000u;
                const float amax = __uint_as_float(top);
                const float up = __uint_as_float(min(255 - (top >> 23), 254u) << 23);
                const float inv = finite && top ? __fdividef(MOST, amax * up) : 0.0f;
#pragma unroll
                for (int k = 0; k < DL; k++) {
                    const int d = 128 * k + 4 * lane;
                    if (DIM % 128 && d >= DIM) break;
                    uint32_t w[4];
                    w[0] = (uint32_t)(__float2int_rn(x[k].x * up * inv) + 0x808080) ^ 0x808080u;
                    w[1] = (uint32_t)(__float2int_rn(x[k].y * up * inv) + 0x808080) ^ 0x808080u;
                    w[2] = (uint32_t)(__float2int_rn(x[k].z * up * inv) + 0x808080) ^ 0x808080u;
                    w[3] = (uint32_t)(__float2int_rn(x[k].w * up * inv) + 0x808080) ^ 0x808080u;
                    const uint32_t a = __byte_perm(w[0], w[1], 0x5140);
                    const uint32_t b = __byte_perm(w[2], w[3], 0x5140);
                    *reinterpret_cast<uint32_t *>(&sm.digits[r][2][d]) =
                        __byte_perm(a, b, 0x5410);
                    *reinterpret_cast<uint32_t *>(&sm.digits[r][1][d]) =
                        __byte_perm(a, b, 0x7632);
                    *reinterpret_cast<uint32_t *>(&sm.digits[r][0][d]) =
                        __byte_perm(__byte_perm(w[0], w[1], 0x0062),
                                    __byte_perm(w[2], w[3], 0x0062), 0x5410);
                }
                if (lane == 0) {
                    constexpr float C65536 = 65536.0f / MOST;
                    sm.unit[r] = !finite       ? __int_as_float(0x7FC00000)
                                 : amax > 1.0f ? amax * C65536 * p.scale2
                                               : amax * (C65536 * p.scale2);
                }
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < RH; r++) {
#pragma unroll
                for (int k = 0; k < ND; k++)
#pragma unroll
                    for (int c = 0; c < DT; c++) {
                        const uint2 w = *reinterpret_cast<const uint2 *>(
                            &sm.digits[g + 8 * r][k][32 * c + 8 * tg]);
                        qa[k][c][2 * r] = w.x;
                        qa[k][c][2 * r + 1] = w.y;
                    }
                unit[r] = sm.unit[g + 8 * r];
                const int tok = (tile * ROWS + g + 8 * r) / p.group;
                const bool on = tok < q.nq;
                const int pos = q.len - q.nq + tok;
                hi[r] = !on ? 0 : p.causal ? min(q.len, pos + 1) : q.len;
                lo[r] = first_seen(p, pos);
                m[r] = big[r] = -INFINITY;
                l[r] = 0.0f;
#pragma unroll
                for (int c = 0; c < DT; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[r][c][i] = 0;
            }
            const int last = min((tile + 1) * ROWS, q.nq * p.group) - 1;  // of the tile's rows
            const int pos_a = q.len - q.nq + tile * ROWS / p.group;
            const int pos_b = q.len - q.nq + last / p.group;
            all_hi = p.causal ? min(q.len, pos_a + 1) : q.len;
            all_lo = first_seen(p, pos_b);
        }

        if (any) {
            const int st = s % STAGES;
            // (each lane polls for itself; all go on, or none: what follows takes whole warps)
            if (!dead)
                dead = !__all_sync(~0u, mbar_wait(&sm.full[warp][st], (phases >> st) & 1,
                                                  &sm.abort_flag, p.err, ERR_ATTN_WAIT));
            if (!dead) phases ^= 1u << st;
        }
        if (any && !dead) {
            const uint8_t *stage = sm.ring[warp][s % STAGES];
            // ---- scores: tokens t0 + 16 i + 8 nt + 2 tg + e of rows g (+ 8) ----
            // (chunks of dims outside, so that an MMA's accumulator comes up again only after
            // those of the other tokens and digits)
            float sc[RH][4 * G];
            int acc[G][2][ND][4] = {};
#pragma unroll
            for (int c = 0; c < DT; c++)
#pragma unroll
                for (int i = 0; i < G; i++)
#pragma unroll
                    for (int nt = 0; nt < 2; nt++) {
                        const uint2 b = *reinterpret_cast<const uint2 *>(
                            stage + i * C::GROUP_BYTES + nt * 8 * DIM + c * 256 + lane * 8);
                        if (RH == 1) {
                            mma_s8(acc[i][nt][0], qa[0][c][0], qa[1][c][0], qa[0][c][1],
                                   qa[1][c][1], b.x, b.y);
                            mma_s8(acc[i][nt][2], qa[2][c][0], 0u, qa[2][c][1], 0u, b.x, b.y);
                        } else {
#pragma unroll
                            for (int k = 0; k < ND; k++)
                                mma_s8(acc[i][nt][k], qa[k][c][0], qa[k][c][2 * RH - 2],
                                       qa[k][c][1], qa[k][c][2 * RH - 1], b.x, b.y);
                        }
                    }
#pragma unroll
            for (int r = 0; r < RH; r++)
#pragma unroll
                for (int i = 0; i < G; i++) {
                    const float f_row = unit[r] * f.sc[i].x;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int(&a)[ND][4] = acc[i][k / 2];
                        const int e = k % 2;
                        const int d0 = RH == 1 ? a[0][e] : a[0][2 * r + e];
                        const int d1 = RH == 1 ? a[0][2 + e] : a[1][2 * r + e];
                        const int d2 = RH == 1 ? a[2][e] : a[2][2 * r + e];
                        sc[r][4 * i + k] =
                            fmaf((float)(d1 * 256 + d2), 1.0f / 65536.0f, (float)d0) * f_row;
                    }
                }
            if (f.t0 < all_lo || f.t0 + C::STEP > all_hi || (G > 1 && !(f.src[0] && f.src[G - 1]))) {
#pragma unroll
                for (int r = 0; r < RH; r++)
#pragma unroll
                    for (int k = 0; k < 4 * G; k++) {
                        const int t = f.t0 + 16 * (k / 4) + 8 * (k / 2 % 2) + 2 * tg + k % 2;
                        if (t < lo[r] || t >= hi[r] || !f.src[k / 4]) sc[r][k] = -INFINITY;
                    }
            }
            // ---- the blocks' value scales: vs = mant * 2^e ----
            float mant[G], e[G];
#pragma unroll
            for (int i = 0; i < G; i++) {
                const uint32_t vb = __float_as_uint(f.sc[i].y);
                e[i] = (float)((int)((vb >> 23) & 255) - 126);
                mant[i] = (vb & 0x7F800000u) ? __uint_as_float((vb & 0x807FFFFFu) | 0x3F000000u)
                                             : 0.0f;
            }
            // ---- softmax step ----
            uint32_t ph[RH][G][2], pl[RH][G][2];
            uint64_t alpha[RH];
#pragma unroll
            for (int r = 0; r < RH; r++) {
                float top[G], mn = m[r];
#pragma unroll
                for (int i = 0; i < G; i++) {
                    const float *x = sc[r] + 4 * i;
                    top[i] = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                    top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 1));
                    top[i] = ceilf(fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 2)));
                    mn = fmaxf(mn, top[i]);
                }
                const float ref = mn == -INFINITY ? 0.0f : mn;
                const float a = ex2(m[r] - ref);
                m[r] = mn;
                float bn = big[r];
#pragma unroll
                for (int i = 0; i < G; i++)  // (weights below 2^-112 count as 0)
                    if (top[i] >= ref - 112.0f) bn = fmaxf(bn, top[i] + e[i]);
                const float bref = bn == -INFINITY ? 0.0f : bn, shift = ex2(big[r] - bref);
                big[r] = bn;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < G; i++) {
                    // at most 2^126, where the weights are below 2^-112
                    const float vmul =
                        top[i] >= ref - 112.0f ? mant[i] * ex2(ref - bref + e[i] + 14.0f) : 0.0f;
                    float w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) w[k] = ex2(sc[r][4 * i + k] - ref);
                    sum += (w[0] + w[1]) + (w[2] + w[3]);
                    split_f16(w[0] * vmul, w[1] * vmul, ph[r][i][0], pl[r][i][0]);
                    split_f16(w[2] * vmul, w[3] * vmul, ph[r][i][1], pl[r][i][1]);
                }
                l[r] = fmaf(l[r], a, sum);
                alpha[r] = pkf(shift, shift);
            }
            // ---- o = o * alpha + p v ----
#pragma unroll
            for (int c = 0; c < DT; c++) {
                uint32_t vw[G][4];
#pragma unroll
                for (int i = 0; i < G; i++) {
                    const uint4 v4 = *reinterpret_cast<const uint4 *>(
                        stage + i * C::GROUP_BYTES + 16 * DIM + c * 512 +
                        (tg * 8 + (g ^ (2 * tg))) * 16);
                    vw[i][0] = v4.x, vw[i][1] = v4.y, vw[i][2] = v4.z, vw[i][3] = v4.w;
                }
                uint32_t b[G][4][2];
#pragma unroll
                for (int i = 0; i < G; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) value_f16(vw[i][j], b[i][j][0], b[i][j][1]);
                float d[4][4];
                if (RH == 1) {  // rows g: high parts, rows g + 8: low parts
#pragma unroll
                    for (int i = 0; i < G; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            if (i == 0)
                                mma_f16<true>(d[j], ph[0][i][0], pl[0][i][0], ph[0][i][1],
                                              pl[0][i][1], b[i][j][0], b[i][j][1]);
                            else
                                mma_f16<false>(d[j], ph[0][i][0], pl[0][i][0], ph[0][i][1],
                                               pl[0][i][1], b[i][j][0], b[i][j][1]);
                        }
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        o[0][c][j] = fma2(o[0][c][j], alpha[0],
                                          add2(pkf(d[j][0], d[j][1]), pkf(d[j][2], d[j][3])));
                } else {
#pragma unroll
                    for (int i = 0; i < G; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            if (i == 0)
                                mma_f16<true>(d[j], pl[0][i][0], pl[RH - 1][i][0], pl[0][i][1],
                                              pl[RH - 1][i][1], b[i][j][0], b[i][j][1]);
                            else
                                mma_f16<false>(d[j], pl[0][i][0], pl[RH - 1][i][0], pl[0][i][1],
                                               pl[RH - 1][i][1], b[i][j][0], b[i][j][1]);
                        }
#pragma unroll
                    for (int i = 0; i < G; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            mma_f16<false>(d[j], ph[0][i][0], ph[RH - 1][i][0], ph[0][i][1],
                                           ph[RH - 1][i][1], b[i][j][0], b[i][j][1]);
#pragma unroll
                    for (int r = 0; r < RH; r++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            o[r][c][j] =
                                fma2(o[r][c][j], alpha[r], pkf(d[j][2 * r], d[j][2 * r + 1]));
                }
            }
        }
        __syncwarp();
        // (a barrier whose phase did not end must not be armed again)
        if (s + STAGES < steps && !dead) issue(s + STAGES, next_src);

        if (!(flags & STEP_LAST)) continue;
        // ---- the piece ends: the warps' (m, l, o) into one ----
        const AttnSeq q = attn_seq(p, f.seq);
        int tiles, first, units;
        seq_units<C>(p, q, tiles, first, units);
        const int head = f.item / tiles, tile = f.item - head * tiles;
#pragma unroll
        for (int r = 0; r < RH; r++) {
            float sum = l[r];
            sum += __shfl_xor_sync(~0u, sum, 1);
            sum += __shfl_xor_sync(~0u, sum, 2);
            if (tg == 0) {
                sm.row_m[warp][g + 8 * r] = m[r];
                sm.row_l[warp][g + 8 * r] = sum;
            }
        }
        __syncthreads();
        float mul[RH];
#pragma unroll
        for (int r = 0; r < RH; r++) {
            float top = -INFINITY;
            for (int w = 0; w < NW; w++) top = fmaxf(top, sm.row_m[w][g + 8 * r]);
            if (top == -INFINITY) top = 0.0f;
            if (tg == 0) sm.row_l[warp][g + 8 * r] *= ex2(m[r] - top);
            mul[r] = ex2(big[r] - 14.0f - top);
        }
        // where this piece's sums go: the output, or its slot in the workspace
        const bool whole = flags & STEP_WHOLE;
        const int rows = min(ROWS, q.nq * p.group - tile * ROWS);
        int cta0 = 0, cta1 = 0;  // that have a piece of this row tile
        const long long start = prefix[f.seq] + (long long)f.item * units;
        if (!whole) {
            cta0 = (int)(start / per);
            cta1 = (int)((start + units - 1) / per);
        }
        auto slot_of = [&](int cta) {
            const int slot = 2 * cta + (cta == cta0 && start != per * cta0 ? 1 : 0);
            return p.partial + (size_t)slot * ROWS * (DIM + 2);
        };
        float *mine = whole ? nullptr : slot_of((int)blockIdx.x);
        auto finish = [&](int row, int d, float4 v, float top, float sum) {
            const int rr = tile * ROWS + row, tok = rr / p.group;
            if (d >= p.dim) return;
            const int h = head * p.group + rr - tok * p.group;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            store4(p, type, (size_t)(q.q0 + tok) * p.out_token + (size_t)h * p.out_head + d,
                   make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
            if (d == 0 && p.lse)
                p.lse[(size_t)(q.q0 + tok) * p.group * p.kv_heads + h] =
                    (top + log2f(sum)) * 0.69314718055994531f;
        };
#pragma unroll
        for (int pass = 0; pass < C::PASSES; pass++) {
#pragma unroll
            for (int c = 0; c < DT; c++) {
#pragma unroll
                for (int r = 0; r < RH; r++) {
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const int d = 32 * c + 8 * tg + 4 * k - pass * C::PASS;
                        if (d >= 0 && d < C::PASS && g + 8 * r < rows) {
                            float x[4];
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                float u, w;
                                upk2(o[r][c][j], u, w);
                                x[j] = (k ? w : u) * mul[r];
                            }
                            const float4 v = make_float4(x[0], x[1], x[2], x[3]);
                            *reinterpret_cast<float4 *>(&sm.merge[warp][g + 8 * r][d]) = v;
                        }
                    }
                }
            }
            __syncthreads();
            for (int i = tid; i < rows * C::PASS / 4; i += 32 * NW) {
                const int row = i / (C::PASS / 4), d = 4 * (i - row * (C::PASS / 4));
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                float top = -INFINITY, sum = 0.0f;
                for (int w = 0; w < NW; w++) {
                    top = fmaxf(top, sm.row_m[w][row]);
                    const float4 x = *reinterpret_cast<const float4 *>(&sm.merge[w][row][d]);
                    v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
                    sum += sm.row_l[w][row];
                }
                const int dd = d + pass * C::PASS;
                if (whole) {
                    finish(row, dd, v, top, sum);
                } else {
                    *reinterpret_cast<float4 *>(mine + row * DIM + dd) = v;
                    if (dd == 0) {
                        mine[ROWS * DIM + row] = top;
                        mine[ROWS * DIM + ROWS + row] = sum;
                    }
                }
            }
            __syncthreads();
        }
        if (whole) continue;
        // ---- JOIN pieces into one at a time: the last of them to arrive does, in order ----
        const int n = cta1 - cta0 + 1;
        int at = (int)blockIdx.x - cta0;  // this CTA has the sum of pieces at .. at + span - 1
        for (int span = 1, level = 0; span < n; span *= JOIN, level++) {
            at -= at % (span * JOIN);
            const int cnt = min(JOIN, (n - at + span - 1) / span);
            if (cnt == 1) continue;
            // (pieces follow in the next CTA too, so no other row tile counts here)
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                int *counter = p.counters + level * gridDim.x + cta0 + at;
                sm.is_last = atomicAdd(counter, 1) == cnt - 1;
                if (sm.is_last) *counter = 0;
            }
            __syncthreads();
            if (!sm.is_last) break;
            __threadfence();
            const bool all = cnt * span >= n;  // (so at == 0)
            float *into = slot_of(cta0 + at);
            for (int i = tid; i < rows * DIM / 4; i += 32 * NW) {
                const int row = i / (DIM / 4), d = 4 * (i - row * (DIM / 4));
                constexpr int NC = 8;  // loads in flight together
                static_assert(JOIN % NC == 0, "");
                float top = -INFINITY, sum = 0.0f;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                for (int c0 = 0; c0 < cnt; c0 += NC) {
                    float m_in[NC], l_in[NC];
                    float4 v_in[NC];
#pragma unroll
                    for (int k = 0; k < NC; k++) {
                        const float *slot = slot_of(cta0 + at + min(c0 + k, cnt - 1) * span);
                        m_in[k] = __ldcg(slot + ROWS * DIM + row);
                        l_in[k] = __ldcg(slot + ROWS * DIM + ROWS + row);
                        v_in[k] = __ldcg(reinterpret_cast<const float4 *>(slot + row * DIM + d));
                    }
                    float mn = top;
#pragma unroll
                    for (int k = 0; k < NC; k++) mn = fmaxf(mn, m_in[k]);
                    const float ref = mn == -INFINITY ? 0.0f : mn;
                    const float a = ex2(top - ref);
                    top = mn;
                    sum *= a;
                    v.x *= a, v.y *= a, v.z *= a, v.w *= a;
#pragma unroll
                    for (int k = 0; k < NC; k++) {
                        if (c0 + k >= cnt) continue;
                        const float w = ex2(m_in[k] - ref);
                        sum = fmaf(w, l_in[k], sum);
                        v.x = fmaf(w, v_in[k].x, v.x);
                        v.y = fmaf(w, v_in[k].y, v.y);
                        v.z = fmaf(w, v_in[k].z, v.z);
                        v.w = fmaf(w, v_in[k].w, v.w);
                    }
                }
                if (all) {
                    finish(row, d, v, top, sum);
                } else {
                    *reinterpret_cast<float4 *>(into + row * DIM + d) = v;
                    if (d == 0) sm.row_m[0][row] = top, sm.row_l[0][row] = sum;
                }
            }
            __syncthreads();
            if (!all && tid < rows) {  // after every thread has read the pieces' own
                into[ROWS * DIM + tid] = sm.row_m[0][tid];
                into[ROWS * DIM + ROWS + tid] = sm.row_l[0][tid];
            }
        }
        __syncthreads();
    }
    if (dead && lane == 0) {  // copies still in flight must land before the CTA's memory goes
        for (int s = 0; s < STAGES; s++) {
            const unsigned long long t0 = globaltimer();
            while (!mbar_try(&sm.full[warp][s], (phases >> s) & 1) &&
                   globaltimer() - t0 < WAIT_NS / 8) {
            }
        }
    }
}

template <class C>
constexpr bool dec_fits() {  // DEC_CTAS an SM, for up to 200 sequences (beyond, one may)
    return DEC_CTAS * (sizeof(DecSmem<C>) + 128 + 8 * 201 + 1024) <= 228 * 1024;
}

template <class C>
int launch_cfg(const AttnParams &p, int type, cudaStream_t st) {
    static_assert(dec_fits<C>(), "");
    static const char *fn = "attention_kv8";
    constexpr size_t fixed = sizeof(DecSmem<C>) + 128;
    constexpr size_t most = fixed + 8 * ((size_t)JKB_KV_MAX_SEQS + 1);
    static_assert(most <= 227 * 1024, "shared memory");
    const size_t smem = fixed + 8 * ((size_t)p.n_seqs + 1);
    // The limit is one for all threads of the process: always the same value, so that no call
    // lowers it under another.
    static thread_local int allowed_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev != allowed_dev) {
        cudaError_t e = cudaFuncSetAttribute(attn_decode_kernel<C>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)most);
        if (e != cudaSuccess) return fail_cuda(e, fn);
        allowed_dev = dev;
    }
    cudaError_t e = launch_pdl(attn_decode_kernel<C>, dim3((unsigned)(num_sms() * DEC_CTAS)),
                               dim3(32 * NW), smem, st, p, type);
    return e == cudaSuccess ? JKB_OK : fail_cuda(e, fn);
}

template <int DT>
int launch_dim(const AttnParams &p, int type, size_t max_rows, cudaStream_t st) {
    if constexpr (DT <= 4) {  // 16 rows of a larger head do not fit the registers
        if (max_rows > 8) return launch_cfg<DecCfg<DT, 16>>(p, type, st);
    }
    return launch_cfg<DecCfg<DT, 8>>(p, type, st);
}

}  // namespace

int attn_decode_launch(const AttnParams &p, int type, int dim_p, size_t max_rows,
                       cudaStream_t st) {
    switch (dim_p) {
    case 64: return launch_dim<2>(p, type, max_rows, st);
    case 96: return launch_dim<3>(p, type, max_rows, st);
    case 128: return launch_dim<4>(p, type, max_rows, st);
    case 192: return launch_dim<6>(p, type, max_rows, st);
    default: return launch_dim<8>(p, type, max_rows, st);
    }
}

}  // namespace jkb

using namespace jkb;

extern "C" {

int jkb_attn_workspace_create(const jkb_kv_cache *cache, jkb_attn_workspace **out) {
    static const char *fn = "attn_workspace";
    if (!out) return fail(JKB_E_INVALID, fn, 0, 0, 0, "null out");
    *out = nullptr;
    int rc = check_kv_cache(cache, fn);
    if (rc) return rc;
    jkb_attn_workspace *w = (jkb_attn_workspace *)calloc(1, sizeof(jkb_attn_workspace));
    if (!w) return fail(JKB_E_INVALID, fn, 0, 0, 0, "host allocation failed");
    w->device = cache->device;
    w->dim_p = cache->dim_p;
    w->ctas = DEC_CTAS * num_sms();
    const size_t sms = (size_t)num_sms(), width = (size_t)w->dim_p + 2;
    const size_t part = Arena::round(2 * (size_t)w->ctas * ATTN_ROWS * width * sizeof(float));
    const size_t tile = w->dim_p <= 128 ? Arena::round(2 * sms * 128 * width * sizeof(float)) : 0;
    const size_t counts = JOIN_LEVELS * (w->ctas + sms) * sizeof(int);
    if (w->ctas > JOIN * JOIN * JOIN) {
        free(w);
        return fail(JKB_E_CAPABILITY, fn, 0, 0, 0, "device has too many SMs");
    }
    cudaError_t e = cudaMalloc(&w->base, part + tile + counts);
    if (e == cudaSuccess) {
        w->partial = (float *)w->base;
        w->tile_partial = tile ? (float *)(w->base + part) : nullptr;
        w->counters = (int *)(w->base + part + tile);
        w->tile_counters = w->counters + JOIN_LEVELS * w->ctas;
        e = cudaMemset(w->counters, 0, counts);
        if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
        if (e != cudaSuccess) cudaFree(w->base);
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        free(w);
        return fail_cuda(e, fn);
    }
    w->magic = ATTN_WS_MAGIC;
    *out = w;
    return JKB_OK;
}

int jkb_attn_workspace_destroy(jkb_attn_workspace *w) {
    if (!w) return JKB_OK;
    if (w->magic != ATTN_WS_MAGIC)
        return fail(JKB_E_INVALID, "attn_workspace", 0, 0, 0,
                    "null or destroyed attention workspace handle");
    w->magic = 0;
    cudaFree(w->base);
    free(w);
    return JKB_OK;
}

int jkb_attention_kv8(const jkb_attn_args *a, void *stream) {
    static const char *fn = "attention_kv8";
    if (!a) return fail(JKB_E_INVALID, fn, 0, 0, 0, "null arguments");
    int rc = check_kv_cache(a->cache, fn);
    if (rc) return rc;
    const jkb_kv_cache *c = a->cache;
    const jkb_attn_workspace *w = a->ws;
    if (!w || w->magic != ATTN_WS_MAGIC)
        return fail(JKB_E_INVALID, fn, 0, 0, 0, "null or destroyed attention workspace handle");
    if (w->device != c->device || w->dim_p != c->dim_p)
        return fail(JKB_E_INVALID, fn, 0, (size_t)w->dim_p, (size_t)c->dim_p,
                    "the workspace was made for another device or head_dim");
    if (a->n_heads == 0 || a->n_heads % c->n_heads || a->n_heads > 65535)
        return fail(JKB_E_BOUNDS, fn, 0, a->n_heads, c->n_heads,
                    "%zu query heads are not a multiple of %zu kv heads", a->n_heads, c->n_heads);
    const int type = a->q.type;
    const size_t eb = type == JKB_F32 ? 4 : type == JKB_F16 || type == JKB_BF16 ? 2 : 0;
    if (!eb || a->out.type != type)
        return fail(JKB_E_CAPABILITY, fn, 0, 0, 0,
                    "query rows of type %s and output rows of type %s: F32, F16 or BF16, both "
                    "alike",
                    quant_name(type), quant_name(a->out.type));
    if (a->n_seqs > JKB_KV_MAX_SEQS)
        return fail(JKB_E_BOUNDS, fn, 0, a->n_seqs, JKB_KV_MAX_SEQS, "%zu sequences, at most %d",
                    a->n_seqs, JKB_KV_MAX_SEQS);
    // (a tile's row numbers go up to 127 beyond the last)
    if (a->n_tokens > (size_t)(INT32_MAX - 128) / a->n_heads)
        return fail(JKB_E_BOUNDS, fn, 0, a->n_tokens, (size_t)(INT32_MAX - 128) / a->n_heads,
                    "%zu query tokens of %zu heads in one call", a->n_tokens, a->n_heads);
    if (a->row_blocks > (size_t)INT32_MAX / c->block_tokens || a->table_stride < a->row_blocks)
        return fail(JKB_E_BOUNDS, fn, 0, a->row_blocks, a->table_stride,
                    "table rows of %zu blocks, %zu apart", a->row_blocks, a->table_stride);
    if (!isfinite(a->scale))
        return fail(JKB_E_BOUNDS, fn, 0, 0, 0, "the softmax scale is not finite");
    if (a->n_tokens == 0 || a->n_seqs == 0) return JKB_OK;
    if (!a->q.data || !a->out.data || !a->block_table || !a->kv_lens || !a->q_starts)
        return fail(JKB_E_INVALID, fn, 0, 0, 0, "null pointer");
    if ((rc = check_align(a->q.data, eb, fn, "q")) ||
        (rc = check_align(a->out.data, eb, fn, "out")) ||
        (rc = check_align(a->lse, 4, fn, "lse")) ||
        (rc = check_align(a->block_table, 4, fn, "block_table")) ||
        (rc = check_align(a->kv_lens, 4, fn, "kv_lens")) ||
        (rc = check_align(a->q_starts, 4, fn, "q_starts")))
        return rc;
    AttnParams p{};
    p.codes = c->codes;
    p.scales = c->scales;
    p.n_blocks = (int)c->n_blocks;
    p.kv_heads = (int)c->n_heads;
    p.log_block = c->block_tokens == 16 ? 4 : c->block_tokens == 32 ? 5
                  : c->block_tokens == 64 ? 6 : 7;
    p.dim = c->dim;
    p.group = (int)(a->n_heads / c->n_heads);
    p.q = a->q.data;
    p.out = const_cast<void *>(a->out.data);
    p.q_token = a->q.token_stride;
    p.q_head = a->q.head_stride;
    p.out_token = a->out.token_stride;
    p.out_head = a->out.head_stride;
    const size_t per16 = 16 / eb;
    p.q_vec = (uintptr_t)p.q % 16 == 0 && p.q_token % per16 == 0 && p.q_head % per16 == 0;
    p.out_vec = (uintptr_t)p.out % 16 == 0 && p.out_token % per16 == 0 && p.out_head % per16 == 0;
    p.lse = a->lse;
    p.n_tokens = (int)a->n_tokens;
    p.table = a->block_table;
    p.kv_lens = a->kv_lens;
    p.q_starts = a->q_starts;
    p.table_stride = a->table_stride;
    p.n_seqs = (int)a->n_seqs;
    p.row_blocks = (int)a->row_blocks;
    p.window = (int)(a->window > (size_t)INT32_MAX ? 0 : a->window);
    p.causal = a->causal != 0;
    p.scale2 = a->scale * 1.4426950408889634f;
    p.min_rows = 1;
    p.max_rows = INT32_MAX;
    p.partial = w->partial;
    p.counters = w->counters;
    p.tile_partial = w->tile_partial;
    p.tile_counters = w->tile_counters;
    p.err = device_error_word();
    if (!p.err) return fail(JKB_E_CUDA, fn, 0, 0, 0, "no device error word");
    cudaStream_t st = as_stream(stream);
    // Sequences of up to ATTN_ROWS query rows a kv head go to the few-row kernel, the others to
    // the prompt kernel; each leaves the other's alone. max_new tells which of them a call needs.
    const size_t most = a->max_new * p.group;
    if (most <= ATTN_ROWS || c->dim_p > 128)
        return attn_decode_launch(p, type, c->dim_p, most, st);
    p.max_rows = ATTN_ROWS;
    if (a->n_seqs > 1 && (rc = attn_decode_launch(p, type, c->dim_p, ATTN_ROWS, st))) return rc;
    p.min_rows = a->n_seqs > 1 ? ATTN_ROWS + 1 : 1;
    p.max_rows = INT32_MAX;
    return attn_prompt_launch(p, type, c->dim_p, st);
}

}  // extern "C"
