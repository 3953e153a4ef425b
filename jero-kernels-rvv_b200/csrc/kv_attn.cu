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
//     two, is split into two f16 (22 bits; the second in the A tile's lower half), the codes are
//     exact in f16. The tensor core truncates its sums, so each 16-token step starts from zero
//     and is added to o in f32 on the FMA pipe, together with the rescale.
//
// A group of 16 tokens (kv_cache.cuh) is one bulk copy and one step of one warp. The four warps
// of a CTA take consecutive groups, each through its own ring of STAGES groups, and keep their
// own (m, l, o): they meet only when a row tile's tokens end. The tokens of all sequences and kv
// heads form one line of 64-token units, cut into equal parts, one a CTA, whatever the lengths
// (which only the device knows): a part that holds a piece of a row tile leaves (m, l, o) in the
// workspace, and the piece that arrives last adds all of them in the order of the line, so the
// result does not depend on which one that is.
#include "kv_attn.cuh"
#include "ptx.cuh"

#include <cuda_bf16.h>

#include <cstdlib>

namespace jkb {

namespace {

constexpr int NW = 4;                  // warps of a CTA
constexpr int UNIT = NW * KV_GROUP;    // tokens of a unit

constexpr int ND = 3;                  // digits of a query element

template <int DT_, int ROWS_>
struct DecCfg {
    static constexpr int DT = DT_;      // 32-element chunks of a head
    static constexpr int ROWS = ROWS_;  // 8: two digits share an MMA; 16: one each
    static constexpr int DIM = 32 * DT;
    static constexpr int STAGES = 3;
    // 12 warps an SM hide the steps' latency; the 16-row tile needs the registers of 8
    static constexpr int CTAS = DT <= 4 && ROWS == 8 ? 3 : 2;
    static constexpr int GROUP_BYTES = 32 * DIM;
    static constexpr int PASS = DIM / 2;  // dims merged at a time
};

struct StepInfo {
    unsigned long long src;  // the group's codes; 0: no visible token in it
    float ks, vs;
    int seq, item;           // item: kv head * row tiles + row tile
    int t0;
    int flags;               // FIRST / LAST of this CTA's piece, WHOLE row tile
};
enum { STEP_FIRST = 1, STEP_LAST = 2, STEP_WHOLE = 4 };

template <class C>
struct DecSmem {
    alignas(128) uint8_t ring[NW][C::STAGES][C::GROUP_BYTES];
    alignas(16) float merge[NW][C::ROWS][C::PASS + 4];
    float row_m[NW][C::ROWS], row_l[NW][C::ROWS];
    StepInfo info[NW][64];  // two batches of 32 steps
    uint64_t full[NW][C::STAGES];
    long long warp_sum[NW];
    int abort_flag, is_last;
};

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                       uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void bulk_load(void *dst, unsigned long long src, uint32_t bytes,
                                          uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
        : "memory");
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

// Elements i .. i + 7 of a query row.
__device__ __forceinline__ void load8(const AttnParams &p, int type, size_t i, float (&x)[8]) {
    if (type == JKB_F32) {
        const float *q = static_cast<const float *>(p.q) + i;
        if (p.q_vec) {
            const float4 a = __ldg(reinterpret_cast<const float4 *>(q));
            const float4 b = __ldg(reinterpret_cast<const float4 *>(q) + 1);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
            x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] = __ldg(q + k);
        }
        return;
    }
    const uint16_t *q = static_cast<const uint16_t *>(p.q) + i;
    uint32_t w[4];
    if (p.q_vec) {
        const uint4 a = __ldg(reinterpret_cast<const uint4 *>(q));
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            w[k] = __ldg(q + 2 * k) | (uint32_t)__ldg(q + 2 * k + 1) << 16;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (type == JKB_F16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
            x[2 * k] = f.x, x[2 * k + 1] = f.y;
        } else {
            x[2 * k] = __uint_as_float(w[k] << 16);
            x[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
        }
    }
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

// A query row is held as integers |n| <= MOST in ND signed base-256 digits: x = unit * n. A row
// with a non-finite element has unit NaN, so that its output is NaN; below 1e-30 the row counts
// as 0 (its scores are 0 to f32's accuracy).
constexpr float MOST = 8355711.0f;  // 127 * (65536 + 256 + 1)

// Units of one sequence and its row tiles.
template <int ROWS>
__device__ __forceinline__ void seq_units(const AttnParams &p, const AttnSeq &s, int &tiles,
                                          int &first_unit, int &units) {
    tiles = (int)(((long long)s.nq * p.group + ROWS - 1) / ROWS);
    first_unit = s.lo / UNIT;
    units = max(1, (s.len + UNIT - 1) / UNIT - first_unit);
}

template <class C>
__global__ void __launch_bounds__(32 * NW, C::CTAS)
    attn_decode_kernel(const __grid_constant__ AttnParams p, const int type) {
    constexpr int ROWS = C::ROWS, DT = C::DT, DIM = C::DIM, STAGES = C::STAGES;
    constexpr int RH = ROWS / 8;  // rows of a thread
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
            seq_units<ROWS>(p, attn_seq(p, i), tiles, first, units);
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
            seq_units<ROWS>(p, attn_seq(p, i), tiles, first, units);
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

    // Fills info[] for steps base .. base + 31 (lane i: step base + i), a multiple of 32: the table
    // entries and scales of 32 steps are fetched together, before the ring needs them.
    auto decode = [&](int base) {
        __syncwarp();
        StepInfo &f = sm.info[warp][(base + lane) & 63];
        f.src = 0;
        f.flags = 0;
        const long long u = u0 + base + lane;
        if (u < u1) {
            int a = 0, b = p.n_seqs - 1;  // the last sequence that starts at or before u
            while (a < b) {
                const int mid = (a + b + 1) >> 1;
                if (prefix[mid] <= u) a = mid;
                else b = mid - 1;
            }
            const AttnSeq s = attn_seq(p, a);
            int tiles, first, units;
            seq_units<ROWS>(p, s, tiles, first, units);
            const long long local = u - prefix[a];
            const int item = (int)(local / units), c = (int)(local - (long long)item * units);
            const int head = item / tiles;
            f.seq = a;
            f.item = item;
            f.t0 = (first + c) * UNIT + warp * KV_GROUP;
            f.flags = (c == 0 || u == u0 ? STEP_FIRST : 0) |
                      (c == units - 1 || u == u1 - 1 ? STEP_LAST : 0);
            const long long start = u - c;
            if (start >= u0 && start + units <= u1) f.flags |= STEP_WHOLE;
            if (f.t0 < s.len && f.t0 + KV_GROUP > s.lo) {
                const int id = __ldg(p.table + (size_t)a * p.table_stride +
                                     (f.t0 >> p.log_block));
                if (id >= 0 && id < p.n_blocks) {
                    const size_t bh = (size_t)id * p.kv_heads + head;
                    const float2 sc = __ldg(p.scales + bh);
                    const int grp = (f.t0 & ((1 << p.log_block) - 1)) / KV_GROUP;
                    f.ks = sc.x;
                    f.vs = sc.y;
                    f.src = (unsigned long long)(p.codes +
                                                 ((bh << p.log_block) / KV_GROUP + grp) *
                                                     (size_t)C::GROUP_BYTES);
                } else {
                    atomicOr(p.err, ERR_KV_RANGE);
                }
            }
        }
        __syncwarp();
    };
    int issued = 0;
    auto issue = [&](int upto) {  // starts the copies of the steps below min(upto, steps)
        for (; issued < min(upto, steps); issued++) {
            if (lane == 0) {
                const unsigned long long src = sm.info[warp][issued & 63].src;
                if (src) {
                    uint64_t *bar = &sm.full[warp][issued % STAGES];
                    mbar_arrive_tx(bar, C::GROUP_BYTES);
                    bulk_load(sm.ring[warp][issued % STAGES], src, C::GROUP_BYTES, bar);
                }
            }
        }
    };

    // ---- running state of the current row tile ----
    uint32_t qa[ND][DT][2 * RH];  // A registers of each digit
    float m[RH], l[RH], unit[RH];
    int lo[RH], hi[RH];
    float o[RH][DT][8];  // dims 32 c + 8 tg + i of row g (+ 8)
    int vexp = 0;
    bool seen = false, dead = false;
    uint32_t phases = 0;

    decode(0);
    issue(STAGES);
    for (int s = 0; s < steps; s++) {
        if ((s & 31) == 24 && s + 8 < steps) decode(s + 8);
        const StepInfo f = sm.info[warp][s & 63];

        if (f.flags & STEP_FIRST) {
            const AttnSeq q = attn_seq(p, f.seq);
            const int tiles = (int)(((long long)q.nq * p.group + ROWS - 1) / ROWS);
            const int head = f.item / tiles, tile = f.item - head * tiles;
#pragma unroll
            for (int r = 0; r < RH; r++) {
                const int row = tile * ROWS + g + 8 * r;
                const int tok = row / p.group;
                const bool on = tok < q.nq;
                const size_t at = (size_t)(q.q0 + tok) * p.q_token +
                                  (size_t)(head * p.group + row - tok * p.group) * p.q_head;
                float x[DT][8], top = 0.0f;
                bool finite = true;
#pragma unroll
                for (int c = 0; c < DT; c++) {
                    const int d = 32 * c + 8 * tg;
#pragma unroll
                    for (int i = 0; i < 8; i++) x[c][i] = 0.0f;
                    if (on && d < p.dim) load8(p, type, at + d, x[c]);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        finite &= isfinite(x[c][i]);
                        top = fmaxf(top, fabsf(x[c][i]));
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                const unsigned all = __ballot_sync(~0u, finite);
                finite = ((all >> (lane & ~3)) & 15u) == 15u;
                const float inv = finite && top > 1e-30f ? __fdividef(MOST, top) : 0.0f;
                unit[r] = (finite ? top / MOST : __int_as_float(0x7FC00000)) * p.scale2;
#pragma unroll
                for (int c = 0; c < DT; c++) {
                    uint32_t dg[ND][2] = {};
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float y = finite ? x[c][i] * inv : 0.0f;
                        int n = __float2int_rn(fminf(fmaxf(y, -MOST), MOST));
#pragma unroll
                        for (int k = ND - 1; k >= 0; k--) {
                            const int low = (int)(int8_t)(n & 255);
                            dg[k][i >> 2] |= (uint32_t)(low & 255) << (8 * (i & 3));
                            n = (n - low) >> 8;
                        }
                    }
#pragma unroll
                    for (int k = 0; k < ND; k++) {
                        qa[k][c][2 * r] = dg[k][0];
                        qa[k][c][2 * r + 1] = dg[k][1];
                    }
                }
                const int pos = q.len - q.nq + tok;
                hi[r] = !on ? 0 : p.causal ? min(q.len, pos + 1) : q.len;
                lo[r] = p.window ? max(0, pos - p.window + 1) : 0;
                m[r] = -INFINITY;
                l[r] = 0.0f;
#pragma unroll
                for (int c = 0; c < DT; c++)
#pragma unroll
                    for (int i = 0; i < 8; i++) o[r][c][i] = 0.0f;
            }
            seen = false;
        }

        if (f.src) {
            const int st = s % STAGES;
            if (!dead && !mbar_wait(&sm.full[warp][st], (phases >> st) & 1, &sm.abort_flag, p.err,
                                    ERR_ATTN_WAIT))
                dead = true;
            phases ^= 1u << st;
        }
        if (f.src && !dead) {
            const uint8_t *stage = sm.ring[warp][s % STAGES];
            // ---- scores: tokens t0 + 8 nt + 2 tg + e of rows g (+ 8) ----
            float sc[RH][4];
#pragma unroll
            for (int nt = 0; nt < 2; nt++) {
                int acc[ND][4] = {};
#pragma unroll
                for (int c = 0; c < DT; c++) {
                    const uint2 b = *reinterpret_cast<const uint2 *>(stage + nt * 8 * DIM +
                                                                     c * 256 + lane * 8);
                    if (RH == 1) {
                        mma_s8(acc[0], qa[0][c][0], qa[1][c][0], qa[0][c][1], qa[1][c][1], b.x,
                               b.y);
                        mma_s8(acc[2], qa[2][c][0], 0u, qa[2][c][1], 0u, b.x, b.y);
                    } else {
#pragma unroll
                        for (int k = 0; k < ND; k++)
                            mma_s8(acc[k], qa[k][c][0], qa[k][c][2 * RH - 2], qa[k][c][1],
                                   qa[k][c][2 * RH - 1], b.x, b.y);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {
#pragma unroll
                    for (int r = 0; r < RH; r++) {
                        const int d0 = RH == 1 ? acc[0][e] : acc[0][2 * r + e];
                        const int d1 = RH == 1 ? acc[0][2 + e] : acc[1][2 * r + e];
                        const int d2 = RH == 1 ? acc[2][e] : acc[2][2 * r + e];
                        const float v =
                            fmaf((float)d0, 65536.0f, fmaf((float)d1, 256.0f, (float)d2));
                        const int t = f.t0 + 8 * nt + 2 * tg + e;
                        sc[r][2 * nt + e] =
                            t >= lo[r] && t < hi[r] ? v * (unit[r] * f.ks) : -INFINITY;
                    }
                }
            }
            // ---- the block's value scale relative to a power of two ----
            const uint32_t vbits = __float_as_uint(f.vs);
            const int e = (int)((vbits >> 23) & 255) - 126;
            const float mant = (vbits & 0x7F800000u)
                                   ? __uint_as_float((vbits & 0x807FFFFFu) | 0x3F000000u)
                                   : 0.0f;  // vs = mant * 2^e
            float shift = 1.0f;
            if (!seen) {
                vexp = e;
                seen = true;
            } else if (e > vexp) {
                shift = ex2((float)(vexp - e));
                vexp = e;
            }
            const float vmul = mant * ex2((float)(e - vexp + 14));
            // ---- softmax step ----
            uint32_t ph[RH][2], pl[RH][2];
            float alpha[RH];
#pragma unroll
            for (int r = 0; r < RH; r++) {
                float top = fmaxf(fmaxf(sc[r][0], sc[r][1]), fmaxf(sc[r][2], sc[r][3]));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                const float mn = fmaxf(m[r], top);
                const float ref = mn == -INFINITY ? 0.0f : mn;
                alpha[r] = ex2(m[r] - ref);
                m[r] = mn;
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = ex2(sc[r][i] - ref);
                l[r] = fmaf(l[r], alpha[r], (w[0] + w[1]) + (w[2] + w[3]));
                alpha[r] *= shift;
                split_f16(w[0] * vmul, w[1] * vmul, ph[r][0], pl[r][0]);
                split_f16(w[2] * vmul, w[3] * vmul, ph[r][1], pl[r][1]);
            }
            // ---- o = o * alpha + p v ----
#pragma unroll
            for (int c = 0; c < DT; c++) {
                const uint4 v4 = *reinterpret_cast<const uint4 *>(
                    stage + 16 * DIM + c * 512 + (tg * 8 + (g ^ (2 * tg))) * 16);
                const uint32_t vw[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t b0, b1;
                    value_f16(vw[j], b0, b1);
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
                    if (RH == 1) {  // rows g: high parts, rows g + 8: low parts
                        mma_f16(d, ph[0][0], pl[0][0], ph[0][1], pl[0][1], b0, b1);
                        o[0][c][j] = fmaf(o[0][c][j], alpha[0], d[0] + d[2]);
                        o[0][c][4 + j] = fmaf(o[0][c][4 + j], alpha[0], d[1] + d[3]);
                    } else {
                        mma_f16(d, pl[0][0], pl[RH - 1][0], pl[0][1], pl[RH - 1][1], b0, b1);
                        mma_f16(d, ph[0][0], ph[RH - 1][0], ph[0][1], ph[RH - 1][1], b0, b1);
#pragma unroll
                        for (int r = 0; r < RH; r++) {
                            o[r][c][j] = fmaf(o[r][c][j], alpha[r], d[2 * r]);
                            o[r][c][4 + j] = fmaf(o[r][c][4 + j], alpha[r], d[2 * r + 1]);
                        }
                    }
                }
            }
        }
        __syncwarp();
        issue(s + 1 + STAGES);

        if (!(f.flags & STEP_LAST)) continue;
        // ---- the piece ends: the warps' (m, l, o) into one ----
        const AttnSeq q = attn_seq(p, f.seq);
        int tiles, first, units;
        seq_units<ROWS>(p, q, tiles, first, units);
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
        const float pow2 = seen ? ldexpf(1.0f, vexp - 14) : 1.0f;
#pragma unroll
        for (int r = 0; r < RH; r++) {
            float top = -INFINITY;
            for (int w = 0; w < NW; w++) top = fmaxf(top, sm.row_m[w][g + 8 * r]);
            mul[r] = ex2(m[r] - (top == -INFINITY ? 0.0f : top));
        }
        // where this piece's sums go: the output, or its slot in the workspace
        const bool whole = f.flags & STEP_WHOLE;
        const long long start = prefix[f.seq] + (long long)f.item * units;
        const int cta0 = (int)(start / per), cta1 = (int)((start + units - 1) / per);
        auto slot_of = [&](int cta) {
            const int slot = 2 * cta + (cta == cta0 && start != per * cta0 ? 1 : 0);
            return p.partial + (size_t)slot * ROWS * (DIM + 2);
        };
        float *mine = whole ? nullptr : slot_of((int)blockIdx.x);
        auto finish = [&](int row, int d, float4 v, float top, float sum) {
            const int rr = tile * ROWS + row, tok = rr / p.group;
            if (tok >= q.nq || d >= p.dim) return;
            const int h = head * p.group + rr - tok * p.group;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            store4(p, type, (size_t)(q.q0 + tok) * p.out_token + (size_t)h * p.out_head + d,
                   make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
            if (d == 0 && p.lse)
                p.lse[(size_t)(q.q0 + tok) * p.group * p.kv_heads + h] =
                    (top + log2f(sum)) * 0.69314718055994531f;
        };
#pragma unroll
        for (int pass = 0; pass < 2; pass++) {
#pragma unroll
            for (int c = 0; c < DT; c++) {
#pragma unroll
                for (int r = 0; r < RH; r++) {
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const int d = 32 * c + 8 * tg + 4 * k - pass * C::PASS;
                        if (d >= 0 && d < C::PASS) {
                            float4 v;
                            v.x = o[r][c][4 * k] * mul[r] * pow2;
                            v.y = o[r][c][4 * k + 1] * mul[r] * pow2;
                            v.z = o[r][c][4 * k + 2] * mul[r] * pow2;
                            v.w = o[r][c][4 * k + 3] * mul[r] * pow2;
                            *reinterpret_cast<float4 *>(&sm.merge[warp][g + 8 * r][d]) = v;
                        }
                    }
                }
            }
            __syncthreads();
            for (int i = tid; i < ROWS * C::PASS / 4; i += 32 * NW) {
                const int row = i / (C::PASS / 4), d = 4 * (i - row * (C::PASS / 4));
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                float top = -INFINITY, sum = 0.0f;
                for (int w = 0; w < NW; w++) top = fmaxf(top, sm.row_m[w][row]);
                const float ref = top == -INFINITY ? 0.0f : top;
                for (int w = 0; w < NW; w++) {
                    const float4 x = *reinterpret_cast<const float4 *>(&sm.merge[w][row][d]);
                    v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
                    sum += sm.row_l[w][row] * ex2(sm.row_m[w][row] - ref);
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
        // ---- the last piece of the row tile to arrive adds them all, in order ----
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            const int before = atomicAdd(&p.counters[cta0], 1);
            sm.is_last = before == cta1 - cta0;
            if (sm.is_last) p.counters[cta0] = 0;
        }
        __syncthreads();
        if (!sm.is_last) continue;
        __threadfence();
        for (int i = tid; i < ROWS * DIM / 4; i += 32 * NW) {
            const int row = i / (DIM / 4), d = 4 * (i - row * (DIM / 4));
            float top = -INFINITY;
#pragma unroll 8
            for (int c = cta0; c <= cta1; c++)
                top = fmaxf(top, __ldcg(slot_of(c) + ROWS * DIM + row));
            const float ref = top == -INFINITY ? 0.0f : top;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float sum = 0.0f;
#pragma unroll 8
            for (int c = cta0; c <= cta1; c++) {
                const float *slot = slot_of(c);
                const float w = ex2(__ldcg(slot + ROWS * DIM + row) - ref);
                const float4 x = __ldcg(reinterpret_cast<const float4 *>(slot + row * DIM + d));
                sum = fmaf(w, __ldcg(slot + ROWS * DIM + ROWS + row), sum);
                v.x = fmaf(w, x.x, v.x);
                v.y = fmaf(w, x.y, v.y);
                v.z = fmaf(w, x.z, v.z);
                v.w = fmaf(w, x.w, v.w);
            }
            finish(row, d, v, top, sum);
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
int launch_cfg(const AttnParams &p, int type, cudaStream_t st) {
    static const char *fn = "attention_kv8";
    const size_t smem = sizeof(DecSmem<C>) + 128 + 8 * ((size_t)p.n_seqs + 1);
    static thread_local size_t allowed = 0;
    static thread_local int allowed_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev != allowed_dev || smem > allowed) {
        cudaError_t e = cudaFuncSetAttribute(attn_decode_kernel<C>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)smem);
        if (e != cudaSuccess) return fail_cuda(e, fn);
        allowed = smem;
        allowed_dev = dev;
    }
    cudaError_t e = launch_pdl(attn_decode_kernel<C>, dim3((unsigned)(num_sms() * C::CTAS)),
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
    w->ctas = 3 * num_sms();
    const size_t sms = (size_t)num_sms(), width = (size_t)w->dim_p + 2;
    const size_t part = Arena::round(2 * (size_t)w->ctas * ATTN_ROWS * width * sizeof(float));
    const size_t tile = w->dim_p <= 128 ? Arena::round(2 * sms * 128 * width * sizeof(float)) : 0;
    const size_t counts = (w->ctas + sms) * sizeof(int);
    cudaError_t e = cudaMalloc(&w->base, part + tile + counts);
    if (e == cudaSuccess) {
        w->partial = (float *)w->base;
        w->tile_partial = tile ? (float *)(w->base + part) : nullptr;
        w->counters = (int *)(w->base + part + tile);
        w->tile_counters = w->counters + w->ctas;
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
    if (a->n_tokens > (size_t)INT32_MAX / a->n_heads)
        return fail(JKB_E_BOUNDS, fn, 0, a->n_tokens, (size_t)INT32_MAX / a->n_heads,
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
