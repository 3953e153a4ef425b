// The 8-bit paged key/value cache (layout: kv_cache.cuh): block tables and slot maps, append with
// its quantization, and copies in and out. All of it moves few bytes; what bounds each kernel is
// at its head.
#include "kv_cache.cuh"

#include <cuda_bf16.h>

#include <cfloat>
#include <cstdlib>

namespace jkb {

namespace {

__device__ __forceinline__ void pdl_enter() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" :::);
}

// ---------------------------------------------------------------- block tables and slot maps

constexpr int TABLE_THREADS = 512;

// One launch for the whole step. Every CTA sums all sequences' lengths itself (two block scans
// over at most JKB_KV_MAX_SEQS entries, read from L2), which is cheaper than a second launch or a
// wait between CTAs; it then writes its share of the rows, lengths and slots. A new token's
// block is looked up in the free list rather than in the row that some other CTA is writing.
// 8 bytes a token move. The launch and the scans' latency bound a decode step (24 sequences of one
// token: 4.3 us), the search of each four tokens' sequence a large one (1500 of 350 tokens on
// average: 10.2 us, 60 % of the issue slots).
__global__ void __launch_bounds__(TABLE_THREADS)
    tables_kernel(int32_t *__restrict__ table, int n_seqs, int row_blocks, size_t table_stride,
                  int32_t *__restrict__ slots, int32_t *__restrict__ positions, int n_slots,
                  int32_t *__restrict__ q_starts, int32_t *__restrict__ kv_lens,
                  int32_t *__restrict__ counts, const int32_t *__restrict__ ctx_lens,
                  const int32_t *__restrict__ new_lens, const int32_t *__restrict__ free_blocks,
                  int n_free, int log_block, int *err) {
    extern __shared__ int32_t table_smem[];
    int32_t *start = table_smem;             // [n_seqs + 1], clamped to INT_MAX
    int32_t *base = table_smem + n_seqs + 1; // [n_seqs] first free-list index; -1: no room
    __shared__ long long warp_new[TABLE_THREADS / 32], warp_need[TABLE_THREADS / 32];
    __shared__ int s_taken, s_refused;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int mask = (1 << log_block) - 1;
    pdl_enter();
    if (tid == 0) s_taken = s_refused = 0;
    const int per = (n_seqs + TABLE_THREADS - 1) / TABLE_THREADS;
    const int lo = min(tid * per, n_seqs), hi = min(lo + per, n_seqs);
    auto lengths = [&](int i, long long &c, long long &n, long long &need, bool &room) {
        c = max(__ldg(ctx_lens + i), 0);
        n = max(__ldg(new_lens + i), 0);
        room = c + n <= (long long)row_blocks << log_block;
        need = room ? ((c + n + mask) >> log_block) - ((c + mask) >> log_block) : 0;
    };
    long long sum_new = 0, sum_need = 0;
    for (int i = lo; i < hi; i++) {
        long long c, n, need;
        bool room;
        lengths(i, c, n, need, room);
        sum_new += n;
        sum_need += need;
    }
    long long inc_new = sum_new, inc_need = sum_need;
    for (int d = 1; d < 32; d <<= 1) {
        const long long a = __shfl_up_sync(~0u, inc_new, d), b = __shfl_up_sync(~0u, inc_need, d);
        if (lane >= d) {
            inc_new += a;
            inc_need += b;
        }
    }
    if (lane == 31) {
        warp_new[warp] = inc_new;
        warp_need[warp] = inc_need;
    }
    __syncthreads();
    long long at_new = inc_new - sum_new, at_need = inc_need - sum_need;
    for (int w = 0; w < warp; w++) {
        at_new += warp_new[w];
        at_need += warp_need[w];
    }
    int taken = 0, refused = 0;
    for (int i = lo; i < hi; i++) {
        long long c, n, need;
        bool room;
        lengths(i, c, n, need, room);
        const bool fits = room && (need == 0 || at_need + need <= n_free);
        start[i] = (int)min(at_new, (long long)INT32_MAX);
        base[i] = fits ? (int)min(at_need, (long long)INT32_MAX) : -1;
        if (fits && need) taken = (int)(at_need + need);
        refused += !fits;
        at_new += n;
        at_need += need;
        if (i == n_seqs - 1) start[n_seqs] = (int)min(at_new, (long long)INT32_MAX);
    }
    if (n_seqs == 0 && tid == 0) start[0] = 0;
    if (blockIdx.x == 0) {
        if (taken) atomicMax(&s_taken, taken);
        if (refused) atomicAdd(&s_refused, refused);
    }
    __syncthreads();

    const int total = start[n_seqs];
    if (blockIdx.x == 0 && tid == 0) {
        counts[0] = total;
        counts[1] = s_taken;
        counts[2] = s_refused;
        q_starts[n_seqs] = total;
    }
    const int nwarps = gridDim.x * (TABLE_THREADS / 32);
    for (int i = blockIdx.x * (TABLE_THREADS / 32) + warp; i < n_seqs; i += nwarps) {
        long long c, n, need;
        bool room;
        lengths(i, c, n, need, room);
        const int b = base[i];
        if (lane == 0) {
            q_starts[i] = start[i];
            kv_lens[i] = (int)min(b >= 0 ? c + n : c, (long long)INT32_MAX);
        }
        if (b < 0) continue;
        int32_t *row = table + (size_t)i * table_stride + (size_t)((c + mask) >> log_block);
        for (int j = lane; j < (int)need; j += 32) row[j] = __ldg(free_blocks + b + j);
    }

    // four consecutive tokens a thread: one search, 16-byte stores
    const bool vec = (((uintptr_t)slots | (uintptr_t)positions) & 15) == 0;
    for (long long t0 = 4 * ((long long)blockIdx.x * TABLE_THREADS + tid); t0 < n_slots;
         t0 += 4ll * gridDim.x * TABLE_THREADS) {
        int s = 0;
        if (t0 < total) {  // the last sequence that starts at or before t0
            int a = 0, b = n_seqs - 1;
            while (a < b) {
                const int mid = (a + b + 1) >> 1;
                if (start[mid] <= (int)t0) a = mid;
                else b = mid - 1;
            }
            s = a;
        }
        int sl[4], po[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int t = (int)min(t0 + k, (long long)INT32_MAX);
            sl[k] = po[k] = -1;
            if (t >= total) continue;
            while (t >= start[s + 1]) s++;
            if (base[s] < 0) continue;
            const int c = max(__ldg(ctx_lens + s), 0), p = c + (t - start[s]);
            const int j = p >> log_block, first = (int)(((long long)c + mask) >> log_block);
            const int id = j < first ? table[(size_t)s * table_stride + j]
                                     : __ldg(free_blocks + base[s] + j - first);
            if (id < 0) continue;
            if (id > INT32_MAX >> log_block) {  // its slots would not fit 32 bits
                atomicOr(err, ERR_KV_RANGE);
                continue;
            }
            sl[k] = (id << log_block) + (p & mask);
            po[k] = p;
        }
        if (vec && t0 + 4 <= n_slots) {
            *reinterpret_cast<int4 *>(slots + t0) = make_int4(sl[0], sl[1], sl[2], sl[3]);
            *reinterpret_cast<int4 *>(positions + t0) = make_int4(po[0], po[1], po[2], po[3]);
        } else {
            for (int k = 0; k < 4 && t0 + k < n_slots; k++) {
                slots[t0 + k] = sl[k];
                positions[t0 + k] = po[k];
            }
        }
    }
}

// ---------------------------------------------------------------- append

constexpr int APPEND_THREADS = 128;

struct AppendSide {
    const void *data;
    size_t token_stride, head_stride;
};

template <int TYPE>
__device__ __forceinline__ float elem(const void *p, size_t i) {
    if (TYPE == JKB_F32) return __ldg(static_cast<const float *>(p) + i);
    if (TYPE == JKB_F16) return __half2float(__ldg(static_cast<const __half *>(p) + i));
    return __bfloat162float(__ldg(static_cast<const __nv_bfloat16 *>(p) + i));
}
// Elements i .. i + 3; VEC: they lie on a boundary of four elements.
template <int TYPE, bool VEC>
__device__ __forceinline__ float4 elem4(const void *p, size_t i) {
    if (!VEC)
        return make_float4(elem<TYPE>(p, i), elem<TYPE>(p, i + 1), elem<TYPE>(p, i + 2),
                           elem<TYPE>(p, i + 3));
    if (TYPE == JKB_F32) return __ldg(reinterpret_cast<const float4 *>((const float *)p + i));
    const uint2 v = __ldg(reinterpret_cast<const uint2 *>((const uint16_t *)p + i));
    if (TYPE == JKB_F16) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u),
                       __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u));
}

__device__ __forceinline__ float finite_or_0(float v) { return isfinite(v) ? v : 0.0f; }

// Code of one element in the low byte: rint(x * inv), ties to even; |x * inv| < 127.5, and adding
// 1.5 * 2^23 rounds to an integer, whose two's complement the low bits are.
__device__ __forceinline__ uint32_t code_of(float x, float inv) {  // x finite
    return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.0f));
}
__device__ __forceinline__ float4 finite_or_0(float4 v) {
    return make_float4(finite_or_0(v.x), finite_or_0(v.y), finite_or_0(v.z), finite_or_0(v.w));
}
// The low bytes of four words.
__device__ __forceinline__ uint32_t low4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return (a & 255) | (b & 255) << 8 | (c & 255) << 16 | (uint32_t)(d & 255) << 24;
}
// The bytes of w with each code rounded again to a larger scale; BIAS: codes are held + 128.
template <bool BIAS>
__device__ __forceinline__ int recode(uint32_t w, int byte, float ratio) {
    const int raw = (w >> (8 * byte)) & 255;
    const int c = BIAS ? raw - 128 : (int)(int8_t)raw;
    return (int)rintf(__fmul_rn((float)c, ratio)) + (BIAS ? 128 : 0);
}

// The tokens of one block in this call: rows t0 .. t0 + n, offsets o .. o + n of block `block`.
struct Run {
    int t0, n, o, block;
};

// Scale and codes of one run, head and side by a team of threads (a warp or the CTA).
// A first pass takes the rows' absmax; the second reads them again (from L1 or L2: a block's rows
// are at most 64 KB) and writes 16 bytes of codes at a time: a key patch is 16 dims of one token,
// a value patch 4 dims of 4 tokens. Old bytes are read only where a patch keeps some of them.
// Instructions bound it, 29 an element (f32) or 25 (bf16), which fill 57 to 66 % of the issue slots,
// the waits between the two passes and, as each instruction runs a few times a run, their fetching:
// the rare paths are loops over little code. (Patches kept in registers between the passes, in eight
// times the code, took twice as long.) 5985 f32 tokens of 8 heads of 128 take 22 us (2.8 TB/s of rows
// and codes), 16,411 bf16 tokens 41 us (2.5 TB/s), 24 single tokens 5 us.
template <int TYPE, bool VEC>
__device__ __forceinline__ void append_run(const Run &r, const AppendSide &src, bool value,
                                           int head, int tid, int team, uint8_t *codes,
                                           float2 *scales, int n_heads, int block_tokens, int dim,
                                           int dim_p, float *red) {
    const size_t row0 = (size_t)r.t0 * src.token_stride + (size_t)head * src.head_stride;
    const size_t bh = (size_t)r.block * n_heads + head;
    float *scale = &scales[bh].x + (value ? 1 : 0);
    const float old = r.o ? *scale : 0.0f;
    const int quads = dim >> 2;
    float amax = 0.0f;
    bool odd = false;  // an element that is not finite
    {
        int t = tid / quads, q = tid - t * quads;
        const int step_t = team / quads, step_q = team - step_t * quads;
        size_t at = row0 + t * src.token_stride + 4 * q;
        const size_t step = step_t * src.token_stride + 4 * step_q;
        const size_t wrap = src.token_stride - 4 * quads;
        float zero = 0.0f;  // NaN once an element is not finite
#pragma unroll 1
        while (t < r.n) {
            constexpr int U = VEC ? 8 : 2;  // loads in flight
            float4 v[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (t < r.n) v[u] = elem4<TYPE, VEC>(src.data, at);
                t += step_t;
                q += step_q;
                at += step;
                if (q >= quads) {
                    q -= quads;
                    t++;
                    at += wrap;
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {  // (fmaxf passes over a NaN)
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(v[u].x), fabsf(v[u].y)),
                                         fmaxf(fabsf(v[u].z), fabsf(v[u].w))));
                zero = fmaf(v[u].x, 0.f, fmaf(v[u].y, 0.f, zero));
                zero = fmaf(v[u].z, 0.f, fmaf(v[u].w, 0.f, zero));
            }
        }
        odd = !(zero == 0.0f);
        if (amax == INFINITY) {  // infinities count as 0: once more without them
            amax = 0.0f;
#pragma unroll 1
            for (int i = tid; i < r.n * quads; i += team) {
                const float4 v = finite_or_0(elem4<TYPE, VEC>(
                    src.data, row0 + i / quads * src.token_stride + 4 * (i % quads)));
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)),
                                         fmaxf(fabsf(v.z), fabsf(v.w))));
            }
        }
    }
    for (int d = 16; d; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, d));
    odd = __any_sync(~0u, odd);
    if (team > 32) {  // (a warp's sign: odd)
        if ((tid & 31) == 0) red[tid >> 5] = odd ? -amax : amax;
        __syncthreads();
        for (int w = 0; w < APPEND_THREADS / 32; w++) {
            odd |= (__float_as_uint(red[w]) >> 31) != 0;
            amax = fmaxf(amax, fabsf(red[w]));
        }
        __syncthreads();
    } else {
        __syncwarp();
    }
    float s = fmaxf(old, __fmul_rn(amax, 1.0f / 127.0f));
    if (!(s >= FLT_MIN)) s = 0.0f;
    const float inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
    const bool grow = r.o > 0 && s > old;
    const float ratio = grow ? __fdiv_rn(old, s) : 1.0f;
    if (tid == 0) *scale = s;
    const int end = r.o + r.n;
    const int g0 = grow ? 0 : r.o / KV_GROUP, g1 = (end + KV_GROUP - 1) / KV_GROUP;
    uint8_t *page = codes + bh * (size_t)block_tokens * 2 * dim_p;
    const int patches = dim_p;  // 16 * dim_p bytes of one side of a group
    // the groups that are new as a whole
    const int f0 = (r.o + KV_GROUP - 1) / KV_GROUP, f1 = max(f0, end / KV_GROUP);
    const int per = dim_p >> 4;  // key patches of a token
    const int n_new = (f1 - f0) * patches;
    const size_t row_f0 = row0 + (size_t)(f0 * KV_GROUP - r.o) * src.token_stride;
    uint8_t *page_f0 = page + (size_t)f0 * 32 * dim_p;
    if (!value) {
        int tok = tid / per, c16 = tid - tok * per;
        const int step_t = team / per, step_c = team - step_t * per;
#pragma unroll 1
        for (int i = tid; i < n_new; i += team) {
            const size_t row = row_f0 + tok * src.token_stride + 16 * c16;
            float4 v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (16 * c16 + 4 * k < dim) v[k] = elem4<TYPE, VEC>(src.data, row + 4 * k);
            }
            if (odd)
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = finite_or_0(v[k]);
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; k++)
                w[k] = low4(code_of(v[k].x, inv), code_of(v[k].y, inv), code_of(v[k].z, inv),
                            code_of(v[k].w, inv));
            *reinterpret_cast<uint4 *>(page_f0 + (size_t)(tok / KV_GROUP) * 32 * dim_p +
                                       kv_key_at(tok % KV_GROUP, 16 * c16, dim_p)) =
                make_uint4(w[0], w[1], w[2], w[3]);
            tok += step_t;
            c16 += step_c;
            if (c16 >= per) {
                c16 -= per;
                tok++;
            }
        }
    } else {
        const int q8 = tid & 31, tt = q8 >> 3, chunks = dim_p >> 5;  // chunks: of 32 dims
        int grp = (tid >> 5) / chunks, chunk = (tid >> 5) - grp * chunks;
        const int d_lane = 4 * ((q8 & 7) ^ (2 * tt));
        const size_t lane_row = row_f0 + 2 * tt * src.token_stride + d_lane;
#pragma unroll 1
        for (int i = tid; i < n_new; i += team) {
            const size_t row = lane_row + (size_t)(grp * KV_GROUP) * src.token_stride + 32 * chunk;
            const bool on = 32 * chunk + d_lane < dim;
            float4 v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (on)
                    v[k] = elem4<TYPE, VEC>(
                        src.data, row + (size_t)((k & 1) + 8 * (k >> 1)) * src.token_stride);
            }
            if (odd)
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = finite_or_0(v[k]);
            uint32_t c[4][4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                c[k][0] = code_of(v[k].x, inv), c[k][1] = code_of(v[k].y, inv);
                c[k][2] = code_of(v[k].z, inv), c[k][3] = code_of(v[k].w, inv);
            }
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                w[j] = 0x80808080u ^ low4(c[0][j], c[1][j], c[2][j], c[3][j]);
            *reinterpret_cast<uint4 *>(page_f0 + (size_t)grp * 32 * dim_p + 16 * dim_p +
                                       512 * chunk + 16 * q8) =
                make_uint4(w[0], w[1], w[2], w[3]);
            chunk += team >> 5;
            while (chunk >= chunks) {
                chunk -= chunks;
                grp++;
            }
        }
    }
    // the groups before and after, which keep bytes or end within
    const int before = max(f0 - g0, 0) * patches, after = (g1 - f1) * patches;
#pragma unroll 1
    for (int j = tid; j < before + after; j += team) {
        const int i = j < before ? j + g0 * patches : j - before + f1 * patches;
        const int grp = i / patches, p = i - grp * patches;
        uint8_t *g = page + (size_t)grp * 32 * dim_p;
        if (!value) {
            const int tok = p / per, d0 = 16 * (p - tok * per);
            const int off = grp * KV_GROUP + tok;
            if (off >= end || (off < r.o && !grow)) continue;
            uint32_t *at = reinterpret_cast<uint32_t *>(g + kv_key_at(tok, d0, dim_p));
            const size_t row = row0 + (size_t)(off - r.o) * src.token_stride + d0;
#pragma unroll 1
            for (int k = 0; k < 4; k++) {
                uint32_t w = 0;
                if (off < r.o) {
                    const uint32_t x = at[k];
                    w = pack4(recode<false>(x, 0, ratio), recode<false>(x, 1, ratio),
                              recode<false>(x, 2, ratio), recode<false>(x, 3, ratio));
                } else if (d0 + 4 * k < dim) {
                    const float4 v = finite_or_0(elem4<TYPE, VEC>(src.data, row + 4 * k));
                    w = low4(code_of(v.x, inv), code_of(v.y, inv), code_of(v.z, inv),
                             code_of(v.w, inv));
                }
                at[k] = w;
            }
        } else {
            const int chunk = p >> 5, q = p & 31, t = q >> 3;
            const int d0 = 32 * chunk + 4 * ((q & 7) ^ (2 * t));
            uint4 *at = reinterpret_cast<uint4 *>(g + 16 * dim_p + 512 * chunk + 16 * q);
            uint4 was = make_uint4(0, 0, 0, 0);
            bool any = false;
#pragma unroll 1
            for (int k = 0; k < 4; k++) {  // byte k of the words: token 2 t + (k & 1) + 8 (k >> 1)
                const int off = grp * KV_GROUP + 2 * t + (k & 1) + 8 * (k >> 1);
                const bool is_new = off >= r.o && off < end, is_old = grow && off < r.o;
                if (!is_new && !is_old) continue;
                if (!any) was = *at;
                any = true;
                uint32_t c[4];
                if (is_new) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (d0 < dim)
                        v = finite_or_0(elem4<TYPE, VEC>(
                            src.data, row0 + (size_t)(off - r.o) * src.token_stride + d0));
                    c[0] = code_of(v.x, inv) + 128, c[1] = code_of(v.y, inv) + 128;
                    c[2] = code_of(v.z, inv) + 128, c[3] = code_of(v.w, inv) + 128;
                } else {
                    c[0] = recode<true>(was.x, k, ratio), c[1] = recode<true>(was.y, k, ratio);
                    c[2] = recode<true>(was.z, k, ratio), c[3] = recode<true>(was.w, k, ratio);
                }
                const uint32_t mask = 255u << (8 * k);
                was.x = (was.x & ~mask) | (c[0] & 255) << (8 * k);
                was.y = (was.y & ~mask) | (c[1] & 255) << (8 * k);
                was.z = (was.z & ~mask) | (c[2] & 255) << (8 * k);
                was.w = (was.w & ~mask) | (c[3] & 255) << (8 * k);
            }
            if (any) *at = was;
        }
    }
}

// CTA (range of `span` tokens, head, side): the runs that start in the range. Few runs (prompts)
// are taken by the whole CTA one after the other, many (decode steps, one token each) by a warp
// each. The kernel moves the rows once from DRAM and a quarter (f32) or half (16-bit) of that
// back; single tokens are bound by latency: slot, then scale and row, then the codes.
template <int TYPE, bool VEC>
__global__ void __launch_bounds__(APPEND_THREADS)
    append_kernel(AppendSide k, AppendSide v, const int32_t *__restrict__ slots, int n_tokens,
                  int span, uint8_t *__restrict__ codes, float2 *__restrict__ scales,
                  long long n_slots, int n_heads, int log_block, int dim, int dim_p, int *err) {
    __shared__ int s_slot[1 + 64 + 128];  // slots of tokens first - 1 .. first + span + 128
    __shared__ float red[APPEND_THREADS / 32];
    __shared__ unsigned s_starts[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = blockIdx.x * span, head = blockIdx.y;
    const bool value = blockIdx.z != 0;
    pdl_enter();
    bool bad = false;
    for (int i = tid; i < 1 + span + 128; i += APPEND_THREADS) {
        const long long t = (long long)first - 1 + i;
        int s = t >= 0 && t < n_tokens ? __ldg(slots + t) : -1;
        if (s >= n_slots) {
            s = -1;
            bad = true;
        }
        s_slot[i] = s;
    }
    __syncthreads();
    // A run starts at a token whose block is not that of the last token before it, skipped ones
    // aside: two runs of one block would rewrite its scale and codes at the same time.
    if (warp < 2) {
        const int s = tid < span ? s_slot[1 + tid] : -1;
        int before = s_slot[tid];
        if (__any_sync(~0u, s >= 0 && before < 0)) {
            const unsigned there0 = __ballot_sync(~0u, lane < span && s_slot[1 + lane] >= 0);
            const unsigned there1 = __ballot_sync(~0u, 32 + lane < span && s_slot[33 + lane] >= 0);
            const unsigned long long earlier =
                (there0 | (unsigned long long)there1 << 32) & ((1ull << tid) - 1);
            before = earlier ? s_slot[64 - __clzll(earlier)] : s_slot[0];
            const bool far = s >= 0 && !earlier && before < 0;  // (the range's first, if any)
            int last = -1;
#pragma unroll 1
            for (int end = __any_sync(~0u, far) ? first - 2 : -1; end >= 0 && last < 0; end -= 32) {
                int x = end >= lane ? __ldg(slots + (end - lane)) : -1;
                if (x >= n_slots) x = -1;
                const unsigned there = __ballot_sync(~0u, x >= 0);
                if (there) last = __shfl_sync(~0u, x, __ffs(there) - 1);
            }
            if (far) before = last;
        }
        const bool joins = before >= 0 && s >= 0 && (before >> log_block) == (s >> log_block);
        if (joins && (s_slot[tid] < 0 || s != before + 1)) bad = true;
        const unsigned b = __ballot_sync(~0u, s >= 0 && !joins);
        if (lane == 0) s_starts[warp] = b;
    }
    if (bad) atomicOr(err, ERR_KV_RANGE);
    __syncthreads();
    unsigned long long starts = s_starts[0] | (unsigned long long)s_starts[1] << 32;
    const int runs = __popcll(starts);
    const bool each = runs >= APPEND_THREADS / 32;
    const AppendSide &src = value ? v : k;
    for (int i = 0; i < runs; i++) {
        const int at = __ffsll(starts) - 1;
        starts &= starts - 1;
        if (each && i % (APPEND_THREADS / 32) != warp) continue;
        const int s = s_slot[1 + at], room = (1 << log_block) - (s & ((1 << log_block) - 1));
        int n = room;  // tokens: the slots that follow on within the block
        for (int j = lane; j < room; j += 32)
            if (s_slot[1 + at + j] != s + j) {
                n = j;
                break;
            }
        for (int d = 16; d; d >>= 1) n = min(n, __shfl_xor_sync(~0u, n, d));
        const Run r{first + at, n, s & ((1 << log_block) - 1), s >> log_block};
        append_run<TYPE, VEC>(r, src, value, head, each ? lane : tid,
                              each ? 32 : APPEND_THREADS, codes, scales, n_heads, 1 << log_block,
                              dim, dim_p, red);
    }
}

// ---------------------------------------------------------------- copies in and out

constexpr int COPY_THREADS = 256;

// Bytes of the keys' half of every group 0 (code 0), of the values' half 128 (code 0).
__global__ void clear_kernel(uint4 *codes, size_t n16, int dim_p) {
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n16;
         i += (size_t)gridDim.x * blockDim.x) {
        const uint32_t w = i % (2 * (size_t)dim_p) < (size_t)dim_p ? 0u : 0x80808080u;
        codes[i] = make_uint4(w, w, w, w);
    }
}

enum { COPY_IMPORT, COPY_EXPORT, COPY_READ };

// One thread a 16-byte patch of codes (a key patch: 16 dims of a token; a value patch: 4 dims of
// 4 tokens). MODE COPY_READ writes 64 bytes of f32 values for it, which bounds the kernel: 257
// blocks of 64 tokens and 8 heads of 128 dims take 34 us, 5.0 TB/s.
template <int MODE, int DP>
__global__ void __launch_bounds__(COPY_THREADS)
    copy_kernel(const int32_t *__restrict__ blocks, uint8_t *__restrict__ codes,
                float2 *__restrict__ scales, int n_blocks, int n_heads, int block_tokens, int dim,
                void *__restrict__ k_any, void *__restrict__ v_any,
                float *__restrict__ k_scales, float *__restrict__ v_scales, int *err) {
    constexpr int dim_p = DP;
    const int head = blockIdx.y;
    const size_t i = blockIdx.x;
    pdl_enter();
    const int id = __ldg(blocks + i);
    if (id < 0 || id >= n_blocks) {
        if (threadIdx.x == 0) atomicOr(err, ERR_KV_RANGE);
        return;
    }
    const size_t bh = (size_t)id * n_heads + head, out_bh = i * n_heads + head;
    uint8_t *page = codes + bh * (size_t)block_tokens * 2 * dim_p;
    const size_t out0 = out_bh * (size_t)block_tokens * dim;
    float2 s = make_float2(0.f, 0.f);
    if (MODE != COPY_IMPORT) s = scales[bh];
    if (threadIdx.x == 0 && MODE == COPY_IMPORT) scales[bh] = make_float2(k_scales[out_bh],
                                                                          v_scales[out_bh]);
    if (threadIdx.x == 0 && MODE == COPY_EXPORT) {
        k_scales[out_bh] = s.x;
        v_scales[out_bh] = s.y;
    }
    const int total = block_tokens / KV_GROUP * 2 * dim_p;
#pragma unroll 2
    for (int p = threadIdx.x; p < total; p += COPY_THREADS) {
        const int grp = p / (2 * dim_p);
        int q = p - grp * 2 * dim_p;
        uint4 *at = reinterpret_cast<uint4 *>(page) + p;
        const bool value = q >= dim_p;
        if (value) q -= dim_p;
        // (token, dim) of the patch's byte `b`: keys token kt, dims kd ..; values 4 x 4
        const int kc = q >> 4, kt = 8 * (q / (dim_p >> 1)) + ((q % (dim_p >> 1)) & 15) / 2;
        const int kd = 32 * (kc % (dim_p >> 5)) + 16 * (q & 1);
        const int vrow = (q >> 3) & 3, vt = 2 * vrow;
        const int vd = 32 * (q >> 5) + 4 * ((q & 7) ^ vt);
        uint32_t w[4] = {0, 0, 0, 0};
        if (MODE != COPY_IMPORT) {
            const uint4 x = *at;
            w[0] = x.x;
            w[1] = x.y;
            w[2] = x.z;
            w[3] = x.w;
        }
        if (!value) {
            const size_t o = out0 + (size_t)(grp * KV_GROUP + kt) * dim + kd;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (kd + 4 * k >= dim) continue;
                if (MODE == COPY_IMPORT) {
                    w[k] = __ldg(reinterpret_cast<const uint32_t *>((const int8_t *)k_any + o +
                                                                    4 * k));
                } else if (MODE == COPY_EXPORT) {
                    *reinterpret_cast<uint32_t *>((int8_t *)k_any + o + 4 * k) = w[k];
                } else {
                    float4 f;
                    f.x = __fmul_rn((float)(int8_t)(w[k] & 255), s.x);
                    f.y = __fmul_rn((float)(int8_t)(w[k] >> 8 & 255), s.x);
                    f.z = __fmul_rn((float)(int8_t)(w[k] >> 16 & 255), s.x);
                    f.w = __fmul_rn((float)(int8_t)(w[k] >> 24), s.x);
                    *reinterpret_cast<float4 *>((float *)k_any + o + 4 * k) = f;
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {  // token vt + (k & 1) + 8 (k >> 1): byte k of each word
                const size_t o =
                    out0 + (size_t)(grp * KV_GROUP + vt + (k & 1) + 8 * (k >> 1)) * dim + vd;
                if (MODE == COPY_IMPORT) {
                    uint32_t x = 0;
                    if (vd < dim)
                        x = __ldg(reinterpret_cast<const uint32_t *>((const int8_t *)v_any + o));
                    x ^= 0x80808080u;
#pragma unroll
                    for (int j = 0; j < 4; j++) w[j] |= ((x >> (8 * j)) & 255) << (8 * k);
                    continue;
                }
                if (vd >= dim) continue;
                int c[4];
#pragma unroll
                for (int j = 0; j < 4; j++) c[j] = (int)((w[j] >> (8 * k)) & 255) - 128;
                if (MODE == COPY_EXPORT)
                    *reinterpret_cast<uint32_t *>((int8_t *)v_any + o) =
                        pack4(c[0], c[1], c[2], c[3]);
                else
                    *reinterpret_cast<float4 *>((float *)v_any + o) = make_float4(
                        __fmul_rn((float)c[0], s.y), __fmul_rn((float)c[1], s.y),
                        __fmul_rn((float)c[2], s.y), __fmul_rn((float)c[3], s.y));
            }
        }
        if (MODE == COPY_IMPORT) *at = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

size_t type_bytes(int type) {
    return type == JKB_F32 ? 4 : type == JKB_F16 || type == JKB_BF16 ? 2 : 0;
}

int check_copy(const jkb_kv_cache *c, const int32_t *blocks, size_t n, const void *a,
               const void *b, size_t align, const char *fn) {
    int rc = check_kv_cache(c, fn);
    if (rc) return rc;
    if (n > c->n_blocks)
        return fail(JKB_E_BOUNDS, fn, 0, n, c->n_blocks, "%s: %zu blocks of a cache of %zu", fn, n,
                    c->n_blocks);
    if (n && (!blocks || !a || !b)) return fail(JKB_E_INVALID, fn, 0, 0, 0, "null pointer");
    if ((rc = check_align(blocks, 4, fn, "blocks")) || (rc = check_align(a, align, fn, "keys")) ||
        (rc = check_align(b, align, fn, "values")))
        return rc;
    return JKB_OK;
}

template <int MODE>
int copy_launch(const jkb_kv_cache *c, const int32_t *blocks, size_t n, void *k, void *v,
                float *ks, float *vs, void *stream, const char *fn) {
    if (n == 0) return JKB_OK;
    int *err = device_error_word();
    if (!err) return fail(JKB_E_CUDA, fn, 0, 0, 0, "no device error word");
    auto go = [&](auto kern) {
        return launch_pdl(kern, dim3((unsigned)n, (unsigned)c->n_heads), dim3(COPY_THREADS), 0,
                          as_stream(stream), blocks, c->codes, c->scales, (int)c->n_blocks,
                          (int)c->n_heads, c->block_tokens, c->dim, k, v, ks, vs, err);
    };
    cudaError_t e = c->dim_p == 64    ? go(copy_kernel<MODE, 64>)
                    : c->dim_p == 96  ? go(copy_kernel<MODE, 96>)
                    : c->dim_p == 128 ? go(copy_kernel<MODE, 128>)
                    : c->dim_p == 192 ? go(copy_kernel<MODE, 192>)
                                      : go(copy_kernel<MODE, 256>);
    return e == cudaSuccess ? JKB_OK : fail_cuda(e, fn);
}

// Whether n ints at p share an element with `rows` rows of `width`, `stride` apart, at `table`.
bool overlaps(const int32_t *table, size_t rows, size_t width, size_t stride, const int32_t *p,
              size_t n) {
    if (!rows || !width || !n) return false;
    const uintptr_t a = (uintptr_t)table / 4, b = (uintptr_t)p / 4;
    if (b < a) return n > a - b;
    if (b - a >= (rows - 1) * stride + width) return false;
    const size_t col = (b - a) % stride;
    return col < width || n > stride - col;
}

// The kernel reads its inputs again after other CTAs have written their outputs, so no output may
// share memory with an input or another output.
int check_tables_apart(const jkb_kv_tables_args *a, const char *fn) {
    const struct {
        const int32_t *p;
        size_t n;
        const char *name;
    } list[] = {{a->slots, a->n_slots, "slots"},         {a->positions, a->n_slots, "positions"},
                {a->q_starts, a->n_seqs + 1, "q_starts"}, {a->kv_lens, a->n_seqs, "kv_lens"},
                {a->counts, 3, "counts"},                 {a->ctx_lens, a->n_seqs, "ctx_lens"},
                {a->new_lens, a->n_seqs, "new_lens"},     {a->free_blocks, a->n_free, "free_blocks"}};
    constexpr int N = sizeof(list) / sizeof(list[0]), OUTPUTS = 5;
    for (int i = 0; i < N; i++) {
        if (overlaps(a->block_table, a->n_seqs, a->row_blocks, a->table_stride, list[i].p,
                     list[i].n))
            return fail(JKB_E_BOUNDS, fn, 0, 0, 0, "%s overlaps block_table", list[i].name);
        for (int j = 0; j < i && j < OUTPUTS; j++)
            if (overlaps(list[j].p, 1, list[j].n, list[j].n, list[i].p, list[i].n))
                return fail(JKB_E_BOUNDS, fn, 0, 0, 0, "%s overlaps %s", list[i].name,
                            list[j].name);
    }
    return JKB_OK;
}

int log2_block(size_t b) { return b == 16 ? 4 : b == 32 ? 5 : b == 64 ? 6 : b == 128 ? 7 : -1; }

}  // namespace

int check_kv_cache(const jkb_kv_cache *c, const char *fn) {
    if (!c || c->magic != KV_MAGIC)
        return fail(JKB_E_INVALID, fn, 0, 0, 0, "null or destroyed kv cache handle");
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev != c->device)
        return fail(JKB_E_INVALID, fn, 0, (size_t)dev, (size_t)c->device,
                    "%s: the cache is on device %d, the current device is %d", fn, c->device, dev);
    return JKB_OK;
}

}  // namespace jkb

using namespace jkb;

extern "C" {

int jkb_kv_cache_create(size_t n_blocks, size_t block_tokens, size_t n_kv_heads, size_t head_dim,
                        jkb_kv_cache **out) {
    static const char *fn = "kv_cache";
    if (!out) return fail(JKB_E_INVALID, fn, 0, 0, 0, "null out");
    *out = nullptr;
    if (log2_block(block_tokens) < 0)
        return fail(JKB_E_BOUNDS, fn, 0, block_tokens, 128,
                    "block_tokens %zu is not 16, 32, 64 or 128", block_tokens);
    if (head_dim == 0 || head_dim > 256 || head_dim % 8)
        return fail(JKB_E_BOUNDS, fn, 0, head_dim, 256,
                    "head_dim %zu is not a multiple of 8 in 8..256", head_dim);
    if (n_kv_heads == 0 || n_kv_heads > 65535)
        return fail(JKB_E_BOUNDS, fn, 0, n_kv_heads, 65535, "n_kv_heads %zu outside 1..65535",
                    n_kv_heads);
    if (n_blocks == 0 || n_blocks > (size_t)INT32_MAX / block_tokens)
        return fail(JKB_E_BOUNDS, fn, 0, n_blocks, (size_t)INT32_MAX / block_tokens,
                    "n_blocks %zu outside 1..%zu", n_blocks, (size_t)INT32_MAX / block_tokens);
    jkb_kv_cache *c = (jkb_kv_cache *)calloc(1, sizeof(jkb_kv_cache));
    if (!c) return fail(JKB_E_INVALID, fn, 0, 0, 0, "host allocation failed");
    c->n_blocks = n_blocks;
    c->n_heads = n_kv_heads;
    c->block_tokens = (int)block_tokens;
    c->dim = (int)head_dim;
    c->dim_p = head_dim <= 64 ? 64 : head_dim <= 96 ? 96 : head_dim <= 128 ? 128
               : head_dim <= 192 ? 192 : 256;
    const size_t code_bytes = n_blocks * n_kv_heads * block_tokens * 2 * (size_t)c->dim_p;
    const size_t bytes = Arena::round(code_bytes) + n_blocks * n_kv_heads * sizeof(float2);
    uint8_t *base = nullptr;
    cudaError_t e = cudaGetDevice(&c->device);
    if (e == cudaSuccess) e = cudaMalloc(&base, bytes);
    if (e != cudaSuccess) {
        cudaGetLastError();
        free(c);
        return fail_cuda(e, fn);
    }
    c->device_bytes = bytes;
    c->codes = base;
    c->scales = (float2 *)(base + Arena::round(code_bytes));
    clear_kernel<<<1184, 256>>>((uint4 *)base, code_bytes / 16, c->dim_p);
    e = cudaGetLastError();
    if (e == cudaSuccess)
        e = cudaMemset(c->scales, 0, n_blocks * n_kv_heads * sizeof(float2));
    if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
    if (e != cudaSuccess) {
        cudaFree(base);
        free(c);
        return fail_cuda(e, fn);
    }
    c->magic = KV_MAGIC;
    *out = c;
    return JKB_OK;
}

int jkb_kv_cache_destroy(jkb_kv_cache *c) {
    if (!c) return JKB_OK;
    if (c->magic != KV_MAGIC)
        return fail(JKB_E_INVALID, "kv_cache", 0, 0, 0, "null or destroyed kv cache handle");
    c->magic = 0;
    cudaFree(c->codes);
    free(c);
    return JKB_OK;
}

int jkb_kv_cache_info(const jkb_kv_cache *c, size_t *n_blocks, size_t *block_tokens,
                      size_t *n_kv_heads, size_t *head_dim, size_t *device_bytes) {
    if (!c || c->magic != KV_MAGIC)
        return fail(JKB_E_INVALID, "kv_cache", 0, 0, 0, "null or destroyed kv cache handle");
    if (n_blocks) *n_blocks = c->n_blocks;
    if (block_tokens) *block_tokens = (size_t)c->block_tokens;
    if (n_kv_heads) *n_kv_heads = c->n_heads;
    if (head_dim) *head_dim = (size_t)c->dim;
    if (device_bytes) *device_bytes = c->device_bytes;
    return JKB_OK;
}

int jkb_kv_cache_import(jkb_kv_cache *c, const int32_t *blocks, size_t n, const int8_t *k_codes,
                        const int8_t *v_codes, const float *k_scales, const float *v_scales,
                        void *stream) {
    static const char *fn = "kv_cache_import";
    int rc = check_copy(c, blocks, n, k_codes, v_codes, 4, fn);
    if (rc) return rc;
    if (n && (!k_scales || !v_scales)) return fail(JKB_E_INVALID, fn, 0, 0, 0, "null pointer");
    if ((rc = check_align(k_scales, 4, fn, "k_scales")) ||
        (rc = check_align(v_scales, 4, fn, "v_scales")))
        return rc;
    return copy_launch<COPY_IMPORT>(c, blocks, n, const_cast<int8_t *>(k_codes),
                                    const_cast<int8_t *>(v_codes), const_cast<float *>(k_scales),
                                    const_cast<float *>(v_scales), stream, fn);
}

int jkb_kv_cache_export(const jkb_kv_cache *c, const int32_t *blocks, size_t n, int8_t *k_codes,
                        int8_t *v_codes, float *k_scales, float *v_scales, void *stream) {
    static const char *fn = "kv_cache_export";
    int rc = check_copy(c, blocks, n, k_codes, v_codes, 4, fn);
    if (rc) return rc;
    if (n && (!k_scales || !v_scales)) return fail(JKB_E_INVALID, fn, 0, 0, 0, "null pointer");
    if ((rc = check_align(k_scales, 4, fn, "k_scales")) ||
        (rc = check_align(v_scales, 4, fn, "v_scales")))
        return rc;
    return copy_launch<COPY_EXPORT>(c, blocks, n, k_codes, v_codes, k_scales, v_scales, stream,
                                    fn);
}

int jkb_kv_cache_read(const jkb_kv_cache *c, const int32_t *blocks, size_t n, float *k_out,
                      float *v_out, void *stream) {
    static const char *fn = "kv_cache_read";
    const int rc = check_copy(c, blocks, n, k_out, v_out, 16, fn);
    if (rc) return rc;
    return copy_launch<COPY_READ>(c, blocks, n, k_out, v_out, nullptr, nullptr, stream, fn);
}

int jkb_kv_append(jkb_kv_cache *c, const jkb_rows *k, const jkb_rows *v, const int32_t *slots,
                  size_t n_tokens, void *stream) {
    static const char *fn = "kv_append";
    int rc = check_kv_cache(c, fn);
    if (rc) return rc;
    if (n_tokens == 0) return JKB_OK;
    if (!k || !v || !slots || !k->data || !v->data)
        return fail(JKB_E_INVALID, fn, 0, 0, 0, "null pointer");
    const size_t eb = type_bytes(k->type);
    if (!eb || v->type != k->type)
        return fail(JKB_E_CAPABILITY, fn, 0, 0, 0,
                    "key rows of type %s and value rows of type %s: F32, F16 or BF16, both alike",
                    quant_name(k->type), quant_name(v->type));
    if (n_tokens > (size_t)INT32_MAX - 256)
        return fail(JKB_E_BOUNDS, fn, 0, n_tokens, INT32_MAX, "%zu tokens in one call", n_tokens);
    bool vec = true;
    for (const jkb_rows *r : {k, v}) {
        if ((rc = check_align(r->data, eb, fn, r == k ? "keys" : "values"))) return rc;
        vec &= ((uintptr_t)r->data % (4 * eb)) == 0 && r->token_stride % 4 == 0 &&
               r->head_stride % 4 == 0;
    }
    if ((rc = check_align(slots, 4, fn, "slots"))) return rc;
    int *err = device_error_word();
    if (!err) return fail(JKB_E_CUDA, fn, 0, 0, 0, "no device error word");
    // tokens a CTA: 64 where that still gives every SM several CTAs, else 4 (a warp each)
    const int span = n_tokens * c->n_heads / 32 >= (size_t)num_sms() * 2 ? 64 : 4;
    const dim3 grid((unsigned)((n_tokens + span - 1) / span), (unsigned)c->n_heads, 2);
    const AppendSide ks{k->data, k->token_stride, k->head_stride};
    const AppendSide vs{v->data, v->token_stride, v->head_stride};
    const long long n_slots = (long long)c->n_blocks * c->block_tokens;
    auto go = [&](auto kern) {
        return launch_pdl(kern, grid, dim3(APPEND_THREADS), 0, as_stream(stream), ks, vs, slots,
                          (int)n_tokens, span, c->codes, c->scales, n_slots, (int)c->n_heads,
                          log2_block((size_t)c->block_tokens), c->dim, c->dim_p, err);
    };
    cudaError_t e;
    if (k->type == JKB_F32)
        e = vec ? go(append_kernel<JKB_F32, true>) : go(append_kernel<JKB_F32, false>);
    else if (k->type == JKB_F16)
        e = vec ? go(append_kernel<JKB_F16, true>) : go(append_kernel<JKB_F16, false>);
    else
        e = vec ? go(append_kernel<JKB_BF16, true>) : go(append_kernel<JKB_BF16, false>);
    return e == cudaSuccess ? JKB_OK : fail_cuda(e, fn);
}

int jkb_kv_build_tables(const jkb_kv_tables_args *a, void *stream) {
    static const char *fn = "kv_build_tables";
    if (!a) return fail(JKB_E_INVALID, fn, 0, 0, 0, "null arguments");
    const int lb = log2_block(a->block_tokens);
    if (lb < 0)
        return fail(JKB_E_BOUNDS, fn, 0, a->block_tokens, 128,
                    "block_tokens %zu is not 16, 32, 64 or 128", a->block_tokens);
    if (a->n_seqs > JKB_KV_MAX_SEQS)
        return fail(JKB_E_BOUNDS, fn, 0, a->n_seqs, JKB_KV_MAX_SEQS, "%zu sequences, at most %d",
                    a->n_seqs, JKB_KV_MAX_SEQS);
    if (a->row_blocks > (size_t)INT32_MAX / a->block_tokens || a->table_stride < a->row_blocks)
        return fail(JKB_E_BOUNDS, fn, 0, a->row_blocks, a->table_stride,
                    "table rows of %zu blocks, %zu apart", a->row_blocks, a->table_stride);
    if (a->n_slots > (size_t)INT32_MAX - 4 || a->n_free > (size_t)INT32_MAX)
        return fail(JKB_E_BOUNDS, fn, 0, a->n_slots, INT32_MAX, "%zu slots, %zu free blocks",
                    a->n_slots, a->n_free);
    if (!a->q_starts || !a->counts || (a->n_slots && (!a->slots || !a->positions)) ||
        (a->n_free && !a->free_blocks) ||
        (a->n_seqs &&
         (!a->kv_lens || !a->ctx_lens || !a->new_lens || (a->row_blocks && !a->block_table))))
        return fail(JKB_E_INVALID, fn, 0, 0, 0, "null pointer");
    const void *ptrs[] = {a->block_table, a->slots,    a->positions, a->q_starts,   a->kv_lens,
                          a->counts,      a->ctx_lens, a->new_lens,  a->free_blocks};
    for (const void *p : ptrs)
        if (int rc = check_align(p, 4, fn, "int32")) return rc;
    if (int rc = check_tables_apart(a, fn)) return rc;
    const size_t smem = (2 * a->n_seqs + 1) * 4;
    if (smem > 48 * 1024) {  // always to the same value: it is one for all threads of the process
        cudaError_t e = cudaFuncSetAttribute(tables_kernel,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (2 * JKB_KV_MAX_SEQS + 1) * 4);
        if (e != cudaSuccess) return fail_cuda(e, fn);
    }
    const size_t want = (a->n_slots + 4 * TABLE_THREADS - 1) / (4 * TABLE_THREADS);
    const size_t most = 2 * (size_t)num_sms();
    const unsigned grid = (unsigned)(want < 1 ? 1 : want > most ? most : want);
    int *err = device_error_word();
    if (!err) return fail(JKB_E_CUDA, fn, 0, 0, 0, "no device error word");
    cudaError_t e = launch_pdl(tables_kernel, dim3(grid), dim3(TABLE_THREADS), smem,
                               as_stream(stream), a->block_table, (int)a->n_seqs,
                               (int)a->row_blocks, a->table_stride, a->slots, a->positions,
                               (int)a->n_slots, a->q_starts, a->kv_lens, a->counts, a->ctx_lens,
                               a->new_lens, a->free_blocks, (int)a->n_free, lb, err);
    return e == cudaSuccess ? JKB_OK : fail_cuda(e, fn);
}

}  // extern "C"
