// hxq_kv8: a key/value cache held in 8 bits - rotary embedding + append of new rows (one token a sequence, or packed
// prompts), single-query grouped attention over it, and its rows back as bf16.  No counterpart in the reference,
// whose decode loop keeps the framework's 16-bit cache (helix_substrate/basin_runtime.py:358-445).
//
// Per (sequence, KV head) the positions form blocks of 64.  A finished block holds codes x = s * code with
//     s = max(up(max |x| / 127), 2^-126),   code = rint(x / s) in -127 .. 127,
// up() rounding up to bf16.  x and s then both have 8 significant bits, so x / s is a tie exactly or at least
// 1/510 off one: x times the rounded reciprocal, snapped to multiples of 1/1024, decides every code as exact arithmetic
// would.  A block with an infinity or a NaN gets s = NaN and reads back as NaN.  The rows of the last, unfinished
// block stay bf16 in the tail (row = position mod 64) and are quantised once, when the 64th arrives: no row is ever
// rounded twice, and what a cache holds does not depend on how a prompt was cut into calls.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <utility>

#include "hxq_common.cuh"

namespace hxq {
namespace kv8 {

constexpr int kBlock = HXQ_KV8_BLOCK;

__device__ __forceinline__ void pdl_enter() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename... KArgs, typename... Args>
static cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, cudaStream_t stream, size_t smem, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = stream;
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

struct Cache {
    int8_t *k, *v;
    float *ks, *vs;
    __nv_bfloat16 *kt, *vt;
    int nkv, D, max_len;
};
static Cache cache_of(const hxq_kv8* c) {
    return Cache{c->k, c->v, c->k_scale, c->v_scale, reinterpret_cast<__nv_bfloat16*>(c->k_tail),
                 reinterpret_cast<__nv_bfloat16*>(c->v_tail), c->nkv, c->D, c->max_len};
}

__device__ __forceinline__ void unpack8(const uint4& q, float (&f)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f[2 * e] = __uint_as_float(w[e] << 16);
        f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const __nv_bfloat162 h2 = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&h2);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 ld16(const void* p) { return *reinterpret_cast<const uint4*>(p); }

// Rotary embedding of the pieces at d and d + D / 2 of one head, packed bf16 in and out: x cos + y sin as 64-bit arithmetic
// has it (its products are exact there), rounded to fp32 and to bf16, so that a value next to a border lands on the side it is
// on.  Nearly always fp32 tells the same: r = fma(x, cos, fl(y sin)) is off by 2^-24 (|y sin| + |r|) at most and the
// true sum's fp32 value by one more rounding, so where r - d and r + d, d = 2^-23 (|y sin| + |r|), round to the same bf16, that is
// it.  One value in some 2^13 takes the 64-bit path.  (All in 64 bits, conversions alone filled half of the time: 86 us for 8191
// tokens of 28 + 4 heads where this takes 36; exact sums of products and their rests in packed fp32 took 42 to 48 when this took 41.)
__device__ __forceinline__ uint32_t turn(float x, float c, float y, float s, bool& sure) {
    const float p = y * s, r = fmaf(x, c, p);
    const float d = fmaf(fabsf(p) + fabsf(r), 1.0001f * 1.1920929e-7f, 2.8e-45f);
    const __nv_bfloat162 h = __floats2bfloat162_rn(r - d, r + d);
    const uint32_t v = *reinterpret_cast<const uint32_t*>(&h);
    sure = sure && v == __byte_perm(v, v, 0x1010);
    return v;
}
__device__ __forceinline__ uint32_t turn_exactly(float x, float c, float y, float s) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(__double2float_rn((double)x * (double)c + (double)y * (double)s)));
}
struct Angles {          // cos and sin of eight dimensions of the lower and of the upper half
    float c0[8], s0[8], c1[8], s1[8];
    __device__ __forceinline__ Angles(const float* cos_row, const float* sin_row, int d, int half) {
        const float* from[4] = {cos_row + d, sin_row + d, cos_row + d + half, sin_row + d + half};
        float* to[4] = {c0, s0, c1, s1};
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const float4 v = *reinterpret_cast<const float4*>(from[k] + 4 * q);
                to[k][4 * q] = v.x; to[k][4 * q + 1] = v.y; to[k][4 * q + 2] = v.z; to[k][4 * q + 3] = v.w;
            }
    }
};
__device__ __forceinline__ void rotate16(uint4& lo, uint4& hi, const Angles& a) {
    float x0[8], x1[8];
    unpack8(lo, x0);
    unpack8(hi, x1);
    uint32_t l[4], h[4];
    bool sure = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        l[e] = __byte_perm(turn(x0[2 * e], a.c0[2 * e], -x1[2 * e], a.s0[2 * e], sure), turn(x0[2 * e + 1], a.c0[2 * e + 1], -x1[2 * e + 1], a.s0[2 * e + 1], sure), 0x5410);
        h[e] = __byte_perm(turn(x1[2 * e], a.c1[2 * e], x0[2 * e], a.s1[2 * e], sure), turn(x1[2 * e + 1], a.c1[2 * e + 1], x0[2 * e + 1], a.s1[2 * e + 1], sure), 0x5410);
    }
    if (!sure) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            l[e] = turn_exactly(x0[2 * e], a.c0[2 * e], -x1[2 * e], a.s0[2 * e]) | turn_exactly(x0[2 * e + 1], a.c0[2 * e + 1], -x1[2 * e + 1], a.s0[2 * e + 1]) << 16;
            h[e] = turn_exactly(x1[2 * e], a.c1[2 * e], x0[2 * e], a.s1[2 * e]) | turn_exactly(x1[2 * e + 1], a.c1[2 * e + 1], x0[2 * e + 1], a.s1[2 * e + 1]) << 16;
        }
    }
    lo = make_uint4(l[0], l[1], l[2], l[3]);
    hi = make_uint4(h[0], h[1], h[2], h[3]);
}
// Largest magnitudes of two bf16 pairs; NaN wins.
__device__ __forceinline__ uint32_t abs_max2(uint32_t m, uint32_t x) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(x & 0x7fff7fffu));
    return r;
}

// ---- append -----------------------------------------------------------------------------------------

struct AppendArgs {
    Cache c;
    const __nv_bfloat16* qkv;
    const int32_t* cu;       // rows of qkv per sequence, or nullptr: row s is sequence s's only token
    const int64_t* pos;      // position of each sequence's first new row (< 0: the sequence is left alone)
    const float *cos_t, *sin_t;
    __nv_bfloat16 *q_out, *k_out;
    int64_t ld_qkv, ld_q, ld_k;
    int pos_stride, T, S, max_q, nq, groups;        // groups: of kHeadsPrompt or kHeadsStep query heads
};

constexpr int kAppendThreads = 256;
constexpr int kMaxD = 128;
constexpr int kHeadsPrompt = 4, kHeadsStep = 2;       // query heads of a thread: few for a single token, whose time is one thread's
constexpr int kUnits = 4 * kMaxD / kAppendThreads;      // pairs of eight-element pieces a thread holds of a block

// Sequence s: its first row of qkv, the number of its new rows that have a place in the cache, its first position.
__device__ __forceinline__ int sequence(const AppendArgs& a, int s, int& row0, int64_t& p0) {
    p0 = a.pos[(int64_t)s * a.pos_stride];
    int r0 = s, r1 = s + 1;
    if (a.cu != nullptr) {
        r0 = a.cu[s];
        r1 = a.cu[s + 1];
    }
    if (r0 < 0) r0 = 0;
    if (r1 > a.T) r1 = a.T;
    row0 = r0;
    if (p0 < 0 || p0 >= a.c.max_len || r1 <= r0) return 0;       // (a position past the cache may be any number)
    const int n = r1 - r0 < a.max_q ? r1 - r0 : a.max_q, room = a.c.max_len - (int)p0;
    return n < room ? n : room;
}

// One block of one KV head's keys or values: rows from r_old on are new, rows before it stand in the tail.
// A whole block is quantised, of an unfinished one the new rows go to the tail.
__device__ void append_block(const AppendArgs& a, bool is_k, int s, int h, int blk, int row0, int64_t p0, int n, uint32_t* red) {
    const int D = a.c.D, half = D >> 1, pieces = D >> 4;
    const int64_t b0 = (int64_t)blk * kBlock;
    const int r_old = p0 > b0 ? (int)(p0 - b0) : 0;
    const int r_end = p0 + n - b0 < kBlock ? (int)(p0 + n - b0) : kBlock;
    const bool whole = r_end == kBlock;
    const int64_t head = (int64_t)s * a.c.nkv + h;
    __nv_bfloat16* tail = (is_k ? a.c.kt : a.c.vt) + head * kBlock * D;
    const int col = (a.nq + (is_k ? 0 : a.c.nkv) + h) * D;

    uint4 lo[kUnits], hi[kUnits];
    uint32_t most = 0u;
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const int u = threadIdx.x + j * kAppendThreads;
        const int r = u / pieces, d = (u - r * pieces) * 8;
        lo[j] = hi[j] = make_uint4(0u, 0u, 0u, 0u);
        if (r >= r_end || (!whole && r < r_old)) continue;
        if (r < r_old) {
            lo[j] = ld16(tail + r * D + d);
            hi[j] = ld16(tail + r * D + d + half);
        } else {
            const __nv_bfloat16* src = a.qkv + (row0 + (b0 + r - p0)) * a.ld_qkv + col;
            lo[j] = ld16(src + d);
            hi[j] = ld16(src + d + half);
        }
    }
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const int u = threadIdx.x + j * kAppendThreads;
        const int r = u / pieces, d = (u - r * pieces) * 8;
        if (r >= r_end || r < r_old) continue;            // a new row
        const int64_t p = b0 + r, t = row0 + (p - p0);
        if (is_k) {
            rotate16(lo[j], hi[j], Angles(a.cos_t + p * D, a.sin_t + p * D, d, half));
            if (a.k_out != nullptr) {
                __nv_bfloat16* dst = a.k_out + t * a.ld_k + h * D + d;
                *reinterpret_cast<uint4*>(dst) = lo[j];
                *reinterpret_cast<uint4*>(dst + half) = hi[j];
            }
        }
        if (!whole) {
            *reinterpret_cast<uint4*>(tail + r * D + d) = lo[j];
            *reinterpret_cast<uint4*>(tail + r * D + d + half) = hi[j];
        }
    }
    if (!whole) return;
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const uint32_t w[8] = {lo[j].x, lo[j].y, lo[j].z, lo[j].w, hi[j].x, hi[j].y, hi[j].z, hi[j].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) most = abs_max2(most, w[e]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = abs_max2(most, __shfl_xor_sync(0xffffffffu, most, o));
    most = abs_max2(most, most >> 16);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) most = abs_max2(most, red[w]);
    __syncthreads();                 // (red is used again, and the tail's rows have been read)
    const float amax = __uint_as_float(most << 16);
    const bool bad = !(amax <= 3.4e38f);
    float scale = __uint_as_float((__float_as_uint(__fdiv_rn(amax, 127.f)) + 0xffffu) & 0xffff0000u);
    scale = fmaxf(scale, 1.17549435e-38f);
    int8_t* codes = (is_k ? a.c.k : a.c.v) + (head * a.c.max_len + b0) * D;
    if (threadIdx.x == 0) (is_k ? a.c.ks : a.c.vs)[head * (a.c.max_len / kBlock) + blk] = bad ? __uint_as_float(0x7fc00000u) : scale;
    // x / s is a tie exactly or at least 1/510 off one (both have 8 significant bits): x * fl(1 / s), off by 2^-16 at most, is
    // snapped to multiples of 1/1024, where ties are ties again, and then rounded; the code is the low byte of 1.5 * 2^23 + it.
    const float inv = bad ? 0.f : __fdiv_rn(1.f, scale);
    auto code = [&](float x) {
        const float q = bad ? 0.f : __fadd_rn(__fmaf_rn(x, inv, 12288.f), -12288.f);
        return __float_as_uint(__fadd_rn(q, 12582912.f));
    };
    auto codes4 = [&](uint32_t w0, uint32_t w1) {
        const uint32_t c0 = code(__uint_as_float(w0 << 16)), c1 = code(__uint_as_float(w0 & 0xffff0000u));
        const uint32_t c2 = code(__uint_as_float(w1 << 16)), c3 = code(__uint_as_float(w1 & 0xffff0000u));
        return __byte_perm(__byte_perm(c0, c1, 0x0040), __byte_perm(c2, c3, 0x0040), 0x5410);
    };
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        const int u = threadIdx.x + j * kAppendThreads;
        const int r = u / pieces, d = (u - r * pieces) * 8;
        if (r >= kBlock) continue;
        *reinterpret_cast<uint2*>(codes + r * D + d) = make_uint2(codes4(lo[j].x, lo[j].y), codes4(lo[j].z, lo[j].w));
        *reinterpret_cast<uint2*>(codes + r * D + d + half) = make_uint2(codes4(hi[j].x, hi[j].y), codes4(hi[j].z, hi[j].w));
    }
}

// The query heads h0, h0 + groups, ... (up to HEADS) of one row, the pieces at d and d + D / 2, under one set of angles.
template <int HEADS>
__device__ __forceinline__ void turn_queries(const AppendArgs& a, int64_t t, int64_t p, int h0, int d) {
    const int D = a.c.D, half = D >> 1;
    const __nv_bfloat16* src = a.qkv + t * a.ld_qkv + h0 * D + d;
    uint4 lo[HEADS], hi[HEADS];
#pragma unroll
    for (int k = 0; k < HEADS; ++k)
        if (h0 + k * a.groups < a.nq) {
            lo[k] = ld16(src + k * a.groups * D);
            hi[k] = ld16(src + k * a.groups * D + half);
        }
    const Angles angles(a.cos_t + p * D, a.sin_t + p * D, d, half);
    __nv_bfloat16* dst = a.q_out + t * a.ld_q + h0 * D + d;
#pragma unroll
    for (int k = 0; k < HEADS; ++k)
        if (h0 + k * a.groups < a.nq) {
            rotate16(lo[k], hi[k], angles);
            *reinterpret_cast<uint4*>(dst + k * a.groups * D) = lo[k];
            *reinterpret_cast<uint4*>(dst + k * a.groups * D + half) = hi[k];
        }
}

// A CTA takes one block of one sequence and either one KV head's keys or values or a group of query heads.
// STEP: one token a sequence, the CTA's block being the token's; a CTA for all query heads.
// Else the blocks that the sequences' new rows touch stand in a row, and every warp works out for itself where its CTA's lies.
// Bound by HBM for prompts (and by instructions nearly as much), by one memory round trip and the launch for single tokens.
// 8191 tokens of 28 + 4 heads: 36 us with three CTAs an SM and 4 heads a thread (a few registers spilled), 41 with two, 43 with four, 38
// with 3 or 5 heads.  32 single tokens: 3.2 us with 2 heads a thread, 4.7 with 4.
template <bool STEP>
__global__ void __launch_bounds__(kAppendThreads, STEP ? 1 : 3) append_kernel(const AppendArgs a) {
    __shared__ uint32_t red[kAppendThreads / 32];
    pdl_enter();
    const int D = a.c.D, pieces = D >> 4, lane = threadIdx.x & 31;
    const int parts = (kBlock * pieces + kAppendThreads - 1) / kAppendThreads;       // of a block, for query heads: one step of the threads each
    const int roles = (STEP ? 1 : a.groups * parts) + 2 * a.c.nkv;
    const int role = blockIdx.x % roles;
    int s = blockIdx.x / roles, row0, blk, n, first, last;
    int64_t p0;
    if (STEP) {
        n = sequence(a, s, row0, p0);
        if (n == 0) return;
        blk = first = last = (int)(p0 / kBlock);
    } else {
        const int at = s;
        if (a.S > 32) {
            // Sequence s has the places from cu[s] / 64 + 2 s on, enough wherever its rows start.  Thirty-two are looked at at a time.
            auto place = [&](int i) {
                const int r0 = a.cu[i];
                return (r0 < 0 ? 0 : (r0 > a.T ? a.T : r0)) / kBlock + 2 * i;
            };
            int lo = 0, hi = a.S;       // place(lo) <= at < place(hi)
            while (hi - lo > 1) {
                const int by = (hi - lo + 31) / 32, i = lo + (lane + 1) * by;
                lo += __popc(__ballot_sync(0xffffffffu, i < hi && place(i) <= at)) * by;
                hi = lo + by < hi ? lo + by : hi;
            }
            s = lo;
            n = sequence(a, s, row0, p0);
            if (n == 0) return;
            first = (int)(p0 / kBlock);
            last = (int)((p0 + n - 1) / kBlock);
            blk = first + at - place(s);
            if (blk < first || blk > last) return;       // (below: a place before the first sequence's, where rows of no sequence precede it)
        } else {
            int rows = 0, r0 = 0, f = 0, l = -1;
            int64_t p = 0;
            if (lane < a.S) rows = sequence(a, lane, r0, p);
            if (rows > 0) { f = (int)(p / kBlock); l = (int)((p + rows - 1) / kBlock); }
            int incl = l - f + 1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, incl > at);
            if (hit == 0u) return;
            s = __ffs(hit) - 1;
            n = __shfl_sync(0xffffffffu, rows, s);
            row0 = __shfl_sync(0xffffffffu, r0, s);
            p0 = __shfl_sync(0xffffffffu, p, s);
            first = __shfl_sync(0xffffffffu, f, s);
            last = __shfl_sync(0xffffffffu, l, s);
            blk = first + at - __shfl_sync(0xffffffffu, incl - (l - f + 1), s);
        }
    }
    if (role < roles - 2 * a.c.nkv) {
        if (STEP) {
            for (int u = threadIdx.x; u < a.groups * pieces; u += kAppendThreads) turn_queries<kHeadsStep>(a, row0, p0, u / pieces, (u % pieces) * 8);
        } else {
            const int64_t p = (int64_t)blk * kBlock + (role % parts) * (kBlock / parts) + threadIdx.x / pieces;
            if ((int)threadIdx.x < kBlock / parts * pieces && p >= p0 && p < p0 + n) turn_queries<kHeadsPrompt>(a, row0 + (p - p0), p, role / parts, (threadIdx.x % pieces) * 8);
        }
        return;
    }
    const int kv = role - (roles - 2 * a.c.nkv), h = kv >> 1;
    const bool is_k = (kv & 1) == 0;
    // An unfinished last block's rows take the place of the tail's rows that the first block takes in: where both
    // happen, the first block's CTA does one after the other.
    const bool waits = !STEP && p0 % kBlock != 0 && last != first && (p0 + n) % kBlock != 0;
    if (waits && blk == last) return;
    append_block(a, is_k, s, h, blk, row0, p0, n, red);
    if (waits && blk == first) append_block(a, is_k, s, h, last, row0, p0, n, red);
}

// ---- rows back as bf16 ------------------------------------------------------------------------------

// One block of one KV head per CTA (keys and values): 16 codes in, 32 bytes out per thread and step.
__global__ void __launch_bounds__(256) rows_kernel(const Cache c, const int64_t* __restrict__ len_p, int len_stride, int rows,
                                                   __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out,
                                                   int64_t ld_seq, int64_t ld_head, int64_t ld_row) {
    const int blk = blockIdx.x, h = blockIdx.y, s = blockIdx.z;
    pdl_enter();
    int64_t len = len_p[(int64_t)s * len_stride];
    if (len > rows) len = rows;
    if (len > c.max_len) len = c.max_len;
    const int64_t b0 = (int64_t)blk * kBlock;
    if (b0 >= len) return;
    const int64_t have = len_p[(int64_t)s * len_stride];
    const bool whole = have - b0 >= kBlock;            // (rows may cut a finished block short)
    const int n = (int)(len - b0 < kBlock ? len - b0 : kBlock);
    const int pieces = c.D >> 4;
    const int64_t head = (int64_t)s * c.nkv + h;
    const int64_t out0 = s * ld_seq + h * ld_head + b0 * ld_row;
    const float ks = whole ? c.ks[head * (c.max_len / kBlock) + blk] : 0.f, vs = whole ? c.vs[head * (c.max_len / kBlock) + blk] : 0.f;
    for (int u = threadIdx.x; u < 2 * n * pieces; u += 256) {
        const bool is_v = u >= n * pieces;
        const int w = is_v ? u - n * pieces : u;
        const int r = w / pieces, d = (w - r * pieces) * 16;
        __nv_bfloat16* dst = (is_v ? v_out : k_out) + out0 + r * ld_row + d;
        if (whole) {
            const uint4 q = ld_stream_u4((is_v ? c.v : c.k) + (head * c.max_len + b0 + r) * c.D + d);
            const uint32_t wd[4] = {q.x, q.y, q.z, q.w};
            const float sc = is_v ? vs : ks;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)(wd[2 * g + (e >> 2)] >> (8 * (e & 3))) * sc;
                *reinterpret_cast<uint4*>(dst + 8 * g) = pack8(f);
            }
        } else {
            const __nv_bfloat16* src = (is_v ? c.vt : c.kt) + (head * kBlock + r) * c.D + d;
            const uint4 a = ld16(src), b = ld16(src + 8);
            *reinterpret_cast<uint4*>(dst) = a;
            *reinterpret_cast<uint4*>(dst + 8) = b;
        }
    }
}

// ---- single-query attention -------------------------------------------------------------------------

constexpr int kWarps = 4;
constexpr int kDecodeCtas = 3;      // per SM
constexpr int kCluster = 8;
constexpr int kHeads = 8;           // query heads of a KV head: the used rows of an MMA's sixteen

// d (+)= a * b, one warp: int8 with 32 dimensions, fp16 and bf16 with 16.
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t bf2_of(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// A pair of bf16 numbers, infinities and NaNs replaced by bf16's largest.
__device__ __forceinline__ uint32_t finite2(uint32_t x) {
    uint32_t r;
    asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x7f7f7f7fu));
    asm("max.bf16x2 %0, %1, %2;" : "=r"(x) : "r"(r), "r"(0xff7fff7fu));
    return x;
}
// Two biased bytes (code + 128), picked by sel out of x, as two fp16 numbers 1024 + byte (0x64nn): the code + 1152, exactly.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t codes2(uint32_t x) { return __byte_perm(x, 0x64646464u, SEL); }
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Units of 64 positions of one sequence, the unfinished block among them.
__device__ __forceinline__ int units_of(int64_t pos, int max_len) {
    if (pos < 0 || pos >= max_len) return 0;
    return (int)(pos / kBlock) + 1;
}

struct DecodeArgs {
    Cache c;
    const __nv_bfloat16* q;
    const int64_t* pos;
    __nv_bfloat16* out;
    float* part;            // [CTAs, 2, G, D + 2]: maximum, sum, un-normalised output
    int64_t ld_q, ld_out;
    int pos_stride, B, nq, G, ctas;
    bool edges;             // more pairs than CTAs: see combine_kernel
    float scale_log2;       // scale * log2(e)
};

// The units of all (sequence, KV head) pairs in a row, sequence by sequence, head by head, each pair followed by kPad empty
// ones, which stand for what a segment costs besides its units (queries, the first copies' way, the sums' meeting; without
// them a CTA with many short pairs would be the last to finish: 32 sequences take 20.4 us with four, 19.1 with eight, 19.6 with twelve).  Where the share of a CTA starts, every warp works
// out for itself from the positions.
constexpr int kPad = 8;
struct Share {
    int64_t per;        // places per CTA
    int64_t before;     // places of the sequences before b, of one head
    int b, units;       // the sequence that holds the given place (or sequence `at`), and its units
};
// The share that place per * cta lies in, or, with at >= 0, sequence `at`.  b < 0: past the end.
__device__ __forceinline__ Share find(const DecodeArgs& a, int cta, int at, int64_t& total) {
    const int lane = threadIdx.x & 31;
    auto padded = [](int u) { return u > 0 ? u + kPad : 0; };
    auto units = [&](int b) { return b < a.B ? units_of(a.pos[(int64_t)b * a.pos_stride], a.c.max_len) : 0; };
    Share r;
    const int first = units(lane);
    int sum = padded(first), pre = lane < at ? sum : 0;         // (what a cache can hold of units stays far below 2^31)
#pragma unroll 4
    for (int b = lane + 32; b < a.B; b += 32) {
        const int u = padded(units(b));
        sum += u;
        pre += b < at ? u : 0;
    }
    total = (int64_t)__reduce_add_sync(0xffffffffu, sum) * a.c.nkv;
    r.per = (total + a.ctas - 1) / a.ctas;
    if (r.per < kWarps) r.per = kWarps;       // a unit for each warp at least
    r.b = -1; r.before = 0; r.units = 0;
    if (at >= 0) {
        r.b = at;
        r.before = __reduce_add_sync(0xffffffffu, pre);
        r.units = units(at);
        return r;
    }
    const int64_t place = r.per * cta;
    if (place >= total) return r;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        const int u = b0 == 0 ? first : units(b0 + lane);
        int incl = padded(u);
        if (b0 + 32 < a.B) {
            const int all = __reduce_add_sync(0xffffffffu, incl);
            if ((r.before + all) * a.c.nkv <= place) {
                r.before += all;
                continue;
            }
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, (r.before + incl) * a.c.nkv > place);
        if (hit == 0u) return r;        // (positions that change meanwhile)
        const int l = __ffs(hit) - 1;
        r.b = b0 + l;
        r.units = __shfl_sync(0xffffffffu, u, l);
        r.before += __shfl_sync(0xffffffffu, incl - padded(u), l);
        return r;
    }
    return r;
}

// Every CTA takes the same share of all units, whatever the sequences' lengths: a few segments, each of one sequence and
// KV head with all of its (up to eight) query heads.  In a segment a warp takes units of 64 positions in turn.  A segment
// that is a whole pair writes the output, the others partial results, which the next launch joins.
// CLUSTER, for few pairs and short caches: a pair has a cluster of eight CTAs, whose results meet over their shared
// memories, and there is no next launch.
//
// Bound by HBM: each code is read once, 2 D bytes a position and KV head.  On the CUDA cores G query heads cost G
// multiply-adds a code, more than the cores have at the memory's pace from G = 5 on, so both products go through
// mma.sync (a tcgen05 tile would want 128 rows of queries; there are eight).
//   * Q K^T runs in int8, the codes as they are.  A query row is rounded to 16 bits, off by 2^-16 of its largest element at
//     most (bf16's rounding is 2^-8 of each: elements below 2^-8 of the largest lose more here), as two int8 planes q = 256 hi + lo: heads' high parts are rows 0-7 of the
//     MMA, low parts rows 8-15, and both sums of a score end in one lane.  They are exact; scales multiply in fp32.
//   * P V runs in fp16 with fp32 sums: a code becomes the fp16 number code + 1152 (byte permutes alone), the sum starts at
//     -1152 times the sum of the probabilities, 32 positions at a time.  The tensor cores cut sums, not round them: that leaves
//     -5e-5 of a code's step in every output, at any length (random values: a hundredth of the output's rounding at 4096 positions
//     of equal weight, a sixteenth at 131072).
//     Dimensions are the MMA's rows and heads its columns, which is how the scores' layout already holds P.  Probabilities are scaled by
//     2^10 and rounded to fp16: 2^-11 relative (an eighth of the output's own rounding) down to 2^-24 of the largest, 2^-35
//     of it absolute below that; the sum that divides takes them in fp32.
//   * the order of a contraction's index is free, so it is chosen such that every lane's operands are 16 consecutive
//     bytes of a cache row, read without bank conflicts.  Rows pass through a ring in shared memory, one per warp, filled by
//     asynchronous copies of whole rows: pieces of 16 bytes trade places only within 128 (spread over a slot per lane, the copies
//     took every sector twice and stopped at 4.3 TB/s).  The next unit's keys are fetched as soon as this one's are used, its values likewise:
//     8 to 16 KB a warp are in flight.  (168 registers are what three CTAs an SM leave; of D > 64 a few are spilled, 12 to 148 bytes a thread.)
//   * the tail's products run in bf16, 16 positions to a warp, with each probability as the sum of two bf16 numbers (2^-16).
//     Infinities and NaNs of its values reach the result, by the first of the two alone.
template <int DP>
struct DecodeSmem { static constexpr int bytes = kWarps * 128 * DP; };

template <int DP, bool FULL, bool CLUSTER>
__global__ void __launch_bounds__(32 * kWarps, kDecodeCtas) decode_kernel(const DecodeArgs a) {
    constexpr int KS = DP / 32;        // k steps of Q K^T
    constexpr int MT = DP / 16;        // m tiles of P V
    constexpr int KC = DP / 64;        // 16-byte pieces of a key row per lane
    constexpr int NT = DP / 8;         // bytes of a value row per lane
    constexpr int RING = 128 * DP;     // a unit of keys, then of values
    extern __shared__ __align__(128) char ring_smem[];
    float (*o_s)[kHeads][DP] = reinterpret_cast<float (*)[kHeads][DP]>(ring_smem);      // at a segment's end, in the rings' place
    static_assert(sizeof(float) * (kWarps + 1) * kHeads * DP <= DecodeSmem<DP>::bytes, "the sums fit");
    __shared__ float m_s[kWarps][kHeads], l_s[kWarps][kHeads], m_c[kHeads], l_c[kHeads];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int D = FULL ? DP : a.c.D;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(ring_smem) + (uint32_t)(warp * RING);
    // In this order: the joining launch, which comes in now, reads the positions before it waits for this one.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int b, kvh, units;
    int64_t flat = 0, flat_end = 0, pair0 = 0;     // this CTA's places, and the place at which the pair starts
    if (CLUSTER) {
        const int pair = blockIdx.x / kCluster, rank = blockIdx.x % kCluster;
        b = pair / a.c.nkv;
        kvh = pair - b * a.c.nkv;
        units = units_of(a.pos[(int64_t)b * a.pos_stride], a.c.max_len);
        const int per = (units + kCluster - 1) / kCluster;
        flat = rank * per < units ? rank * per : units;
        flat_end = flat + per < units ? flat + per : units;
    } else {
        if (a.edges)            // sequences with nothing to see: the joining launch does not come by
            for (int i = blockIdx.x; i < a.B; i += gridDim.x)
                if (units_of(a.pos[(int64_t)i * a.pos_stride], a.c.max_len) == 0)
                    for (int d = threadIdx.x; d < a.nq * D; d += 32 * kWarps) a.out[(int64_t)i * a.ld_out + d] = __float2bfloat16_rn(0.f);
        int64_t total;
        const Share at = find(a, blockIdx.x, -1, total);
        if (at.b < 0) return;
        flat = at.per * blockIdx.x;
        flat_end = flat + at.per < total ? flat + at.per : total;
        b = at.b;
        units = at.units;
        pair0 = at.before * a.c.nkv;
        kvh = (int)((flat - pair0) / (units + kPad));
        pair0 += (int64_t)kvh * (units + kPad);
    }
    const int64_t start = flat;

    while (true) {          // segments
        const int64_t pos = a.pos[(int64_t)b * a.pos_stride];
        const int u0 = flat - pair0 < units ? (int)(flat - pair0) : units;
        const int u1 = flat_end - pair0 < units ? (int)(flat_end - pair0) : units;
        if (CLUSTER || u0 < u1) {
        const int tail_n = (int)((pos + 1) % kBlock);        // rows of the unfinished block
        const int whole = tail_n ? units - 1 : units;        // units below this one are finished blocks
        const int u_end = u1 < whole ? u1 : whole;
        const int64_t head = (int64_t)b * a.c.nkv + kvh;
        const __nv_bfloat16* q = a.q + (int64_t)b * a.ld_q + ((int64_t)kvh * a.G + (g < a.G ? g : 0)) * D;
        const int8_t* kp = a.c.k + head * a.c.max_len * D;
        const int8_t* vp = a.c.v + head * a.c.max_len * D;
        const float* ksp = a.c.ks + head * (a.c.max_len / kBlock);
        const float* vsp = a.c.vs + head * (a.c.max_len / kBlock);
        const int first = u0 + warp;
        // The copies of a unit's keys, or values, into their half of the ring: always one group.  Rows stay rows, eight lanes
        // to 128 bytes; pieces of 16 bytes trade places within 128 (by the row, as the reads below want it).
        const int c_cp = DP == 128 ? lane & 7 : lane & 3, r_cp = DP == 128 ? lane >> 3 : lane >> 2;        // this lane's piece and row
        const int64_t off_cp = (int64_t)r_cp * D + 16 * c_cp;
        const uint32_t k_cp = ring + (uint32_t)(DP == 128 ? r_cp * 128 + ((c_cp ^ ((r_cp & 1) << 2 | r_cp >> 1)) << 4) : lane * 16);
        const uint32_t v_cp = ring + (uint32_t)(64 * DP + (DP == 128 ? r_cp * 128 + ((c_cp ^ r_cp) << 4)
                                                                     : (lane >> 3) * 128 + (((lane & 7) ^ ((lane >> 3 & 1) << 2 | (lane >> 4) << 1)) << 4)));
        auto fetch_k = [&](int unit) {
            if (unit < u_end && (FULL || 16 * c_cp < D)) {
                const int8_t* k = kp + (int64_t)unit * kBlock * D + off_cp;
#pragma unroll
                for (int i = 0; i < 8 * KC; ++i)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                 :: "r"((k_cp ^ (uint32_t)(DP == 128 ? (i & 1) * 32 : 0)) + (uint32_t)(i * 512)), "l"(k + i * (DP == 128 ? 4 : 8) * D) : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        auto fetch_v = [&](int unit) {
            if (unit < u_end && (FULL || 16 * c_cp < D)) {
                const int8_t* v = vp + (int64_t)unit * kBlock * D + off_cp;
#pragma unroll
                for (int i = 0; i < 8 * KC; ++i)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                 :: "r"((v_cp ^ (uint32_t)(DP == 128 ? (i & 1) * 64 : 0)) + (uint32_t)(i * 512)), "l"(v + i * (DP == 128 ? 4 : 8) * D) : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        // where this lane's operands are: keys of row 8 n + g, piece 4 i + t, and values of rows 8 k + 2 t + b, bytes NT g ..
        const uint32_t k_rd = ring + (uint32_t)(DP == 128 ? g * 128 + ((t ^ ((g & 1) << 2 | g >> 1)) << 4) : lane * 16);
        const uint32_t v_rd = ring + (uint32_t)(64 * DP + (DP == 128 ? t * 256 + ((g ^ 2 * t) << 4)
                                                                     : t * 128 + (((g >> 1) ^ ((t & 1) << 2 | (t >> 1) << 1)) << 4) + 8 * (g & 1)));
        auto take = [&](uint32_t addr) {
            uint4 v;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
            return v;
        };
        if (!FULL) {        // the slots of dimensions that there are not: zeros
            for (int i = 0; i < RING / 512; ++i)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" :: "r"(ring + (uint32_t)(i * 512 + lane * 16)), "r"(0u) : "memory");
            __syncwarp();
        }
        // (the queries and the first scales before them: behind sixteen kilobytes a warp they would be three microseconds coming)
        uint4 qw[KC][2];
        float ks = 0.f, vs = 0.f;
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                qw[i][hh] = make_uint4(0u, 0u, 0u, 0u);
                if (64 * i + 16 * t + 8 * hh < D && g < a.G) qw[i][hh] = ld16(q + 64 * i + 16 * t + 8 * hh);
            }
        if (first < u_end) { ks = ksp[first]; vs = vsp[first]; }
        fetch_k(first);
        fetch_v(first);

        float o[MT][4];        // dimensions 16 g + 2 i and + 1 (rows g, g + 8) of heads 2 t and 2 t + 1
#pragma unroll
        for (int i = 0; i < MT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float m = -INFINITY, l = 0.f;           // of head g: m the same in its four lanes, l this lane's positions

        // Running softmax of S scores; rescales o when the maximum moved.  Returns the probabilities in s.
        auto softmax = [&](float* s, int S) {
            float mx = m;
#pragma unroll
            for (int i = 0; i < S; ++i) mx = fmaxf(mx, s[i]);
            mx = quad_max(mx);
            const float ref = mx == -INFINITY ? 0.f : mx;
            const float corr = ex2(m - ref);
            l *= corr;
#pragma unroll
            for (int i = 0; i < S; ++i) {
                s[i] = ex2(s[i] - ref);
                l += s[i];
            }
            if (__any_sync(0xffffffffu, mx != m)) {
                const float c0 = __shfl_sync(0xffffffffu, corr, 8 * t), c1 = __shfl_sync(0xffffffffu, corr, 8 * t + 4);
#pragma unroll
                for (int i = 0; i < MT; ++i) { o[i][0] *= c0; o[i][1] *= c1; o[i][2] *= c0; o[i][3] *= c1; }
            }
            m = mx;
        };

        // the unfinished block first, while the copies are under way: bf16 rows, sixteen positions to a warp
        if (u0 < u1 && u1 == units && 16 * warp < tail_n) {
            const __nv_bfloat16* kt = a.c.kt + head * kBlock * D;
            const __nv_bfloat16* vt = a.c.vt + head * kBlock * D;
            const int p = 16 * warp;
            float s[4];
            uint32_t qb[KC * 2][4];
#pragma unroll
            for (int i = 0; i < 2 * KC; ++i) {
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (32 * i + 8 * t < D && g < a.G) w = ld16(q + 32 * i + 8 * t);
                qb[i][0] = w.x; qb[i][1] = w.y; qb[i][2] = w.z; qb[i][3] = w.w;
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int row = p + 8 * n + g;
                float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 2 * KC; ++i) {
                    uint4 w = make_uint4(0u, 0u, 0u, 0u);
                    if (32 * i + 8 * t < D && row < tail_n) w = ld16(kt + row * D + 32 * i + 8 * t);
                    mma_bf16(c, qb[i][0], 0u, qb[i][1], 0u, w.x, w.y);
                    mma_bf16(c, qb[i][2], 0u, qb[i][3], 0u, w.z, w.w);
                }
                const int col = p + 8 * n + 2 * t;
                s[2 * n] = col < tail_n ? c[0] * a.scale_log2 : -INFINITY;
                s[2 * n + 1] = col + 1 < tail_n ? c[1] * a.scale_log2 : -INFINITY;
            }
            softmax(s, 4);
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const float h0 = __bfloat162float(__float2bfloat16_rn(s[2 * n])), h1 = __bfloat162float(__float2bfloat16_rn(s[2 * n + 1]));
                hi[n] = bf2_of(h0, h1);
                lo[n] = bf2_of(s[2 * n] - h0, s[2 * n + 1] - h1);
            }
#pragma unroll
            for (int n0 = 0; n0 < NT; n0 += 8) {          // eight dimensions of four rows at a time
                uint4 w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int row = p + 2 * t + (k & 1) + 8 * (k >> 1);
                    w[k] = make_uint4(0u, 0u, 0u, 0u);
                    if (NT * g + n0 < D && row < tail_n) w[k] = ld16(vt + row * D + NT * g + n0);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {             // a word is two dimensions: rows g and g + 8 of an m tile
                    const uint32_t x0 = (&w[0].x)[e], x1 = (&w[1].x)[e], x2 = (&w[2].x)[e], x3 = (&w[3].x)[e];
                    const uint32_t a0 = __byte_perm(x0, x1, 0x5410), a1 = __byte_perm(x0, x1, 0x7632);
                    const uint32_t a2 = __byte_perm(x2, x3, 0x5410), a3 = __byte_perm(x2, x3, 0x7632);
                    mma_bf16(o[n0 / 2 + e], a0, a1, a2, a3, hi[0], hi[1]);
                    // (an infinity is the high part's alone: the low one, zero or of the other sign, would make a NaN of it)
                    mma_bf16(o[n0 / 2 + e], finite2(a0), finite2(a1), finite2(a2), finite2(a3), lo[0], lo[1]);
                }
            }
        }

        if (first < u_end) {
            float ks_next = 0.f, vs_next = 0.f;
            // query rows as int8 A operands: lane (g, t) holds the dimensions of the key pieces it loads
            uint32_t qa[KS][4];
            float q_back;
            {
                float f[KC][2][8];
                float amax = 0.f;
                bool bad = false;
#pragma unroll
                for (int i = 0; i < KC; ++i)
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        unpack8(qw[i][hh], f[i][hh]);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            amax = fmaxf(amax, fabsf(f[i][hh][e]));
                            bad |= !(fabsf(f[i][hh][e]) <= 3.4e38f);
                        }
                    }
                bad = (__ballot_sync(0xffffffffu, bad) >> (lane & 28) & 15u) != 0u;      // in any of the head's four lanes
                amax = quad_max(amax);
                int ex = (int)(__float_as_uint(amax) >> 23);
                if (ex == 0 || bad) { ex = 127; amax = 0.f; }       // zeros (or less than a normal number)
                if (ex > 253) ex = 253;
                const float up = __uint_as_float((uint32_t)(254 - ex) << 23);          // largest element into [1, 4)
                const float to16 = amax > 0.f ? 32512.f / (amax * up) : 0.f;
                q_back = __uint_as_float((uint32_t)ex << 23) * (amax * up / 32512.f) * a.scale_log2;
                if (bad) q_back = __uint_as_float(0x7fc00000u);
#pragma unroll
                for (int i = 0; i < KC; ++i)
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            uint32_t hi = 0u, lo = 0u;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int v = __float2int_rn(f[i][hh][4 * w + e] * up * to16);
                                const int h = (v + 128) >> 8;
                                hi |= ((uint32_t)h & 0xffu) << (8 * e);
                                lo |= ((uint32_t)(v - 256 * h) & 0xffu) << (8 * e);
                            }
                            qa[2 * i + hh][2 * w] = hi;
                            qa[2 * i + hh][2 * w + 1] = lo;
                        }
            }
#pragma unroll 1
            for (int u = first; u < u_end; u += kWarps) {
                const int next = u + kWarps;
                if (next < u_end) { ks_next = ksp[next]; vs_next = vsp[next]; }
                asm volatile("cp.async.wait_group 1;" ::: "memory");      // the keys have landed, their values are under way
                __syncwarp();
                float s[16];
                int c4[8][4];
#pragma unroll
                for (int n = 0; n < 8; ++n) c4[n][0] = c4[n][1] = c4[n][2] = c4[n][3] = 0;
#pragma unroll
                for (int i = 0; i < KC; ++i) {
                    uint4 kr[8];
#pragma unroll
                    for (int n = 0; n < 8; ++n) kr[n] = take((k_rd ^ (uint32_t)(i * 64)) + (uint32_t)(n * KC * 512));
#pragma unroll
                    for (int n = 0; n < 8; ++n) mma_s8(c4[n], qa[2 * i], kr[n].x, kr[n].y);
#pragma unroll
                    for (int n = 0; n < 8; ++n) mma_s8(c4[n], qa[2 * i + 1], kr[n].z, kr[n].w);
                }
                const float back = ks * q_back;
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    s[2 * n] = (float)(c4[n][0] * 256 + c4[n][2]) * back;
                    s[2 * n + 1] = (float)(c4[n][1] * 256 + c4[n][3]) * back;
                }
                __syncwarp();
                fetch_k(next);                  // where these keys were
                softmax(s, 16);
                uint32_t p[8];
#pragma unroll
                for (int n = 0; n < 8; ++n) p[n] = half2_of(s[2 * n] * 1024.f, s[2 * n + 1] * 1024.f);
                const float vb = vs * (1.f / 1024.f);
                asm volatile("cp.async.wait_group 1;" ::: "memory");      // and now the values
                __syncwarp();
#pragma unroll
                for (int h = 0; h < 2; ++h) {                 // 32 positions
                    uint4 vr[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t src = (v_rd ^ (uint32_t)((j & 1) * (DP == 128 ? 16 : 64))) + (uint32_t)((4 * h + (j >> 1)) * 8 * DP + (DP == 128 ? (j & 1) * 128 : 0));
                        if constexpr (NT == 16) {
                            vr[j] = take(src);
                        } else {
                            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(vr[j].x), "=r"(vr[j].y) : "r"(src) : "memory");
                            vr[j].z = vr[j].w = 0u;
                        }
                    }
                    float off[4] = {0.f, 0.f, 0.f, 0.f};       // sums of the rounded probabilities of heads 2 t and 2 t + 1: what the 1152 adds
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        mma_f16(off, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, p[4 * h + 2 * j], p[4 * h + 2 * j + 1]);
                    off[0] *= -1152.f;
                    off[1] *= -1152.f;
#pragma unroll
                    for (int w = 0; w < NT / 4; ++w) {            // four dimensions: two m tiles
                        float c[2][4];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            c[i][0] = c[i][2] = off[0];
                            c[i][1] = c[i][3] = off[1];
                        }
#pragma unroll
                        for (int j = 0; j < 2; ++j) {             // sixteen positions
                            uint32_t x[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint32_t v4[4] = {vr[4 * j + k].x, vr[4 * j + k].y, vr[4 * j + k].z, vr[4 * j + k].w};
                                x[k] = v4[w] ^ 0x80808080u;
                            }
                            const uint32_t p0 = p[4 * h + 2 * j], p1 = p[4 * h + 2 * j + 1];
                            const uint32_t a01 = __byte_perm(x[0], x[1], 0x5140), a23 = __byte_perm(x[0], x[1], 0x7362);
                            const uint32_t b01 = __byte_perm(x[2], x[3], 0x5140), b23 = __byte_perm(x[2], x[3], 0x7362);
                            mma_f16(c[0], codes2<0x4140>(a01), codes2<0x4342>(a01), codes2<0x4140>(b01), codes2<0x4342>(b01), p0, p1);
                            mma_f16(c[1], codes2<0x4140>(a23), codes2<0x4342>(a23), codes2<0x4140>(b23), codes2<0x4342>(b23), p0, p1);
                        }
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[2 * w + i][e] = fmaf(vb, c[i][e], o[2 * w + i][e]);
                    }
                }
                __syncwarp();
                fetch_v(next);                  // where these values were
                ks = ks_next;
                vs = vs_next;
            }
        }

        // ---- the four warps' (m, l, o) meet
        asm volatile("cp.async.wait_all;" ::: "memory");
        l = quad_sum(l);
        __syncthreads();              // every warp is through with its ring
        if (t == 0) { m_s[warp][g] = m; l_s[warp][g] = l; }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            *reinterpret_cast<float2*>(&o_s[warp][2 * t][NT * g + 2 * i]) = make_float2(o[i][0], o[i][2]);
            *reinterpret_cast<float2*>(&o_s[warp][2 * t + 1][NT * g + 2 * i]) = make_float2(o[i][1], o[i][3]);
        }
        __syncthreads();
        const bool all = u0 == 0 && u1 == units;
        float* o_c = reinterpret_cast<float*>(ring_smem) + kWarps * kHeads * DP;      // CLUSTER: this CTA's [G][D]
        for (int i = threadIdx.x; i < a.G * D / 4; i += 32 * kWarps) {        // four dimensions
            const int hd = 4 * i / D, d = 4 * i - hd * D;
            float mx = m_s[0][hd];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, m_s[w][hd]);
            const float ref = mx == -INFINITY ? 0.f : mx;
            float4 ov = make_float4(0.f, 0.f, 0.f, 0.f);
            float lv = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float e = ex2(m_s[w][hd] - ref);
                const float4 x = *reinterpret_cast<const float4*>(&o_s[w][hd][d]);
                ov.x += e * x.x; ov.y += e * x.y; ov.z += e * x.z; ov.w += e * x.w;
                lv += e * l_s[w][hd];
            }
            if (CLUSTER) {
                *reinterpret_cast<float4*>(o_c + 4 * i) = ov;
                if (d == 0) { m_c[hd] = mx; l_c[hd] = lv; }
            } else if (all) {
                __nv_bfloat16* dst = a.out + (int64_t)b * a.ld_out + ((int64_t)kvh * a.G + hd) * D + d;
                dst[0] = __float2bfloat16_rn(ov.x / lv);
                dst[1] = __float2bfloat16_rn(ov.y / lv);
                dst[2] = __float2bfloat16_rn(ov.z / lv);
                dst[3] = __float2bfloat16_rn(ov.w / lv);
            } else {
                // (of a pair that started before this CTA, or with it, and of the one that it leaves unfinished)
                float* dst = a.part + (((int64_t)blockIdx.x * 2 + (pair0 <= start ? 0 : 1)) * a.G + hd) * (D + 2);
                *reinterpret_cast<float2*>(dst + 2 + d) = make_float2(ov.x, ov.y);
                *reinterpret_cast<float2*>(dst + 4 + d) = make_float2(ov.z, ov.w);
                if (d == 0) *reinterpret_cast<float2*>(dst) = make_float2(mx, lv);
            }
        }
        __syncthreads();              // the sums have been read
        }
        if (CLUSTER) break;
        flat = pair0 + units + kPad;  // the next pair
        if (flat >= flat_end) return;
        pair0 = flat;
        if (++kvh == a.c.nkv) {
            kvh = 0;
            do units = units_of(a.pos[(int64_t)(++b) * a.pos_stride], a.c.max_len); while (units == 0);
        }
    }
    if (CLUSTER) {
        const uint32_t o_at = (uint32_t)__cvta_generic_to_shared(ring_smem) + sizeof(float) * kWarps * kHeads * DP;
        const uint32_t m_at = (uint32_t)__cvta_generic_to_shared(m_c), l_at = (uint32_t)__cvta_generic_to_shared(l_c);
        auto peer = [](uint32_t addr, int rank) {       // a float of another CTA of the cluster
            uint32_t at;
            float v;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
            return v;
        };
        asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
        const int rank = blockIdx.x % kCluster, n = a.G * D, share = (n + kCluster - 1) / kCluster;
        const int end = (rank + 1) * share < n ? (rank + 1) * share : n;
        for (int i = rank * share + threadIdx.x; i < end; i += 32 * kWarps) {
            const int hd = i / D;
            float mv[kCluster], mx = -INFINITY, ov = 0.f, lv = 0.f;
#pragma unroll
            for (int c = 0; c < kCluster; ++c) { mv[c] = peer(m_at + 4u * hd, c); mx = fmaxf(mx, mv[c]); }
            const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
            for (int c = 0; c < kCluster; ++c) {
                const float e = ex2(mv[c] - ref);
                ov += e * peer(o_at + 4u * i, c);
                lv += e * peer(l_at + 4u * hd, c);
            }
            // (a sequence with nothing to see: zeros; NaN passes)
            a.out[(int64_t)b * a.ld_out + (int64_t)kvh * n + i] = __float2bfloat16_rn(units == 0 ? 0.f : ov / lv);
        }
        asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");     // nobody leaves while it is read
    }
}

// Joins the partial results of the pairs that more than one CTA had a segment of:
// out = sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c; sequences with nothing to see get zeros.  kFew results are one round
// trip to memory.  A long context has a hundred and more, and a large CTA.
// With more pairs than CTAs (EDGES) there is a CTA for each place where a share starts instead, and the first in a pair joins it.
// (32 sequences: 128 threads a CTA, so that all CTAs are there and have found their pairs when the last result is written, and
// one round trip: 10 -> 3 us.)
constexpr int kJoin = 8, kFew = 8, kHeld = 28;
static_assert(kJoin * kMaxD >= kDecodeCtas * 148 + 1, "a thread to a result");
template <bool EDGES>
__global__ void __launch_bounds__(EDGES ? kMaxD : kJoin * kMaxD) combine_kernel(const DecodeArgs a) {
    __shared__ float w_s[kDecodeCtas * 148 + 1], o_s[kJoin][kMaxD], red[2][kJoin * kMaxD / 32];
    const int hd = blockIdx.y, tid = threadIdx.x, D = a.c.D;
    int kvh = blockIdx.x, b = blockIdx.z;
    const int d = tid & (kMaxD - 1), j = tid / kMaxD, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int64_t total;
    const Share at = EDGES ? find(a, blockIdx.x + 1, -1, total) : find(a, 0, b, total);
    int64_t s = at.before * a.c.nkv;
    if (EDGES) {
        b = at.b;
        kvh = b < 0 ? 0 : (int)((at.per * (blockIdx.x + 1) - s) / (at.units + kPad));
    }
    s += (int64_t)kvh * (at.units + kPad);
    const int64_t e = s + at.units;
    const int c0 = (int)(s / at.per);
    int n = at.units == 0 ? 0 : (int)((e - 1) / at.per) - c0 + 1;
    if (EDGES && (b < 0 || c0 != (int)blockIdx.x || n < 2)) n = 1;        // (c0 < the share that starts here <= the pair's last)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __nv_bfloat16* out = a.out + (int64_t)b * a.ld_out + ((int64_t)kvh * a.G + hd) * D;
    if (n == 0) {
        if (tid < D) out[tid] = __float2bfloat16_rn(0.f);
        return;
    }
    if (n == 1) return;           // one CTA had it all and wrote it
    // the CTA that a pair starts in has it in its first slot if it starts there, too, the others always
    const int64_t step = 2 * (int64_t)a.G * (D + 2);
    const float* base = a.part + c0 * step + (int64_t)hd * (D + 2);
    const int64_t skip = s == c0 * at.per ? 0 : step / 2;
    auto part = [&](int c) { return base + c * step + (c == 0 ? skip : 0); };
    if (n <= kFew || blockDim.x < kJoin * kMaxD) {
        if (tid >= D) return;
        float top = -INFINITY, lv = 0.f, ov = 0.f;
        for (int at0 = 0; at0 < n; at0 += kFew) {
            float m[kFew], l[kFew], o[kFew], mx = top;
#pragma unroll
            for (int i = 0; i < kFew; ++i) {
                const int c = at0 + i;
                m[i] = c < n ? part(c)[0] : -INFINITY;
                l[i] = c < n ? part(c)[1] : 0.f;
                o[i] = c < n ? part(c)[2 + tid] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < kFew; ++i) mx = fmaxf(mx, m[i]);
            const float ref = mx == -INFINITY ? 0.f : mx, corr = ex2(top - ref);
            lv *= corr;
            ov *= corr;
#pragma unroll
            for (int i = 0; i < kFew; ++i) {
                const float w = ex2(m[i] - ref);
                lv += w * l[i];
                ov += w * o[i];
            }
            top = mx;
        }
        out[tid] = __float2bfloat16_rn(ov / lv);
        return;
    }
    // a thread to a result's maximum and sum, a group of threads to every kJoin-th result's outputs, all under way at once
    float v[kHeld], m = -INFINITY, l = 0.f;
    if (tid < n) { m = part(tid)[0]; l = part(tid)[1]; }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) v[i] = d < D && j + kJoin * i < n ? part(j + kJoin * i)[2 + d] : 0.f;
    float mx = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) red[0][warp] = mx;
    __syncthreads();
    mx = red[0][0];
#pragma unroll
    for (int w = 1; w < kJoin * kMaxD / 32; ++w) mx = fmaxf(mx, red[0][w]);
    const float weight = ex2(m - (mx == -INFINITY ? 0.f : mx));
    if (tid < n) w_s[tid] = weight;
    l *= weight;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) red[1][warp] = l;
    __syncthreads();
    float o = 0.f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        if (j + kJoin * i < n) o += w_s[j + kJoin * i] * v[i];
    if (d < D)
#pragma unroll 8
        for (int c = j + kJoin * kHeld; c < n; c += kJoin) o += w_s[c] * part(c)[2 + d];
    o_s[j][d] = o;
    __syncthreads();
    if (tid < D) {
        float lv = 0.f, ov = 0.f;
#pragma unroll
        for (int w = 0; w < kJoin * kMaxD / 32; ++w) lv += red[1][w];
#pragma unroll
        for (int w = 0; w < kJoin; ++w) ov += o_s[w][d];
        out[d] = __float2bfloat16_rn(ov / lv);
    }
}

// ---- host side --------------------------------------------------------------------------------------

static int check_cache(const hxq_kv8* c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail) return HXQ_E_ARG;
    if (c->slots <= 0 || c->nkv <= 0 || c->nkv > 65535 || c->D < 16 || c->D > kMaxD || c->D % 16 != 0 || c->max_len <= 0 || c->max_len % kBlock != 0)
        return HXQ_E_SHAPE;
    if (!aligned_to(c->k, 16) || !aligned_to(c->v, 16) || !aligned_to(c->k_tail, 16) || !aligned_to(c->v_tail, 16) ||
        !aligned_to(c->k_scale, 4) || !aligned_to(c->v_scale, 4))
        return HXQ_E_ALIGN;
    return HXQ_OK;
}

static int run_append(const hxq_kv8* c, const void* qkv, int64_t ld_qkv, int32_t T, const int32_t* cu, int32_t S, int32_t max_q,
                      const int64_t* pos, int32_t pos_stride, const float* cos_table, const float* sin_table, void* q_out, int64_t ld_q,
                      void* k_out, int64_t ld_k, int32_t nq, cudaStream_t stream) {
    if (!qkv || !pos || !cos_table || !sin_table || !q_out || T < 0 || S <= 0 || max_q < 0 || nq <= 0) return HXQ_E_ARG;
    const int st = check_cache(c);
    if (st != HXQ_OK) return st;
    const int64_t width = (int64_t)(nq + 2 * c->nkv) * c->D;
    if (S > c->slots || nq % c->nkv != 0 || (pos_stride != 0 && pos_stride != 1)) return HXQ_E_SHAPE;
    if (ld_qkv < width || ld_q < (int64_t)nq * c->D || (k_out && ld_k < (int64_t)c->nkv * c->D)) return HXQ_E_SHAPE;
    if (!aligned_to(qkv, 16) || !aligned_to(q_out, 16) || !aligned_to(cos_table, 16) || !aligned_to(sin_table, 16) || ld_qkv % 8 != 0 ||
        ld_q % 8 != 0 || (k_out && (!aligned_to(k_out, 16) || ld_k % 8 != 0)))
        return HXQ_E_ALIGN;
    if (T == 0 || max_q == 0) return HXQ_OK;
    AppendArgs a;
    a.c = cache_of(c);
    a.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv);
    a.cu = cu;
    a.pos = pos;
    a.cos_t = cos_table;
    a.sin_t = sin_table;
    a.q_out = reinterpret_cast<__nv_bfloat16*>(q_out);
    a.k_out = reinterpret_cast<__nv_bfloat16*>(k_out);
    a.ld_qkv = ld_qkv; a.ld_q = ld_q; a.ld_k = ld_k;
    a.pos_stride = pos_stride; a.T = T; a.S = S; a.nq = nq;
    a.max_q = max_q < c->max_len ? max_q : c->max_len;
    a.groups = cu ? (nq + kHeadsPrompt - 1) / kHeadsPrompt : (nq + kHeadsStep - 1) / kHeadsStep;
    // blocks that n rows touch: n / 64 and up to two more, wherever they start
    const int64_t blocks = cu ? (int64_t)T / kBlock + 2 * (int64_t)S : S, grid = blocks * ((cu ? a.groups * ((kBlock * (c->D / 16) + kAppendThreads - 1) / kAppendThreads) : 1) + 2 * c->nkv);
    if (grid > 0x7fffffffLL) return HXQ_E_SHAPE;
    const cudaError_t e = cu ? launch_pdl(append_kernel<false>, dim3((unsigned)grid), dim3(kAppendThreads), stream, 0, a)
                             : launch_pdl(append_kernel<true>, dim3((unsigned)grid), dim3(kAppendThreads), stream, 0, a);
    return e == cudaSuccess ? HXQ_OK : HXQ_E_LAUNCH;
}

// A cluster of eight CTAs for each (sequence, KV head) pair, where that many are resident at once and no warp has more than
// four units of a full cache to walk.
static bool decode_clustered(int B, int nkv, int max_len) {
    return (int64_t)B * nkv * kCluster <= kDecodeCtas * 148 && max_len <= kBlock * kCluster * kWarps * 4;
}
// Otherwise CTAs as many as fit, fewer where a full cache has not that many times four units.
static int decode_ctas(int B, int nkv, int max_len) {
    const int64_t units = (int64_t)(max_len / kBlock + kPad) * B * nkv, n = (units + kWarps - 1) / kWarps;
    const int most = kDecodeCtas * 148;
    return (int)(n < most ? n : most);
}

template <int DP, bool FULL, bool CLUSTER>
static cudaError_t run_decode(const DecodeArgs& a, cudaStream_t stream) {
    static bool attr_set[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    const auto kernel = decode_kernel<DP, FULL, CLUSTER>;
    if (!attr_set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodeSmem<DP>::bytes);
        if (e != cudaSuccess) return e;
        attr_set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(CLUSTER ? a.B * a.c.nkv * kCluster : a.ctas);
    cfg.blockDim = dim3(32 * kWarps);
    cfg.stream = stream;
    cfg.dynamicSmemBytes = DecodeSmem<DP>::bytes;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kCluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CLUSTER ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}
template <bool CLUSTER>
static cudaError_t run_decode(const DecodeArgs& a, cudaStream_t stream) {
    const int D = a.c.D;
    return D == 128 ? run_decode<128, true, CLUSTER>(a, stream) : D > 64 ? run_decode<128, false, CLUSTER>(a, stream)
           : D == 64 ? run_decode<64, true, CLUSTER>(a, stream) : run_decode<64, false, CLUSTER>(a, stream);
}

}  // namespace kv8
}  // namespace hxq

using namespace hxq::kv8;

extern "C" int hxq_rope_append_kv8(const hxq_kv8* cache, const void* qkv, int64_t ld_qkv, const int64_t* pos, int32_t pos_stride,
                                   const float* cos_table, const float* sin_table, void* q_out, int64_t ld_q, int32_t B, int32_t nq,
                                   hxq_stream_t stream) {
    if (B <= 0) return HXQ_E_ARG;
    return run_append(cache, qkv, ld_qkv, B, nullptr, B, 1, pos, pos_stride, cos_table, sin_table, q_out, ld_q, nullptr, 0, nq,
                      reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int hxq_rope_append_prompt_kv8(const hxq_kv8* cache, const void* qkv, int64_t ld_qkv, int32_t T, const int32_t* cu, int32_t S,
                                          int32_t max_q, const int64_t* pos, int32_t pos_stride, const float* cos_table, const float* sin_table,
                                          void* q_out, int64_t ld_q, void* k_out, int64_t ld_k, int32_t nq, hxq_stream_t stream) {
    if (!cu) return HXQ_E_ARG;
    return run_append(cache, qkv, ld_qkv, T, cu, S, max_q, pos, pos_stride, cos_table, sin_table, q_out, ld_q, k_out, ld_k, nq,
                      reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int hxq_kv8_rows(const hxq_kv8* cache, const int64_t* len, int32_t len_stride, int32_t S, int32_t rows, void* k_out, void* v_out,
                            int64_t ld_seq, int64_t ld_head, int64_t ld_row, hxq_stream_t stream) {
    if (!len || !k_out || !v_out || S <= 0 || rows < 0) return HXQ_E_ARG;
    const int st = check_cache(cache);
    if (st != HXQ_OK) return st;
    if (S > cache->slots || S > 65535 || (len_stride != 0 && len_stride != 1) || ld_row < cache->D) return HXQ_E_SHAPE;
    if (!hxq::aligned_to(k_out, 16) || !hxq::aligned_to(v_out, 16) || ld_seq % 8 != 0 || ld_head % 8 != 0 || ld_row % 8 != 0) return HXQ_E_ALIGN;
    const int n = rows < cache->max_len ? rows : cache->max_len;
    if (n == 0) return HXQ_OK;
    const cudaError_t e = launch_pdl(rows_kernel, dim3((n + kBlock - 1) / kBlock, cache->nkv, S), dim3(256), reinterpret_cast<cudaStream_t>(stream), 0,
                                     cache_of(cache), len, (int)len_stride, n, reinterpret_cast<__nv_bfloat16*>(k_out),
                                     reinterpret_cast<__nv_bfloat16*>(v_out), ld_seq, ld_head, ld_row);
    return e == cudaSuccess ? HXQ_OK : HXQ_E_LAUNCH;
}

extern "C" size_t hxq_attn_decode_kv8_workspace_bytes(int32_t B, int32_t nq, int32_t nkv, int32_t D, int32_t max_len) {
    if (B <= 0 || nq <= 0 || nkv <= 0 || D <= 0 || max_len <= 0) return 0;
    if (decode_clustered(B, nkv, max_len)) return 0;
    return (size_t)decode_ctas(B, nkv, max_len) * 2 * (nq / nkv) * (D + 2) * sizeof(float);
}

extern "C" int hxq_attn_decode_kv8(const hxq_kv8* cache, const void* q, int64_t ld_q, const int64_t* pos, int32_t pos_stride, void* out,
                                   int64_t ld_out, void* workspace, size_t workspace_bytes, int32_t B, int32_t nq, float scale,
                                   hxq_stream_t stream_) {
    if (!q || !pos || !out || B <= 0 || nq <= 0) return HXQ_E_ARG;
    const int st = check_cache(cache);
    if (st != HXQ_OK) return st;
    if (B > cache->slots || B > 65535 || nq % cache->nkv != 0 || nq / cache->nkv > kHeads || (pos_stride != 0 && pos_stride != 1)) return HXQ_E_SHAPE;
    if (ld_q < (int64_t)nq * cache->D || ld_out < (int64_t)nq * cache->D) return HXQ_E_SHAPE;
    if (!hxq::aligned_to(q, 16) || ld_q % 8 != 0) return HXQ_E_ALIGN;
    const bool clustered = decode_clustered(B, cache->nkv, cache->max_len);
    if (!clustered && (!workspace || !hxq::aligned_to(workspace, 8) || workspace_bytes < hxq_attn_decode_kv8_workspace_bytes(B, nq, cache->nkv, cache->D, cache->max_len)))
        return HXQ_E_WORKSPACE;
    DecodeArgs a;
    a.c = cache_of(cache);
    a.q = reinterpret_cast<const __nv_bfloat16*>(q);
    a.pos = pos;
    a.out = reinterpret_cast<__nv_bfloat16*>(out);
    a.part = reinterpret_cast<float*>(workspace);
    a.ld_q = ld_q; a.ld_out = ld_out;
    a.pos_stride = pos_stride; a.B = B; a.nq = nq; a.G = nq / cache->nkv;
    a.ctas = decode_ctas(B, cache->nkv, cache->max_len);
    a.edges = (int64_t)B * cache->nkv > a.ctas && a.ctas > 1;
    a.scale_log2 = scale * 1.4426950408889634f;
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    if (clustered) return run_decode<true>(a, stream) == cudaSuccess ? HXQ_OK : HXQ_E_LAUNCH;
    cudaError_t e = run_decode<false>(a, stream);
    // (about ctas / (B nkv) results a pair)
    const bool few = (int64_t)a.ctas <= (int64_t)B * cache->nkv * (kFew - 2);
    if (e == cudaSuccess && a.edges) e = launch_pdl(combine_kernel<true>, dim3(a.ctas - 1, a.G), dim3(kMaxD), stream, 0, a);
    else if (e == cudaSuccess) e = launch_pdl(combine_kernel<false>, dim3(cache->nkv, a.G, B), dim3(few ? kMaxD : kJoin * kMaxD), stream, 0, a);
    return e == cudaSuccess ? HXQ_OK : HXQ_E_LAUNCH;
}
