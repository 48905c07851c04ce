// hxq_attn_prompt: attention of whole prompts - causal, grouped heads, packed sequences of different lengths, keys
// and values packed like the queries or in the slabs of a cache (a later piece of a prompt over the rows before it).
// The reference leaves this to the framework's attention inside its HF models
// (helix_substrate/basin_runtime.py:281-330).
//
//     out[i, h] = sum_j softmax_j(scale q[i, h] . k[j, h / G]) v[j, h / G],   j < count(i),
//     count(i) = lk - lq + i + 1 (causal) or lk;  a row with count(i) <= 0 is zero.
//
// A tile is 128 rows.  A row is (token, head of the group): the G query heads of a KV head share its keys, so a tile
// spans 128 / G tokens, the causal edge wastes that much less, and a short prompt fills its tiles G times better than
// with a head per CTA.  Per 64 keys and tile, all on the tensor cores (tcgen05):
//
//     S = Q K^T       both operands in shared memory (TMA, 128-byte swizzle), S in tensor memory
//     P = 2^(scale' S - m)      one thread per row, in registers: running maximum m and sum; P goes back to tensor
//                               memory as bf16, over S
//     O += P V        A operand from tensor memory, V as it lies in memory (its rows are the contraction), O in
//                     tensor memory for the whole row
//
// Roles: four warps a tile are its softmax and epilogue, one warp feeds K and V through a ring, one issues the MMAs, two
// clean V tiles.  P is rounded to bf16, V's type (the MMA takes no other beside it): 2^-8 at most per weight, as much as
// the output's own rounding; the sum that divides takes the weights before rounding.
//
// Bound by the tensor cores for long prompts, by each CTA's start and end for short ones.  A step's products, its softmax
// and the signals between them depend on one another (about 1000 cycles of the last two each), so two tiles take turns, in one
// CTA or in two on an SM, and S has two buffers a tile, of 64 keys, tensor memory being full with them and O: the next step's
// scores are there when a warp comes for them.  (Products of 64 keys cost a third more, 670 cycles a step and tile instead of 512: a
// Q tile is read from shared memory for half the work.  With 128 keys a step and one buffer, S of the next waiting for P V of
// this one, a step took 3900 cycles, its products 2048.)  Both tiles' 64 keys take 1530 to 1750 cycles, their products 1345; a
// tile by itself takes 1241, its softmax's latency.  16384 tokens of 28 + 4 heads of 128 take 1.51 ms in a short run (1270
// TFLOP/s), 1.76 in one of a second, at the 1.6 GHz that the power limit leaves.
//
// A CTA's start (finding its tokens 1 to 2 us, first loads and scores 1.3) and end (V's edge 0.7, outputs by way of shared memory
// 1.7) cost as much as six steps; of 2048 tokens and less they are half of the time.
//
// The reference point m moves only when the maximum has grown by more than 2^8: weights stay below 256, nothing
// overflows, the result is the same, and O is rarely rescaled.
//
// What a row does not see must not reach it, whatever it holds: scores are replaced, not added to; a V tile with rows past
// the sequence's end, or past what some row of the CTA sees, is looked at before its product: rows past the end become
// zero, infinities and NaNs in rows that only some see are taken out and, in the epilogue, given back to the rows that do.
//
// Every mbarrier wait is bounded and raises the status word.  No multicast loads.

#include <cuda.h>

#include <type_traits>

#include "hxq_common.cuh"
#include "hxq_sm100.cuh"

namespace hxq {
namespace gemm {
bool make_map_nd(CUtensorMap* map, CUtensorMapDataType dt, int rank, const void* base, const uint64_t* dims,
                 const uint64_t* strides_bytes, const uint32_t* box, CUtensorMapSwizzle sw);
}  // namespace gemm

namespace attnp {

constexpr int BM = 128;                     // rows of a tile
constexpr int BN = 64;                      // keys of a step
constexpr int kMaxStages = 8;
constexpr int kBarBytes = 768;
constexpr int kSorted = 128;                // sequences whose items stand in order of their work
constexpr int kMany = 4 * 148;              // items of two tiles from which on the tiles stay together
constexpr int kShare = 8;                   // key tiles that a CTA of a shared item has at least
constexpr int kPolyOf4 = 1;                 // of four pairs of weights, how many are made on the multiply-add units

template <int DP, int TILES>
struct Sizes {
    static constexpr int kSoftmaxWarps = 4 * TILES, kThreads = 32 * (kSoftmaxWarps + 4);
    // Registers of a thread: at launch, and after the roles have parted.  (16384 tokens in a long run: 1727 us with 176, 1738 with 184,
    // 1768 with 208, 1770 without the exchange; packed prompts 71.5 with 168 of a single tile, 72.3 with 192, 73.5 without.)
    static constexpr int kRegsLaunch = TILES == 2 ? 168 : 128;
    static constexpr int kRegsSoftmax = TILES == 2 ? 176 : 168, kRegsOther = TILES == 2 ? 136 : 88;
    static constexpr int kQ = BM * DP * 2, kTile = BN * DP * 2;               // a Q tile, a K or V tile
    static constexpr int kStages = TILES == 2 ? (DP == 128 ? 5 : 8) : (DP == 128 ? 2 : 6);      // of two tiles: the first two of K, then one of V and one of K
    static constexpr int kSmem = TILES * kQ + 2 * kStages * kTile + kBarBytes;
};

struct Args {
    const int32_t *cu_q, *cu_k;
    const int64_t* k_len;
    const __nv_bfloat16* v;
    __nv_bfloat16* out;
    int32_t* status;
    int64_t v_seq, v_head, v_row, o_tok, o_head;
    float* part;            // splits > 1: [items][splits][DP + 2][2 * BM]: reference point, sum, output before the division
    int32_t Tq, Tk, S, max_q, nkv, G, D, tpg, rows, n_ct, causal, splits, alone, groups;     // max_q: tokens of a sequence that are computed; rows: tokens of an item; alone: key tiles up to which a sequence's items are not shared; groups of 32 rows of an item that any token can fill
    float scale_log2;
};

// ---- what a CTA is for

struct Seq {
    int q0, lq, k0, lk;     // first row and number of its queries, of its keys
};
__device__ __forceinline__ Seq sequence(const Args& a, int s) {
    Seq r = {0, 0, 0, 0};
    if (s >= a.S) return r;
    const int q0 = a.cu_q[s], q1 = a.cu_q[s + 1];
    if (a.cu_k == nullptr) {
        const int64_t n = a.k_len[s];
        r.lk = n < 0 ? 0 : (n > a.Tk ? a.Tk : (int)n);
    } else {
        const int k0 = a.cu_k[s], k1 = a.cu_k[s + 1];
        r.k0 = k0 < 0 ? 0 : k0;
        r.lk = (k1 > a.Tk ? a.Tk : k1) - r.k0;
    }
    r.q0 = q0 < 0 ? 0 : q0;
    r.lq = (q1 > a.Tq ? a.Tq : q1) - r.q0;
    if (r.lq < 0) r.lq = 0;
    if (r.lk < 0) r.lk = 0;
    return r;
}
__device__ __forceinline__ int reach(const Args& a, int lq, int keys, int i) {      // keys that token i sees
    if (!a.causal || i >= lq) return keys;
    const int n = keys - lq + i + 1;
    return n > 0 ? n : 0;
}
// An item's key tiles are shared out among `used` CTAs, `per` tiles each, unless its sequence has few.  A larger a.splits than
// `used` changes nothing: the same bits from a slab of any length.
struct Share {
    int used, per;
};
__device__ __forceinline__ Share find_share(const Args& a, int lq, int keys, int i0) {
    if (a.splits == 1 || keys <= a.alone * BN) return {1, 0};
    const int last = i0 + a.rows < lq ? i0 + a.rows - 1 : lq - 1;
    const int total = (reach(a, lq, keys, last) + BN - 1) / BN, each = (total + a.splits - 1) / a.splits;
    const int per = each > kShare ? each : kShare;
    return {total > 0 ? (total + per - 1) / per : 1, per};
}
// Item i: a CTA's tokens (from ct * rows on) of one sequence and KV head.  The items of all sequences stand in a row by
// falling ct, the longest work (of causal attention) first, with no gaps for sequences that are shorter than others.
// A warp finds the item: F(c), the number of items with ct >= c of one head, falls in c.  (kSorted sequences at most: the lanes hold
// their lengths.)  Of more, sequence s has the places from first_row / rows + s on, enough for its items and its last one first;
// thirty-two sequences are looked at at a time.
__device__ __forceinline__ bool find_item(const Args& a, int i, Seq& q, int& s, int& ct, int& kvh) {
    const int lane = threadIdx.x & 31;
    kvh = i % a.nkv;
    i /= a.nkv;
    auto items = [&](int lq) {
        const int n = (lq + a.rows - 1) / a.rows;
        return n < a.n_ct ? n : a.n_ct;
    };
    if (a.S == 1) {             // (0.7 us less, of 5)
        s = 0;
        q = sequence(a, 0);
        ct = items(q.lq) - 1 - i;
        return ct >= 0;
    }
    if (a.S > kSorted) {
        auto place = [&](int s) {
            const int q0 = a.cu_q[s];
            return (q0 < 0 ? 0 : (q0 > a.Tq ? a.Tq : q0)) / a.rows + s;
        };
        int lo = 0, hi = a.S;           // place(lo) <= i < place(hi)
        while (hi - lo > 1) {
            const int by = (hi - lo + 31) / 32, at = lo + (lane + 1) * by;
            const int n = __popc(__ballot_sync(0xffffffffu, at < hi && place(at) <= i));
            lo += n * by;
            hi = lo + by < hi ? lo + by : hi;
        }
        s = lo;
        q = sequence(a, lo);
        ct = items(q.lq) - 1 - (i - place(lo));
        return ct >= 0 && i >= place(lo);       // (before the first sequence's places, where rows of no sequence precede it: none)
    }
    constexpr int HELD = kSorted / 32;      // (loads that run together)
    int held[HELD];
#pragma unroll
    for (int b = 0; b < HELD; ++b) held[b] = 32 * b < a.S ? items(sequence(a, 32 * b + lane).lq) : 0;
    auto from = [&](int c) {
        int sum = 0;
#pragma unroll
        for (int b = 0; b < HELD; ++b) sum += held[b] > c ? held[b] - c : 0;
        return __reduce_add_sync(0xffffffffu, sum);
    };
    if (from(0) <= i) return false;
    int lo = 0, hi = a.n_ct, before = 0;        // F(lo) > i >= F(hi) = before
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1, n = from(mid);
        if (n > i) lo = mid; else { hi = mid; before = n; }
    }
    ct = lo;
    i -= before;                                // the i-th of the sequences that are long enough
    for (int b = 0; b < a.S; b += 32) {
        const Seq here = sequence(a, b + lane);
        uint32_t has = __ballot_sync(0xffffffffu, items(here.lq) > lo);
        const int n = __popc(has);
        if (i < n) {
            for (; i > 0; --i) has &= has - 1;
            const int at = __ffs(has) - 1;
            s = b + at;
            q.q0 = __shfl_sync(0xffffffffu, here.q0, at);
            q.lq = __shfl_sync(0xffffffffu, here.lq, at);
            q.k0 = __shfl_sync(0xffffffffu, here.k0, at);
            q.lk = __shfl_sync(0xffffffffu, here.lk, at);
            return true;
        }
        i -= n;
    }
    return false;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(sm100::smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(sm100::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// D[tmem] (+)= A * B[smem], A in shared memory or in tensor memory, and the arrival when all products so far have retired; by the
// lane whose `leader` is set.
__device__ __forceinline__ void umma_ss(uint32_t leader, uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t leader, uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
__device__ __forceinline__ void commit(uint32_t leader, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(leader) : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
}
// The wait for loads from tensor memory, through which their registers pass: nothing that uses them can be moved in front of it.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}
// ... and a second load's registers, behind the same wait
__device__ __forceinline__ void tmem_ld_tie(uint32_t (&r)[32]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) :: "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t elect_one() {       // one lane of the whole warp
    uint32_t p;
    asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
    return p;
}
__device__ __forceinline__ uint32_t peek(uint32_t bar, uint32_t parity) {       // has the phase completed?
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done;
}
// As sm100::mbar_wait, bounded by the number of tries (each of which the hardware may stretch to microseconds) and in few
// instructions: every role's loop shares a small instruction cache.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* abort) {
#pragma unroll 1
    for (int i = 0; i < (1 << 19); ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
        if (*abort != 0) return false;
    }
    *abort = 1;
    return false;
}
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, volatile int* abort) { return bar_wait(sm100::smem_u32(bar), parity, abort); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// ---- pairs of fp32 numbers
typedef uint64_t f2;
__device__ __forceinline__ f2 pair(float lo, float hi) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void split(f2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ float max3(float a, float b, float c) {       // NaN wins
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^x of a pair on the multiply-add units: x = n + f with n whole, |f| <= 1/2 (adding and taking off 1.5 * 2^23 leaves n, in
// the low bits too); 2^f by a polynomial of least largest relative error, 1.0e-4 (a fortieth of P's rounding), with the
// constant term 1; n added to the exponent.  From x = -127 down, and at -inf, it is 0 (there f = 0, and 1's exponent is
// 127).  x <= 127.
__device__ __forceinline__ f2 ex2_pair(f2 x) {
    float lo, hi;
    split(x, lo, hi);
    x = pair(fmaxf(lo, -127.f), fmaxf(hi, -127.f));
    const f2 t = add2(x, pair(12582912.f, 12582912.f));
    const f2 f = fma2(add2(t, pair(-12582912.f, -12582912.f)), pair(-1.f, -1.f), x);
    f2 p = fma2(f, pair(0.0550089329f, 0.0550089329f), pair(0.242210969f, 0.242210969f));
    p = fma2(f, p, pair(0.693282902f, 0.693282902f));
    p = fma2(f, p, pair(1.f, 1.f));
    float tl, th;
    split(t, tl, th);
    split(p, lo, hi);
    return pair(__uint_as_float((__float_as_uint(tl) << 23) + __float_as_uint(lo)), __uint_as_float((__float_as_uint(th) << 23) + __float_as_uint(hi)));
}
__device__ __forceinline__ uint32_t bf2(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// V's descriptor: the contraction's index (keys) is the row, 64 elements of N a 128-byte swizzled row, 8 rows 1024 B
// apart, the next 64 elements of N a whole half tile on.
__device__ __forceinline__ uint64_t make_desc_mn_sw128(uint32_t smem_addr, uint32_t half_bytes) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(half_bytes >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

template <int DP, int TILES>
__global__ void __launch_bounds__(Sizes<DP, TILES>::kThreads, 3 - TILES)
attn_prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const Args a) {
    using Z = Sizes<DP, TILES>;
    constexpr int SM_WARPS = Z::kSoftmaxWarps, NUM_THREADS = Z::kThreads;
    constexpr int NS = Z::kStages, QT = Z::kQ, TILE = Z::kTile;
    constexpr int QHALF = BM * 128, HALF = BN * 128;      // 64 of the dimensions of a Q tile, of a K or V tile
    extern __shared__ __align__(1024) char smem[];        // (no room for slack: the swizzled tiles need that alignment, checked here)
    if (sm100::smem_u32(smem) % 1024 != 0) {
        if (threadIdx.x == 0 && a.status != nullptr) atomicExch(a.status, HXQ_E_ALIGN);
        return;
    }
    char* ring = smem + TILES * QT;
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + NS * 2 * TILE);      // [NS] a stage has landed, ready for its products
    uint64_t* empty = full + kMaxStages;        // [NS] its products have retired
    uint64_t* raw = empty + kMaxStages;         // [NS] a stage whose V tile is to be cleaned has landed (full is not signalled) ...
    uint64_t* clean = raw + kMaxStages;         // [NS] ... and has been cleaned
    uint64_t* q_full = clean + kMaxStages;
    uint64_t* s_full = q_full + 1;              // [2 tiles][2 buffers] S is complete
    uint64_t* p_ready = s_full + 4;             // [2][2] P is written, O is rescaled
    uint64_t* o_done = p_ready + 4;             // [2][2] the last P V but one has retired; the last (a phase each: a wait for the first of two
                                                // could come after the second)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 4);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* odd_v = abort_flag + 1;       // a V tile held an infinity or a NaN that some row does not see
    volatile int* job = odd_v + 1;              // [8] this CTA's sequence, first token and head
    static_assert((4 * kMaxStages + 13) * 8 + 12 + 8 * 4 <= kBarBytes, "barrier area");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = a.G * a.tpg;               // of a tile; the rest is zero
    const int item = a.splits == 1 ? blockIdx.x : blockIdx.x / a.splits, share = blockIdx.x - item * a.splits;
    // The warp that loads looks for what this CTA is for, and loads the first tiles, while others set up.
    if (warp == SM_WARPS) {
        constexpr int BARS = 4 * kMaxStages + 13, CLEAN = 3 * kMaxStages, P_READY = 4 * kMaxStages + 5;
        for (int i = lane; i < BARS; i += 32)
            sm100::mbar_init(full + i, i >= CLEAN && i < CLEAN + kMaxStages ? 2 : (i >= P_READY && i < P_READY + 4 ? 4 : 1));
        if (lane == 0) {
            *abort_flag = 0;
            *odd_v = 0;
            sm100::prefetch_tensormap(&map_q);
            sm100::prefetch_tensormap(&map_k);
            sm100::prefetch_tensormap(&map_v);
        }
        sm100::fence_barrier_init();
        __syncwarp();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == SM_WARPS) {
        Seq seq;
        int s, ct, kvh;
        bool found = find_item(a, item, seq, s, ct, kvh);
        if (found && lane == 0) {
            const Share sh = find_share(a, seq.lq, seq.lk, ct * a.rows);
            found = share < sh.used;
            const int i0 = ct * a.rows, last = i0 + a.rows < seq.lq ? i0 + a.rows - 1 : seq.lq - 1, skip = share * sh.per * BN;
            int n = reach(a, seq.lq, seq.lk, last) - skip;
            if (sh.used > 1 && n > sh.per * BN) n = sh.per * BN;
            if (found && n > 0) {
                sm100::mbar_arrive_expect_tx(&full[0], n > BN ? 2 * TILE : TILE);
                for (int t = 0; t < (n > BN ? 2 : 1); ++t)
                    for (int h = 0; h < DP / 64; ++h)
                        tma_load_4d(sm100::smem_u32(ring + t * TILE + h * HALF), &map_k, &full[0], 64 * h, seq.k0 + skip + t * BN, kvh, a.cu_k != nullptr ? 0 : s);
                sm100::mbar_arrive_expect_tx(q_full, (uint32_t)TILES * (DP / 64) * (uint32_t)rows * 128u);
                for (int x = 0; x < TILES; ++x)
                    for (int h = 0; h < DP / 64; ++h)
                        tma_load_3d(sm100::smem_u32(smem + x * QT + h * QHALF), &map_q, q_full, 64 * h, kvh * a.G, seq.q0 + i0 + x * a.tpg);
            }
        }
        if (lane == 0) {
            job[0] = found;
            job[1] = seq.q0;
            job[2] = seq.lq;
            job[3] = seq.k0;
            job[4] = seq.lk;
            job[5] = s;
            job[6] = ct * a.rows;
            job[7] = kvh;
        }
    } else if (warp == SM_WARPS + 1) {
        sm100::tmem_alloc(tmem_slot, 256 * TILES);
        sm100::tmem_relinquish();
    } else {        // rows of the Q tiles that no token fills
        const int idle = (BM - rows) * 8, i0 = threadIdx.x - (warp > SM_WARPS ? 64 : 0);
        for (int part = 0; part < TILES * (DP / 64); ++part)
            for (int i = i0; i < idle; i += NUM_THREADS - 64)
                *reinterpret_cast<uint4*>(smem + part * QHALF + (rows + (i >> 3)) * 128 + (i & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    sm100::fence_proxy_async_smem();
    sm100::tc_fence_before_sync();
    __syncthreads();
    sm100::tc_fence_after_sync();
    // The next kernel may come in only now: one that took tensor memory before this CTA did would keep it waiting.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = *tmem_slot;       // S of tile 0: two buffers of 64 columns; of tile 1; O of either, 128 columns each
    if (job[0] == 0) {
        if (warp == SM_WARPS + 1) sm100::tmem_dealloc(tmem, 256 * TILES);
        return;
    }
    const int q0 = job[1], lq = job[2], all_keys = job[4], s = job[5], i0 = job[6], kvh = job[7];
    const Share sh = find_share(a, lq, all_keys, i0);
    const int skip = share * sh.per * BN, lk = all_keys - skip;        // keys before this CTA's first, and from it on
    const int k0 = job[3] + skip;
    auto count = [&](int i) {           // of this CTA's keys, those that token i sees
        const int n = reach(a, lq, all_keys, i) - skip;
        return n < 0 ? 0 : (sh.used > 1 && n > sh.per * BN ? sh.per * BN : n);
    };
    auto steps = [&](int x) {           // key tiles of Q tile x
        const int first = i0 + x * a.tpg;
        if (first >= lq) return 0;
        return (count(first + a.tpg < lq ? first + a.tpg - 1 : lq - 1) + BN - 1) / BN;
    };
    const int n0 = steps(0), n1 = TILES == 2 ? steps(1) : 0, n = n0 > n1 ? n0 : n1;
    const int seen_by_all = count(i0);          // keys that every token of this CTA sees
    const int jc = seen_by_all / BN;            // V tiles from here on are looked at
    bool ok = true;

    static_assert(32 * SM_WARPS * Z::kRegsSoftmax + 128 * Z::kRegsOther <= NUM_THREADS * Z::kRegsLaunch, "no more registers than the launch brings");
    if (warp >= SM_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Z::kRegsOther));
    if (warp == SM_WARPS) {
        // ------------------------------------------------------------ loads, in the order of their use: K0 K1 (above) | V0 K2 | V1 K3 | ...
        if (lane == 0 && n > 0) {
            const int slab = a.cu_k != nullptr ? 0 : s;
            int slot = 1;
            uint32_t ph = 1;
            for (int i = 0; i < n; ++i) {           // stage i + 1: V of step i and K of step i + 2
                ok = bar_wait(&empty[slot], ph, abort_flag);
                if (!ok) break;
                const bool two = i + 2 < n;
                uint64_t* bar = i >= jc ? &raw[slot] : &full[slot];
                sm100::mbar_arrive_expect_tx(bar, two ? 2 * TILE : TILE);
                const uint32_t dst = sm100::smem_u32(ring + slot * 2 * TILE);
                for (int h = 0; h < DP / 64; ++h)
                    tma_load_4d(dst + h * HALF, &map_v, bar, 64 * h, k0 + i * BN, kvh, slab);
                if (two)
                    for (int h = 0; h < DP / 64; ++h) tma_load_4d(dst + TILE + h * HALF, &map_k, bar, 64 * h, k0 + (i + 2) * BN, kvh, slab);
                if (++slot == NS) { slot = 0; ph ^= 1u; }
            }
        }
    } else if (warp == SM_WARPS + 1) {
        // ------------------------------------------------------------ MMAs
        // The whole warp walks the steps without a branch that its lanes could part at, and a predicate picks the lane that issues:
        // what the loop computes is then known to be the same in every lane and stays in uniform registers, where the products
        // want it.  A barrier is looked at before the products in front of its use are issued, and waited for
        // only if it was not done then: issuing is in order, so a wait holds up what comes after it, 150 cycles and more even
        // when there is nothing to wait for.  (Products alone 670 cycles a step and tile, their own time; with the loop inside an
        // "if (lane == 0)" 1000 and more, each descriptor being moved between register files, with four waits a step 1000.)
        const int un = __shfl_sync(0xffffffffu, n, 0), un0 = __shfl_sync(0xffffffffu, n0, 0), un1 = __shfl_sync(0xffffffffu, n1, 0);
        const int ujc = __shfl_sync(0xffffffffu, jc, 0);
        const uint32_t ut = __shfl_sync(0xffffffffu, tmem, 0);
        if (un > 0) {
            const uint32_t leader = elect_one();
            const uint32_t idesc_s = sm100::make_idesc_bf16(BM, BN);
            const uint32_t idesc_o = sm100::make_idesc_bf16(BM, DP) | (1u << 16);      // B is N-major
            const uint32_t full_at = sm100::smem_u32(full), empty_at = sm100::smem_u32(empty), clean_at = sm100::smem_u32(clean);
            const uint32_t s_at = sm100::smem_u32(s_full), p_at = sm100::smem_u32(p_ready), o_at = sm100::smem_u32(o_done);
            const uint64_t dq = sm100::make_desc_k_sw128(sm100::smem_u32(smem)), dk = sm100::make_desc_k_sw128(sm100::smem_u32(ring));
            const uint64_t dv = make_desc_mn_sw128(sm100::smem_u32(ring), HALF);
            uint32_t stage = 0, full_ph = 0, clean_ph = 0;       // full_ph, clean_ph: of each stage its next phase, not every round signals both
            auto scores = [&](int x, int buf, uint32_t at) {     // at: of the K tile in the ring
#pragma unroll
                for (int k = 0; k < DP / 16; ++k)
                    umma_ss(leader, ut + (uint32_t)(128 * x + 64 * buf), dq + (uint32_t)((x * QT + (k >> 2) * QHALF) / 16 + 2 * (k & 3)),
                            dk + (uint32_t)(at / 16) + (uint32_t)((k >> 2) * HALF / 16 + 2 * (k & 3)), idesc_s, k > 0);
                commit(leader, s_at + (uint32_t)(8 * (2 * x + buf)));        // (and the products before it)
            };
            ok = bar_wait(q_full, 0, abort_flag) && bar_wait(full_at, 0, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            full_ph = 1u;
            if (ok) {
                sm100::tc_fence_after_sync();
                if (un0 > 0) scores(0, 0, 0);
                if (un1 > 0) scores(1, 0, 0);
                if (un0 > 1) scores(0, 1, TILE);
                if (un1 > 1) scores(1, 1, TILE);
                commit(leader, empty_at);
            }
            stage = 1;
            uint32_t kv_done = 0, p_done = 0;
            // One step.  PLAIN: both tiles take part in it and in the one after the next, no V tile is cleaned.
            auto step = [&](int j, auto plain_, auto buf_) {
                constexpr bool PLAIN = decltype(plain_)::value;
                constexpr int buf = decltype(buf_)::value;
                const uint32_t here = stage, at = here * (uint32_t)(2 * TILE), p_phase = (uint32_t)(j >> 1) & 1u;
                const bool cleaned = !PLAIN && j >= ujc;
                if (!kv_done) ok = bar_wait((cleaned ? clean_at : full_at) + 8 * here, ((cleaned ? clean_ph : full_ph) >> here) & 1u, abort_flag) && ok;
                if (cleaned) clean_ph ^= 1u << here; else full_ph ^= 1u << here;
                stage = here + 1 == NS ? 0 : here + 1;
#pragma unroll
                for (int x = 0; x < TILES; ++x) {
                    const int nx = x ? un1 : un0;
                    const bool live = PLAIN || j < nx;
                    if (live && !p_done) ok = bar_wait(p_at + (uint32_t)(8 * (2 * x + buf)), p_phase, abort_flag) && ok;
                    sm100::tc_fence_after_sync();
                    // the next looks: at the other tile's weights of this step, or the first's of the next and the next stage
                    if (x + 1 < TILES) {
                        p_done = peek(p_at + (uint32_t)(8 * (2 + buf)), p_phase);
                    } else {
                        const bool next_cleaned = !PLAIN && j + 1 >= ujc;
                        p_done = peek(p_at + (uint32_t)(8 * (buf ^ 1)), (uint32_t)((j + 1) >> 1) & 1u);
                        kv_done = peek((next_cleaned ? clean_at : full_at) + 8 * stage, ((next_cleaned ? clean_ph : full_ph) >> stage) & 1u);
                    }
                    if (live) {
#pragma unroll
                        for (int k = 0; k < BN / 16; ++k)
                            umma_ts(leader, ut + (uint32_t)(128 * TILES + 128 * x), ut + (uint32_t)(128 * x + 64 * buf + 8 * k), dv + at / 16 + (uint32_t)(k * (2048 / 16)), idesc_o,
                                    (j > 0 || k > 0) ? 1u : 0u);
                        if (!PLAIN && j + 2 >= nx) commit(leader, o_at + (uint32_t)(16 * x) + (j + 1 == nx ? 8u : 0u));
                    }
                    if (PLAIN || j + 2 < nx) scores(x, buf, at + TILE);       // over P, which the product before it reads: issued in order
                }
                commit(leader, empty_at + 8 * here);
                ok = __all_sync(0xffffffffu, ok);
            };
            int j = 0;
            const int plain = min((TILES == 2 ? min(un0, un1) : un0) - 2, ujc);
            for (; j + 2 <= plain && ok; j += 2) {
                step(j, std::true_type{}, std::integral_constant<int, 0>{});
                if (ok) step(j + 1, std::true_type{}, std::integral_constant<int, 1>{});
            }
            kv_done = 0;        // (the last plain step's look did not reckon with cleaning)
            for (; j < un && ok; ++j) {
                if (j & 1) step(j, std::false_type{}, std::integral_constant<int, 1>{});
                else step(j, std::false_type{}, std::integral_constant<int, 0>{});
            }
        }
    } else {
        // ------------------------------------------------------------ V tiles that some row sees only in part
        uint32_t raw_ph = 0;
        for (int j = jc; j < n; ++j) {
            const int slot = (j + 1) % NS;
            ok = __all_sync(0xffffffffu, bar_wait(&raw[slot], (raw_ph >> slot) & 1u, abort_flag));
            raw_ph ^= 1u << slot;
            if (!ok) break;
            char* tile = ring + slot * 2 * TILE;
            const int from = seen_by_all - j * BN > 0 ? seen_by_all - j * BN : 0;         // rows before it are everybody's
            bool odd = false;
            // a lane's column of 16 bytes, in rows eight apart, four rows of both halves at a time
            for (int row0 = from + (warp - SM_WARPS - 2) * 4 + (lane >> 3); row0 < BN; row0 += 32) {
                uint4 w[4][DP / 64];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int h = 0; h < DP / 64; ++h)
                        if (row0 + 8 * i < BN) w[i][h] = *reinterpret_cast<const uint4*>(tile + h * HALF + (row0 + 8 * i) * 128 + (lane & 7) * 16);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int h = 0; h < DP / 64; ++h) {
                        const int row = row0 + 8 * i;
                        if (row >= BN) continue;
                        uint4* p = reinterpret_cast<uint4*>(tile + h * HALF + row * 128 + (lane & 7) * 16);
                        if (j * BN + row >= lk) {
                            *p = make_uint4(0u, 0u, 0u, 0u);
                            continue;
                        }
                        uint32_t* e = &w[i][h].x;
                        bool hit = false;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {        // exponent of all ones
                            if ((e[c] & 0x7f80u) == 0x7f80u) { e[c] &= 0xffff0000u; hit = true; }
                            if ((e[c] & 0x7f800000u) == 0x7f800000u) { e[c] &= 0xffffu; hit = true; }
                        }
                        if (hit) { *p = w[i][h]; odd = true; }
                    }
            }
            if (odd) *odd_v = 1;
            sm100::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&clean[slot]);
        }
    }
    } else {
        // ------------------------------------------------------------ softmax and epilogue: TMEM lane == row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Z::kRegsSoftmax));
        const int x = warp >> 2, row = 32 * (warp & 3) + lane;
        const int nx = x ? n1 : n0;
        const int cnt = count(i0 + x * a.tpg + row / a.G);
        const int seen = nx > 0 ? count(i0 + x * a.tpg) : 0;        // keys that every row of the tile sees
        const uint32_t t_lane = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t to = t_lane + 128u * TILES + 128u * x;
        const float sc = a.scale_log2;
        float ref = -INFINITY, l = 0.f;         // in units of S
        float first = 0.f, bias = 0.f;          // weights are 2^((S - first) sc + bias)
        bool far = false;                       // first is not zero in some lane
        for (int j = 0; j < nx; ++j) {
            const int buf = j & 1;
            const uint32_t ts = t_lane + 128u * x + 64u * buf;
            ok = __all_sync(0xffffffffu, bar_wait(&s_full[2 * x + buf], (uint32_t)(j >> 1) & 1u, abort_flag));
            if (!ok) break;
            sm100::tc_fence_after_sync();
            uint32_t r[BN];
#pragma unroll
            for (int c = 0; c < BN; c += 32) sm100::tmem_ld_32x32(ts + c, reinterpret_cast<uint32_t(&)[32]>(r[c]));
            tmem_ld_wait(reinterpret_cast<uint32_t(&)[32]>(r[0]));
            tmem_ld_tie(reinterpret_cast<uint32_t(&)[32]>(r[32]));
            if ((j + 1) * BN > seen) {
                const int lim = cnt - j * BN;
#pragma unroll
                for (int e = 0; e < BN; ++e) if (e >= lim) r[e] = 0xff800000u;
            }
            float m4[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                m4[k] = max3(__uint_as_float(r[k]), __uint_as_float(r[4 + k]), __uint_as_float(r[8 + k]));
#pragma unroll
                for (int e = 12 + k; e < BN - 4; e += 8) m4[k] = max3(m4[k], __uint_as_float(r[e]), __uint_as_float(r[e + 4]));
            }
            static_assert((BN - 16) % 8 == 0, "the pairs above end four before the end");
            const float mx = max3(max3(m4[0], m4[1], __uint_as_float(r[BN - 4])), max3(m4[2], m4[3], __uint_as_float(r[BN - 3])),
                                  max3(__uint_as_float(r[BN - 2]), __uint_as_float(r[BN - 1]), -INFINITY));
            // a new reference point where the maximum has grown by more than 2^8
            const bool move = (mx - ref) * sc > 8.f;        // (-inf - -inf is NaN: no)
            if (__any_sync(0xffffffffu, move || !(mx < INFINITY))) {
                if (!(mx < INFINITY)) l = __uint_as_float(0x7fc00000u);        // a score that is infinite or none: so is the row
                const float corr = move ? ex2((ref - mx) * sc) : 1.f;
                if (move) ref = mx;
                l *= corr;
                // 2^(S sc - ref sc) in one multiply-add.  The rounding of ref sc divides out only among the keys of one reference point;
                // up to 1024 it is 2^-15 at most, 2.1e-5 of a weight (P's own rounding is 2^-8), beyond, the difference is taken
                // first.  A row by itself: its neighbours in the warp may be other sequences' and have no say in its bits.
                const bool large = ref != -INFINITY && fabsf(ref * sc) > 1024.f;
                far = __any_sync(0xffffffffu, large);
                first = large ? ref : 0.f;
                bias = large || ref == -INFINITY ? 0.f : -ref * sc;
                if (j > 0) {
                    // the product before has retired: the next step's scores come after it, or, at the end, its own signal does
                    const bool next = j + 1 < nx;
                    ok = __all_sync(0xffffffffu, bar_wait(next ? &s_full[2 * x + (buf ^ 1)] : &o_done[2 * x], next ? (uint32_t)((j + 1) >> 1) & 1u : 0u, abort_flag));
                    if (!ok) break;
                    sm100::tc_fence_after_sync();
#pragma unroll 1
                    for (int c = 0; c < DP; c += 16) {
                        uint32_t o[16];
                        tmem_ld_32x16(to + c, o);
                        tmem_ld_wait(o);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                        tmem_st_32x16(to + c, o);
                    }
                }
            }
            if (far) {
#pragma unroll
                for (int e = 0; e < BN; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) - first);
            }
            const f2 sc2 = pair(sc, sc), bias2 = pair(bias, bias);
            f2 l2[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
            for (int c = 0; c < BN; c += 32) {
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    f2 y = fma2(pair(__uint_as_float(r[c + 2 * e]), __uint_as_float(r[c + 2 * e + 1])), sc2, bias2);
                    float y0, y1;
                    if (e % 4 < kPolyOf4) {
                        y = ex2_pair(y);
                        split(y, y0, y1);
                    } else {
                        split(y, y0, y1);
                        y0 = ex2(y0);
                        y1 = ex2(y1);
                        y = pair(y0, y1);
                    }
                    l2[e & 1] = add2(l2[e & 1], y);
                    p[e] = bf2(y0, y1);
                }
                tmem_st_32x16(ts + c / 2, p);        // over scores that this warp has taken
            }
            float l0, l1;
            split(add2(l2[0], l2[1]), l0, l1);
            l += l0 + l1;
            tmem_st_wait();
            sm100::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&p_ready[2 * x + buf]);
        }
        if (ok && nx > 0) ok = __all_sync(0xffffffffu, bar_wait(&o_done[2 * x + 1], 0, abort_flag));
        if (ok) {
            sm100::tc_fence_after_sync();
            const int tok = job[6] + x * a.tpg + row / a.G, head = job[7];
            const bool live = row < a.G * a.tpg && tok < job[2] && tok < a.max_q, shared = TILES == 2 && a.splits > 1 && find_share(a, job[2], job[4], job[6]).used > 1;
            const float inv = shared ? 1.f : 1.f / l;
            const bool odd = nx > 0 && *odd_v != 0;
            __nv_bfloat16* dst = a.out + (int64_t)(job[1] + tok) * a.o_tok + (int64_t)(head * a.G + row % a.G) * a.o_head;
            float* part = a.part + (int64_t)blockIdx.x * (DP + 2) * 2 * BM + x * BM + row;
            char* stage = smem + warp * (32 * DP * 2);      // 32 rows; Q has been read: the tile's last product has retired
            if (shared && live) {
                part[0] = ref;
                part[2 * BM] = l;
            }
#pragma unroll 1
            for (int d = 0; d < DP; d += 32) {
                uint32_t r[32];
                if (nx > 0) {
                    sm100::tmem_ld_32x32(to + d, r);
                    tmem_ld_wait(r);
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) r[e] = cnt <= 0 ? 0u : __float_as_uint(__uint_as_float(r[e]) * inv);     // (scores of -inf alone: NaN)
                if (odd && live) {      // infinities and NaNs that were taken out of V, back to the rows that see them
                    const __nv_bfloat16* vp = a.v + (a.cu_k != nullptr ? 0 : (int64_t)job[5] * a.v_seq) + (int64_t)head * a.v_head + (int64_t)k0 * a.v_row;
                    for (int kk = seen_by_all; kk < cnt; ++kk)
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float y = d + e < a.D ? __bfloat162float(vp[(int64_t)kk * a.v_row + d + e]) : 0.f;
                            if (!(fabsf(y) <= 3.4e38f)) r[e] = __float_as_uint(__uint_as_float(r[e]) + y);
                        }
                }
                if (shared) {
                    if (live) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) part[(2 + d + e) * 2 * BM] = __uint_as_float(r[e]);
                    }
                } else if (nx == 0) {               // (Q may still be landing)
                    if (live) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (d + 8 * e < a.D) *reinterpret_cast<uint4*>(dst + d + 8 * e) = make_uint4(0u, 0u, 0u, 0u);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<uint4*>(stage + lane * (DP * 2) + (((d >> 3) + e) ^ (lane & 7)) * 16) =
                            make_uint4(bf2(__uint_as_float(r[8 * e]), __uint_as_float(r[8 * e + 1])), bf2(__uint_as_float(r[8 * e + 2]), __uint_as_float(r[8 * e + 3])),
                                       bf2(__uint_as_float(r[8 * e + 4]), __uint_as_float(r[8 * e + 5])), bf2(__uint_as_float(r[8 * e + 6]), __uint_as_float(r[8 * e + 7])));
                }
            }
            // Rows by way of shared memory: a store of 16 bytes to each of 32 rows is 32 half sectors, and was the longest part of
            // a short CTA.
            if (!shared && nx > 0) {
                __syncwarp();
                constexpr int PER = DP / 8, AT_ONCE = 32 / PER;     // lanes to a row, rows to a store
                const int64_t mine = live ? dst - a.out : -1;
#pragma unroll 1
                for (int i0 = 0; i0 < PER; i0 += 8) {       // (all eight read before the first is written: nothing says that they differ)
                    uint4 w[8];
                    int64_t off[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int from = (i0 + i) * AT_ONCE + lane / PER, c = lane % PER;
                        off[i] = __shfl_sync(0xffffffffu, mine, from);
                        if (8 * c >= a.D) off[i] = -1;
                        w[i] = *reinterpret_cast<const uint4*>(stage + from * (DP * 2) + (c ^ (from & 7)) * 16);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (off[i] >= 0) *reinterpret_cast<uint4*>(a.out + off[i] + 8 * (lane % PER)) = w[i];
                }
            }
        }
    }

    if (!ok && (warp == SM_WARPS || warp == SM_WARPS + 1)) {     // gave up: let copies and products already in flight land
        const long long t0 = clock64();
        while (clock64() - t0 < 20000000LL) { }
    }
    sm100::tc_fence_before_sync();
    __syncthreads();
    if (warp == SM_WARPS + 1) {
        sm100::tc_fence_after_sync();
        sm100::tmem_dealloc(tmem, 256 * TILES);
    }
    if (threadIdx.x == 0 && *abort_flag != 0 && a.status != nullptr) atomicExch(a.status, HXQ_E_TIMEOUT);
}

// The shares' results of one row: out = sum_p 2^((m_p - M) sc) o_p / sum_p 2^((m_p - M) sc) l_p.  A CTA has 32 rows of a
// tile, a lane each (in memory the rows are innermost), and kJoin dimensions; its warps take every eighth share and meet in
// shared memory.
constexpr int kJoin = 16;
template <int DP>
__global__ void __launch_bounds__(256) join_kernel(const Args a) {
    __shared__ float meet[8][2 + kJoin][32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int d = blockIdx.x % (DP / kJoin) * kJoin, group = blockIdx.x / (DP / kJoin) % a.groups, item = blockIdx.x / (DP / kJoin) / a.groups;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Seq seq;
    int s, ct, kvh;
    if (!find_item(a, item, seq, s, ct, kvh)) return;
    const int used = find_share(a, seq.lq, seq.lk, ct * a.rows).used;
    if (used == 1) return;              // written already
    const int x = group >> 2, first = (2 * ct + x) * a.tpg, left = (seq.lq < a.max_q ? seq.lq : a.max_q) - first, rows = a.G * (left < a.tpg ? left : a.tpg);
    const int in = (group & 3) * 32 + lane;
    float m = -INFINITY, l = 0.f, o[kJoin] = {};
    if (in < rows) {
        const float* part = a.part + (int64_t)item * a.splits * (DP + 2) * 2 * BM + x * BM + in;
#pragma unroll 2
        for (int p = warp; p < used; p += 8) {
            const float* q = part + (int64_t)p * (DP + 2) * 2 * BM;
            float v[kJoin];
            const float ref = q[0], sum = q[2 * BM];
#pragma unroll
            for (int e = 0; e < kJoin; ++e) v[e] = q[(2 + d + e) * 2 * BM];
            const float top = fmaxf(m, ref), c = m == -INFINITY ? 0.f : ex2((m - top) * a.scale_log2), w = ref == -INFINITY ? 0.f : ex2((ref - top) * a.scale_log2);
            m = top;
            l = c * l + w * sum;        // (NaN, a row's that sees one, stays one whatever the weights)
#pragma unroll
            for (int e = 0; e < kJoin; ++e) o[e] = c * o[e] + w * v[e];
        }
    }
    meet[warp][0][lane] = m;
    meet[warp][1][lane] = l;
#pragma unroll
    for (int e = 0; e < kJoin; ++e) meet[warp][2 + e][lane] = o[e];
    __syncthreads();
    if (in >= rows || d + 2 * warp >= a.D) return;        // a warp, two dimensions
    float top = -INFINITY;
#pragma unroll
    for (int p = 0; p < 8; ++p) top = fmaxf(top, meet[p][0][lane]);
    float sum = 0.f, y0 = 0.f, y1 = 0.f;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const float w = meet[p][0][lane] == -INFINITY ? 0.f : ex2((meet[p][0][lane] - top) * a.scale_log2);
        sum += w * meet[p][1][lane];
        y0 += w * meet[p][2 + 2 * warp][lane];
        y1 += w * meet[p][3 + 2 * warp][lane];
    }
    const bool none = reach(a, seq.lq, seq.lk, first + in / a.G) == 0;
    const float inv = 1.f / sum;
    __nv_bfloat16* dst = a.out + (int64_t)(seq.q0 + first + in / a.G) * a.o_tok + (int64_t)(kvh * a.G + in % a.G) * a.o_head + d + 2 * warp;
    *reinterpret_cast<uint32_t*>(dst) = none ? 0u : bf2(y0 * inv, y1 * inv);
}

// ---- host side ---------------------------------------------------------------------

struct Plan {
    int tpg, rows, n_ct, items, splits, alone, groups;
};
// Items: the tokens' tiles, two to a CTA, and one more for each sequence's last.
// Few of them before many keys leave SMs idle: then their key tiles are shared out, to as many CTAs (room) as there are SMs
// for.  Sharing costs a launch and the shares' way through memory, and pays from some number of key tiles on, the sooner the more
// room there is (28 + 4 heads, 16 queries, room 37, behind 32768 keys: 360 -> 28 us; 256, room 4: 349 -> 145, but 19 -> 28
// behind 1024; 512, room 2: 352 -> 276, but 50 -> 63 behind 4096).  max_q has no say in any of this: it would in the result's last bits.
// Items that stay whole have one tile each and come two to an SM, where one's start and end pass behind the other's products
// (813 tokens behind 8111: 106 -> 95 us; 908 tokens of 3 heads: 18.9 -> 13.8 us), unless there are so many that these matter less than
// keys and values read twice as often (16384 tokens: 1543 us together, 1636 apart).
static bool make_plan(const hxq_attn* p, Plan& plan) {
    plan.tpg = BM / (p->nq / p->nkv);
    const int64_t max_q = p->max_q < p->Tq ? p->max_q : p->Tq;
    const int64_t all = ((int64_t)p->Tq / (2 * plan.tpg) + p->S) * p->nkv, room = 148 / all;
    const int64_t keys = p->cu_k == p->cu_q && max_q < p->Tk ? max_q : p->Tk;        // of one sequence, at most
    const int64_t steps = (keys + BN - 1) / BN, parts = (steps + kShare - 1) / kShare;
    plan.alone = room > 1 ? 16 + (int)(384 / (room * room)) : 0;
    plan.splits = room > 1 && steps > plan.alone ? (int)(parts < room ? parts : room) : 1;
    plan.rows = plan.splits > 1 || all >= kMany ? 2 * plan.tpg : plan.tpg;
    const int64_t n_ct = (max_q + plan.rows - 1) / plan.rows;
    const int64_t some = (int64_t)p->Tq / plan.rows + p->S, most = n_ct * p->S, n = (some < most || p->S > kSorted ? some : most) * p->nkv;
    plan.n_ct = (int)n_ct;
    plan.items = (int)n;
    plan.groups = max_q > plan.tpg ? 8 : (int)((max_q * (p->nq / p->nkv) + 31) / 32);
    return n <= 0x7fffffffLL / 128;
}
static size_t part_bytes(const hxq_attn* p, const Plan& plan) {
    return plan.splits == 1 ? 0 : (size_t)plan.items * plan.splits * 2 * BM * ((p->D <= 64 ? 64 : 128) + 2) * sizeof(float);
}

template <int DP, int TILES>
static int run_tiles(const hxq_attn* p, const Plan& plan, void* workspace, int32_t* status, cudaStream_t stream) {
    using Z = Sizes<DP, TILES>;
    Args a;
    a.cu_q = p->cu_q; a.cu_k = p->cu_k; a.k_len = p->k_len;
    a.v = reinterpret_cast<const __nv_bfloat16*>(p->v);
    a.out = reinterpret_cast<__nv_bfloat16*>(p->out);
    a.status = status;
    a.v_seq = p->v_seq; a.v_head = p->v_head; a.v_row = p->v_row; a.o_tok = p->o_tok; a.o_head = p->o_head;
    a.Tq = p->Tq; a.Tk = p->Tk; a.S = p->S; a.max_q = p->max_q; a.nkv = p->nkv; a.G = p->nq / p->nkv; a.D = p->D; a.causal = p->causal != 0;
    a.tpg = plan.tpg;
    a.rows = plan.rows;
    a.n_ct = plan.n_ct;
    a.splits = plan.splits;
    a.alone = plan.alone;
    a.groups = plan.groups;
    a.part = reinterpret_cast<float*>(workspace);
    a.scale_log2 = p->scale * 1.4426950408889634f;

    CUtensorMap mq, mk, mv;
    // (the stride of a dimension of one element is never used, but has to be a valid one)
    auto st = [](int64_t elements, int64_t extent) { return extent > 1 ? (uint64_t)elements * 2 : (uint64_t)16; };
    const uint64_t qd[3] = {(uint64_t)p->D, (uint64_t)p->nq, (uint64_t)p->Tq}, qs[2] = {st(p->q_head, p->nq), st(p->q_tok, p->Tq)};
    const uint32_t qb[3] = {64, (uint32_t)a.G, (uint32_t)a.tpg};
    const uint64_t slabs = p->cu_k ? 1 : (uint64_t)p->S;
    const uint64_t kd[4] = {(uint64_t)p->D, (uint64_t)p->Tk, (uint64_t)p->nkv, slabs};
    const uint64_t ks[3] = {st(p->k_row, p->Tk), st(p->k_head, p->nkv), st(p->k_seq, (int64_t)slabs)};
    const uint64_t vs[3] = {st(p->v_row, p->Tk), st(p->v_head, p->nkv), st(p->v_seq, (int64_t)slabs)};
    const uint32_t kb[4] = {64, BN, 1, 1};
    const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (!gemm::make_map_nd(&mq, dt, 3, p->q, qd, qs, qb, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !gemm::make_map_nd(&mk, dt, 4, p->k, kd, ks, kb, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !gemm::make_map_nd(&mv, dt, 4, p->v, kd, vs, kb, CU_TENSOR_MAP_SWIZZLE_128B))
        return HXQ_E_DEVICE;
    static bool attr_set[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return HXQ_E_DEVICE;
    if (!attr_set[dev]) {
        cudaFuncAttributes fa;        // the warps' exchange of registers counts on what the launch brings
        if (cudaFuncGetAttributes(&fa, attn_prompt_kernel<DP, TILES>) != cudaSuccess || (fa.numRegs + 7) / 8 * 8 < Z::kRegsLaunch) return HXQ_E_DEVICE;
        if (cudaFuncSetAttribute(attn_prompt_kernel<DP, TILES>, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::kSmem) != cudaSuccess) return HXQ_E_DEVICE;
        attr_set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(plan.items * plan.splits));
    cfg.blockDim = dim3(Z::kThreads);
    cfg.dynamicSmemBytes = Z::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, attn_prompt_kernel<DP, TILES>, mq, mk, mv, a);
    if (e == cudaSuccess && plan.splits > 1) {
        cfg.gridDim = dim3((unsigned)(plan.items * plan.groups * (DP / kJoin)));
        cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = 0;
        e = cudaLaunchKernelEx(&cfg, join_kernel<DP>, a);
    }
    return e == cudaSuccess ? HXQ_OK : HXQ_E_LAUNCH;
}
template <int DP>
static int run(const hxq_attn* p, const Plan& plan, void* workspace, int32_t* status, cudaStream_t stream) {
    return plan.rows == plan.tpg ? run_tiles<DP, 1>(p, plan, workspace, status, stream) : run_tiles<DP, 2>(p, plan, workspace, status, stream);
}

}  // namespace attnp
}  // namespace hxq

static int check(const hxq_attn* p) {
    if (!p || !p->q || !p->k || !p->v || !p->out || !p->cu_q || (!p->cu_k) == (!p->k_len)) return HXQ_E_ARG;
    if (p->Tq < 0 || p->Tk < 0 || p->S <= 0 || p->max_q < 0 || !(p->scale > 0.f) || !(p->scale <= 3.4e38f)) return HXQ_E_ARG;
    if (p->Tq > 1 << 30 || p->Tk > 1 << 30) return HXQ_E_SHAPE;        // (coordinates past the end stay in 32 bits)
    if (p->nq <= 0 || p->nkv <= 0 || p->nq % p->nkv != 0 || p->nq / p->nkv > 64) return HXQ_E_SHAPE;
    if (p->D < 8 || p->D > 128 || p->D % 8 != 0) return HXQ_E_SHAPE;
    const int64_t strides[10] = {p->q_tok, p->q_head, p->k_seq, p->k_head, p->k_row, p->v_seq, p->v_head, p->v_row, p->o_tok, p->o_head};
    for (int64_t s : strides)
        if (s < 0 || s >= (int64_t(1) << 38) || s % 8 != 0) return HXQ_E_ALIGN;
    if (!hxq::aligned_to(p->q, 16) || !hxq::aligned_to(p->k, 16) || !hxq::aligned_to(p->v, 16) || !hxq::aligned_to(p->out, 16)) return HXQ_E_ALIGN;
    return HXQ_OK;
}

extern "C" size_t hxq_attn_prompt_workspace_bytes(const hxq_attn* p) {
    hxq::attnp::Plan plan;
    return check(p) == HXQ_OK && hxq::attnp::make_plan(p, plan) ? hxq::attnp::part_bytes(p, plan) : 0;
}

extern "C" int hxq_attn_prompt(const hxq_attn* p, void* workspace, size_t workspace_bytes, int32_t* status_word, hxq_stream_t stream) {
    const int bad = check(p);
    if (bad != HXQ_OK) return bad;
    hxq::attnp::Plan plan;
    if (!hxq::attnp::make_plan(p, plan)) return HXQ_E_SHAPE;
    if (plan.items == 0) return HXQ_OK;
    if (p->Tk == 0) return HXQ_E_SHAPE;
    const size_t need = hxq::attnp::part_bytes(p, plan);
    if (need > 0 && (!workspace || !hxq::aligned_to(workspace, 8) || workspace_bytes < need)) return HXQ_E_WORKSPACE;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return p->D <= 64 ? hxq::attnp::run<64>(p, plan, workspace, status_word, st) : hxq::attnp::run<128>(p, plan, workspace, status_word, st);
}
