// Causal attention over a paged 4-bit KV cache (include/ckb200_cache.h), one or several new tokens of each sequence, on the tensor cores at fp32
// accuracy.
//
// Mathematics.  A block of 32 key channels is k = d c + m with 4-bit codes c, so a score is the sum over blocks of d (q . c) + m (sum q); a
// block of value channels is v = d (c - 8) + (m + 8 d), so its part of the output is the sum over keys of (p d) (c - 8) + p (m + 8 d).  Every inner
// product has a small integer or a number of the block on one side, exact in fp16 (the middle m + 8 d as two pieces), and on the other an fp32 number
// that goes in as two fp16 pieces, x = hi + lo, 22 bits, whose products add up in the same fp32 accumulator.
//   * Key codes are not converted at all: a nibble in bits 4..7 of a half IS the subnormal 16 c * 2^-24, so masks and shifts of a word of codes make
//     operands, and the power of two is taken out of the result.  (Not in bits 0..3: the tensor cores line products up without normalising them, and what a
//     subnormal has in leading zeros is lost below: 2e-5 of the result at 500 keys.)
//   * Value codes are taken from their middle.  With c in place of c - 8 all terms of the sum have one sign, the tensor cores cut what they add to an accumulator
//     instead of rounding it, and the error adds up: 2.3e-5 of the result at 131072 keys, 7e-7 as it is here.
//   * Ranges: queries are scaled so that the largest of a row is in [2^14, 2^15), weights, relative to a reference that may lag 2^3 behind the largest, by 2^10.  Steps and middles (which
//     reach 9 * 65504) are scaled chunk by chunk, so that the largest step is below 4 and the largest middle below 2^15: no piece passes fp16's range.  Blocks whose step is about 2^10 below the
//     chunk's largest would lose bits with that scale.  They are left out of the products and weighed in fp32, key by key, and every block is as exact as it would be alone (32 sequences of up
//     to 4096 tokens: 51 us without such blocks, 60 us with one key of 64, 262 us with 31 keys of 32).  A weight times a step is a rounded half-precision product and its exact remainder.
//
//   scores  S^T = K Q^T   mma.m16n8k16: 16 keys x 8 query rows; a thread's A words are 4 bytes of codes of keys g and g + 8 (lane = 4 g + t), which
//                         settles which channel sits at which k: the query's fragments are laid out to match
//           from S^T to the operand P^T: a thread's weights of one key and two rows are a word of each piece, and a transpose of 8 x 8 halves between lanes makes
//                         them those of one row and two keys
//   output  O^T = V^T P^T 16 channels x 8 query rows; A words are the same two bytes (four channels) of two keys, joined by one byte permute
//
// A query row is a (token, head) of the kv head's group: up to 8 NB rows share every code that is unpacked (NB = 1 for decoding, more for
// drafts and portions of prompts).  Up to four rows take one product instead of two: its eight columns are their hi and their lo pieces.
//
// Work.  A unit is 128 keys of one (sequence, block of 8 NB rows, kv head); the units of all sequences form one line that is cut evenly among the CTAs that
// the GPU holds at once, so long and short sequences load it alike and nothing but the lengths on the device decides.  Each of the four warps takes
// a quarter of a unit through a ring of its own (untiled bulk copies: 32 rows of K and of V, or 16 where pages may end between), without meeting the
// others until a sequence's stretch ends; then each warp joins a quarter of the accumulators while the next queries load.  Stretches that lie within one CTA are
// written out at once, the others as partial results that a second kernel joins (log-sum-exp).
//
// What bounds it.  Not HBM: the ring alone, without the arithmetic, takes 113 us for four sequences of 131072 tokens (64 heads over 8 of 128 channels,
// 667 MB, 102 us at the measured copy rate), the whole call 215 us, 3.1 TB/s (32 heads: 187 us, 3.6 TB/s).  A chunk of 32 keys is 1045 warp instructions, 74 of them
// products (38 with four rows), issued at 2.5 an SM and cycle: products, half-precision instructions and integer multiplications share one pipe, half-rate logic (codes, 300
// instructions) has another, each is busy for 20 to 40 % of the time, and a warp waits 1.8 cycles an instruction for the one before it.
// Two, three or four CTAs an SM (8 to 16 warps, 255 to 128 registers): 235 / 215 / 207 us inside a graph.
#include <cuda_fp16.h>
#include <math.h>

#include "../../include/ckb200_cache.h"
#include "device_common.cuh"
#include "kv_q4.cuh"
#include "launch.h"
#include "pdl.cuh"
#include "runtime.h"

namespace ckb {

constexpr int AQ_WARPS = 4, AQ_THREADS = 32 * AQ_WARPS;

// BLOCKS 4: one block and four CTAs an SM, for long caches; 0: up to four query rows, whose hi pieces are columns 0 .. 3 of a product and whose lo pieces are columns 4 .. 7
template <int HD, int BLOCKS>
struct AqShape {
    static constexpr bool PACK = BLOCKS == 0, FOUR = BLOCKS == 4;
    static constexpr int NB = PACK || FOUR ? 1 : BLOCKS, G4 = HD / 32, KS = HD / 16, ROW = G4 * KQ4_BLOCK, ROWS = PACK ? 4 : 8 * NB;
    static constexpr int XT = 2, CHUNK = 16 * XT, UNIT = AQ_WARPS * CHUNK;      // a warp takes XT tiles of 16 keys at a time
    static constexpr int STAGE = 2 * CHUNK * ROW;                              // K rows, then V rows
    static constexpr int CTAS = NB > 1 || HD > 128 ? 2 : (FOUR ? 4 : 3);                       // resident on an SM, for which registers and shared memory are kept
    static constexpr int STAGES = HD <= 64 ? 4 : (HD <= 128 && NB < 3 && !FOUR ? 3 : 2);
    // the next stretch's queries load while one is joined, where there are registers: three blocks 97 us with it and 96 us without (20 rows of 16 sequences), four rows 187 and 186 us
    static constexpr bool EARLY = !PACK && NB < 3;
    static constexpr int MINE = NB * G4 * 2;                                  // each warp joins a quarter of the four warps' accumulators; it gives away the others
    static constexpr int GIVEN = AQ_WARPS * (3 * MINE * 32 + NB * 16) * 4;
    static constexpr int RING = AQ_WARPS * STAGES * STAGE, QF = NB * KS * 32 * 16, QS = NB * 32 * 8, TAB = AQ_WARPS * 3 * G4 * 2 * CHUNK;
    static constexpr int SMEM = RING + (QF + QS + TAB > GIVEN ? QF + QS + TAB : GIVEN);      // the exchange between warps lies over the queries
    static_assert(CTAS * (SMEM + 2048) <= 227 * 1024, "shared memory");
};

struct AqParams {
    const float *q;
    const uint8_t *k, *v;
    float *out;
    long long q_stride, out_stride;
    KvQ4 c;
    int G, R, RC, window, *err;                // G heads a kv head, R = tokens * G query rows a kv head, RC blocks of them
    float scale;
    KvDivide by_page, by_group;                // by page_tokens and by G
    int2 *desc;                                // [batch][Hkv][RC]: the first and the last CTA of a stretch that several work on; last < 0: one did
    float *part;                               // [2 CTAs][ROWS][HD + 2]: the stretch that began before the CTA, the one that goes on after it
};

// where a CTA is on the line of units
struct AqWalk {
    int b, h, rc, u, n, begin, end, len;       // unit u of n; keys [begin, end), begin a multiple of 32
};
// tokens r0 / G .. of block rc: the keys that any of them sees
__device__ __forceinline__ void aq_range(const AqParams &p, int nrows, int unit, AqWalk &w)
{
    const int t0 = p.by_group(w.rc * nrows), t1 = p.by_group(min(p.R, (w.rc + 1) * nrows) - 1), at = w.len - p.c.tokens;
    w.end = max(0, at + t1 + 1);
    w.begin = p.window > 0 ? max(0, at + t0 - p.window + 1) & ~31 : 0;      // a chunk's beginning
    w.n = w.end > w.begin ? (w.end - w.begin + unit - 1) / unit : 0;
}
__device__ __forceinline__ int aq_length(const AqParams &p, int b) { return kv_len(__ldcg(p.c.lens + b), p.c.stride, p.c.page_tokens); }
// the next block of rows
__device__ __forceinline__ void aq_next_block(const AqParams &p, int nrows, int unit, AqWalk &w)
{
    if (++w.rc == p.RC) {
        w.rc = 0;
        ++w.b;
        w.len = w.b < p.c.batch ? aq_length(p, w.b) : 0;
    }
    aq_range(p, nrows, unit, w);
}
// the first unit of the next stretch that has units, if there is one
__device__ __forceinline__ void aq_next_stretch(const AqParams &p, int nrows, int unit, AqWalk &w)
{
    w.u = 0;
    if (++w.h < p.c.Hkv) return;
    w.h = 0;
    do aq_next_block(p, nrows, unit, w);
    while (w.n == 0 && w.b < p.c.batch);
}

__device__ __forceinline__ void aq_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void aq_mma_k8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b)
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};" : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(b));
}
__device__ __forceinline__ void aq_mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// two fp32 operations in one instruction
__device__ __forceinline__ float2 aq_sub2(float2 a, float2 b)
{
    unsigned long long d;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<unsigned long long *>(&a)), "l"(*reinterpret_cast<unsigned long long *>(&b)));
    return *reinterpret_cast<float2 *>(&d);
}
// p = hi + lo, both fp16
__device__ __forceinline__ void aq_split(float2 p, uint32_t &hi, uint32_t &lo)
{
    const __half2 h = __floats2half2_rn(p.x, p.y);
    const float2 r = aq_sub2(p, __half22float2(h));
    const __half2 l = __floats2half2_rn(r.x, r.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
__device__ __forceinline__ float aq_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));       // two units in the last place
    return y;
}
// of a matrix of 8 x 8 halves, thread 4 g + t: (row g, columns 2t, 2t + 1) in, (column g, rows 2t, 2t + 1) out
__device__ __forceinline__ uint32_t aq_transpose(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t aq_u32(const uint8_t *p) { return *reinterpret_cast<const uint32_t *>(p); }
__device__ __forceinline__ uint32_t aq_u16(const uint8_t *p) { return *reinterpret_cast<const uint16_t *>(p); }
// nibble P of each half of the word, as 16 c * 2^-24
template <int P>
__device__ __forceinline__ uint32_t aq_codes(uint32_t w) { return (P == 0 ? w << 4 : w >> (P ? 4 * (P - 1) : 0)) & 0x00f000f0u; }
// nibble P of each half of the word, as the number c - 8
template <int P>
__device__ __forceinline__ uint32_t aq_centred(uint32_t w)
{
    uint32_t x, y;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(x) : "r"(P & 2 ? w >> 8 : w), "r"(P & 1 ? 0x00f000f0u : 0x000f000fu), "r"(0x64006400u));      // and, or: 1024 + c, or 1024 + 16 c
    if constexpr (P & 1) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(x), "r"(0x2c002c00u), "r"(0xd480d480u));      // x / 16 - 72
    else asm("add.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0xe408e408u));                                              // x - 1032
    return y;
}
__device__ __forceinline__ __half2 aq_h2(uint32_t x) { return *reinterpret_cast<const __half2 *>(&x); }
__device__ __forceinline__ uint32_t aq_bits(__half2 x) { return *reinterpret_cast<const uint32_t *>(&x); }
// (hi + lo) d of two keys = h + l: h the rounded product, l what it lacks, exact, and lo d
__device__ __forceinline__ void aq_weigh(uint32_t hi, uint32_t lo, uint32_t d, uint32_t &h, uint32_t &l)
{
    const __half2 p = __hmul2_rn(aq_h2(hi), aq_h2(d));
    l = aq_bits(__hfma2(aq_h2(lo), aq_h2(d), __hfma2(aq_h2(hi), aq_h2(d), __hneg2(p))));
    h = aq_bits(p);
}
constexpr float AQ_UNSCALE = 1048576.0f;       // 2^20
__device__ __forceinline__ float aq_lo(uint32_t dm) { return __low2float(*reinterpret_cast<const __half2 *>(&dm)); }
__device__ __forceinline__ float aq_hi(uint32_t dm) { return __high2float(*reinterpret_cast<const __half2 *>(&dm)); }
// For scales (d, m) of the blocks of a lane's key: the biased exponent of the chunk's largest |m| plus eight of its largest |d|, below 2^20 for what the store makes, and
// the lane's smallest |d|.  Numbers that are none do not count.
template <int G4>
__device__ __forceinline__ int aq_size(const uint32_t (&dm)[G4], float &least)
{
    __half2 top = __habs2(aq_h2(dm[0])), low = top;
#pragma unroll
    for (int j = 1; j < G4; ++j) {
        top = __hmax2(top, __habs2(aq_h2(dm[j])));
        low = __hmin2(low, __habs2(aq_h2(dm[j])));
    }
    least = __low2float(low);
    const float size = fmaxf(0.0f, fmaf(8.0f, __low2float(top), __high2float(top)));
    return max(127 - 24, min(127 + 19, (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(size)) >> 23)));
}
// what brings that into [16, 32), and back
__device__ __forceinline__ float aq_up(int size) { return __uint_as_float((uint32_t)(258 - size) << 23); }
__device__ __forceinline__ float aq_down(int size) { return __uint_as_float((uint32_t)(size - 4) << 23); }
// A block that is so much smaller that products with its step (or, where that is zero, with its one value) would lose bits.
constexpr float AQ_LEAST = 0x1p-10f;
__device__ __forceinline__ bool aq_late(uint32_t dm, float up)
{
    const float d = fabsf(aq_lo(dm)) * up, m = fabsf(aq_hi(dm)) * up;
    return fmaf(8.0f, d, m) < 2.0f && (d > 0.0f ? d < AQ_LEAST : m > 0.0f && m < 0x1p-13f);
}
__device__ __forceinline__ bool aq_no_number(uint32_t dm) { return (dm & 0x7c00u) == 0x7c00u || (dm & 0x7c000000u) == 0x7c000000u; }

template <int HD, int BLOCKS>
__global__ void __launch_bounds__(AQ_THREADS, AqShape<HD, BLOCKS>::CTAS) attn_q4_kernel(const AqParams p)
{
    using S = AqShape<HD, BLOCKS>;
    constexpr bool PACK = S::PACK;
    constexpr int NB = S::NB, G4 = S::G4, KS = S::KS, ROW = S::ROW, ROWS = S::ROWS, STAGES = S::STAGES;
    extern __shared__ __align__(128) uint8_t aq_smem[];
    __shared__ __align__(8) uint64_t full[AQ_WARPS][STAGES];
    __shared__ int pieces[AQ_WARPS][STAGES];
    __shared__ long long s_sum[AQ_WARPS];
    __shared__ AqWalk s_walk;
    uint4 *qf = reinterpret_cast<uint4 *>(aq_smem + S::RING);                     // [NB][KS][lane] {hi b0, hi b1, lo b0, lo b1}; PACK: [KS][lane] {b0, b1}
    const uint2 *qf2 = reinterpret_cast<const uint2 *>(qf);
    uint2 *qsum = reinterpret_cast<uint2 *>(aq_smem + S::RING + S::QF);           // [NB][lane] {hi, lo} sums of the scaled query over blocks 2t and 2t + 1, times 2^-6: both in fp16's normal range
    __shared__ float q_factor[ROWS];
    float *given = reinterpret_cast<float *>(aq_smem + S::RING), *given_ref = given + AQ_WARPS * 3 * S::MINE * 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, col = PACK ? 2 * t & 3 : 2 * t;      // a thread has query rows col and col + 1 of each block
    // for each key of the warp's chunk: d times 2^b, and the middle m + 8 d of the values that a block can say, scaled too, as two pieces; [G4][keys] halves each
    __half *tab = reinterpret_cast<__half *>(aq_smem + S::RING + S::QF + S::QS) + warp * 3 * G4 * S::CHUNK;
    const int tab_at = (lane & 16) | (lane & 6) << 1 | (lane & 8) >> 2 | (lane & 1);      // keys 2t, 2t + 1, 2t + 8 and 2t + 9 of a tile side by side: one load for a thread
    const int N = gridDim.x, me = blockIdx.x;

    if (lane == 0) {
        for (int i = 0; i < STAGES; ++i) mbar_init(smem_u32(&full[warp][i]), 1);
        mbar_fence_init();
    }
    pdl_wait();                                                // lengths, table, rows and cache come from the kernels before this one: read through L2

    // ---- this CTA's part of the line.  On it lie the sequences, their blocks of rows, for each its stretches of the kv heads; each thread counts the units of
    // some consecutive blocks.
    const int blocks = p.c.batch * p.RC, each = (blocks + AQ_THREADS - 1) / AQ_THREADS, x0 = min(blocks, tid * each), x1 = min(blocks, x0 + each);
    auto at_block = [&](int x, AqWalk &w) {
        w.b = x / p.RC;
        w.rc = x - w.b * p.RC;
        w.len = aq_length(p, w.b);
        aq_range(p, ROWS, S::UNIT, w);
    };
    long long mine = 0;
    if (x0 < x1) {
        AqWalk w;
        at_block(x0, w);
        mine = w.n;
        for (int x = x0 + 1; x < x1; ++x) {
            aq_next_block(p, ROWS, S::UNIT, w);
            mine += w.n;
        }
        mine *= p.c.Hkv;
    }
    long long before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
    }
    if (lane == 31) s_sum[warp] = before;
    before -= mine;
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < AQ_WARPS; ++w) {
        if (w < warp) before += s_sum[w];
        total += s_sum[w];
    }
    const int parts = (int)min((long long)N, total);                              // every CTA below has at least one unit
    long long first = 0, last = 0;                                                // its units [first, last)
    if (me < parts) {
        if (total < 1 << 20) {                                                    // 64-bit divisions take as long as a trip to memory
            first = (uint32_t)total * (uint32_t)me / (uint32_t)parts;
            last = (uint32_t)total * (uint32_t)(me + 1) / (uint32_t)parts;
        } else {
            first = total * me / parts;
            last = total * (me + 1) / parts;
        }
    }
    if (first < last && mine && before <= first && first < before + mine) {
        long long rest = first - before;
        AqWalk w;
        for (at_block(x0, w); rest >= (long long)w.n * p.c.Hkv; aq_next_block(p, ROWS, S::UNIT, w)) rest -= (long long)w.n * p.c.Hkv;
        w.h = rest >> 31 ? (int)(rest / w.n) : (int)((uint32_t)rest / (uint32_t)w.n);
        w.u = (int)(rest - (long long)w.h * w.n);
        s_walk = w;
    }
    __syncthreads();
    bool ok = true;
    if (first < last) {
        AqWalk w = s_walk;                                     // the unit being computed
        // Lane 0 fetches, up to STAGES - 1 units ahead: the table's entry for a chunk's beginning is read one chunk ahead.  A chunk that cannot span pages is one copy
        // of K rows and one of V rows, another one as many as it has pieces of 16.  What stays the same in a stretch is worked out once for it.
        AqWalk f = w;
        int f_left = (int)(last - first), f_stage = 0, f_pos, f_slot = 0, entry = -1;
        const int *f_table;
        uint32_t f_head;
        const bool one_page = p.c.page_tokens % S::CHUNK == 0;
        const uint32_t page_bytes = (uint32_t)kv_row(1, 0, 0, p.c.Hkv, p.c.page_tokens, G4), ring = smem_u32(aq_smem) + warp * STAGES * S::STAGE, bars = smem_u32(&full[warp][0]);
        auto look = [&](int pos, int &slot) {                  // the page of a position, and its place in it
            if (pos >= f.end) return -1;
            const int column = p.by_page(pos);
            slot = pos - column * p.c.page_tokens;
            return kv_entry(__ldcg(f_table + column), p.c.pages);
        };
        auto enter = [&]() {                                   // a stretch
            f_table = p.c.table + (size_t)f.b * p.c.stride;
            f_head = (uint32_t)(f.h * p.c.page_tokens * ROW);
            f_pos = f.begin + f.u * S::UNIT + warp * S::CHUNK;
        };
        auto fetch = [&]() {                                   // the next unit into the next stage
            if (f_left == 0) return;
            if (lane == 0) {
                const uint32_t bar = bars + 8 * f_stage, to = ring + f_stage * S::STAGE;
                auto copy = [&](uint32_t at, int page, int slot, uint32_t bytes) {
                    const size_t src = (size_t)page * page_bytes + (f_head + (uint32_t)(slot * ROW));
                    bulk_g2s(at, p.k + src, bytes, bar);
                    bulk_g2s(at + S::CHUNK * ROW, p.v + src, bytes, bar);
                };
                if (one_page) {
                    const int n = entry < 0 ? 0 : min(S::XT, (f.end - f_pos + 15) >> 4);
                    pieces[warp][f_stage] = (1 << n) - 1;
                    mbar_arrive_expect_tx(bar, n * 2 * 16 * ROW);
                    if (n) copy(to, entry, f_slot, n * 16 * ROW);
                } else {
                    int e[S::XT], at[S::XT], there = 0;
#pragma unroll
                    for (int x = 0; x < S::XT; ++x) {
                        at[x] = f_slot;
                        e[x] = x ? look(f_pos + 16 * x, at[x]) : entry;
                        there |= (e[x] >= 0) << x;
                    }
                    pieces[warp][f_stage] = there;
                    mbar_arrive_expect_tx(bar, __popc(there) * 2 * 16 * ROW);
#pragma unroll
                    for (int x = 0; x < S::XT; ++x)
                        if (e[x] >= 0) copy(to + 16 * x * ROW, e[x], at[x], 16 * ROW);
                }
            }
            if (++f_stage == STAGES) f_stage = 0;
            f_pos += S::UNIT;
            if (--f_left == 0) return;
            if (++f.u >= f.n) {
                aq_next_stretch(p, ROWS, S::UNIT, f);
                enter();
            }
            if (lane == 0) entry = look(f_pos, f_slot);
        };
        enter();
        if (lane == 0) entry = look(f_pos, f_slot);
        for (int i = 0; i < STAGES - 1; ++i) fetch();

        float qx[ROWS / AQ_WARPS][G4];                         // rows of a stretch's queries
        auto load_q = [&]() {
#pragma unroll
            for (int i = 0; i < ROWS / AQ_WARPS; ++i) {
                const int row = w.rc * ROWS + warp + i * AQ_WARPS, tok = p.by_group(row);
                const float *src = p.q + ((long long)w.b * p.c.tokens + tok) * p.q_stride + (long long)(w.h * p.G + row - tok * p.G) * HD;
#pragma unroll
                for (int j = 0; j < G4; ++j) qx[i][j] = row < p.R ? __ldcg(src + 32 * j + lane) : 0.0f;
            }
        };
        if (S::EARLY) load_q();
        int stage = 0;
        uint32_t phase = 0;
        for (int left = (int)(last - first); left;) {
            // ---- a stretch: query fragments of its rows
            const int r0 = w.rc * ROWS, u_first = w.u;
            if (!S::EARLY) load_q();
            __syncthreads();                                   // the stretch before is done with them
#pragma unroll
            for (int i = 0; i < ROWS / AQ_WARPS; ++i) {      // a warp per row, a lane the channels 4 (lane % 4 ..) of its blocks
                const int r = warp + i * AQ_WARPS;
                const float (&x)[G4] = qx[i];
                float top = 0.0f;
#pragma unroll
                for (int j = 0; j < G4; ++j) top = fmaxf(top, fabsf(x[j]));
                const int ex_top = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23);      // biased exponent of the row's largest
                const int sh = max(-126, min(126, 141 - ex_top));                                           // largest into [2^14, 2^15)
                const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
                if (lane == 0) q_factor[r] = __uint_as_float((uint32_t)(127 - sh) << 23) * p.scale * (1.44269504088896340736f * AQ_UNSCALE);
                float sum0 = 0.0f, sum1 = 0.0f;                // lane t: of blocks 2t and 2t + 1
#pragma unroll
                for (int j = 0; j < G4; ++j) {
                    const float y = x[j] * up;
                    const float sum = group_sum<32>(y) * 0.015625f;
                    if (lane == j / 2) (j & 1 ? sum1 : sum0) = sum;
                    // channel c of the block: k-step c / 16, thread t = (c % 16) / 4, place c % 4: b0 holds places 0 and 2, b1 places 1 and 3
                    const __half hi = __float2half_rn(y), lo = __float2half_rn(y - __half2float(hi));
                    const int place = lane & 3, to = ((((r >> 3) * KS + 2 * j + (lane >> 4)) * 32 + 4 * (r & 7) + ((lane & 15) >> 2)) * 8) + (place & 1) * 2 + (place >> 1);
                    if constexpr (PACK) {
                        const int at = ((2 * j + (lane >> 4)) * 32 + 4 * r + ((lane & 15) >> 2)) * 4 + (place & 1) * 2 + (place >> 1);
                        reinterpret_cast<__half *>(qf)[at] = hi;
                        reinterpret_cast<__half *>(qf)[at + 64] = lo;          // four columns on
                    } else {
                        reinterpret_cast<__half *>(qf)[to] = hi;
                        reinterpret_cast<__half *>(qf)[to + 4] = lo;
                    }
                }
                if (lane < 4) {
                    uint2 v;
                    aq_split(make_float2(sum0, sum1), v.x, v.y);
                    qsum[(r >> 3) * 32 + 4 * (r & 7) + lane] = v;
                    if constexpr (PACK) qsum[16 + 4 * r + lane].x = v.y;
                }
            }
            __syncthreads();
            float om[NB][2];                                   // row g: block g's sum of weight times middle
            float o[NB][G4][2][4], m_run[NB][2], l_run[NB][2], fac[NB][2];      // m_run: the reference of the weights, in powers of two; l_run: of this thread's keys
            int pos_row[NB][2];                                 // pos_row: the position of a row, -1 where there is none
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = r0 + 8 * nb + col + e;
                    pos_row[nb][e] = row < p.R ? w.len - p.c.tokens + p.by_group(row) : -1;
                    fac[nb][e] = q_factor[8 * nb + col + e];
                    m_run[nb][e] = -INFINITY;
                    l_run[nb][e] = om[nb][e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < G4 * 8; ++e) o[nb][e >> 3][e >> 2 & 1][e & 3] = 0.0f;
            }
            // chunks in [all_from, all_to) are seen by every row
            const int pos_first = w.len - p.c.tokens + p.by_group(r0), pos_last = w.len - p.c.tokens + p.by_group(min(p.R, r0 + ROWS) - 1);
            const int all_to = pos_first + 1, all_from = p.window > 0 ? pos_last - p.window + 1 : 0;

            for (int key0 = w.begin + w.u * S::UNIT + warp * S::CHUNK;; key0 += S::UNIT) {
                fetch();
                if (ok && !mbar_wait_spin(bars + 8 * stage, phase)) {
                    ok = false;
                    if (lane == 0) atomicExch(p.err, DEV_ERR_FULL_WAIT);
                }
                const uint32_t there = pieces[warp][stage];
                if (there) {
                    const uint8_t *kb = aq_smem + (warp * STAGES + stage) * S::STAGE, *vb = kb + S::CHUNK * ROW;
                    const bool mixed = there != (1u << S::XT) - 1u || key0 < all_from || key0 + S::CHUNK > all_to;
                    // ---- the values' scales, a lane a key
                    static_assert(S::CHUNK == 32, "a lane a key");
                    uint32_t dm[G4];
#pragma unroll
                    for (int j = 0; j < G4; ++j) dm[j] = aq_u32(vb + lane * ROW + j * KQ4_BLOCK);
                    auto keep_seen = [&](bool mark) {          // in a chunk that not every row sees whole
                        // What no row sees must not reach the products even with weight zero (0 x NaN), what some rows see only those: scales that are no
                        // numbers are taken out, and the rows that see them marked.
                        const bool in = (there >> (lane >> 4) & 1u) && key0 + lane < w.end;
#pragma unroll
                        for (int j = 0; j < G4; ++j) {
                            const bool nan = in && aq_no_number(dm[j]);
                            if (!in || nan) dm[j] = 0;
                            if (!mark) continue;
                            for (uint32_t bad = __ballot_sync(0xffffffffu, nan); bad; bad &= bad - 1) {
                                const int at_key = key0 + __ffs(bad) - 1;
#pragma unroll
                                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                                    for (int e = 0; e < 2; ++e) {
                                        const int pos = pos_row[nb][e];
                                        if (at_key <= pos && (p.window == 0 || at_key > pos - p.window))
#pragma unroll
                                            for (int x = 0; x < 2; ++x) o[nb][j][x][e] = o[nb][j][x][e + 2] = __int_as_float(0x7fffffff);
                                    }
                            }
                        }
                    };
                    if (mixed) keep_seen(true);
                    // The chunk's size times `up` is in [16, 32): steps are below 4, so that their products with weights of up to 2^13 stay in fp16's range, middles times 2^10 below 2^15.
                    float least;
                    const int size = aq_size(dm, least);
                    const float up = aq_up(size);
                    const bool small = least * up < AQ_LEAST;      // there may be blocks that do not go with this scale
#pragma unroll
                    for (int j = 0; j < G4; ++j) {
                        const float d = aq_lo(dm[j]) * up, mid = fmaf(8192.0f, d, aq_hi(dm[j]) * (1024.0f * up));
                        const __half hi = __float2half_rn(mid);
                        tab[j * S::CHUNK + tab_at] = __float2half_rn(d);
                        tab[(G4 + j) * S::CHUNK + tab_at] = hi;
                        tab[(2 * G4 + j) * S::CHUNK + tab_at] = __float2half_rn(mid - __half2float(hi));
                    }
                    // ---- scores of tiles of 16 keys.  A product waits long for the one before it in its sum: those of several tiles and blocks take turns.
                    float s[S::XT][NB][4];                     // keys 16 x + g and 8 further on, rows col and col + 1
                    {
                        const uint8_t *key_row = kb + g * ROW;
#pragma unroll
                        for (int x = 0; x < S::XT; ++x) {
                            const uint8_t *at0 = key_row + 16 * x * ROW + min(2 * t, G4 - 1) * KQ4_BLOCK, *at1 = key_row + 16 * x * ROW + min(2 * t + 1, G4 - 1) * KQ4_BLOCK;
                            const uint32_t m0 = __byte_perm(aq_u32(at0), aq_u32(at1), 0x7632), m1 = __byte_perm(aq_u32(at0 + 8 * ROW), aq_u32(at1 + 8 * ROW), 0x7632);
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                const uint2 b = qsum[nb * 32 + lane];
                                s[x][nb][0] = s[x][nb][1] = s[x][nb][2] = s[x][nb][3] = 0.0f;
                                if (!PACK) aq_mma_k8(s[x][nb], m0, m1, b.y);
                                aq_mma_k8(s[x][nb], m0, m1, b.x);
#pragma unroll
                                for (int e = 0; e < 4; ++e) s[x][nb][e] *= 64.0f / AQ_UNSCALE;
                            }
                        }
#pragma unroll
                        for (int j = 0; j < G4; ++j) {
                            uint32_t c[S::XT][2];
                            float d[S::XT][2];
#pragma unroll
                            for (int x = 0; x < S::XT; ++x)
#pragma unroll
                                for (int y = 0; y < 2; ++y) {
                                    const uint8_t *at = key_row + (16 * x + 8 * y) * ROW + j * KQ4_BLOCK;
                                    c[x][y] = aq_u32(at + 4 + 4 * t);
                                    d[x][y] = aq_lo(aq_u32(at));
                                }
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                uint4 q0, q1;
                                if constexpr (PACK) {
                                    const uint2 u = qf2[2 * j * 32 + lane], w2 = qf2[(2 * j + 1) * 32 + lane];
                                    q0 = make_uint4(0, 0, u.x, u.y);
                                    q1 = make_uint4(0, 0, w2.x, w2.y);
                                } else {
                                    q0 = qf[(nb * KS + 2 * j) * 32 + lane];
                                    q1 = qf[(nb * KS + 2 * j + 1) * 32 + lane];
                                }
                                float acc[S::XT][4];
#pragma unroll
                                for (int half = 0; half < 2; ++half)           // of the block
#pragma unroll
                                    for (int x = 0; x < S::XT; ++x) {
                                        const uint4 &q = half ? q1 : q0;
                                        const uint32_t a[4] = {half ? aq_codes<1>(c[x][0]) : aq_codes<0>(c[x][0]), half ? aq_codes<1>(c[x][1]) : aq_codes<0>(c[x][1]),
                                                               half ? aq_codes<3>(c[x][0]) : aq_codes<2>(c[x][0]), half ? aq_codes<3>(c[x][1]) : aq_codes<2>(c[x][1])};
                                        if (half == 0) aq_mma_first(acc[x], a, q.z, q.w);
                                        else aq_mma(acc[x], a, q.z, q.w);
                                        if (!PACK) aq_mma(acc[x], a, q.x, q.y);
                                    }
#pragma unroll
                                for (int x = 0; x < S::XT; ++x)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) s[x][nb][e] = fmaf(d[x][e >> 1], acc[x][e], s[x][nb][e]);
                            }
                        }
                    }
                    // ---- weights times 2^10, as two pieces.  The reference follows the maximum when that is more than 2^3 ahead: each time costs every accumulator a product,
                    // and only then the maximum over the keys is found.
                    bool moved = false;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        if constexpr (PACK) {                  // what hi and lo pieces gave, columns c and c + 4
#pragma unroll
                            for (int x = 0; x < S::XT; ++x)
#pragma unroll
                                for (int e = 0; e < 4; ++e) s[x][nb][e] += __shfl_xor_sync(0xffffffffu, s[x][nb][e], 2);
                        }
                        if (mixed) {
#pragma unroll
                            for (int x = 0; x < S::XT; ++x)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int key = key0 + 16 * x + 8 * (e >> 1) + g, pos = pos_row[nb][e & 1];
                                    if (!(there >> x & 1u) || key > pos || (p.window > 0 && key <= pos - p.window)) s[x][nb][e] = -INFINITY;
                                }
                        }
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float top = -INFINITY;
#pragma unroll
                            for (int x = 0; x < S::XT; ++x) top = fmaxf(top, fmaxf(s[x][nb][e], s[x][nb][e + 2]));
                            moved |= top * fac[nb][e] > m_run[nb][e] + 3.0f;
                        }
                    }
                    if (__any_sync(0xffffffffu, moved)) {      // rare once the first keys have been seen
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            float alpha[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float top = -INFINITY;
#pragma unroll
                                for (int x = 0; x < S::XT; ++x) top = fmaxf(top, fmaxf(s[x][nb][e], s[x][nb][e + 2]));
#pragma unroll
                                for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                                top *= fac[nb][e];
                                const float m_new = top > m_run[nb][e] + 3.0f ? top : m_run[nb][e];
                                alpha[e] = m_run[nb][e] == -INFINITY ? 0.0f : aq_exp2(m_run[nb][e] - m_new);
                                m_run[nb][e] = m_new;
                                l_run[nb][e] *= alpha[e];
                                om[nb][e] *= alpha[e];
                            }
#pragma unroll
                            for (int e = 0; e < G4 * 8; ++e) o[nb][e >> 3][e >> 2 & 1][e & 3] *= alpha[e & 1];
                        }
                    }
                    uint32_t ph[NB][2 * S::XT], pl[NB][2 * S::XT];             // of row g: keys 8y + 2t and 8y + 2t + 1
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const float c0 = 10.0f - (m_run[nb][0] == -INFINITY ? 0.0f : m_run[nb][0]), c1 = 10.0f - (m_run[nb][1] == -INFINITY ? 0.0f : m_run[nb][1]);
                        float sum0 = 0.0f, sum1 = 0.0f;        // of the chunk: a long sequence's sum rounds once a chunk
#pragma unroll
                        for (int y = 0; y < 2 * S::XT; ++y) {
                            const float2 e = make_float2(aq_exp2(fmaf(s[y >> 1][nb][2 * (y & 1)], fac[nb][0], c0)), aq_exp2(fmaf(s[y >> 1][nb][2 * (y & 1) + 1], fac[nb][1], c1)));
                            sum0 += e.x;
                            sum1 += e.y;
                            aq_split(e, ph[nb][y], pl[nb][y]);
                            ph[nb][y] = aq_transpose(ph[nb][y]);
                            pl[nb][y] = aq_transpose(pl[nb][y]);
                        }
                        l_run[nb][0] += sum0;
                        l_run[nb][1] += sum1;
                    }
                    __syncwarp();                              // the table below is complete
                    // ---- values.  The tensor cores cut what they add to an accumulator instead of rounding it: a chunk's sums start from zero and are
                    // added up by the rounding adder, and codes are taken from their middle, so that the terms do not all have one sign.
                    const uint8_t *at_t = reinterpret_cast<const uint8_t *>(tab) + 8 * t;
                    if (__any_sync(0xffffffffu, small)) {
                        // Blocks that would lose bits beside the chunk's largest leave the table; their values are weighed in fp32, key by key.
#pragma unroll
                        for (int j = 0; j < G4; ++j) dm[j] = aq_u32(vb + lane * ROW + j * KQ4_BLOCK);
                        if (mixed) keep_seen(false);
                        uint32_t mine = 0;
#pragma unroll
                        for (int j = 0; j < G4; ++j) {
                            if (!aq_late(dm[j], aq_up(size))) continue;
                            mine |= 1u << j;
#pragma unroll
                            for (int i = 0; i < 3; ++i) tab[(i * G4 + j) * S::CHUNK + tab_at] = __float2half_rn(0.0f);
                        }
#pragma unroll 1
                        for (uint32_t keys = __ballot_sync(0xffffffffu, mine != 0); keys; keys &= keys - 1) {
                            const int key = __ffs(keys) - 1;
                            const uint32_t of_key = __shfl_sync(0xffffffffu, mine, key);
                            float weight[NB][2];               // of rows col and col + 1
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                uint32_t hi = 0, lo = 0;
#pragma unroll
                                for (int y = 0; y < 2 * S::XT; ++y) {      // by masks: an array that is indexed would lie in memory
                                    const uint32_t is = key >> 3 == y ? 0xffffffffu : 0u;
                                    hi |= ph[nb][y] & is;
                                    lo |= pl[nb][y] & is;
                                }
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const int from = 4 * (col + e) + (key >> 1 & 3);
                                    const uint32_t h = __shfl_sync(0xffffffffu, hi, from), l = __shfl_sync(0xffffffffu, lo, from);
                                    weight[nb][e] = PACK && t >= 2 ? 0.0f : (key & 1 ? aq_hi(h) + aq_hi(l) : aq_lo(h) + aq_lo(l));
                                }
                            }
#pragma unroll
                            for (int j = 0; j < G4; ++j) {
                                if (!(of_key >> j & 1u)) continue;
                                const uint8_t *at = vb + key * ROW + j * KQ4_BLOCK;
                                const uint32_t scales = aq_u32(at), codes = aq_u16(at + 4 + 2 * g);
#pragma unroll
                                for (int e = 0; e < 4; ++e) {  // byte e / 2, nibble e % 2
                                    const float v = fmaf(aq_lo(scales), (float)(codes >> 4 * e & 15u), aq_hi(scales));
#pragma unroll
                                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                                        for (int r = 0; r < 2; ++r) o[nb][j][e >> 1][2 * (e & 1) + r] = fmaf(weight[nb][r], v, o[nb][j][e >> 1][2 * (e & 1) + r]);
                                }
                            }
                        }
                        __syncwarp();
                    }
                    const float down = aq_down(size);
                    {
                        float acc[NB][4];
#pragma unroll
                        for (int x = 0; x < S::XT; ++x) {
                            const uint8_t *at_m = at_t + 32 * x + (G4 + min(g, G4 - 1)) * 2 * S::CHUNK;
                            const uint2 mh = *reinterpret_cast<const uint2 *>(at_m), ml = *reinterpret_cast<const uint2 *>(at_m + G4 * 2 * S::CHUNK);
                            const uint32_t hi[4] = {mh.x, 0, mh.y, 0}, lo[4] = {ml.x, 0, ml.y, 0};
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                const uint32_t b0 = PACK && g >= 4 ? pl[nb][2 * x] : ph[nb][2 * x], b1 = PACK && g >= 4 ? pl[nb][2 * x + 1] : ph[nb][2 * x + 1];
                                if (x == 0) aq_mma_first(acc[nb], lo, b0, b1);
                                else aq_mma(acc[nb], lo, b0, b1);
                                if (!PACK) aq_mma(acc[nb], hi, pl[nb][2 * x], pl[nb][2 * x + 1]);
                                aq_mma(acc[nb], hi, b0, b1);
                            }
                        }
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            om[nb][0] = fmaf(acc[nb][0], down, om[nb][0]);
                            om[nb][1] = fmaf(acc[nb][1], down, om[nb][1]);
                        }
                    }
                    const uint8_t *key_row = vb + 2 * t * ROW + 4 + 2 * g;
#pragma unroll
                    for (int j = 0; j < G4; ++j) {
                        float acc[NB][2][4];
#pragma unroll
                        for (int x = 0; x < S::XT; ++x) {
                            uint32_t w[2];
                            const uint2 d = *reinterpret_cast<const uint2 *>(at_t + j * 2 * S::CHUNK + 32 * x);
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const uint8_t *at = key_row + (16 * x + 8 * y) * ROW + j * KQ4_BLOCK;
                                w[y] = __byte_perm(aq_u16(at), aq_u16(at + ROW), 0x5410);
                            }
                            const uint32_t a0[4] = {aq_centred<0>(w[0]), aq_centred<1>(w[0]), aq_centred<0>(w[1]), aq_centred<1>(w[1])};
                            const uint32_t a1[4] = {aq_centred<2>(w[0]), aq_centred<3>(w[0]), aq_centred<2>(w[1]), aq_centred<3>(w[1])};
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                uint32_t h0, l0, h1, l1;
                                aq_weigh(ph[nb][2 * x], pl[nb][2 * x], d.x, h0, l0);
                                aq_weigh(ph[nb][2 * x + 1], pl[nb][2 * x + 1], d.y, h1, l1);
                                if constexpr (PACK) {
                                    const uint32_t b0 = g >= 4 ? l0 : h0, b1 = g >= 4 ? l1 : h1;
                                    if (x == 0) {
                                        aq_mma_first(acc[nb][0], a0, b0, b1);
                                        aq_mma_first(acc[nb][1], a1, b0, b1);
                                    } else {
                                        aq_mma(acc[nb][0], a0, b0, b1);
                                        aq_mma(acc[nb][1], a1, b0, b1);
                                    }
                                    continue;
                                }
                                if (x == 0) {
                                    aq_mma_first(acc[nb][0], a0, l0, l1);
                                    aq_mma_first(acc[nb][1], a1, l0, l1);
                                } else {
                                    aq_mma(acc[nb][0], a0, l0, l1);
                                    aq_mma(acc[nb][1], a1, l0, l1);
                                }
                                aq_mma(acc[nb][0], a0, h0, h1);
                                aq_mma(acc[nb][1], a1, h0, h1);
                            }
                        }
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                            for (int e = 0; e < 8; ++e) o[nb][j][e >> 2][e & 3] = fmaf(acc[nb][e >> 2][e & 3], down, o[nb][j][e >> 2][e & 3]);
                    }
                }
                __syncwarp();                                  // the stage and its word and the table are free again
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                --left;
                if (++w.u >= w.n || left == 0) break;
            }

            // ---- the stretch ends here: the four warps' results, relative to 2^ref, become one
            const bool whole = u_first == 0 && w.u >= w.n;
            if (u_first == 0 && tid == 0)                      // its last unit is n - u units behind the end of this CTA's part
                p.desc[((size_t)w.b * p.c.Hkv + w.h) * p.RC + w.rc] = make_int2(me, whole ? -1 : (int)(((last + w.n - w.u) * parts - 1) / total));
            float *part = whole ? nullptr : p.part + (size_t)(2 * me + (u_first == 0)) * ROWS * (HD + 2), *out = p.out + (long long)w.b * p.c.tokens * p.out_stride + (long long)w.h * p.G * HD;
            if (left) {
                aq_next_stretch(p, ROWS, S::UNIT, w);
                if (S::EARLY) load_q();
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    l_run[nb][0] += __shfl_xor_sync(0xffffffffu, l_run[nb][0], d);
                    l_run[nb][1] += __shfl_xor_sync(0xffffffffu, l_run[nb][1], d);
                }
#pragma unroll
                for (int j = 0; j < G4; ++j) {
                    const float a0 = __shfl_sync(0xffffffffu, om[nb][0], 4 * j + t), a1 = __shfl_sync(0xffffffffu, om[nb][1], 4 * j + t);
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[nb][j][e >> 2][e & 3] += (e & 1 ? a1 : a0) * 0x1p-10f;
                    if constexpr (PACK) {                      // what hi and lo pieces gave, column c and c + 4
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[nb][j][e >> 2][e & 3] += __shfl_xor_sync(0xffffffffu, o[nb][j][e >> 2][e & 3], 2);
                    }
                }
            }
            // quarter d of a block's registers goes to warp d: pairs d G4 .. of (channel block, x, y)
            auto given_by = [&](int from, int to) { return given + (from * 3 + ((to - from - 1) & 3)) * S::MINE * 32 + lane; };
            __syncthreads();                                   // the queries are no longer needed
#pragma unroll
            for (int d = 0; d < AQ_WARPS; ++d) {
                if (d == warp) continue;
                float *to = given_by(warp, d);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < G4 * 2; ++e) {
                        const int at = d * G4 * 2 + e;
                        to[(nb * G4 * 2 + e) * 32] = o[nb][at >> 3][at >> 2 & 1][at & 3];
                    }
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
                if (g == 0) *reinterpret_cast<float4 *>(given_ref + (warp * NB + nb) * 16 + 4 * t) = make_float4(m_run[nb][0], l_run[nb][0], m_run[nb][1], l_run[nb][1]);
            __syncthreads();
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float4 ref[AQ_WARPS];                          // reference and sum of the two rows
                float both[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, f[AQ_WARPS][2], sum[G4 * 2];
#pragma unroll
                for (int s = 0; s < AQ_WARPS; ++s) {
                    ref[s] = *reinterpret_cast<const float4 *>(given_ref + (s * NB + nb) * 16 + 4 * t);
                    both[0] = fmaxf(both[0], ref[s].x);
                    both[1] = fmaxf(both[1], ref[s].z);
                }
#pragma unroll
                for (int s = 0; s < AQ_WARPS; ++s) {
                    f[s][0] = ref[s].x == -INFINITY ? 0.0f : aq_exp2(ref[s].x - both[0]);
                    f[s][1] = ref[s].z == -INFINITY ? 0.0f : aq_exp2(ref[s].z - both[1]);
                    l[0] = fmaf(f[s][0], ref[s].y, l[0]);
                    l[1] = fmaf(f[s][1], ref[s].w, l[1]);
                }
#pragma unroll
                for (int e = 0; e < G4 * 2; ++e) sum[e] = 0.0f;
#pragma unroll
                for (int s = 0; s < AQ_WARPS; ++s) {           // in the same order whichever warp joins
                    const float *from = given_by(s, warp) + nb * G4 * 2 * 32;
#pragma unroll
                    for (int e = 0; e < G4 * 2; ++e) {
                        float x;
                        if (s == warp) x = o[nb][(s * G4 * 2 + e) >> 3][(s * G4 * 2 + e) >> 2 & 1][(s * G4 * 2 + e) & 3];
                        else x = from[e * 32];
                        sum[e] = fmaf(f[s][e & 1], x, sum[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = 8 * nb + 2 * t + e, row = r0 + r, tok = p.by_group(row);
                    const float inv = l[e] == 0.0f ? 0.0f : 1.0f / l[e];
                    if (part && warp == 0 && g == 0 && r < ROWS) {
                        part[r * (HD + 2) + HD] = both[e];
                        part[r * (HD + 2) + HD + 1] = l[e];
                    }
                    if (r >= ROWS || row >= p.R) continue;
                    float *to = part ? part + r * (HD + 2) : out + tok * p.out_stride + (long long)(row - tok * p.G) * HD;
#pragma unroll
                    for (int k = 0; k < G4; ++k) {
                        const int at = warp * G4 + k;
                        to[32 * (at >> 2) + 2 * g + (at >> 1 & 1) + 16 * (at & 1)] = part ? sum[2 * k + e] : sum[2 * k + e] * inv;
                    }
                }
            }
        }
        // a wait ran out: the copies still on their way, of the last STAGES units, end before the CTA does
        if (!ok)
            for (int i = 0; i < STAGES; ++i) {
                if (i < (int)(last - first)) {
                    const int at = stage ? stage - 1 : STAGES - 1;
                    mbar_wait_spin(bars + 8 * at, stage ? phase : phase ^ 1u);
                }
                if (stage-- == 0) { stage = STAGES - 1; phase ^= 1u; }
            }
    }
    pdl_trigger();                                             // not earlier: what comes behind would only wait in this kernel's place
    // blocks of query rows that see no key
    for (int x = me; x < p.c.batch * p.RC; x += N) {
        AqWalk w;
        at_block(x, w);
        if (w.n) continue;
        for (int h = tid; h < p.c.Hkv; h += AQ_THREADS) p.desc[((size_t)w.b * p.c.Hkv + h) * p.RC + w.rc] = make_int2(me, -1);
        const int r0 = w.rc * ROWS, rows = min(p.R, r0 + ROWS) - r0;
        for (int y = tid; y < rows * p.c.Hkv * HD; y += AQ_THREADS) {
            const int c = y % HD, hr = y / HD, h = hr / rows, row = r0 + hr - h * rows, tok = row / p.G;
            p.out[((long long)w.b * p.c.tokens + tok) * p.out_stride + (long long)(h * p.G + row - tok * p.G) * HD + c] = 0.0f;
        }
    }
}

// The results of a stretch that several CTAs worked on become one, row by row.  Two forms: few stretches are in many parts each, many in two or three.
struct AqParts {
    const float *first, *base;                 // the first CTA's is its second one
    size_t step;
    int count;
    float *out;
};
template <int HD>
__device__ __forceinline__ bool aq_parts(const AqParams &p, int nrows, int x, int r, AqParts &a)
{
    const int2 d = __ldcg(p.desc + x);
    const int bh = x / p.RC, row = (x - bh * p.RC) * nrows + r;
    if (d.y < 0 || row >= p.R) return false;
    a.count = d.y - d.x + 1;
    a.step = (size_t)2 * nrows * (HD + 2);
    a.base = p.part + (size_t)(2 * d.x) * nrows * (HD + 2) + r * (HD + 2);
    a.first = a.base + a.step / 2;
    const int b = bh / p.c.Hkv, h = bh - b * p.c.Hkv, tok = p.by_group(row);
    a.out = p.out + ((long long)b * p.c.tokens + tok) * p.out_stride + (long long)(h * p.G + row - tok * p.G) * HD;
    return true;
}

// A warp for a row, four parts at a time.
template <int HD>
__global__ void __launch_bounds__(128) attn_q4_merge_rows_kernel(const AqParams p, int nrows, int rows)
{
    constexpr int PARTS = 4;
    pdl_wait();
    const int lane = threadIdx.x & 31, all = p.c.batch * p.c.Hkv * p.RC;
    const int warp = (int)(threadIdx.x >> 5), x = blockIdx.x, r0 = blockIdx.y * 4 + warp;
    for (int s = x; s < all; s += gridDim.x) {
        AqParts a;
        if (r0 >= rows || !aq_parts<HD>(p, nrows, s, r0, a)) continue;
        float top = -INFINITY, l = 0.0f, acc[HD / 32] = {};
        for (int i0 = 0; i0 < a.count; i0 += PARTS) {
            float ref[PARTS], part_l[PARTS], v[PARTS][HD / 32], now = top;
#pragma unroll
            for (int u = 0; u < PARTS; ++u) {
                const float *from = i0 + u ? a.base + (i0 + u) * a.step : a.first;
                const bool is = i0 + u < a.count;
                ref[u] = is ? __ldcg(from + HD) : -INFINITY;
                part_l[u] = is ? __ldcg(from + HD + 1) : 0.0f;
#pragma unroll
                for (int k = 0; k < HD / 32; ++k) v[u][k] = is ? __ldcg(from + 32 * k + lane) : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < PARTS; ++u) now = fmaxf(now, ref[u]);
            const float keep = top == -INFINITY ? 0.0f : aq_exp2(top - now);
            top = now;
            l *= keep;
#pragma unroll
            for (int k = 0; k < HD / 32; ++k) acc[k] *= keep;
#pragma unroll
            for (int u = 0; u < PARTS; ++u) {
                const float f = ref[u] == -INFINITY ? 0.0f : aq_exp2(ref[u] - top);
                l = fmaf(f, part_l[u], l);                      // 0 x NaN: scores that are no numbers have no maximum, and must be seen
#pragma unroll
                for (int k = 0; k < HD / 32; ++k) acc[k] = fmaf(f, v[u][k], acc[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < HD / 32; ++k) a.out[32 * k + lane] = l == 0.0f ? 0.0f : acc[k] / l;
    }
}

// A CTA for a row: a warp has the weights of 32 parts in its lanes and a channel for each lane, whose parts it adds up LOADS at a time; groups of HD threads take
// every GROUPS-th 32 parts.
template <int HD>
__global__ void __launch_bounds__(512 / HD * HD) attn_q4_merge_kernel(const AqParams p, int nrows)
{
    constexpr int GROUPS = 512 / HD, LOADS = 16;
    __shared__ float acc_s[GROUPS][HD], top_s[GROUPS], l_s[GROUPS];
    pdl_wait();
    const int r = blockIdx.y, lane = threadIdx.x & 31, grp = threadIdx.x / HD, c = threadIdx.x - grp * HD;
    for (int x = blockIdx.x; x < p.c.batch * p.c.Hkv * p.RC; x += gridDim.x) {
        AqParts a;
        if (!aq_parts<HD>(p, nrows, x, r, a)) continue;
        float top = -INFINITY, l = 0.0f, acc = 0.0f;
        for (int i0 = 32 * grp; i0 < a.count; i0 += 32 * GROUPS) {
            const int n = min(32, a.count - i0);
            const float *mine = i0 + lane == 0 ? a.first : a.base + (i0 + min(lane, n - 1)) * a.step;
            const float ref = lane < n ? __ldcg(mine + HD) : -INFINITY, part_l = __ldcg(mine + HD + 1);
            float v[LOADS], now = ref;
            auto load = [&](int k0) {
#pragma unroll
                for (int u = 0; u < LOADS; ++u) v[u] = k0 + u < n ? __ldcg((i0 + k0 + u ? a.base + (i0 + k0 + u) * a.step : a.first) + c) : 0.0f;
            };
            load(0);                                            // on their way while the weights are found
#pragma unroll
            for (int o = 16; o; o >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, o));
            now = fmaxf(now, top);
            const float keep = top == -INFINITY ? 0.0f : aq_exp2(top - now), f = ref == -INFINITY ? 0.0f : aq_exp2(ref - now);
            top = now;
            float sum = lane < n ? f * part_l : 0.0f;           // 0 x NaN, as above
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l = l * keep + sum;
            acc *= keep;
            for (int k0 = 0;;) {
#pragma unroll
                for (int u = 0; u < LOADS; ++u) acc = fmaf(__shfl_sync(0xffffffffu, f, k0 + u), v[u], acc);
                if ((k0 += LOADS) >= n) break;
                load(k0);
            }
        }
        if (a.count > 32 && GROUPS > 1) {
            acc_s[grp][c] = acc;
            if (c == 0) { top_s[grp] = top; l_s[grp] = l; }
            __syncthreads();
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) top = fmaxf(top, top_s[g]);
            acc = l = 0.0f;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const float f = top_s[g] == -INFINITY ? 0.0f : aq_exp2(top_s[g] - top);
                l += l_s[g] * f;
                acc += acc_s[g][c] * f;
            }
            __syncthreads();
        }
        if (grp == 0) a.out[c] = l == 0.0f ? 0.0f : acc / l;
    }
}

template <int HD, int BLOCKS>
static size_t aq_desc_bytes(int batch, int Hkv, int R) { return ((size_t)batch * Hkv * ((R + AqShape<HD, BLOCKS>::ROWS - 1) / AqShape<HD, BLOCKS>::ROWS) * sizeof(int2) + 15) & ~(size_t)15; }

template <int HD, int BLOCKS>
static int aq_launch(AqParams p, void *ws, cudaStream_t st)
{
    using S = AqShape<HD, BLOCKS>;
    static_assert(S::SMEM <= 227 * 1024, "shared memory");
    p.RC = (p.R + S::ROWS - 1) / S::ROWS;
    // as many CTAs as can be resident, no more than units that the table has room for
    const long long stretches = (long long)p.c.batch * p.c.Hkv * p.RC, units = stretches * ((p.c.stride * p.c.page_tokens + S::UNIT - 1) / S::UNIT);
    const int most = ckb_sm_count() * S::CTAS, N = units < most ? (int)units : most;
    p.desc = (int2 *)ws;
    p.part = (float *)((uint8_t *)ws + aq_desc_bytes<HD, BLOCKS>(p.c.batch, p.c.Hkv, p.R));
    static bool attr_set = false;
    if (!attr_set) {
        if (ckb_check_cuda((int)cudaFuncSetAttribute(attn_q4_kernel<HD, BLOCKS>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM), "attention_q4cache")) return CKB_ERR_CUDA;
        attr_set = true;
    }
    const int rc = launch_pdl("attention_q4cache", attn_q4_kernel<HD, BLOCKS>, dim3(N), dim3(AQ_THREADS), (size_t)S::SMEM, st, p);
    if (rc || p.c.stride * p.c.page_tokens <= S::UNIT) return rc;      // no stretch has two units
    // 128 channels, the whole call by CTAs and by warps: 8 stretches of 32 parts 10.0 and 12.1 us, 16 of 27 13.0 and 14.8, 24 of 18 16.0 and 15.5, 32 of 14 16.8 and 16.0,
    // 40 with 16 rows of 7 21.6 and 17.6
    const int rows = S::ROWS < p.R ? S::ROWS : p.R;
    if (stretches * 22 < N) return launch_pdl("attention_q4cache", attn_q4_merge_kernel<HD>, dim3((unsigned)stretches, rows), dim3(512 / HD * HD), 0, st, p, S::ROWS);
    return launch_pdl("attention_q4cache", attn_q4_merge_rows_kernel<HD>, dim3((unsigned)(stretches < N ? stretches : N), (rows + 3) / 4), dim3(128), 0, st, p, S::ROWS, rows);
}

template <int HD, int BLOCKS>
static size_t aq_bytes(int batch, int Hkv, int R)
{
    using S = AqShape<HD, BLOCKS>;
    return aq_desc_bytes<HD, BLOCKS>(batch, Hkv, R) + (size_t)ckb_sm_count() * S::CTAS * 2 * sizeof(float) * S::ROWS * (HD + 2);
}

// Blocks of 8 query rows that share the codes a CTA unpacks; 0: up to four, with both pieces of a row in one product (32 heads over 8, four sequences of 131072
// tokens 186 us, 213 us in a block of 8; 32 of up to 4096 47 and 52).  Three blocks leave no register free and are worth it only where they hold all the rows: 20 rows of
// 16 sequences (five drafts, up to 8190 tokens) 96 us with three, 108 us one by one, 128 us with two and two; 516 rows 39 us in blocks of two, 42 us one by one, 41 us in threes.
// Above 128 channels two blocks leave one CTA an SM (256) or spill (192): 16 rows of 8 sequences of 4096 tokens 24 us one by one and 30 us in twos (192: 19 and 21), 516 rows behind 1024 42 and 58 (32 and 38).
static int aq_blocks(long long rows, int hd) { return rows <= 4 ? 0 : rows <= 8 || hd > 128 ? 1 : (rows > 16 && rows <= 24 ? 3 : 2); }

// Eight rows of 128 channels: four CTAs an SM, with 128 registers a thread, hide more of the waiting than three with 168, but take longer for a chunk.  They are taken where the table has
// room for eight units a CTA and sixteen a stretch.  Of lengths the host sees the table's columns alone.  With tables that just fit (four and three CTAs, inside a graph, 64 heads over 8): four
// sequences of 131072 tokens 207 and 215 us, 128 of up to 3000 113 and 117, 32 of up to 4096 52 and 53, 48 of up to 2047 37 and 38; the rule leaves 16 of up to 4096 (26.4 and 26.2), 8 (21.7 and 19.0),
// 4 (17.6 and 16.6) and 256 of up to 600 (74 and 73) to three.  With tables that have room for 131072 tokens it takes four for these too: 26.5 and 26.2 us, 22.1 and 18.8, 17.7 and 16.6, 74 and 73; one of 20000 20.6
// and 18.4, two of up to 8000 13.8 and 15.3.
static bool aq_four(long long stretches, int units, int hd) { return hd == 128 && units >= 16 && stretches * units >= 8LL * 4 * ckb_sm_count(); }

}  // namespace ckb

using namespace ckb;

#define AQ_EACH(hd, nb, F)                                                                                              \
    (hd == 64 ? (nb == 0 ? F<64, 0> : nb == 1 ? F<64, 1> : nb == 2 ? F<64, 2> : F<64, 3>)                               \
     : hd == 96 ? (nb == 0 ? F<96, 0> : nb == 1 ? F<96, 1> : nb == 2 ? F<96, 2> : F<96, 3>)                             \
     : hd == 128 ? (nb == 0 ? F<128, 0> : nb == 1 ? F<128, 1> : nb == 2 ? F<128, 2> : nb == 3 ? F<128, 3> : F<128, 4>)                        \
     : hd == 192 ? (nb == 0 ? F<192, 0> : F<192, 1>)                                                                    \
                 : (nb == 0 ? F<256, 0> : F<256, 1>))

extern "C" size_t ckb200_attention_q4cache_workspace_bytes(int batch, int num_tokens, int num_heads, int num_kv_heads, int head_dim)
{
    if (batch <= 0 || num_tokens <= 0 || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads || (long long)batch * num_tokens * num_heads > 1 << 30 || !ckb200_kv_q4_page_bytes(1, 16, head_dim)) return 0;
    int nb = aq_blocks((long long)num_tokens * (num_heads / num_kv_heads), head_dim);
    if (nb == 1 && head_dim == 128) nb = 4;                    // whichever the call takes: four CTAs an SM need more
    return AQ_EACH(head_dim, nb, aq_bytes)(batch, num_kv_heads, num_tokens * (num_heads / num_kv_heads));
}

extern "C" int ckb200_dev_attention_q4cache(const float *q, long long q_stride, const void *k_pages, const void *v_pages, float *out, long long out_stride, const int *page_table,
                                            int table_stride, const int *kv_lens, int batch, int num_tokens, int num_pages, int page_tokens, int num_heads, int num_kv_heads,
                                            int head_dim, int sliding_window, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *what = "attention_q4cache";
    int rc = ckb_check_kv_q4(what, k_pages, v_pages, page_table, table_stride, kv_lens, batch, num_tokens, num_pages, page_tokens, num_kv_heads, head_dim);
    if (rc) return rc;
    if (!q || !out) return ckb_fail(CKB_ERR_STATE, "%s: a pointer is NULL", what);
    if (num_heads <= 0 || num_heads % num_kv_heads) return ckb_fail(CKB_ERR_SHAPE, "%s: %d heads over %d kv heads", what, num_heads, num_kv_heads);
    if (sliding_window < 0) return ckb_fail(CKB_ERR_SHAPE, "%s: window of %d tokens", what, sliding_window);
    const long long rows = (long long)batch * num_tokens;
    if (rows > 1 && (q_stride < (long long)num_heads * head_dim || out_stride < (long long)num_heads * head_dim))
        return ckb_fail(CKB_ERR_SHAPE, "%s: rows of %lld values lie %lld and %lld apart", what, (long long)num_heads * head_dim, q_stride, out_stride);
    if (((uintptr_t)q | (uintptr_t)out) & 3) return ckb_fail(CKB_ERR_ALIGN, "%s: rows must be aligned to 4 bytes", what);
    if (rows * num_heads > 1 << 30 || num_heads > 1 << 20) return ckb_fail(CKB_ERR_LIMIT, "%s: %lld query rows in one call", what, rows * num_heads);
    if (!rows) return 0;
    if (!workspace || workspace_bytes < ckb200_attention_q4cache_workspace_bytes(batch, num_tokens, num_heads, num_kv_heads, head_dim))
        return ckb_fail(CKB_ERR_STATE, "%s: the workspace is too small", what);
    if ((uintptr_t)workspace & 15) return ckb_fail(CKB_ERR_ALIGN, "%s: the workspace must be aligned to 16 bytes", what);
    if (ckb_ensure_init()) return CKB_ERR_NO_DEVICE;
    if ((rc = ckb_check_device(what))) return rc;
    AqParams p = {};
    p.q = q;
    p.k = (const uint8_t *)k_pages;
    p.v = (const uint8_t *)v_pages;
    p.out = out;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.c = {page_table, kv_lens, table_stride, batch, num_tokens, num_pages, page_tokens, num_kv_heads, head_dim / 32};
    p.G = num_heads / num_kv_heads;
    p.R = num_tokens * p.G;
    p.window = sliding_window < 1 << 30 ? sliding_window : 0;      // no sequence is longer
    p.scale = 1.0f / sqrtf((float)head_dim);
    p.err = ckb_device_error_word();
    p.by_page = kv_divide((uint32_t)page_tokens);
    p.by_group = kv_divide((uint32_t)p.G);
    int nb = aq_blocks(p.R, head_dim);
    if (nb == 1 && aq_four((long long)batch * num_kv_heads, (table_stride * page_tokens + 127) / 128, head_dim)) nb = 4;
    return AQ_EACH(head_dim, nb, aq_launch)(p, workspace, ckb_stream(stream));
}
