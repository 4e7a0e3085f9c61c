// Rows of a paged 4-bit KV cache: quantised into it, and read back.
//
// A block of 32 values is the work of four lanes, for K and for V: lane l has values 4l .. 4l + 3 and 16 + 4l .. 16 + 4l + 3, which are the nibbles of code bytes
// 4l .. 4l + 3, so that only the block's least and largest value cross lanes (two shuffles each).  A warp's loads and stores are of whole 32-byte sectors.
// Bound by HBM, 4.625 bytes a value either way: reading 4 bytes when storing, writing them when loading.  8192 rows of K and V of 1024 values: 14.4 us loaded
// (5.4 TB/s), 16.4 us stored (4.7 TB/s, 1.4 of its floor: the quantiser's comparisons and shifts keep their pipe busy for more than half the time, so that they and the loads do not hide one another
// wholly).  A turn (rotate and store, 64 heads over 8 of 128): 5.8 us for 32 sequences inside a graph, 5.0 us for one, against 0.4 us of bytes: a launch, and the length, the table's entry and the
// rows one after the other.
#include <cuda_fp16.h>
#include <float.h>
#include <math.h>

#include "../../include/ckb200_cache.h"
#include "device_common.cuh"
#include "kv_q4.cuh"
#include "launch.h"
#include "pdl.cuh"
#include "runtime.h"

namespace ckb {

constexpr int KR_THREADS = 256;

__device__ __forceinline__ float kr_min3(float a, float b, float c)
{
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float kr_max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// the word of codes of lane l of the four, and the block's (d, m)
__device__ __forceinline__ uint32_t kr_quantise(const float4 &x, const float4 &y, uint32_t &dm)
{
    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    float lo = fminf(v[0], v[1]), hi = fmaxf(v[0], v[1]), zero = 0.0f;
#pragma unroll
    for (int i = 2; i < 8; i += 2) {
        lo = kr_min3(lo, v[i], v[i + 1]);
        hi = kr_max3(hi, v[i], v[i + 1]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) zero = __fmaf_rn(v[i], 0.0f, zero);      // minimum and maximum pass over NaN: it is looked for by itself, with infinities
    if (zero != 0.0f) hi = INFINITY;                           // no code can say the block: d becomes infinite, below
#pragma unroll
    for (int o = 2; o; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    // the two roundings to fp16 that the format asks for; codes are then taken against the rounded pair, so that each is the nearest that the block can say
    const __half mh = __float2half_rn(lo), dh = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f));
    const float m = __half2float(mh), d = __half2float(dh), inv = d > 0.0f ? __frcp_rn(d) : 0.0f;
    // The floor of a number of [0, 16) is in the last bits of its sixteenth's sum with 2^19, rounded down; what the sums' other bits add up to is taken off at the end.
    // (Comparisons and shifts are what bounds the store: here a value costs two of them, and floor, clamp, convert and shift six.)
    uint32_t codes = 0, others = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = __saturatef(fminf(__fadd_rn(__fmul_rn(__fsub_rn(v[i], m), inv), 0.5f), 15.5f) * 0.0625f);
        const int at = 8 * (i & 3) + 4 * (i >> 2);
        codes += __float_as_uint(__fadd_rd(t, 524288.0f)) << at;
        others += 0x49000000u << at;
    }
    codes -= others;
    const bool good = fabsf(m) <= 65504.0f && d <= 65504.0f;
    dm = good ? (uint32_t)__half_as_ushort(mh) << 16 | __half_as_ushort(dh) : 0x7fff7fffu;
    return good ? codes : 0;
}

template <bool VEC>
__device__ __forceinline__ float4 kr_load4(const float *p)
{
    if constexpr (VEC) return __ldcs(reinterpret_cast<const float4 *>(p));
    return make_float4(__ldcs(p), __ldcs(p + 1), __ldcs(p + 2), __ldcs(p + 3));
}
template <bool VEC>
__device__ __forceinline__ void kr_store4(float *p, const float4 &v)
{
    if constexpr (VEC) {
        __stcs(reinterpret_cast<float4 *>(p), v);
    } else {
        __stcs(p, v.x);
        __stcs(p + 1, v.y);
        __stcs(p + 2, v.z);
        __stcs(p + 3, v.w);
    }
}

struct KrRows {
    KvQ4 c;
    long long k_stride, v_stride;
    uint32_t groups;                           // blocks of 32 values of all rows
    KvDivide by_items, by_tokens, by_nb, by_page;
};

// where block `grp` of all rows lies: its row's number, its place in the row, and its place in the pools in bytes (-1: nowhere)
// FRESH: the lengths come from a kernel that may still have been running when this one was launched
template <bool FRESH>
__device__ __forceinline__ void kr_where(const KrRows &p, uint32_t grp, int &row, int &block, long long &at)
{
    row = p.by_items(grp);
    block = (int)(grp - (uint32_t)row * p.by_items.d);
    const int b = p.by_tokens(row), t = row - b * p.c.tokens, head = p.by_nb(block);
    const int pos = kv_len(FRESH ? __ldcg(p.c.lens + b) : __ldg(p.c.lens + b), p.c.stride, p.c.page_tokens) - p.c.tokens + t;
    at = -1;
    if (pos < 0) return;
    const int column = p.by_page(pos), page = kv_entry(FRESH ? __ldcg(p.c.table + (size_t)b * p.c.stride + column) : __ldg(p.c.table + (size_t)b * p.c.stride + column), p.c.pages);      // pos is below the length: the column exists
    if (page >= 0) at = (long long)kv_row(page, head, pos - column * p.c.page_tokens, p.c.Hkv, p.c.page_tokens, p.c.nb) + (block - head * p.c.nb) * KQ4_BLOCK;
}

template <bool VEC>
__global__ void __launch_bounds__(KR_THREADS) kv_store_q4_kernel(uint8_t *__restrict__ kp, uint8_t *__restrict__ vp, const float *__restrict__ k, const float *__restrict__ v, KrRows p)
{
    const int l = threadIdx.x & 3;
    const uint32_t grp = blockIdx.x * (KR_THREADS / 4) + (threadIdx.x >> 2);
    float4 a[2], b[2];
    a[0] = a[1] = b[0] = b[1] = make_float4(0.f, 0.f, 0.f, 0.f);
    long long at = -1;
    if (grp < p.groups) {
        int row = p.by_items(grp), block = (int)(grp - (uint32_t)row * p.by_items.d);
        const float *x = k + row * p.k_stride + block * 32 + 4 * l, *y = v + row * p.v_stride + block * 32 + 4 * l;
        a[0] = kr_load4<VEC>(x);                               // on their way while the length and the table's entry are looked up
        a[1] = kr_load4<VEC>(x + 16);
        b[0] = kr_load4<VEC>(y);
        b[1] = kr_load4<VEC>(y + 16);
        kr_where<false>(p, grp, row, block, at);
    }
    uint32_t dmk, dmv;
    const uint32_t wk = kr_quantise(a[0], a[1], dmk), wv = kr_quantise(b[0], b[1], dmv);
    if (at < 0) return;
    uint32_t *x = reinterpret_cast<uint32_t *>(kp + at), *y = reinterpret_cast<uint32_t *>(vp + at);
    x[1 + l] = wk;
    y[1 + l] = wv;
    if (l == 0) x[0] = dmk;
    if (l == 1) y[0] = dmv;
}

// the code of byte `byte`, low nibble, as a number: in the last bits of 2^23, which is taken off again
__device__ __forceinline__ float kr_code(uint32_t w, int byte) { return __fsub_rn(__uint_as_float((w >> 8 * byte & 15u) | 0x4b000000u), 8388608.0f); }
__device__ __forceinline__ float4 kr_values(uint32_t dm, uint32_t w)       // of the low nibbles of w; d times a code is exact
{
    const float d = half_bits_to_float(dm & 0xffffu), m = half_bits_to_float(dm >> 16);
    return make_float4(__fmaf_rn(d, kr_code(w, 0), m), __fmaf_rn(d, kr_code(w, 1), m), __fmaf_rn(d, kr_code(w, 2), m), __fmaf_rn(d, kr_code(w, 3), m));
}

template <bool VEC>
__global__ void __launch_bounds__(KR_THREADS) kv_load_q4_kernel(float *__restrict__ k, float *__restrict__ v, const uint8_t *__restrict__ kp, const uint8_t *__restrict__ vp, KrRows p)
{
    const int l = threadIdx.x & 3;
    const uint32_t grp = blockIdx.x * (KR_THREADS / 4) + (threadIdx.x >> 2);
    if (grp >= p.groups) return;
    long long at;
    int row, block;
    kr_where<false>(p, grp, row, block, at);
    uint32_t dmk = 0, dmv = 0, wk = 0, wv = 0;
    if (at >= 0) {
        const uint32_t *x = reinterpret_cast<const uint32_t *>(kp + at), *y = reinterpret_cast<const uint32_t *>(vp + at);
        dmk = __ldg(x);
        wk = __ldg(x + 1 + l);
        dmv = __ldg(y);
        wv = __ldg(y + 1 + l);
    }
    float *x = k + row * p.k_stride + block * 32 + 4 * l, *y = v + row * p.v_stride + block * 32 + 4 * l;
    kr_store4<VEC>(x, kr_values(dmk, wk));
    kr_store4<VEC>(x + 16, kr_values(dmk, wk >> 4));
    kr_store4<VEC>(y, kr_values(dmv, wv));
    kr_store4<VEC>(y + 16, kr_values(dmv, wv >> 4));
}

// One new token of each sequence: q rotated in place, k rotated and quantised, v quantised.  Four lanes a block as above; those of q come after those of the cache.
// Channels i and i + head_dim / 2 turn together, and a lane's four channels lie on one side of the middle: their partners are one load more.
__global__ void __launch_bounds__(KR_THREADS) rope_kv_store_q4_kernel(float *__restrict__ q, uint8_t *__restrict__ kp, uint8_t *__restrict__ vp, const float *__restrict__ k,
                                                                      const float *__restrict__ v, const float *__restrict__ cos_cache, const float *__restrict__ sin_cache,
                                                                      int positions, int H, int pairs, KrRows p)
{
    pdl_trigger();
    pdl_wait();
    const int l = threadIdx.x & 3, hd = 32 * p.c.nb, half = hd / 2;
    const uint32_t grp = blockIdx.x * (KR_THREADS / 4) + (threadIdx.x >> 2);
    const uint32_t stored = (p.groups + 7) & ~7u;              // whole warps: the shuffles below
    if (grp >= stored) {
        // eight channels of the first half of a row of q, and their partners
        const uint32_t i = (grp - stored) * 4 + l, per_row = half / 8;
        if (i >= (uint32_t)pairs) return;
        const int row = (int)(i / per_row), c0 = (int)(i - row * per_row) * 8, b = row / H;
        const int pos = kv_len(__ldcg(p.c.lens + b), p.c.stride, p.c.page_tokens) - 1;
        if (pos < 0 || pos >= positions) return;
        float *x = q + (size_t)row * hd + c0;
        const float *cs = cos_cache + (size_t)pos * half + c0, *sn = sin_cache + (size_t)pos * half + c0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = __ldcg(x + e), z = __ldcg(x + e + half), c = cs[e], s = sn[e];
            x[e] = __fsub_rn(__fmul_rn(a, c), __fmul_rn(z, s));
            x[e + half] = __fadd_rn(__fmul_rn(a, s), __fmul_rn(z, c));
        }
        return;
    }
    float a[8] = {}, b[8] = {};
    long long at = -1;
    if (grp < p.groups) {
        int row, block;
        kr_where<true>(p, grp, row, block, at);
        const int pos = kv_len(__ldcg(p.c.lens + row), p.c.stride, p.c.page_tokens) - 1, head = p.by_nb(block), first = 32 * (block - head * p.c.nb) + 4 * l;
        if (pos >= positions) at = -1;
        if (at >= 0) {
            const float *x = k + ((size_t)row * p.c.Hkv + head) * hd, *y = v + ((size_t)row * p.c.Hkv + head) * hd + first;
            const float *cs = cos_cache + (size_t)pos * half, *sn = sin_cache + (size_t)pos * half;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = first + (e & 3) + 16 * (e >> 2), turn = i < half ? i : i - half;
                const float u = __ldcg(x + turn), w = __ldcg(x + turn + half), c = cs[turn], s = sn[turn];
                a[e] = i < half ? __fsub_rn(__fmul_rn(u, c), __fmul_rn(w, s)) : __fadd_rn(__fmul_rn(u, s), __fmul_rn(w, c));
                b[e] = __ldcg(y + (e & 3) + 16 * (e >> 2));
            }
        }
    }
    uint32_t dmk, dmv;
    const uint32_t wk = kr_quantise(make_float4(a[0], a[1], a[2], a[3]), make_float4(a[4], a[5], a[6], a[7]), dmk);
    const uint32_t wv = kr_quantise(make_float4(b[0], b[1], b[2], b[3]), make_float4(b[4], b[5], b[6], b[7]), dmv);
    if (at < 0) return;
    uint32_t *x = reinterpret_cast<uint32_t *>(kp + at), *y = reinterpret_cast<uint32_t *>(vp + at);
    x[1 + l] = wk;
    y[1 + l] = wv;
    if (l == 0) x[0] = dmk;
    if (l == 1) y[0] = dmv;
}

// lengths of `batch` sequences that are all at *pos: its token counted
__global__ void kv_lens_from_pos_kernel(int *lens, const int *pos, int batch)
{
    for (int b = threadIdx.x; b < batch; b += blockDim.x) lens[b] = *pos + 1;
}

}  // namespace ckb

using namespace ckb;

static bool kq4_head_dim(int hd) { return hd == 64 || hd == 96 || hd == 128 || hd == 192 || hd == 256; }

extern "C" size_t ckb200_kv_q4_page_bytes(int num_kv_heads, int page_tokens, int head_dim)
{
    if (num_kv_heads <= 0 || page_tokens <= 0 || page_tokens % 16 || !kq4_head_dim(head_dim)) return 0;
    return (size_t)num_kv_heads * page_tokens * (head_dim / 32) * KQ4_BLOCK;
}

extern "C" long long ckb200_kv_q4_row_offset(const int *table_row, int table_stride, int num_pages, int page_tokens, int num_kv_heads, int head_dim, int head, int pos)
{
    if (!table_row || table_stride <= 0 || !ckb200_kv_q4_page_bytes(num_kv_heads, page_tokens, head_dim) || head < 0 || head >= num_kv_heads) return -1;
    const int page = kv_page(table_row, table_stride, num_pages, page_tokens, pos);
    return page < 0 ? -1 : (long long)kv_row(page, head, pos % page_tokens, num_kv_heads, page_tokens, head_dim / 32);
}

extern "C" int ckb_check_kv_q4(const char *what, const void *k_pages, const void *v_pages, const int *page_table, int table_stride, const int *kv_lens, int batch,
                               int num_tokens, int num_pages, int page_tokens, int num_kv_heads, int head_dim)
{
    if (!k_pages || !v_pages || !page_table || !kv_lens) return ckb_fail(CKB_ERR_STATE, "%s: a pointer is NULL", what);
    if (batch < 0 || num_tokens < 0 || num_pages <= 0 || table_stride <= 0) return ckb_fail(CKB_ERR_SHAPE, "%s: batch %d, tokens %d, pages %d, table columns %d", what, batch, num_tokens, num_pages, table_stride);
    if (!ckb200_kv_q4_page_bytes(num_kv_heads, page_tokens, head_dim))
        return ckb_fail(CKB_ERR_SHAPE, "%s: %d kv heads, pages of %d tokens, head size %d (64, 96, 128, 192 or 256; pages of a multiple of 16 tokens)", what, num_kv_heads, page_tokens, head_dim);
    if (num_kv_heads > 1024) return ckb_fail(CKB_ERR_LIMIT, "%s: %d kv heads, at most 1024", what, num_kv_heads);
    if (ckb200_kv_q4_page_bytes(num_kv_heads, page_tokens, head_dim) > 0x7fffffffu) return ckb_fail(CKB_ERR_LIMIT, "%s: a page of 2 GB or more", what);
    if ((long long)table_stride * page_tokens > 1 << 30 || num_tokens > 1 << 30) return ckb_fail(CKB_ERR_LIMIT, "%s: a sequence may have up to 2^30 tokens", what);
    if ((long long)batch * num_tokens > 0x7fffffffLL) return ckb_fail(CKB_ERR_LIMIT, "%s: %lld rows in one call", what, (long long)batch * num_tokens);
    if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) return ckb_fail(CKB_ERR_ALIGN, "%s: pools must be aligned to 16 bytes", what);
    if (((uintptr_t)page_table | (uintptr_t)kv_lens) & 3) return ckb_fail(CKB_ERR_ALIGN, "%s: table and lengths must be aligned to 4 bytes", what);
    return 0;
}

static int check_rows(const char *what, const float *k, const float *v, long long ks, long long vs, int rows_of, int n)
{
    if (!k || !v) return ckb_fail(CKB_ERR_STATE, "%s: a pointer is NULL", what);
    if (((uintptr_t)k | (uintptr_t)v) & 3) return ckb_fail(CKB_ERR_ALIGN, "%s: rows must be aligned to 4 bytes", what);
    if (rows_of > 1 && (ks < n || vs < n)) return ckb_fail(CKB_ERR_SHAPE, "%s: rows of %d values lie %lld and %lld apart", what, n, ks, vs);
    return 0;
}

static bool rows_vectors(const float *k, const float *v, long long ks, long long vs) { return !(((uintptr_t)k | (uintptr_t)v) & 15) && !((ks | vs) & 3); }

// 0 and the launch's parameters, or an error
static int rows_params(const char *what, const KvQ4 &c, long long rows, long long ks, long long vs, KrRows *p, unsigned *grid)
{
    const long long groups = rows * c.Hkv * c.nb;
    if (groups > 0x7fffffffLL) return ckb_fail(CKB_ERR_LIMIT, "%s: %lld rows in one call", what, rows);
    *p = {c, ks, vs, (uint32_t)groups, kv_divide((uint32_t)(c.Hkv * c.nb)), kv_divide((uint32_t)(c.tokens > 0 ? c.tokens : 1)), kv_divide((uint32_t)c.nb), kv_divide((uint32_t)c.page_tokens)};
    *grid = (unsigned)((groups + KR_THREADS / 4 - 1) / (KR_THREADS / 4));
    return 0;
}

extern "C" int ckb200_dev_kv_cache_store_q4(void *k_pages, void *v_pages, const float *k, const float *v, long long k_stride, long long v_stride, const int *page_table,
                                            int table_stride, const int *kv_lens, int batch, int num_tokens, int num_pages, int page_tokens, int num_kv_heads, int head_dim,
                                            void *stream)
{
    const char *what = "kv_cache_store_q4";
    int rc = ckb_check_kv_q4(what, k_pages, v_pages, page_table, table_stride, kv_lens, batch, num_tokens, num_pages, page_tokens, num_kv_heads, head_dim);
    const long long rows = (long long)batch * num_tokens;
    if (rc || (rc = check_rows(what, k, v, k_stride, v_stride, rows > 1 ? 2 : 1, num_kv_heads * head_dim))) return rc;
    const KvQ4 c = {page_table, kv_lens, table_stride, batch, num_tokens, num_pages, page_tokens, num_kv_heads, head_dim / 32};
    KrRows p;
    unsigned grid;
    if ((rc = rows_params(what, c, rows, k_stride, v_stride, &p, &grid))) return rc;
    if (!rows) return 0;
    if (ckb_ensure_init()) return CKB_ERR_NO_DEVICE;
    if ((rc = ckb_check_device(what))) return rc;
    if (rows_vectors(k, v, k_stride, v_stride))
        kv_store_q4_kernel<true><<<grid, KR_THREADS, 0, ckb_stream(stream)>>>((uint8_t *)k_pages, (uint8_t *)v_pages, k, v, p);
    else
        kv_store_q4_kernel<false><<<grid, KR_THREADS, 0, ckb_stream(stream)>>>((uint8_t *)k_pages, (uint8_t *)v_pages, k, v, p);
    return ckb_check_launch(what);
}

extern "C" int ckb200_dev_kv_cache_load_q4(float *k, float *v, long long k_stride, long long v_stride, const void *k_pages, const void *v_pages, const int *page_table,
                                           int table_stride, const int *kv_lens, int batch, int num_tokens, int num_pages, int page_tokens, int num_kv_heads, int head_dim,
                                           void *stream)
{
    const char *what = "kv_cache_load_q4";
    int rc = ckb_check_kv_q4(what, k_pages, v_pages, page_table, table_stride, kv_lens, batch, num_tokens, num_pages, page_tokens, num_kv_heads, head_dim);
    const long long rows = (long long)batch * num_tokens;
    if (rc || (rc = check_rows(what, k, v, k_stride, v_stride, rows > 1 ? 2 : 1, num_kv_heads * head_dim))) return rc;
    const KvQ4 c = {page_table, kv_lens, table_stride, batch, num_tokens, num_pages, page_tokens, num_kv_heads, head_dim / 32};
    KrRows p;
    unsigned grid;
    if ((rc = rows_params(what, c, rows, k_stride, v_stride, &p, &grid))) return rc;
    if (!rows) return 0;
    if (ckb_ensure_init()) return CKB_ERR_NO_DEVICE;
    if ((rc = ckb_check_device(what))) return rc;
    if (rows_vectors(k, v, k_stride, v_stride))
        kv_load_q4_kernel<true><<<grid, KR_THREADS, 0, ckb_stream(stream)>>>(k, v, (const uint8_t *)k_pages, (const uint8_t *)v_pages, p);
    else
        kv_load_q4_kernel<false><<<grid, KR_THREADS, 0, ckb_stream(stream)>>>(k, v, (const uint8_t *)k_pages, (const uint8_t *)v_pages, p);
    return ckb_check_launch(what);
}

extern "C" int ckb200_dev_rope_kv_store_q4(float *q, const float *k, const float *v, void *k_pages, void *v_pages, const float *cos_cache, const float *sin_cache, int rope_positions,
                                           const int *page_table, int table_stride, const int *kv_lens, int batch, int num_pages, int page_tokens, int num_heads, int num_kv_heads,
                                           int head_dim, void *stream)
{
    const char *what = "rope_kv_store_q4";
    int rc = ckb_check_kv_q4(what, k_pages, v_pages, page_table, table_stride, kv_lens, batch, 1, num_pages, page_tokens, num_kv_heads, head_dim);
    if (rc || (rc = check_rows(what, k, v, 0, 0, 1, num_kv_heads * head_dim))) return rc;
    if (!q || !cos_cache || !sin_cache) return ckb_fail(CKB_ERR_STATE, "%s: a pointer is NULL", what);
    if (num_heads <= 0 || rope_positions <= 0) return ckb_fail(CKB_ERR_SHAPE, "%s: %d heads, tables of %d positions", what, num_heads, rope_positions);
    if (((uintptr_t)q | (uintptr_t)cos_cache | (uintptr_t)sin_cache) & 3) return ckb_fail(CKB_ERR_ALIGN, "%s: rows must be aligned to 4 bytes", what);
    const long long pairs = (long long)batch * num_heads * (head_dim / 16);
    if (pairs > 0x3fffffffLL) return ckb_fail(CKB_ERR_LIMIT, "%s: %d sequences of %d heads", what, batch, num_heads);
    const KvQ4 c = {page_table, kv_lens, table_stride, batch, 1, num_pages, page_tokens, num_kv_heads, head_dim / 32};
    KrRows p;
    unsigned grid;
    if ((rc = rows_params(what, c, batch, 0, 0, &p, &grid))) return rc;
    if (!batch) return 0;
    if (ckb_ensure_init()) return CKB_ERR_NO_DEVICE;
    if ((rc = ckb_check_device(what))) return rc;
    grid = (unsigned)((((long long)p.groups + 7) / 8 * 8 + (pairs + 3) / 4 + KR_THREADS / 4 - 1) / (KR_THREADS / 4));
    return launch_pdl(what, rope_kv_store_q4_kernel, dim3(grid), dim3(KR_THREADS), 0, ckb_stream(stream), q, (uint8_t *)k_pages, (uint8_t *)v_pages, k, v, cos_cache, sin_cache,
                      rope_positions, num_heads, (int)pairs, p);
}

// kv_lens of sequences that are all at *pos_dev, for a step that begins (model_kquant.c)
extern "C" int ckb_kv_lens_from_pos(int *kv_lens, const int *pos_dev, int batch, void *stream)
{
    kv_lens_from_pos_kernel<<<1, 256, 0, ckb_stream(stream)>>>(kv_lens, pos_dev, batch);
    return ckb_check_launch("kv_lens_from_pos");
}
