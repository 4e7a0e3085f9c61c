// Rows of a paged 4-bit KV cache: quantised into it, and read back.
//
// A block of 32 values is the work of eight lanes, four values (16 bytes) each, for K and for V: the lanes find the block's least and
// largest value by shuffles; a lane's four codes make four bytes' nibbles, and since byte j holds values j and j + 16, lane l and lane l + 4
// share them: one more shuffle, and lanes 0..3 write the 16 code bytes, lane 4 the (d, m) pair.  A warp's writes are consecutive.
// Bound by HBM, 4.625 bytes a value either way: reading 4 bytes when storing, writing them when loading.
#include <cuda_fp16.h>
#include <float.h>
#include <math.h>

#include "../../include/ckb200_cache.h"
#include "device_common.cuh"
#include "kv_q4.cuh"
#include "launch.h"
#include "runtime.h"

namespace ckb {

constexpr int KR_THREADS = 256;

// lanes 0..7 of a group hold values 4l .. 4l + 3 of a block; the word that lane l < 4 (codes 4l ..) or lane 4 (d, m) writes
__device__ __forceinline__ uint32_t kr_quantise(const float4 &x, int l)
{
    float lo = fminf(fminf(x.x, x.y), fminf(x.z, x.w)), hi = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
    // minimum and maximum pass over NaN: it is looked for by itself
    int bad = !(fabsf(x.x) <= FLT_MAX && fabsf(x.y) <= FLT_MAX && fabsf(x.z) <= FLT_MAX && fabsf(x.w) <= FLT_MAX);
#pragma unroll
    for (int o = 4; o; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        bad |= __shfl_xor_sync(0xffffffffu, bad, o);
    }
    // the two roundings to fp16 that the format asks for; codes are then taken against the rounded pair, so that each is the nearest that the block can say
    const __half mh = __float2half_rn(lo), dh = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f));
    const float m = __half2float(mh), d = __half2float(dh);
    bad |= !(fabsf(m) <= 65504.0f && d <= 65504.0f);
    const float inv = d > 0.0f ? __frcp_rn(d) : 0.0f;
    const float v[4] = {x.x, x.y, x.z, x.w};
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float t = floorf(__fadd_rn(__fmul_rn(__fsub_rn(v[i], m), inv), 0.5f));
        codes |= (uint32_t)fminf(fmaxf(t, 0.0f), 15.0f) << (8 * i);
    }
    if (bad) codes = 0;
    const uint32_t other = __shfl_xor_sync(0xffffffffu, codes, 4);
    const uint32_t dm = bad ? 0x7fff7fffu : ((uint32_t)__half_as_ushort(mh) << 16 | __half_as_ushort(dh));
    return l < 4 ? codes | other << 4 : dm;
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

// group (8 lanes) -> (row, block of the row); where the row lies in the pools, -1: nowhere
__device__ __forceinline__ bool kr_where(const KvQ4 &c, long long rows, long long &row, int &block, long long &at)
{
    const long long grp = ((long long)blockIdx.x * KR_THREADS + threadIdx.x) >> 3;
    const int items = c.Hkv * c.nb;
    row = grp / items;
    block = (int)(grp - row * items);
    at = -1;
    if (row >= rows) return false;
    const int b = (int)(row / c.tokens), t = (int)(row - (long long)b * c.tokens);
    const int pos = kv_len(__ldg(c.lens + b), c.stride, c.page_tokens) - c.tokens + t;
    const int page = kv_page(c.table + (size_t)b * c.stride, c.stride, c.pages, c.page_tokens, pos);
    const int head = block / c.nb;
    if (page >= 0) at = (long long)kv_row(page, head, pos % c.page_tokens, c.Hkv, c.page_tokens, c.nb) + (block - head * c.nb) * KQ4_BLOCK;
    return true;
}

template <bool VEC>
__global__ void __launch_bounds__(KR_THREADS) kv_store_q4_kernel(uint8_t *__restrict__ kp, uint8_t *__restrict__ vp, const float *__restrict__ k, const float *__restrict__ v,
                                                                 long long ks, long long vs, KvQ4 c, long long rows)
{
    long long row, at;
    int block;
    const int l = threadIdx.x & 7;
    const bool in = kr_where(c, rows, row, block, at);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (in) {
        a = kr_load4<VEC>(k + row * ks + block * 32 + 4 * l);
        b = kr_load4<VEC>(v + row * vs + block * 32 + 4 * l);
    }
    const uint32_t wk = kr_quantise(a, l), wv = kr_quantise(b, l);
    if (at < 0 || l > 4) return;
    const size_t to = (size_t)at + (l < 4 ? 4 + 4 * l : 0);
    *reinterpret_cast<uint32_t *>(kp + to) = wk;
    *reinterpret_cast<uint32_t *>(vp + to) = wv;
}

__device__ __forceinline__ float4 kr_values(const uint8_t *p, int l)
{
    const uint32_t dm = __ldg(reinterpret_cast<const uint32_t *>(p)), w = __ldg(reinterpret_cast<const uint32_t *>(p + 4 + 4 * (l & 3))) >> (l < 4 ? 0 : 4);
    const float d = half_bits_to_float(dm & 0xffffu), m = half_bits_to_float(dm >> 16);
    return make_float4(__fadd_rn(__fmul_rn(d, (float)(w & 15u)), m), __fadd_rn(__fmul_rn(d, (float)(w >> 8 & 15u)), m), __fadd_rn(__fmul_rn(d, (float)(w >> 16 & 15u)), m),
                       __fadd_rn(__fmul_rn(d, (float)(w >> 24 & 15u)), m));
}

template <bool VEC>
__global__ void __launch_bounds__(KR_THREADS) kv_load_q4_kernel(float *__restrict__ k, float *__restrict__ v, long long ks, long long vs, const uint8_t *__restrict__ kp,
                                                                const uint8_t *__restrict__ vp, KvQ4 c, long long rows)
{
    long long row, at;
    int block;
    const int l = threadIdx.x & 7;
    if (!kr_where(c, rows, row, block, at)) return;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (at >= 0) {
        a = kr_values(kp + at, l);
        b = kr_values(vp + at, l);
    }
    kr_store4<VEC>(k + row * ks + block * 32 + 4 * l, a);
    kr_store4<VEC>(v + row * vs + block * 32 + 4 * l, b);
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

static int rows_grid(const char *what, const KvQ4 &c, long long rows, unsigned *grid)
{
    const long long n = (rows * c.Hkv * c.nb * 8 + KR_THREADS - 1) / KR_THREADS;
    if (n > 0x7fffffffLL) return ckb_fail(CKB_ERR_LIMIT, "%s: %lld rows in one call", what, rows);
    *grid = (unsigned)n;
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
    unsigned grid;
    if ((rc = rows_grid(what, c, rows, &grid))) return rc;
    if (!rows) return 0;
    if (ckb_ensure_init()) return CKB_ERR_NO_DEVICE;
    if ((rc = ckb_check_device(what))) return rc;
    if (rows_vectors(k, v, k_stride, v_stride))
        kv_store_q4_kernel<true><<<grid, KR_THREADS, 0, ckb_stream(stream)>>>((uint8_t *)k_pages, (uint8_t *)v_pages, k, v, k_stride, v_stride, c, rows);
    else
        kv_store_q4_kernel<false><<<grid, KR_THREADS, 0, ckb_stream(stream)>>>((uint8_t *)k_pages, (uint8_t *)v_pages, k, v, k_stride, v_stride, c, rows);
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
    unsigned grid;
    if ((rc = rows_grid(what, c, rows, &grid))) return rc;
    if (!rows) return 0;
    if (ckb_ensure_init()) return CKB_ERR_NO_DEVICE;
    if ((rc = ckb_check_device(what))) return rc;
    if (rows_vectors(k, v, k_stride, v_stride))
        kv_load_q4_kernel<true><<<grid, KR_THREADS, 0, ckb_stream(stream)>>>(k, v, k_stride, v_stride, (const uint8_t *)k_pages, (const uint8_t *)v_pages, c, rows);
    else
        kv_load_q4_kernel<false><<<grid, KR_THREADS, 0, ckb_stream(stream)>>>(k, v, k_stride, v_stride, (const uint8_t *)k_pages, (const uint8_t *)v_pages, c, rows);
    return ckb_check_launch(what);
}
