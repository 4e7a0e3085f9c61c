// Causal attention over a paged 4-bit KV cache (include/ckb200_cache.h).
//
// One CTA per (query token, head): its warps take every fourth visible key, a lane the codes of head_dim / 32 values, with a running
// maximum and sum each; the four are merged at the end.
#include <cuda_fp16.h>
#include <math.h>

#include "../../include/ckb200_cache.h"
#include "device_common.cuh"
#include "kv_q4.cuh"
#include "launch.h"
#include "runtime.h"

namespace ckb {

constexpr int AQ_WARPS = 4, AQ_THREADS = 32 * AQ_WARPS;

template <int NB>
__global__ void __launch_bounds__(AQ_THREADS) attn_q4_kernel(const float *__restrict__ q, long long q_stride, const uint8_t *__restrict__ kp, const uint8_t *__restrict__ vp,
                                                             float *__restrict__ out, long long out_stride, KvQ4 c, int H, int window, float scale)
{
    __shared__ float acc_s[AQ_WARPS][32 * NB], m_s[AQ_WARPS], l_s[AQ_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = blockIdx.x % H;
    const long long row = blockIdx.x / H;
    const int b = (int)(row / c.tokens), t = (int)(row - (long long)b * c.tokens), kvh = h / (H / c.Hkv);
    const int pos = kv_len(c.lens[b], c.stride, c.page_tokens) - c.tokens + t, first = window > 0 ? max(0, pos - window + 1) : 0;
    float qv[NB], acc[NB], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        qv[i] = q[row * q_stride + (long long)h * 32 * NB + 32 * i + lane] * scale;
        acc[i] = 0.0f;
    }
    const int byte = 4 + (lane & 15), shift = lane < 16 ? 0 : 4;
    for (int key = first + warp; key <= pos; key += AQ_WARPS) {
        const int page = kv_page(c.table + (size_t)b * c.stride, c.stride, c.pages, c.page_tokens, key);
        if (page < 0) continue;
        const size_t at = kv_row(page, kvh, key % c.page_tokens, c.Hkv, c.page_tokens, NB);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const uint8_t *p = kp + at + i * KQ4_BLOCK;
            const uint32_t dm = *reinterpret_cast<const uint32_t *>(p);
            s = fmaf(qv[i], fmaf(half_bits_to_float(dm & 0xffffu), (float)(p[byte] >> shift & 15), half_bits_to_float(dm >> 16)), s);
        }
        s = group_sum<32>(s);
        const float m_new = fmaxf(m, s), m_ref = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = m == -INFINITY ? 0.0f : expf(m - m_ref), p = expf(s - m_ref);
        m = m_new;
        l = l * alpha + p;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const uint8_t *pv = vp + at + i * KQ4_BLOCK;
            const uint32_t dm = *reinterpret_cast<const uint32_t *>(pv);
            acc[i] = fmaf(p, fmaf(half_bits_to_float(dm & 0xffffu), (float)(pv[byte] >> shift & 15), half_bits_to_float(dm >> 16)), acc[i] * alpha);
        }
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) acc_s[warp][32 * i + lane] = acc[i];
    if (lane == 0) { m_s[warp] = m; l_s[warp] = l; }
    __syncthreads();
    float mm = -INFINITY;
    for (int w = 0; w < AQ_WARPS; ++w) mm = fmaxf(mm, m_s[w]);
    const float m_ref = mm == -INFINITY ? 0.0f : mm;
    for (int x = threadIdx.x; x < 32 * NB; x += AQ_THREADS) {
        float a = 0.0f, ll = 0.0f;
        for (int w = 0; w < AQ_WARPS; ++w) {
            const float f = m_s[w] == -INFINITY ? (l_s[w] == 0.0f ? 0.0f : 1.0f) : expf(m_s[w] - m_ref);      // a sum without a maximum: NaN scores
            a = fmaf(acc_s[w][x], f, a);
            ll = fmaf(l_s[w], f, ll);
        }
        out[row * out_stride + (long long)h * 32 * NB + x] = ll == 0.0f ? 0.0f : a / ll;
    }
}

}  // namespace ckb

using namespace ckb;

extern "C" size_t ckb200_attention_q4cache_workspace_bytes(int batch, int num_tokens, int num_heads, int num_kv_heads, int head_dim)
{
    (void)batch; (void)num_tokens; (void)num_heads; (void)num_kv_heads; (void)head_dim;
    return 0;
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
    if (workspace_bytes < ckb200_attention_q4cache_workspace_bytes(batch, num_tokens, num_heads, num_kv_heads, head_dim))
        return ckb_fail(CKB_ERR_STATE, "%s: the workspace is too small", what);
    if (rows * num_heads > 0x7fffffffLL) return ckb_fail(CKB_ERR_LIMIT, "%s: %lld query rows in one call", what, rows * num_heads);
    if (!rows) return 0;
    if (ckb_ensure_init()) return CKB_ERR_NO_DEVICE;
    if ((rc = ckb_check_device(what))) return rc;
    (void)workspace;
    const KvQ4 c = {page_table, kv_lens, table_stride, batch, num_tokens, num_pages, page_tokens, num_kv_heads, head_dim / 32};
    const float scale = 1.0f / sqrtf((float)head_dim);
    const unsigned grid = (unsigned)(rows * num_heads);
    cudaStream_t st = ckb_stream(stream);
#define AQ_RUN(NB) attn_q4_kernel<NB><<<grid, AQ_THREADS, 0, st>>>(q, q_stride, (const uint8_t *)k_pages, (const uint8_t *)v_pages, out, out_stride, c, num_heads, sliding_window, scale)
    switch (head_dim) {
    case 64: AQ_RUN(2); break;
    case 96: AQ_RUN(3); break;
    case 128: AQ_RUN(4); break;
    case 192: AQ_RUN(6); break;
    default: AQ_RUN(8); break;
    }
#undef AQ_RUN
    return ckb_check_launch(what);
}
