// A paged KV cache of Q4_1 rows (include/ckb200_cache.h): where a row lies, and what every kernel over it is given.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ckb {

constexpr int KQ4_BLOCK = 20;                 // block_q4_1: fp16 d, fp16 m, 16 bytes of nibbles for 32 values

struct KvQ4 {
    const int *table, *lens;
    int stride, batch, tokens, pages, page_tokens, Hkv, nb;      // nb: blocks of a row
};

__host__ __device__ __forceinline__ int kv_len(int len, int stride, int page_tokens)      // stride * page_tokens fits an int
{
    const int most = stride * page_tokens;
    return len < 0 ? 0 : (len > most ? most : len);
}
__host__ __device__ __forceinline__ int kv_columns(int len, int page_tokens) { return (len + page_tokens - 1) / page_tokens; }
// the page of a table entry, -1 for none
__host__ __device__ __forceinline__ int kv_entry(int entry, int pages) { return entry >= 0 && entry < pages ? entry : -1; }
__host__ __device__ __forceinline__ int kv_page(const int *row, int stride, int pages, int page_tokens, int pos)
{
    if (pos < 0 || pos / page_tokens >= stride) return -1;
    return kv_entry(row[pos / page_tokens], pages);
}
// bytes from the start of a pool of K or V to the row of `slot` in a page: 64 bits, a pool may be larger than 4 GB
__host__ __device__ __forceinline__ size_t kv_row(int page, int head, int slot, int Hkv, int page_tokens, int nb)
{
    return (((size_t)page * Hkv + head) * page_tokens + slot) * (size_t)(nb * KQ4_BLOCK);
}

// n / d by a multiplication, n below 2^31
struct KvDivide {
    uint32_t d, mul, shift;
    __device__ __forceinline__ int operator()(uint32_t n) const { return (int)(d == 1 ? n : __umulhi(n, mul) >> shift); }
};
inline KvDivide kv_divide(uint32_t d)
{
    KvDivide x = {d, 0, 0};
    if (d > 1) {
        while (2u << x.shift < d) ++x.shift;                   // 2^shift < d <= 2^(shift + 1)
        x.mul = (uint32_t)((((uint64_t)1 << (32 + x.shift)) + d - 1) / d);
    }
    return x;
}

}  // namespace ckb

#ifdef __cplusplus
extern "C" {
#endif
/* 0, or the recorded error: sizes that every call over such a cache needs (kv_q4_rows.cu) */
int ckb_check_kv_q4(const char *what, const void *k_pages, const void *v_pages, const int *page_table, int table_stride, const int *kv_lens, int batch,
                    int num_tokens, int num_pages, int page_tokens, int num_kv_heads, int head_dim);
#ifdef __cplusplus
}
#endif
