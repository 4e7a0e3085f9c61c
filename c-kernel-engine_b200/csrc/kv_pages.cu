// Pages of a KV cache that sequences share (include/ckb200_cache.h): growing, shrinking, freeing, forking, compacting, copying.
//
// Tables and reference counts stay on the device, so that a decode step's turn of them can be part of its graph and nothing waits for the
// host.  What a call decides is the same in every run: free pages are handed out by number, the order of the atomics on the counts cannot
// be seen in their sums.  Each call is one kernel that decides, by one CTA where an order over all pages or sequences is needed (latency: a few
// dependent trips to L2), and one that moves the bytes of the pages chosen, at copy bandwidth, reading the list that the first one left.
// Kernels start while the one before is still running and wait for it: tables are read through L2.
#include "../../include/ckb200_cache.h"
#include "device_common.cuh"
#include "kv_q4.cuh"
#include "launch.h"
#include "pdl.cuh"
#include "runtime.h"

namespace ckb {

constexpr int KP_THREADS = 1024, KP_WARPS = KP_THREADS / 32, KP_MAX_BATCH = 4096, KP_KEPT = 32 * 8, KP_LIST = 2048, KP_FORK = 2;
constexpr int KC_THREADS = 256, KC_UNROLL = 8;

struct KvTables {
    int *table, *lens, *refs;
    int stride, batch, pages, page_tokens;
};
struct KvPool {
    uint8_t *base;
    long long plane_stride, page_bytes;
    int planes, pages;
};

// sums over the CTA of N numbers of the threads before this one; total: of all.  `sh`: N rows of KP_WARPS + 1 ints, free again after the call
template <int N>
__device__ __forceinline__ void kp_before(const int (&v)[N], int (&before)[N], int (&total)[N], int (*sh)[KP_WARPS + 1])
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = v[i];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x[i], o);
            if (lane >= o) x[i] += y;
        }
        if (lane == 31) sh[i][warp] = x[i];
    }
    __syncthreads();
    if (warp < N) {
        const int w = lane < KP_WARPS ? sh[warp][lane] : 0;
        int s = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        sh[warp][lane] = s - w;
        if (lane == 31) sh[warp][KP_WARPS] = s;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        before[i] = sh[i][warp] + x[i] - v[i];
        total[i] = sh[i][KP_WARPS];
    }
    __syncthreads();
}

// A warp's stretch [lo, hi) of the reference counts, and which of them are zero: up to 256 pages as bits that stay in registers, a longer stretch is read again
// where it is needed.
struct KpStretch {
    int lo, hi;
    uint32_t free_bits[8];
};
__device__ __forceinline__ void kp_load(const int *refs, int p0, int hi, int (&ref)[8])
{
#pragma unroll
    for (int i = 0; i < 8; ++i) ref[i] = p0 + 32 * i + (threadIdx.x & 31) < hi ? __ldcg(refs + p0 + 32 * i + (threadIdx.x & 31)) : 1;
}
__device__ __forceinline__ int kp_bits(const int (&ref)[8], uint32_t (&bits)[8])
{
    int n = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        bits[i] = __ballot_sync(0xffffffffu, ref[i] == 0);
        n += __popc(bits[i]);
    }
    return n;
}
__device__ __forceinline__ int kp_count_free(const int *refs, KpStretch &s)
{
    int n = 0;
    for (int p0 = s.lo; p0 < s.hi; p0 += KP_KEPT) {
        int ref[8];
        kp_load(refs, p0, s.hi, ref);
        n += kp_bits(ref, s.free_bits);
    }
    return n;
}
// Numbers of the pages of [lo, hi), a part of the stretch, that are free (or in use) into list[at ..), in their order, up to `most` entries of the list in all.
__device__ __forceinline__ void kp_list(const int *refs, const KpStretch &s, int lo, int hi, bool in_use, int *list, int at, int most)
{
    const int lane = threadIdx.x & 31;
    const bool kept = s.hi - s.lo <= KP_KEPT;
    for (int p0 = s.lo; p0 < hi && at < most; p0 += KP_KEPT) {
        uint32_t bits[8];
        if (kept) {
#pragma unroll
            for (int i = 0; i < 8; ++i) bits[i] = s.free_bits[i];
        } else {
            int ref[8];
            kp_load(refs, p0, hi, ref);
            kp_bits(ref, bits);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int p = p0 + 32 * i + lane;
            const bool is = p >= lo && p < hi && ((bits[i] >> lane & 1u) == 0) == in_use;
            const uint32_t mask = __ballot_sync(0xffffffffu, is);
            const int to = at + __popc(mask & ((1u << lane) - 1u));
            if (is && to < most) list[to] = p;
            at += __popc(mask);
        }
    }
}
// how many of [s.lo, cut) are zero
__device__ __forceinline__ int kp_free_below(const int *refs, const KpStretch &s, int cut)
{
    const int lane = threadIdx.x & 31;
    int n = 0;
    for (int p = s.lo + lane; p < cut; p += 32) n += __ldcg(refs + p) == 0;
    return __reduce_add_sync(0xffffffffu, n);
}
__device__ __forceinline__ KpStretch kp_stretch(int pages)
{
    const int span = (pages + KP_WARPS - 1) / KP_WARPS, lo = min(pages, (int)(threadIdx.x >> 5) * span);
    return {lo, min(pages, lo + span), {}};
}

// ---------------------------------------------------------------- the bytes

// Warps take pieces of 4 KB (KC_UNROLL 16-byte loads a lane in flight) of (pair, plane) rows.  With `t` set, the entries of the tables
// from page `live` on are renamed on the way (compaction).
__global__ void __launch_bounds__(KC_THREADS) kv_pages_copy_kernel(KvPool pool, const int *__restrict__ src, const int *__restrict__ dst, const int *__restrict__ count_dev, int count,
                                                                   KvTables t, const int *__restrict__ place)
{
    pdl_wait();
    const int lane = threadIdx.x & 31;
    if (t.table) {
        const int live = __ldcg(count_dev + 1);
        for (int b = blockIdx.x; b < t.batch; b += gridDim.x) {
            int *row = t.table + (size_t)b * t.stride;
            const int n = kv_columns(kv_len(__ldcg(t.lens + b), t.stride, t.page_tokens), t.page_tokens);
            for (int i = threadIdx.x; i < n; i += KC_THREADS) {
                const int e = __ldcg(row + i);
                if (e < live || e >= t.pages) continue;
                const int to = __ldcg(place + e);
                if (to >= 0) row[i] = to;
            }
        }
    }
    if (count_dev) count = __ldcg(count_dev);
    const long long vecs = pool.page_bytes / 16, pieces = (vecs + 32 * KC_UNROLL - 1) / (32 * KC_UNROLL), all = (long long)count * pool.planes * pieces;
    for (long long i = (long long)blockIdx.x * (KC_THREADS / 32) + (threadIdx.x >> 5); i < all; i += (long long)gridDim.x * (KC_THREADS / 32)) {
        const long long row = i / pieces, piece = i - row * pieces;
        const int pair = (int)(row / pool.planes), plane = (int)(row - (long long)pair * pool.planes);
        const int s = __ldcg(src + pair), d = __ldcg(dst + pair);
        if ((unsigned)s >= (unsigned)pool.pages || (unsigned)d >= (unsigned)pool.pages || s == d) continue;
        uint8_t *base = pool.base + plane * pool.plane_stride;
        const uint4 *from = reinterpret_cast<const uint4 *>(base + s * pool.page_bytes);
        uint4 *to = reinterpret_cast<uint4 *>(base + d * pool.page_bytes);
        const long long v0 = piece * (32 * KC_UNROLL) + lane;
        uint4 x[KC_UNROLL];
#pragma unroll
        for (int u = 0; u < KC_UNROLL; ++u)
            if (v0 + 32 * u < vecs) x[u] = __ldcs(from + v0 + 32 * u);
#pragma unroll
        for (int u = 0; u < KC_UNROLL; ++u)
            if (v0 + 32 * u < vecs) __stcs(to + v0 + 32 * u, x[u]);
    }
}

// ---------------------------------------------------------------- resize

// ws: [0] number of pages to copy, [4 ..) their sources, [4 + batch ..) their copies, [4 + 2 batch ..) free pages where they are more than KP_LIST
__global__ void __launch_bounds__(KP_THREADS) kv_pages_resize_kernel(KvTables t, const int *__restrict__ new_lens, int *__restrict__ status, int *__restrict__ ws)
{
    extern __shared__ int kp_sm[];
    __shared__ int sh[3][KP_WARPS + 1], s_copies, s_slow, list_s[KP_LIST];
    const int B = t.batch, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pt = t.page_tokens;
    // for each sequence: its length now and then, the shared page that it would write into (-1: none), pages wanted (-1: stays as it is), where its pages begin in the list
    int *len_s = kp_sm, *new_s = len_s + B, *part_s = new_s + B, *want_s = part_s + B, *first_s = want_s + B, *cow_s = first_s + B;
    int *src = ws + 4, *dst = src + B;
    pdl_trigger();
    pdl_wait();
    if (threadIdx.x == 0) s_slow = 0;
    int shrinks = 0;
    for (int b = threadIdx.x; b < B; b += KP_THREADS) {
        const int len = kv_len(__ldcg(t.lens + b), t.stride, pt);
        int nl = __ldcg(new_lens + b), bad = 0;
        if (nl > t.stride * pt) { nl = -1; bad = 1; }
        len_s[b] = len;
        new_s[b] = nl = nl < 0 ? len : nl;
        status[b] = bad;
        shrinks |= nl < len;
    }
    shrinks = __syncthreads_or(shrinks);
    // those that shrink give back their pages
    for (int b = warp; shrinks && b < B; b += KP_WARPS) {
        const int have = kv_columns(len_s[b], pt), need = kv_columns(new_s[b], pt);
        int *row = t.table + (size_t)b * t.stride;
        for (int i = need + lane; i < have; i += 32) {
            const int e = kv_entry(__ldcg(row + i), t.pages);
            if (e >= 0) atomicSub(t.refs + e, 1);
            row[i] = -1;
        }
    }
    if (shrinks) __syncthreads();
    // those that grow: is the page that the next row goes into shared?  Meanwhile the counts of a pool of up to 8192 pages are on their way
    KpStretch pages = kp_stretch(t.pages);
    const bool kept = t.pages <= KP_WARPS * KP_KEPT;
    int ref[8], shares = 0;
    if (kept) kp_load(t.refs, pages.lo, pages.hi, ref);
    for (int b = threadIdx.x; b < B; b += KP_THREADS) {
        int page = -1;
        if (new_s[b] > len_s[b] && len_s[b] % pt) {
            page = kv_entry(__ldcg(t.table + (size_t)b * t.stride + len_s[b] / pt), t.pages);
            if (page >= 0 && __ldcg(t.refs + page) <= 1) page = -1;
        }
        part_s[b] = page;
        shares |= page >= 0;
    }
    shares = __syncthreads_or(shares);
    int mine = 0, copies = 0;                                   // this thread's sequences are consecutive: the scans below are in their order
    const int each = (B + KP_THREADS - 1) / KP_THREADS, b0 = min(B, (int)threadIdx.x * each), b1 = min(B, b0 + each);
    for (int b = b0; b < b1; ++b) {
        const int grows = new_s[b] > len_s[b];
        int cow = 0;
        if (shares && part_s[b] >= 0) {
            int before = 0;                                     // sharers that have taken their copy when it is b's turn
            for (int o = 0; o < b; ++o) before += part_s[o] == part_s[b];
            cow = __ldcg(t.refs + part_s[b]) - before > 1;
        }
        cow_s[b] = cow;
        want_s[b] = grows ? cow + kv_columns(new_s[b], pt) - kv_columns(len_s[b], pt) : -1;
        mine += max(0, want_s[b]);
        copies += cow;
    }
    // the first page of the list that is this thread's, its first copy, its warp's first free page
    int sums[3] = {mine, copies, 0}, before[3], all[3];
    if (kept) {
        const int n = kp_bits(ref, pages.free_bits);
        if (lane == 0) sums[2] = n;
    }
    kp_before(sums, before, all, sh);
    const int total = all[0];
    int at = before[0], cat = before[1];
    for (int b = b0; b < b1; ++b) {
        first_s[b] = at;
        at += max(0, want_s[b]);
        if (cow_s[b]) cow_s[b] = 1 + cat++;                     // 1 + its place in the list of copies
    }
    if (threadIdx.x == 0) s_copies = all[1];
    int *list = total <= KP_LIST ? list_s : dst + B;
    if (total > 0) {
        if (!kept) {
            const int n = kp_count_free(t.refs, pages), mine_free[1] = {lane == 0 ? n : 0};
            int at_free[1], all_free[1];
            kp_before(mine_free, at_free, all_free, sh);
            before[2] = at_free[0];
            all[2] = all_free[0];
        }
        const int have_free = all[2];
        if (have_free < total) __syncthreads();                 // what the threads have written about the sequences
        if (have_free < total) {                                // one by one: who finds no room leaves its claim to those behind
            if (threadIdx.x == 0) {
                int used = 0, nc = 0;
                for (int b = 0; b < B; ++b) {
                    if (want_s[b] < 0) continue;
                    int page = len_s[b] % pt ? kv_entry(__ldcg(t.table + (size_t)b * t.stride + len_s[b] / pt), t.pages) : -1, cow = 0;
                    if (page >= 0) cow = __ldcg(t.refs + page) > 1;
                    const int want = cow + kv_columns(new_s[b], pt) - kv_columns(len_s[b], pt);
                    cow_s[b] = 0;
                    if (want > have_free - used) {
                        want_s[b] = -1;
                        new_s[b] = len_s[b];
                        status[b] = 1;
                        continue;
                    }
                    part_s[b] = page;
                    want_s[b] = want;
                    first_s[b] = used;
                    used += want;
                    if (cow) {
                        cow_s[b] = 1 + nc++;
                        atomicSub(t.refs + page, 1);
                    }
                }
                s_copies = nc;
                s_slow = 1;
            }
        }
        // the free pages themselves; a page whose count the loop above took down was shared before and still has a holder
        const int base = __shfl_sync(0xffffffffu, before[2], 0);
        kp_list(t.refs, pages, pages.lo, pages.hi, false, list, base, min(total, have_free));
    }
    __syncthreads();
    for (int b = warp; b < B; b += KP_WARPS) {
        int *row = t.table + (size_t)b * t.stride;
        if (want_s[b] > 0) {
            const int have = kv_columns(len_s[b], pt), need = kv_columns(new_s[b], pt), cow = cow_s[b] > 0;
            for (int i = have + lane; i < need; i += 32) {
                const int page = list[first_s[b] + cow + i - have];
                row[i] = page;
                t.refs[page] = 1;
            }
            if (cow && lane == 0) {
                const int page = list[first_s[b]], old = part_s[b];
                src[cow_s[b] - 1] = old;
                dst[cow_s[b] - 1] = page;
                t.refs[page] = 1;
                if (!s_slow) atomicSub(t.refs + old, 1);
                row[have - 1] = page;
            }
        }
        if (lane == 0) t.lens[b] = new_s[b];
    }
    if (threadIdx.x == 0) ws[0] = s_copies;
}

// ---------------------------------------------------------------- fork

// ws: [batch] lengths to come (-1: stays as it is), [batch][stride] rows to come
__global__ void __launch_bounds__(128) kv_pages_fork_read_kernel(KvTables t, const int *__restrict__ parent, int *__restrict__ ws)
{
    pdl_trigger();
    pdl_wait();
    const int b = blockIdx.x, from = __ldcg(parent + b);
    if (from < 0 || from >= t.batch || from == b) {
        if (threadIdx.x == 0) ws[b] = -1;
        return;
    }
    const int len = kv_len(__ldcg(t.lens + from), t.stride, t.page_tokens), n = kv_columns(len, t.page_tokens);
    const int *row = t.table + (size_t)from * t.stride;
    int *to = ws + t.batch + (size_t)b * t.stride;
    for (int i = threadIdx.x; i < n; i += 128) {
        const int e = kv_entry(__ldcg(row + i), t.pages);
        to[i] = e;
        if (e >= 0) atomicAdd(t.refs + e, 1);
    }
    if (threadIdx.x == 0) ws[b] = len;
}
__global__ void __launch_bounds__(128) kv_pages_fork_write_kernel(KvTables t, const int *__restrict__ ws)
{
    pdl_trigger();
    pdl_wait();
    const int b = blockIdx.x, len = __ldcg(ws + b);
    if (len < 0) return;
    const int n = kv_columns(len, t.page_tokens), had = kv_columns(kv_len(__ldcg(t.lens + b), t.stride, t.page_tokens), t.page_tokens);
    const int *from = ws + t.batch + (size_t)b * t.stride;
    int *row = t.table + (size_t)b * t.stride;
    for (int i = threadIdx.x; i < max(n, had); i += 128) {
        const int e = i < had ? kv_entry(__ldcg(row + i), t.pages) : -1;
        if (e >= 0) atomicSub(t.refs + e, 1);
        row[i] = i < n ? __ldcg(from + i) : -1;
    }
    __syncthreads();
    if (threadIdx.x == 0) t.lens[b] = len;
}

// Tables of up to KP_THREADS * KP_FORK entries, by one CTA that holds what every entry was: one launch.  (2048 entries 3.6 us in a graph, 3.7 us by the two kernels
// above and a launch more for the caller; 8192 entries 8.5 and 3.6 us.)
__global__ void __launch_bounds__(KP_THREADS) kv_pages_fork_kernel(KvTables t, const int *__restrict__ parent)
{
    extern __shared__ int kp_sm[];
    pdl_trigger();
    pdl_wait();
    int *len_s = kp_sm, *parent_s = len_s + t.batch;            // a parent: -1 for none
    for (int b = threadIdx.x; b < t.batch; b += KP_THREADS) {
        const int from = __ldcg(parent + b);
        len_s[b] = kv_len(__ldcg(t.lens + b), t.stride, t.page_tokens);
        parent_s[b] = from < 0 || from >= t.batch || from == b ? -1 : from;
    }
    __syncthreads();
    int now[KP_FORK], next[KP_FORK];                            // -1: no page; -2: stays as it is
#pragma unroll
    for (int u = 0; u < KP_FORK; ++u) {
        const int x = threadIdx.x + u * KP_THREADS, b = x / t.stride, i = x - b * t.stride;
        now[u] = -1;
        next[u] = -2;
        if (b >= t.batch || parent_s[b] < 0) continue;
        const int had = kv_columns(len_s[b], t.page_tokens), n = kv_columns(len_s[parent_s[b]], t.page_tokens);
        if (i < had) now[u] = __ldcg(t.table + x);
        if (i < n) next[u] = __ldcg(t.table + parent_s[b] * t.stride + i);
        else if (i < had) next[u] = -1;
        if (i < n) next[u] = max(-1, next[u]);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < KP_FORK; ++u) {
        if (next[u] == -2) continue;
        const int to = kv_entry(next[u], t.pages), old = kv_entry(now[u], t.pages);
        if (to >= 0) atomicAdd(t.refs + to, 1);
        if (old >= 0) atomicSub(t.refs + old, 1);
        t.table[threadIdx.x + u * KP_THREADS] = to;
    }
    for (int b = threadIdx.x; b < t.batch; b += KP_THREADS)
        if (parent_s[b] >= 0) t.lens[b] = len_s[parent_s[b]];
}

// ---------------------------------------------------------------- compact

// ws: [0] pages that move, [1] pages in use, [4 ..) which, [4 + pages ..) where to, [4 + 2 pages ..) for each page from [1] on: where it goes or -1
__global__ void __launch_bounds__(KP_THREADS) kv_pages_plan_kernel(KvTables t, int *__restrict__ live_out, int *__restrict__ ws)
{
    __shared__ int sh[2][KP_WARPS + 1], src_s[KP_LIST], dst_s[KP_LIST];
    const int lane = threadIdx.x & 31;
    int *src = ws + 4, *dst = src + t.pages, *place = dst + t.pages;
    pdl_trigger();
    pdl_wait();
    KpStretch pages = kp_stretch(t.pages);
    const int lo = pages.lo, hi = pages.hi, n = kp_count_free(t.refs, pages);
    const int free_here[1] = {lane == 0 ? n : 0};
    int free_before[1], free_all[1];
    kp_before(free_here, free_before, free_all, sh);
    const int live = t.pages - free_all[0], cut = min(hi, max(lo, live));
    // free ones below `live`, used ones from there on: as many of the one kind as of the other
    const int holes = cut == hi ? n : (cut == lo ? 0 : kp_free_below(t.refs, pages, cut)), movers = (hi - cut) - (n - holes);
    const int sums[2] = {lane == 0 ? holes : 0, lane == 0 ? movers : 0};
    int before[2], all[2];
    kp_before(sums, before, all, sh);
    const int count = all[0];
    const bool near = count <= KP_LIST;                         // the lists are read back from shared memory
    kp_list(t.refs, pages, lo, cut, false, near ? dst_s : dst, __shfl_sync(0xffffffffu, before[0], 0), count);
    kp_list(t.refs, pages, cut, hi, true, near ? src_s : src, __shfl_sync(0xffffffffu, before[1], 0), count);
    for (int p = cut + lane; p < hi; p += 32) place[p] = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += KP_THREADS) {
        const int s = near ? src_s[i] : src[i], d = near ? dst_s[i] : dst[i];
        if (near) {
            src[i] = s;
            dst[i] = d;
        }
        place[s] = d;
        t.refs[d] = __ldcg(t.refs + s);
        t.refs[s] = 0;
    }
    if (threadIdx.x == 0) {
        ws[0] = count;
        ws[1] = live;
        if (live_out) *live_out = live;
    }
}

}  // namespace ckb

using namespace ckb;

extern "C" size_t ckb200_kv_pages_workspace_bytes(int batch, int table_stride, int num_pages)
{
    if (batch <= 0 || table_stride <= 0 || num_pages <= 0) return 0;
    const size_t resize = 4 + 2 * (size_t)batch + num_pages, fork = (size_t)batch * (1 + (size_t)table_stride), compact = 4 + 3 * (size_t)num_pages;
    const size_t most = resize > fork ? (resize > compact ? resize : compact) : (fork > compact ? fork : compact);
    return (most * sizeof(int) + 255) & ~(size_t)255;
}

static int check_tables(const char *what, const int *table, int stride, const int *lens, const int *refs, int batch, int pages, int page_tokens, const void *ws, size_t ws_bytes)
{
    if (!table || !lens || !refs) return ckb_fail(CKB_ERR_STATE, "%s: a pointer is NULL", what);
    if (batch < 0 || stride <= 0 || pages <= 0 || page_tokens <= 0) return ckb_fail(CKB_ERR_SHAPE, "%s: batch %d, table columns %d, pages %d of %d tokens", what, batch, stride, pages, page_tokens);
    if (batch > KP_MAX_BATCH) return ckb_fail(CKB_ERR_LIMIT, "%s: %d sequences, at most %d", what, batch, KP_MAX_BATCH);
    if ((long long)stride * page_tokens > 1 << 30 || pages > 1 << 30) return ckb_fail(CKB_ERR_LIMIT, "%s: a sequence may have up to 2^30 tokens, a pool 2^30 pages", what);
    if ((long long)batch * stride > 0x7fffffffLL) return ckb_fail(CKB_ERR_LIMIT, "%s: a table of %lld entries, at most 2^31 - 1", what, (long long)batch * stride);
    if (((uintptr_t)table | (uintptr_t)lens | (uintptr_t)refs) & 3) return ckb_fail(CKB_ERR_ALIGN, "%s: tables must be aligned to 4 bytes", what);
    if (batch && (!ws || ws_bytes < ckb200_kv_pages_workspace_bytes(batch, stride, pages))) return ckb_fail(CKB_ERR_STATE, "%s: the workspace is too small", what);
    if ((uintptr_t)ws & 15) return ckb_fail(CKB_ERR_ALIGN, "%s: the workspace must be aligned to 16 bytes", what);
    return 0;
}
static int check_pool(const char *what, const void *pages, int planes, long long plane_stride, long long page_bytes, int num_pages)
{
    if (planes < 0 || (planes > 0 && (page_bytes <= 0 || page_bytes % 16 || plane_stride % 16)) || num_pages <= 0)
        return ckb_fail(CKB_ERR_SHAPE, "%s: %d planes %lld bytes apart, %d pages of %lld bytes (multiples of 16)", what, planes, plane_stride, num_pages, page_bytes);
    if (planes > 0 && !pages) return ckb_fail(CKB_ERR_STATE, "%s: a pointer is NULL", what);
    if (planes > 1 && (plane_stride < 0 || plane_stride / page_bytes < num_pages)) return ckb_fail(CKB_ERR_SHAPE, "%s: planes of %d pages lie %lld bytes apart", what, num_pages, plane_stride);
    if ((uintptr_t)pages & 15) return ckb_fail(CKB_ERR_ALIGN, "%s: pools must be aligned to 16 bytes", what);
    return 0;
}
// CTAs for up to `pairs` pages of every plane: no more than can be resident, no more than have a piece to copy
static unsigned copy_grid(long long pairs, int planes, long long page_bytes)
{
    const long long most = (long long)ckb_sm_count() * (2048 / KC_THREADS), pieces = pairs * planes * ((page_bytes + 512 * KC_UNROLL - 1) / (512 * KC_UNROLL)), n = (pieces + KC_THREADS / 32 - 1) / (KC_THREADS / 32);
    return (unsigned)(n < 1 ? 1 : (n < most ? n : most));
}

extern "C" int ckb200_dev_kv_pages_copy(void *pages, int planes, long long plane_stride, long long page_bytes, const int *src, const int *dst, int count, int num_pages, void *stream)
{
    const char *what = "kv_pages_copy";
    int rc = check_pool(what, pages, planes, plane_stride, page_bytes, num_pages);
    if (rc) return rc;
    if (count < 0) return ckb_fail(CKB_ERR_SHAPE, "%s: %d pages", what, count);
    if (count && (!src || !dst)) return ckb_fail(CKB_ERR_STATE, "%s: a pointer is NULL", what);
    if (((uintptr_t)src | (uintptr_t)dst) & 3) return ckb_fail(CKB_ERR_ALIGN, "%s: lists must be aligned to 4 bytes", what);
    if (!count || !planes) return 0;
    if (ckb_ensure_init()) return CKB_ERR_NO_DEVICE;
    if ((rc = ckb_check_device(what))) return rc;
    const KvPool pool = {(uint8_t *)pages, plane_stride, page_bytes, planes, num_pages};
    kv_pages_copy_kernel<<<copy_grid(count, planes, page_bytes), KC_THREADS, 0, ckb_stream(stream)>>>(pool, src, dst, NULL, count, KvTables{}, NULL);
    return ckb_check_launch(what);
}

extern "C" int ckb200_dev_kv_pages_resize(int *page_table, int table_stride, int *kv_lens, int *page_refs, const int *new_lens, int batch, int num_pages, int page_tokens,
                                          void *pages, int planes, long long plane_stride, long long page_bytes, int *status, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *what = "kv_pages_resize";
    int rc = check_tables(what, page_table, table_stride, kv_lens, page_refs, batch, num_pages, page_tokens, workspace, workspace_bytes);
    if (rc || (rc = check_pool(what, pages, planes, plane_stride, page_bytes, num_pages))) return rc;
    if (!new_lens || !status) return ckb_fail(CKB_ERR_STATE, "%s: a pointer is NULL", what);
    if (((uintptr_t)new_lens | (uintptr_t)status) & 3) return ckb_fail(CKB_ERR_ALIGN, "%s: lists must be aligned to 4 bytes", what);
    if (!batch) return 0;
    if (ckb_ensure_init()) return CKB_ERR_NO_DEVICE;
    if ((rc = ckb_check_device(what))) return rc;
    const KvTables t = {page_table, kv_lens, page_refs, table_stride, batch, num_pages, page_tokens};
    const size_t smem = 6 * sizeof(int) * (size_t)batch;
    if (smem > 32 * 1024 && ckb_check_cuda((int)cudaFuncSetAttribute(kv_pages_resize_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 6 * (int)sizeof(int) * KP_MAX_BATCH), what))
        return CKB_ERR_CUDA;
    cudaStream_t st = ckb_stream(stream);
    int *ws = (int *)workspace;
    if ((rc = launch_pdl(what, kv_pages_resize_kernel, dim3(1), dim3(KP_THREADS), smem, st, t, new_lens, status, ws)) || !planes) return rc;
    const KvPool pool = {(uint8_t *)pages, plane_stride, page_bytes, planes, num_pages};
    return launch_pdl(what, kv_pages_copy_kernel, dim3(copy_grid(batch, planes, page_bytes)), dim3(KC_THREADS), 0, st, pool, (const int *)(ws + 4), (const int *)(ws + 4 + batch), (const int *)ws, 0, KvTables{},
                      (const int *)NULL);
}

extern "C" int ckb200_dev_kv_pages_fork(int *page_table, int table_stride, int *kv_lens, int *page_refs, const int *parent, int batch, int num_pages, int page_tokens,
                                        void *workspace, size_t workspace_bytes, void *stream)
{
    const char *what = "kv_pages_fork";
    int rc = check_tables(what, page_table, table_stride, kv_lens, page_refs, batch, num_pages, page_tokens, workspace, workspace_bytes);
    if (rc) return rc;
    if (!parent) return ckb_fail(CKB_ERR_STATE, "%s: a pointer is NULL", what);
    if ((uintptr_t)parent & 3) return ckb_fail(CKB_ERR_ALIGN, "%s: lists must be aligned to 4 bytes", what);
    if (!batch) return 0;
    if (ckb_ensure_init()) return CKB_ERR_NO_DEVICE;
    if ((rc = ckb_check_device(what))) return rc;
    const KvTables t = {page_table, kv_lens, page_refs, table_stride, batch, num_pages, page_tokens};
    cudaStream_t st = ckb_stream(stream);
    if ((long long)batch * table_stride <= KP_THREADS * KP_FORK)
        return launch_pdl(what, kv_pages_fork_kernel, dim3(1), dim3(KP_THREADS), 2 * sizeof(int) * (size_t)batch, st, t, parent);
    if ((rc = launch_pdl(what, kv_pages_fork_read_kernel, dim3(batch), dim3(128), 0, st, t, parent, (int *)workspace))) return rc;
    return launch_pdl(what, kv_pages_fork_write_kernel, dim3(batch), dim3(128), 0, st, t, (const int *)workspace);
}

extern "C" int ckb200_dev_kv_pages_compact(int *page_table, int table_stride, const int *kv_lens, int *page_refs, int batch, int num_pages, int page_tokens, void *pages,
                                           int planes, long long plane_stride, long long page_bytes, int *live, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *what = "kv_pages_compact";
    int rc = check_tables(what, page_table, table_stride, kv_lens, page_refs, batch, num_pages, page_tokens, workspace, workspace_bytes);
    if (rc || (rc = check_pool(what, pages, planes, plane_stride, page_bytes, num_pages))) return rc;
    if ((uintptr_t)live & 3) return ckb_fail(CKB_ERR_ALIGN, "%s: lists must be aligned to 4 bytes", what);
    if (!batch) return 0;
    if (ckb_ensure_init()) return CKB_ERR_NO_DEVICE;
    if ((rc = ckb_check_device(what))) return rc;
    const KvTables t = {page_table, const_cast<int *>(kv_lens), page_refs, table_stride, batch, num_pages, page_tokens};
    cudaStream_t st = ckb_stream(stream);
    int *ws = (int *)workspace;
    if ((rc = launch_pdl(what, kv_pages_plan_kernel, dim3(1), dim3(KP_THREADS), 0, st, t, live, ws))) return rc;
    const KvPool pool = {(uint8_t *)pages, plane_stride, page_bytes, planes, num_pages};
    const unsigned pieces = copy_grid(num_pages / 2, planes, page_bytes), grid = pieces > (unsigned)batch ? pieces : (unsigned)batch;      // each also takes rows of the table
    return launch_pdl(what, kv_pages_copy_kernel, dim3(grid), dim3(KC_THREADS), 0, st, pool, (const int *)(ws + 4), (const int *)(ws + 4 + num_pages), (const int *)ws, 0, t,
                      (const int *)(ws + 4 + 2 * (size_t)num_pages));
}
