// Pages and cache slots for the new tokens of many requests, and the rotary embedding that stores their keys and values
// there: the two steps that keep a paged key/value cache, beside the contiguous cache of decode_glue.cu.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "pair16.cuh"

namespace eptq {
namespace {

// ---- plan ----------------------------------------------------------------------------------------
// Two prefix sums over the requests: of the new tokens (the requests' rows) and of the pages they need (their place in
// the free list); everything else follows from them row by row and page by page.
//
// A few bytes per request and 16 per row: the time is the launch and the chain of dependent reads, so it is one launch.
// Every block forms the sums over all requests itself, 1024 at a time (512 requests are 4 KB from L2), instead of
// waiting for another block's, and then writes its share of the rows and pages, found by bisection in the sums.  4.6 us for 64
// requests of one token, 6.0 us for 512 requests and 49904 rows, replayed.
constexpr int kPlanThreads = 1024;
constexpr int kPlanRowsPerBlock = 1024;

struct PlanArgs {
    const int *cached, *fresh, *free_pages, *n_free;
    int *tables, *cu_rows, *kv_lens, *n_free_out;
    long long *positions, *slots;
    long long table_stride;
    int B, width, free_cap, page_size, rows;
};

// Inclusive prefix sum over the block; `warp_sums` holds 33 values, the last of them the total afterwards.
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
    }
    __syncthreads();                                   // the previous scan's sums may still be read
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
        long long w = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += up;
        }
        __syncwarp();
        warp_sums[lane] = w;
        if (lane == 31) warp_sums[32] = w;
    }
    __syncthreads();
    return v + (warp > 0 ? warp_sums[warp - 1] : 0);
}

// First index of ends[0..n) whose value is above x (n if none).
__device__ __forceinline__ int first_above(const long long* ends, int n, long long x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > x) hi = mid; else lo = mid + 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_pages_kernel(const PlanArgs p) {
    __shared__ long long warp_sums[33];
    __shared__ long long row_end[kPlanThreads], page_end[kPlanThreads];
    __shared__ int held_s[kPlanThreads], cached_s[kPlanThreads];
    __shared__ bool served_s[kPlanThreads];
    __shared__ int taken;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, ps = p.page_size;
    const long long n_free = min(max(*p.n_free, 0), p.free_cap);
    const bool first_block = blockIdx.x == 0;
    const long long step = static_cast<long long>(gridDim.x) * kPlanThreads;
    if (tid == 0) taken = 0;
    if (first_block && tid == 0) p.cu_rows[0] = 0;
    long long rows_before = 0, pages_before = 0;
    for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
        const int b = b0 + tid, n = min(kPlanThreads, p.B - b0);
        const long long cached = b < p.B ? max(p.cached[b], 0) : 0;
        const long long fresh = b < p.B ? max(p.fresh[b], 0) : 0;
        const long long total = cached + fresh;
        const long long ends = rows_before + block_scan(fresh, warp_sums);
        const long long chunk_rows = warp_sums[32];
        const bool fits = total <= static_cast<long long>(p.width) * ps && ends <= p.rows;
        const long long held = (cached + ps - 1) / ps;
        const long long need = fits ? (total + ps - 1) / ps - held : 0;
        const long long upto = pages_before + block_scan(need, warp_sums);
        const long long chunk_pages = warp_sums[32];
        const bool served = fits && (need == 0 || upto <= n_free);
        row_end[tid] = ends;
        page_end[tid] = upto;
        held_s[tid] = static_cast<int>(held);
        cached_s[tid] = static_cast<int>(cached);
        served_s[tid] = served;
        if (served && need > 0) atomicMax(&taken, static_cast<int>(upto));      // a maximum: the order does not matter
        if (first_block && b < p.B) {
            p.cu_rows[b + 1] = static_cast<int>(min(ends, static_cast<long long>(p.rows)));
            p.kv_lens[b] = served ? static_cast<int>(total) : 0;
        }
        __syncthreads();
        // this block's share of the rows of these requests
        const long long r_end = min(rows_before + chunk_rows, static_cast<long long>(p.rows));
        for (long long r = blockIdx.x * static_cast<long long>(kPlanThreads) + tid; r < r_end; r += step) {
            if (r < rows_before) continue;
            const int i = first_above(row_end, n, r);
            const long long before = i > 0 ? row_end[i - 1] : rows_before;
            const long long pos = cached_s[i] + (r - before);
            long long slot = -1;
            if (served_s[i]) {
                const long long at = pos / ps, nth = at - held_s[i];
                const long long pages_of_others = i > 0 ? page_end[i - 1] : pages_before;
                const long long page = nth >= 0 ? p.free_pages[n_free - 1 - (pages_of_others + nth)]
                                                : p.tables[(b0 + i) * p.table_stride + at];
                slot = page * ps + pos % ps;
            }
            p.positions[r] = pos;
            p.slots[r] = slot;
        }
        // and of their new pages
        for (long long g = pages_before + blockIdx.x * static_cast<long long>(kPlanThreads) + tid; g < min(pages_before + chunk_pages, n_free); g += step) {
            const int i = first_above(page_end, n, g);
            if (!served_s[i]) continue;
            const long long before = i > 0 ? page_end[i - 1] : pages_before;
            p.tables[(b0 + i) * p.table_stride + held_s[i] + (g - before)] = p.free_pages[n_free - 1 - g];
        }
        rows_before += chunk_rows;
        pages_before += chunk_pages;
        __syncthreads();
    }
    for (long long r = blockIdx.x * static_cast<long long>(kPlanThreads) + tid; r < p.rows; r += step)
        if (r >= rows_before) { p.positions[r] = 0; p.slots[r] = -1; }
    __syncthreads();
    if (first_block && tid == 0) *p.n_free_out = static_cast<int>(n_free) - taken;
}

// ---- rotary embedding + store into the pages ---------------------------------------------------------
// One block per row.  cos and sin of the row's angles are formed once, in shared memory, for all its heads; an item is 8
// neighbouring pairs of one head (two 16-byte reads, two 16-byte writes).  The angle position * inv_freq is exact in 64
// bits and reduced there to [-pi, pi]: in 32 bits it would be off by position * 2^-24, more than a rounding of the
// outputs from a few thousand tokens on.  cos and sin stay in 32 bits: they are rounded once, with the product.  Bound by memory:
// 4847 rows of 32 + 8 + 8 heads of 128 in 21.0 us (5.7 TB/s), 8 rows in 3.9 us, replayed.  (Aligned
// to 16 bytes, the pairs of cos and sin are read four at a time, and the same rows take 22.0 us.)
constexpr int kAppendThreads = 128;
constexpr int kAppendMaxHeadDim = 256;

struct AppendArgs {
    const uint16_t *q, *k, *v;
    uint16_t *q_out, *k_cache, *v_cache;
    const long long *positions, *slots;
    const float* inv_freq;
    long long q_stride, k_stride, v_stride, page_stride;
    int nh, nkv, hd, n_pages, page_size;
    float scaling;
};

template <typename T>
__global__ void __launch_bounds__(kAppendThreads) rope_append_paged_kernel(const AppendArgs p) {
    __shared__ __align__(8) float cos_s[kAppendMaxHeadDim / 2], sin_s[kAppendMaxHeadDim / 2];      // read in pairs
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long r = blockIdx.x;
    const int half = p.hd >> 1, ipr = p.hd >> 4;                    // items per head
    const long long pos = p.positions[r], slot = p.slots[r];
    for (int i = threadIdx.x; i < half; i += kAppendThreads) {
        constexpr double kTurn = 6.283185307179586476925;
        const double angle = static_cast<double>(pos) * static_cast<double>(p.inv_freq[i]);
        float s, c;
        sincosf(static_cast<float>(angle - rint(angle * (1.0 / kTurn)) * kTurn), &s, &c);
        cos_s[i] = c * p.scaling;
        sin_s[i] = s * p.scaling;
    }
    __syncthreads();
    const bool stored = slot >= 0 && slot < static_cast<long long>(p.n_pages) * p.page_size;
    const long long in_cache = stored ? (slot / p.page_size) * p.page_stride + (slot % p.page_size) * p.hd : 0;
    const int items = (p.nh + 2 * (stored ? p.nkv : 0)) * ipr;
    for (int it = threadIdx.x; it < items; it += kAppendThreads) {
        const int head = it / ipr, i = (it - head * ipr) * 8;
        const uint16_t* src;
        uint16_t* dst;
        if (head < p.nh) {
            src = p.q + r * p.q_stride + head * p.hd;
            dst = p.q_out + (r * p.nh + head) * p.hd;
        } else {
            const bool value = head >= p.nh + p.nkv;
            const int h = head - p.nh - (value ? p.nkv : 0);
            src = (value ? p.v + r * p.v_stride : p.k + r * p.k_stride) + h * p.hd;
            dst = (value ? p.v_cache : p.k_cache) + in_cache + static_cast<long long>(h) * p.page_size * p.hd;
        }
        uint4 lo = *reinterpret_cast<const uint4*>(src + i), hi = *reinterpret_cast<const uint4*>(src + half + i);
        if (head < p.nh + p.nkv) {
            unsigned* const a = reinterpret_cast<unsigned*>(&lo);
            unsigned* const b = reinterpret_cast<unsigned*>(&hi);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 x = Pair16<T>::unpack(a[e]), y = Pair16<T>::unpack(b[e]);
                const float2 c = *reinterpret_cast<const float2*>(cos_s + i + 2 * e), s = *reinterpret_cast<const float2*>(sin_s + i + 2 * e);
                a[e] = Pair16<T>::pack(x.x * c.x - y.x * s.x, x.y * c.y - y.y * s.y);
                b[e] = Pair16<T>::pack(y.x * c.x + x.x * s.x, y.y * c.y + x.y * s.y);
            }
        }
        *reinterpret_cast<uint4*>(dst + i) = lo;
        *reinterpret_cast<uint4*>(dst + half + i) = hi;
    }
}

bool page_size_ok(int ps) { return ps >= 16 && ps <= 128 && (ps & (ps - 1)) == 0; }

template <typename Args>
int launch(void (*kernel)(Args), unsigned blocks, unsigned threads, const Args& args, void* stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, args) != cudaSuccess) {
        cudaGetLastError();
        return EPTQ_ERR_LAUNCH;
    }
    count_launch(EPTQ_KERNEL_OTHER);
    return EPTQ_OK;
}

}  // namespace
}  // namespace eptq

using namespace eptq;

extern "C" int eptq_plan_pages(const int32_t* cached, const int32_t* fresh, int B, int32_t* tables, int64_t table_stride,
                               int width, const int32_t* free_pages, int free_cap, const int32_t* n_free, int page_size,
                               int rows, int32_t* cu_rows, int32_t* kv_lens, int64_t* positions, int64_t* slots,
                               int32_t* n_free_out, void* stream) {
    if (B < 0 || width < 0 || free_cap < 0 || rows < 0 || table_stride < width || !page_size_ok(page_size)) return EPTQ_ERR_SHAPE;
    if (cu_rows == nullptr || n_free == nullptr || n_free_out == nullptr) return EPTQ_ERR_NULL;
    if ((B > 0 && (cached == nullptr || fresh == nullptr || kv_lens == nullptr)) || (B > 0 && width > 0 && tables == nullptr) ||
        (free_cap > 0 && free_pages == nullptr) || (rows > 0 && (positions == nullptr || slots == nullptr))) return EPTQ_ERR_NULL;
    PlanArgs a;
    a.cached = cached; a.fresh = fresh; a.free_pages = free_pages; a.n_free = n_free;
    a.tables = tables; a.cu_rows = cu_rows; a.kv_lens = kv_lens; a.n_free_out = n_free_out;
    a.positions = reinterpret_cast<long long*>(positions); a.slots = reinterpret_cast<long long*>(slots);
    a.table_stride = table_stride;
    a.B = B; a.width = width; a.free_cap = free_cap; a.page_size = page_size; a.rows = rows;
    const long long blocks = (static_cast<long long>(rows) + kPlanRowsPerBlock - 1) / kPlanRowsPerBlock;
    return launch(plan_pages_kernel, static_cast<unsigned>(blocks < 1 ? 1 : blocks > kSms ? kSms : blocks), kPlanThreads, a, stream);
}

extern "C" int eptq_rope_append_paged(int dtype, const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride,
                                      const uint16_t* v, int64_t v_stride, uint16_t* q_out, uint16_t* k_cache,
                                      uint16_t* v_cache, int64_t page_stride, const int64_t* positions, const int64_t* slots,
                                      const float* inv_freq, int rows, int n_heads, int n_kv_heads, int head_dim,
                                      int n_pages, int page_size, float scaling, void* stream) {
    if (dtype != EPTQ_FP16 && dtype != EPTQ_BF16) return EPTQ_ERR_UNSUPPORTED;
    if (rows < 0 || n_heads < 1 || n_kv_heads < 1 || n_heads > 65535 || n_kv_heads > 65535 || n_pages < 0 || !page_size_ok(page_size))
        return EPTQ_ERR_SHAPE;
    if (head_dim < 16 || head_dim > kAppendMaxHeadDim || (head_dim % 16) != 0) return EPTQ_ERR_UNSUPPORTED;
    if (q_stride < static_cast<int64_t>(n_heads) * head_dim || k_stride < static_cast<int64_t>(n_kv_heads) * head_dim ||
        v_stride < static_cast<int64_t>(n_kv_heads) * head_dim ||
        page_stride < static_cast<int64_t>(n_kv_heads) * page_size * head_dim) return EPTQ_ERR_SHAPE;
    if (rows == 0) return EPTQ_OK;
    if (q == nullptr || k == nullptr || v == nullptr || q_out == nullptr || positions == nullptr || slots == nullptr ||
        inv_freq == nullptr || (n_pages > 0 && (k_cache == nullptr || v_cache == nullptr))) return EPTQ_ERR_NULL;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_out) || !aligned16(k_cache) || !aligned16(v_cache) ||
        ((q_stride | k_stride | v_stride | page_stride) % 8) != 0) return EPTQ_ERR_ALIGN;
    AppendArgs a;
    a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.k_cache = k_cache; a.v_cache = v_cache;
    a.positions = reinterpret_cast<const long long*>(positions); a.slots = reinterpret_cast<const long long*>(slots);
    a.inv_freq = inv_freq;
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride; a.page_stride = page_stride;
    a.nh = n_heads; a.nkv = n_kv_heads; a.hd = head_dim; a.n_pages = n_pages; a.page_size = page_size;
    a.scaling = scaling;
    return launch(dtype == EPTQ_FP16 ? rope_append_paged_kernel<__half> : rope_append_paged_kernel<__nv_bfloat16>, rows, kAppendThreads, a, stream);
}
