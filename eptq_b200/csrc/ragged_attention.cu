// Causal attention of many requests' rows, over a paged key/value cache or over packed keys and values.
//
// For row t of a request with n rows and L keys, and head h with the keys of head g = h / (n_heads / n_kv_heads):
//     o_t = sum_j exp(s_tj - m_t) v_j / sum_j exp(s_tj - m_t),   s_tj = scale q_t . k_j,   j = 0 .. L - n + t,
// with the maximum m_t and the sum kept while the keys go by once.

#include "common.cuh"
#include "pair16.cuh"

namespace eptq {

size_t attention_tcgen05_bytes(const EptqAttention& a);
int launch_attention_tcgen05(const EptqAttention& a, void* workspace, size_t workspace_bytes, cudaStream_t stream);

namespace {

constexpr int kSimpleWarps = 4;

// One warp per row and head, one key after the other.
template <typename T, int HD>
__global__ void __launch_bounds__(kSimpleWarps * 32) ragged_attention_simple_kernel(const EptqAttention a) {
    constexpr int W = HD / 64;                               // 32-bit words of a head that a lane holds
    const int lane = threadIdx.x & 31;
    const long long unit = blockIdx.x * static_cast<long long>(kSimpleWarps) + (threadIdx.x >> 5);
    const int r = static_cast<int>(unit / a.n_heads), h = static_cast<int>(unit % a.n_heads);
    if (r >= a.rows) return;
    int lo = 0, hi = a.batch;                                // the request whose rows hold r
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.cu_rows[mid + 1] > r) hi = mid; else lo = mid + 1;
    }
    if (lo == a.batch) return;
    const int b = lo, first = a.cu_rows[b], n = a.cu_rows[b + 1] - first, t = r - first;
    const long long keys = a.page_size != 0 ? min(static_cast<long long>(a.kv_lens[b]), static_cast<long long>(a.table_width) * a.page_size) : n;
    const long long seen = keys - n + t + 1;
    const int g = h / (a.n_heads / a.n_kv_heads);
    float q[2 * W], o[2 * W], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float2 f = Pair16<T>::unpack(reinterpret_cast<const unsigned*>(a.q + r * a.q_stride + h * HD)[w * 32 + lane]);
        q[2 * w] = f.x * a.scale; q[2 * w + 1] = f.y * a.scale;
        o[2 * w] = o[2 * w + 1] = 0.f;
    }
    for (long long j = 0; j < seen; ++j) {
        long long k_at, v_at;
        if (a.page_size != 0) {
            const int page = a.tables[b * a.table_stride + j / a.page_size];
            if (page < 0 || page >= a.n_pages) continue;
            const long long in_page = (static_cast<long long>(g) * a.page_size + j % a.page_size) * HD;
            k_at = page * a.k_stride + in_page;
            v_at = page * a.v_stride + in_page;
        } else {
            k_at = (first + j) * a.k_stride + g * HD;
            v_at = (first + j) * a.v_stride + g * HD;
        }
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 f = Pair16<T>::unpack(reinterpret_cast<const unsigned*>(a.k + k_at)[w * 32 + lane]);
            s = fmaf(q[2 * w], f.x, fmaf(q[2 * w + 1], f.y, s));
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        const float m2 = fmaxf(m, s);
        const float keep = m2 == -INFINITY ? 1.f : __expf(m - m2), p = m2 == -INFINITY ? 0.f : __expf(s - m2);
        l = l * keep + p;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 f = Pair16<T>::unpack(reinterpret_cast<const unsigned*>(a.v + v_at)[w * 32 + lane]);
            o[2 * w] = o[2 * w] * keep + p * f.x;
            o[2 * w + 1] = o[2 * w + 1] * keep + p * f.y;
        }
        m = m2;
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w)
        reinterpret_cast<unsigned*>(a.out + (static_cast<long long>(r) * a.n_heads + h) * HD)[w * 32 + lane] = Pair16<T>::pack(o[2 * w] * inv, o[2 * w + 1] * inv);
}

int check(const EptqAttention& a) {
    if (a.dtype != EPTQ_FP16 && a.dtype != EPTQ_BF16) return EPTQ_ERR_UNSUPPORTED;
    if (a.rows < 0 || a.batch < 0 || a.n_heads < 1 || a.n_heads > 65535 || a.n_kv_heads < 1 || (a.n_heads % a.n_kv_heads) != 0 || a.max_rows < 0)
        return EPTQ_ERR_SHAPE;
    if (a.head_dim != 64 && a.head_dim != 128) return EPTQ_ERR_UNSUPPORTED;
    const bool paged = a.page_size != 0;
    if (paged && (a.page_size < 16 || a.page_size > 128 || (a.page_size & (a.page_size - 1)) != 0 || a.n_pages < 0 || a.table_width < 0 ||
                  a.table_stride < a.table_width)) return EPTQ_ERR_SHAPE;
    const int64_t kv_row = static_cast<int64_t>(a.n_kv_heads) * a.head_dim * (paged ? a.page_size : 1);
    if (a.q_stride < static_cast<int64_t>(a.n_heads) * a.head_dim || a.k_stride < kv_row || a.v_stride < kv_row) return EPTQ_ERR_SHAPE;
    if (a.rows > 0 && a.batch > 0 && (a.q == nullptr || a.out == nullptr || a.cu_rows == nullptr || (paged && (a.kv_lens == nullptr || (a.tables == nullptr && a.table_width > 0))) ||
                                      ((!paged || a.n_pages > 0) && (a.k == nullptr || a.v == nullptr)))) return EPTQ_ERR_NULL;
    if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.out) || ((a.q_stride | a.k_stride | a.v_stride) % 8) != 0)
        return EPTQ_ERR_ALIGN;
    return EPTQ_OK;
}

}  // namespace
}  // namespace eptq

using namespace eptq;

// Rows of one key/value head of a request from which the tensor-core kernel takes a paged call.
constexpr int kTensorRows = 32;

static bool on_tensor_cores(const EptqAttention& a) {
    if (a.page_size == 0) return true;
    return a.n_pages > 0 && static_cast<long long>(a.max_rows) * (a.n_heads / a.n_kv_heads) > kTensorRows;
}

extern "C" size_t eptq_ragged_attention_workspace_bytes(const EptqAttention* a) {
    return a == nullptr || check(*a) != EPTQ_OK || !on_tensor_cores(*a) ? 0 : attention_tcgen05_bytes(*a);
}

extern "C" int eptq_ragged_attention(const EptqAttention* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (a == nullptr) return EPTQ_ERR_NULL;
    if (const int st = check(*a); st != EPTQ_OK) return st;
    if (a->rows == 0 || a->batch == 0) return EPTQ_OK;
    if (on_tensor_cores(*a)) return launch_attention_tcgen05(*a, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
    const long long blocks = (static_cast<long long>(a->rows) * a->n_heads + kSimpleWarps - 1) / kSimpleWarps;
    if (blocks > 2147483647LL) return EPTQ_ERR_SHAPE;
    auto* kernel = a->dtype == EPTQ_FP16 ? (a->head_dim == 128 ? ragged_attention_simple_kernel<__half, 128> : ragged_attention_simple_kernel<__half, 64>)
                                         : (a->head_dim == 128 ? ragged_attention_simple_kernel<__nv_bfloat16, 128> : ragged_attention_simple_kernel<__nv_bfloat16, 64>);
    kernel<<<static_cast<unsigned>(blocks), kSimpleWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(*a);
    count_launch(EPTQ_KERNEL_OTHER);
    return cudaGetLastError() == cudaSuccess ? EPTQ_OK : EPTQ_ERR_LAUNCH;
}
