// Causal attention of many requests' rows, over a paged key/value cache or over packed keys and values: the entry point,
// the choice of the kernel, and the join of row tiles whose keys several blocks have taken.
//
// For row t of a request with n rows and L keys, and head h with the keys of head g = h / (n_heads / n_kv_heads):
//     o_t = sum_j exp(s_tj - m_t) v_j / sum_j exp(s_tj - m_t),   s_tj = scale q_t . k_j,   j = 0 .. L - n + t.
// A piece of the keys gives (reference m, sum, o); pieces join as sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) sum_i.

#include <mutex>

#include "attention_host.cuh"
#include "pair16.cuh"

namespace eptq {

PFN_cuTensorMapEncodeTiled_v12000 attention_map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, []() {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) == cudaSuccess &&
            qres == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

namespace {

// Block (share, 16 rows of its cut tile), 8 columns of one row per thread.  Where the tile has 8 rows or 4 -- a long request of one
// token has 50 pieces of 4 rows -- two or four sets of threads take every second or fourth piece.  Pieces are added in an order
// that depends on the tile and its cuts alone.  About 4 us where little is cut (launch, descriptor, reads in turn), 7 us for 55
// pieces of 8 tiles of 4 rows, 13 us for a cut tile of 256 rows in every share (39 MB of pieces).  Where a tile has fewer pieces than are
// read together, its last one is read for those it lacks: branches around the reads made calls of 24.2, 40.7 and 32.1 us (32 rows
// on 6000 keys, 5 times 64 on 3000, 256 on 2000; 32 over 8 heads) 24.8, 44.1 and 35.3 us.
constexpr int kJoinRows = 16;

template <typename T, int HD>
__global__ void __launch_bounds__(kJoinRows * HD / 8) attention_join_kernel(const __grid_constant__ AttentionArgs p) {
    constexpr int kCols = HD / 8;
    __shared__ float parts[10][kJoinRows * kCols];
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const CutTile c = p.cut_tiles[blockIdx.x];
    if (c.of == 0) return;
    const int tile_rows = p.tile_rows < 256 ? min(c.tokens, p.tokens_per_half) * p.heads_per_tile : kJoinRows;
    const int sets = tile_rows <= kJoinRows / 4 ? 4 : tile_rows <= kJoinRows / 2 ? 2 : 1, set_rows = kJoinRows / sets;
    const int in_block = threadIdx.x % kJoinRows, set = in_block / set_rows;
    const int at_row = blockIdx.y * kJoinRows + in_block % set_rows, col = threadIdx.x / kJoinRows * 8;
    const int half = at_row >> 7, row = at_row & 127;
    const int token = half * p.tokens_per_half + row / p.heads_per_tile, head = row % p.heads_per_tile;
    const bool live = row < p.heads_per_tile * p.tokens_per_half && token < c.tokens;
    const long long size = piece_floats(p.tile_rows, HD);
    const float* const first = p.partial + (2 * blockIdx.x + 1) * size;
    const float* const others = p.partial + 2 * blockIdx.x * size;      // piece i at 2 i pieces behind, i = 1 ..
    const int stat = p.tile_rows * HD + at_row;
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, all = 0.f, top = -INFINITY;
    constexpr int kAtOnce = 8;                                          // pieces whose reads are in flight together
    for (int i0 = set; live && i0 < c.of; i0 += kAtOnce * sets) {
        float bias[kAtOnce], sum[kAtOnce];
        float4 x[kAtOnce], y[kAtOnce];
        float high = top;
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            const int i = min(i0 + n * sets, c.of - 1);
            const float* const piece = i == 0 ? first : others + 2 * i * size;
            bias[n] = __ldcg(piece + stat);
            sum[n] = i0 + n * sets < c.of ? __ldcg(piece + stat + p.tile_rows) : 0.f;
            x[n] = __ldcg(reinterpret_cast<const float4*>(piece) + col / 4 * p.tile_rows + at_row);
            y[n] = __ldcg(reinterpret_cast<const float4*>(piece) + (col / 4 + 1) * p.tile_rows + at_row);
        }
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n)
            if (sum[n] != 0.f) high = fmaxf(high, bias[n]);
        const float keep = top == -INFINITY ? 0.f : exp2_approx(top - high);
        top = high;
        all *= keep;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] *= keep;
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            if (sum[n] == 0.f) continue;                                // no key seen: its o was not written
            const float w = exp2_approx(bias[n] - top);
            all += sum[n] * w;
            o[0] += x[n].x * w; o[1] += x[n].y * w; o[2] += x[n].z * w; o[3] += x[n].w * w;
            o[4] += y[n].x * w; o[5] += y[n].y * w; o[6] += y[n].z * w; o[7] += y[n].w * w;
        }
    }
    if (sets > 1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) parts[e][threadIdx.x] = o[e];
        parts[8][threadIdx.x] = all;
        parts[9][threadIdx.x] = top;
        __syncthreads();
        if (set > 0 || !live) return;
        for (int s = 1; s < sets; ++s) {
            const int other = threadIdx.x + s * set_rows;
            const float sum = parts[8][other];
            if (sum == 0.f) continue;
            const float high = fmaxf(top, parts[9][other]);
            const float keep = all == 0.f ? 0.f : exp2_approx(top - high), w = exp2_approx(parts[9][other] - high);
            top = high;
            all = all * keep + sum * w;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = o[e] * keep + parts[e][other] * w;
        }
    }
    if (!live) return;
    const float inv = all == 0.f ? 0.f : 1.f / all;
    uint4 v;
    v.x = Pair16<T>::pack(o[0] * inv, o[1] * inv);
    v.y = Pair16<T>::pack(o[2] * inv, o[3] * inv);
    v.z = Pair16<T>::pack(o[4] * inv, o[5] * inv);
    v.w = Pair16<T>::pack(o[6] * inv, o[7] * inv);
    *reinterpret_cast<uint4*>(p.out + (static_cast<long long>(c.row + token) * p.n_heads + c.head + head) * HD + col) = v;
}

int launch_join(const EptqAttention& a, const AttentionPlan& plan, const AttentionArgs& p, cudaStream_t stream) {
    const dim3 grid(plan.shares, plan.tile_rows / kJoinRows);
    const int threads = kJoinRows * a.head_dim / 8;
    if (a.dtype == EPTQ_FP16)
        return a.head_dim == 128 ? launch_dependent(attention_join_kernel<__half, 128>, grid, threads, 0, stream, p)
                                 : launch_dependent(attention_join_kernel<__half, 64>, grid, threads, 0, stream, p);
    return a.head_dim == 128 ? launch_dependent(attention_join_kernel<__nv_bfloat16, 128>, grid, threads, 0, stream, p)
                             : launch_dependent(attention_join_kernel<__nv_bfloat16, 64>, grid, threads, 0, stream, p);
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
    if (a.rows > 0 && a.clear_rest != 0 && a.out == nullptr) return EPTQ_ERR_NULL;
    if (a.rows > 0 && a.batch > 0 && (a.q == nullptr || a.out == nullptr || a.cu_rows == nullptr ||
                                      (paged && (a.kv_lens == nullptr || (a.tables == nullptr && a.table_width > 0))) ||
                                      ((!paged || a.n_pages > 0) && (a.k == nullptr || a.v == nullptr)))) return EPTQ_ERR_NULL;
    if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.out) || ((a.q_stride | a.k_stride | a.v_stride) % 8) != 0)
        return EPTQ_ERR_ALIGN;
    return EPTQ_OK;
}

// Tiles of 16 rows (whole tokens of one key/value head) up to which a request counts as few rows.  One is bound by the cache's reads; more
// read the keys again, which pays as long as the smaller shares win more: with heads of 64 up to two tiles, with heads of 128 no longer.
// Few rows against tcgen05, us, replayed:
//   heads of 64, 32 rows: 12 heads, 16 requests of 1000 keys 30 / 40, 64 of 2000 138 / 161; 8 heads, 64 of 2000 98 / 122, 1 of 16000 25 / 24,
//     16 of 1000 25 / 21; 40 rows: 39 / 40, 210 / 161, 136 / 122, 27 / 23, 28 / 21
//   heads of 128, 16 rows: 12 heads, 16 of 1000 32 / 43, 64 of 2000 145 / 186; 8 heads, 64 of 2000 102 / 141, 1 of 16000 31 / 29, 16 of 1000
//     26 / 26; 20 rows: 45 / 43, 268 / 189, 183 / 142, 36 / 29, 36 / 26
// One or four short requests (1000 keys) would be faster with few rows at 64 rows still, 12 to 18 against 19 to 24 us, but lengths stand
// on the device.
bool on_tensor_cores(const EptqAttention& a) {
    const int group = a.n_heads / a.n_kv_heads, heads = heads_in(group, 16), tokens = 16 / heads;
    const long long tiles = (static_cast<long long>(a.max_rows) + tokens - 1) / tokens * (group / heads);
    return a.page_size == 0 || tiles > (a.head_dim == 64 ? 2 : 1);
}

AttentionPlan plan_of(const EptqAttention& a) { return on_tensor_cores(a) ? attention_tcgen05_plan(a) : attention_rows_plan(a); }

size_t cut_tile_bytes(const AttentionPlan& plan) { return (plan.shares * sizeof(CutTile) + 255) / 256 * 256; }

size_t bytes_of(const EptqAttention& a, const AttentionPlan& plan) {
    return plan.may_cut ? cut_tile_bytes(plan) + 2 * plan.shares * piece_floats(plan.tile_rows, a.head_dim) * sizeof(float) : 0;
}

}  // namespace
}  // namespace eptq

using namespace eptq;

extern "C" size_t eptq_ragged_attention_workspace_bytes(const EptqAttention* a) {
    return a == nullptr || check(*a) != EPTQ_OK ? 0 : bytes_of(*a, plan_of(*a));
}

extern "C" int eptq_ragged_attention(const EptqAttention* args, void* workspace, size_t workspace_bytes, void* stream) {
    if (args == nullptr) return EPTQ_ERR_NULL;
    const EptqAttention& a = *args;
    if (const int st = check(a); st != EPTQ_OK) return st;
    if (a.rows == 0) return EPTQ_OK;
    if (a.batch == 0) {
        const size_t bytes = static_cast<size_t>(a.rows) * a.n_heads * a.head_dim * 2;
        return a.clear_rest == 0 || cudaMemsetAsync(a.out, 0, bytes, static_cast<cudaStream_t>(stream)) == cudaSuccess ? EPTQ_OK : EPTQ_ERR_LAUNCH;
    }
    const AttentionPlan plan = plan_of(a);
    if (plan.may_cut && (workspace == nullptr || workspace_bytes < bytes_of(a, plan))) return EPTQ_ERR_WORKSPACE;
    if (plan.may_cut && (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return EPTQ_ERR_ALIGN;
    int dev = 0;
    if (attention_map_encoder() == nullptr || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return EPTQ_ERR_LAUNCH;
    AttentionArgs p = {};
    p.tables = a.tables; p.kv_lens = a.kv_lens; p.cu_rows = a.cu_rows;
    p.q = a.q; p.q_stride = a.q_stride;
    p.out = a.out; p.status = a.status;
    p.cut_tiles = plan.may_cut ? static_cast<CutTile*>(workspace) : nullptr;
    p.partial = plan.may_cut ? reinterpret_cast<float*>(static_cast<char*>(workspace) + cut_tile_bytes(plan)) : nullptr;
    p.tile_rows = plan.tile_rows;
    p.table_width = a.n_pages > 0 ? a.table_width : 0;           // no pages: no keys
    p.table_stride = a.table_stride;
    p.table_keys = static_cast<long long>(p.table_width) * a.page_size;
    p.rows = a.rows; p.batch = a.batch; p.n_heads = a.n_heads;
    p.kv_group = a.n_heads / a.n_kv_heads;
    p.page_size = a.page_size; p.n_pages = a.n_pages;
    // A scale of zero stays a step above it: masked scores are -infinity and must stay so.
    p.scale_log2 = a.scale == 0.f ? 1e-30f : (a.scale < 0.f ? -a.scale : a.scale) * kLog2e;
    p.negative = a.scale < 0.f;
    p.clear_rest = a.clear_rest != 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int status = on_tensor_cores(a) ? launch_attention_tcgen05(a, p, dev, st) : launch_attention_rows(a, p, dev, st);
    return status != EPTQ_OK || !plan.may_cut ? status : launch_join(a, plan, p, st);
}
