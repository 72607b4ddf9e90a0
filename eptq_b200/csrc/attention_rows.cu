// Causal attention of few rows over a paged cache, sm_100a: the single token of every running request, or a few of them.
//
// Every key and value is read once and meets at most 16 rows (the query heads of one key/value head times the request's
// tokens), so the kernel is bound by how fast the cache can be read; the products run on mma.sync (16 rows x 8 keys x 16),
// whose rate is far above what the reads can feed.  What counts is bytes in flight: each of a block's four warps works alone,
// on its own 16 keys (32 of head 64) of every block of keys, with its own ring of TMA stages (4 KB of keys and 4 KB of values
// each) that its own lanes refill; no warp waits for another before the end of a row tile, where the four results meet in
// shared memory.  Three blocks an SM cover each other's ends and starts (refilling on into the next tile, with shared memory
// of its own for the results, was 5 to 8 % slower).  Which keys a block takes: attention_schedule.cuh.
//
// Measured on one B200, replayed (join included), keys and values read by that time: 64 requests of 100 to 16000 keys, 32 over 8 heads
// of 128, 132 us (5.8 TB/s); the same over 32 heads 477 us (6.4 TB/s); 256 requests of 100 to 1000 keys 76 us (5.4 TB/s); one request
// of 907 keys 10.1 us, which is launch, share, page table, first reads and the join.

#include <mutex>

#include "attention_args.cuh"
#include "attention_host.cuh"
#include "pair16.cuh"

namespace eptq {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = 4;
constexpr int kRows = 16;
constexpr int kBlocksPerSm = 3;
constexpr int kStages = 2;
constexpr int kStageBytes = 8192;
constexpr int kBoxBytes = 16 * 128;                       // 16 keys x 64 columns
constexpr int kPad = 8;                                   // floats behind a row of results: rows begin in different banks
__host__ __device__ constexpr int unit_keys(int hd) { return 2048 / hd; }
__host__ __device__ constexpr int key_block(int hd) { return kWarps * unit_keys(hd); }
constexpr int kSmemBytes = kWarps * kStages * kStageBytes + 1024;

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    if constexpr (__is_same(T, __half))
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// o += w v over the unit's keys, with `limit` set over its first `keys` keys; with SOME only for the rows that are named (of g
// and of g + 8).
template <typename T, int HD, bool SOME>
__device__ __forceinline__ void product(float (&o)[HD / 8][4], const unsigned (&w)[unit_keys(HD) / 16][4], unsigned v_at, bool limit, int keys, bool lower, bool upper) {
    constexpr int kSub = unit_keys(HD) / 16, kCols = HD / 64;
    const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
    for (int b = 0; b < kSub; ++b) {
        unsigned keep0 = 0xffffffffu, keep1 = 0xffffffffu;
        if (limit) {
            const int live = keys - b * 16 - 2 * t;
            keep0 = live >= 2 ? 0xffffffffu : live == 1 ? 0xffffu : 0u;
            keep1 = live >= 10 ? 0xffffffffu : live == 9 ? 0xffffu : 0u;
        }
#pragma unroll
        for (int n = 0; n < HD / 16; ++n) {
            unsigned r[4];
            const int key = ((lane >> 3) & 1) * 8 + (lane & 7), chunk = (n & 3) * 2 + (lane >> 4);
            ldmatrix4_trans(r, v_at + (b * kCols + (n >> 2)) * kBoxBytes + key * 128 + ((chunk ^ (key & 7)) << 4));
            if (limit) { r[0] &= keep0; r[1] &= keep1; r[2] &= keep0; r[3] &= keep1; }
            if (SOME) {
                float x[4], y[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) { x[c] = o[2 * n][c]; y[c] = o[2 * n + 1][c]; }
                mma<T>(x, w[b], r[0], r[1]);
                mma<T>(y, w[b], r[2], r[3]);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c < 2 ? lower : upper) { o[2 * n][c] = x[c]; o[2 * n + 1][c] = y[c]; }
            } else {
                mma<T>(o[2 * n], w[b], r[0], r[1]);
                mma<T>(o[2 * n + 1], w[b], r[2], r[3]);
            }
        }
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
attention_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ AttentionArgs p, CutRule rule) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ __align__(8) unsigned long long full[kWarps][kStages];
    __shared__ ShareScratch<kThreads> share_scratch;
    __shared__ float2 stats[kWarps][kRows];                // reference and sum of a warp's rows
    __shared__ int stop;
    constexpr int kUnit = unit_keys(HD), kBlock = key_block(HD);
    constexpr int kSub = kUnit / 16, kCols = HD / 64;      // boxes of 16 keys, of 64 columns: two in all for keys, two for values
    constexpr int kPitch = HD + kPad;
    static_assert(kSub * kCols == 2 && kRows * kPitch * 4 <= kStages * kStageBytes, "stage layout");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    unsigned char* const ring = smem + ((1024u - (smem_u32(smem) & 1023u)) & 1023u) + warp * (kStages * kStageBytes);
    const unsigned ring_at = smem_u32(ring);
    const int tile_tokens = p.tokens_per_half;
    const int page_shift = 31 - __clz(p.page_size);

    if (tid == 0) {
        for (int w = 0; w < kWarps; ++w)
            for (int s = 0; s < kStages; ++s) mbar_init(smem_u32(&full[w][s]), 1);
        stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(&map_k)) : "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(&map_v)) : "memory");
    }
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Share share = find_share<kThreads, 4>(p, tile_tokens, kBlock, rule, share_scratch);
    bool cut_written = false;
    unsigned issued = 0, used = 0;                         // units of this warp's ring
    bool ok = true;

    ShareWalk walk;
    if (share.begin < share.end) walk.start(p, share); else walk.left = 0;
    for (;;) {
        Item it;
        if (!walk.next(p, tile_tokens, kBlock, rule, it)) break;
        if (it.of > 0 && tid == 0) {
            write_cut_tile(p, it);
            cut_written = true;
        }
        // this warp's units: the warp-th of every block whose first key exists
        const int unit0 = kWarps * it.block + warp;
        const int units = max(0, min(it.blocks, ((it.keys + kUnit - 1) / kUnit - unit0 + kWarps - 1) / kWarps));
        const int kv_head = it.head / p.kv_group;
        const int* const table = p.tables + it.request * p.table_stride;
        // lanes 0-3 each load one box of a unit: of keys or values, and which of the two
        const int sub = kSub == 2 ? lane & 1 : 0, col64 = kSub == 2 ? 0 : lane & 1;
        auto page_of = [&](int i) {                        // page of this lane's box of unit i
            const int key = (unit0 + i * kWarps) * kUnit + sub * 16;
            return lane < 4 && i < units && key < it.keys ? table[key >> page_shift] : 0;
        };
        unsigned lost = 0;                                 // two bits a stage: 16-key groups on no page of the cache
        auto load = [&](int i, int page) {
            const int s = issued % kStages, key = (unit0 + i * kWarps) * kUnit + sub * 16;
            const bool there = lane < 4 && key < it.keys;
            const bool gone = there && (page < 0 || page >= p.n_pages);
            const unsigned boxes = __ballot_sync(0xffffffffu, there), bad = __ballot_sync(0xffffffffu, gone) & 3u;
            lost = (lost & ~(3u << (2 * s))) | ((kSub == 2 ? bad : (bad & 1u)) << (2 * s));
            const unsigned bar = smem_u32(&full[warp][s]);
            if (lane == 0) mbar_arrive_expect_tx(bar, __popc(boxes) * kBoxBytes);
            __syncwarp();
            if (there)
                tma_4d(ring_at + s * kStageBytes + lane * kBoxBytes, lane < 2 ? &map_k : &map_v, col64 * 64, key & (p.page_size - 1), kv_head,
                       gone ? p.n_pages : page, bar);
            ++issued;
        };
        int page[kStages + 1];
#pragma unroll
        for (int i = 0; i <= kStages; ++i) page[i] = page_of(i);
#pragma unroll
        for (int i = 0; i < kStages; ++i)
            if (i < units) load(i, page[i]);
        int next_page = page[kStages];

        // q as the product's left operand, and what each of this thread's rows sees
        unsigned q[HD / 16][4];
        int seen[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = e * 8 + g, token = row / p.heads_per_tile;
            const bool live = row < p.heads_per_tile * tile_tokens && token < it.tokens;
            seen[e] = it.seen + min(token, it.tokens - 1);
            const uint16_t* const src = p.q + (it.row + token) * p.q_stride + (it.head + row % p.heads_per_tile) * HD + 2 * t;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    q[k][2 * c + e] = live ? *reinterpret_cast<const unsigned*>(src + k * 16 + c * 8) : 0u;
        }
        // Up to eight rows leave the tile's upper eight to the second parts of their weights (see below).
        const bool folded = p.heads_per_tile * min(it.tokens, tile_tokens) <= 8;
        if (folded) seen[1] = seen[0];
        float o[HD / 8][4], top[2], bias[2], sum[2];
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) { top[e] = -INFINITY; bias[e] = 0.f; sum[e] = 0.f; }

        for (int i = 0; i < units; ++i) {
            const int s = used % kStages;
            ok = warp_wait(smem_u32(&full[warp][s]), (used / kStages) & 1u, &stop);
            if (!ok) break;
            ++used;
            const unsigned k_at = ring_at + s * kStageBytes, v_at = k_at + kStageBytes / 2;
            const int key0 = (unit0 + i * kWarps) * kUnit;
            const unsigned gone = (lost >> (2 * s)) & 3u;
            float z[2 * kSub][4];
#pragma unroll
            for (int n = 0; n < 2 * kSub; ++n) z[n][0] = z[n][1] = z[n][2] = z[n][3] = 0.f;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
#pragma unroll
                for (int b = 0; b < kSub; ++b) {
                    unsigned r[4];
                    const int key = (lane >> 4) * 8 + (lane & 7), chunk = (k & 3) * 2 + ((lane >> 3) & 1);
                    ldmatrix4(r, k_at + (b * kCols + (k >> 2)) * kBoxBytes + key * 128 + ((chunk ^ (key & 7)) << 4));
                    mma<T>(z[2 * b], q[k], r[0], r[1]);
                    mma<T>(z[2 * b + 1], q[k], r[2], r[3]);
                }
            if (p.negative) {
#pragma unroll
                for (int n = 0; n < 2 * kSub; ++n)
#pragma unroll
                    for (int c = 0; c < 4; ++c) z[n][c] = -z[n][c];
            }
            if (it.seen + 1 - key0 < kUnit || gone != 0) {     // the first token sees the fewest keys
#pragma unroll
                for (int n = 0; n < 2 * kSub; ++n)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (key0 + n * 8 + 2 * t + (c & 1) > seen[c >> 1] || ((gone >> (n >> 1)) & 1u)) z[n][c] = -INFINITY;
            }
            float high[2];
            bool any = false;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float v = z[0][2 * e];
#pragma unroll
                for (int n = 0; n < 2 * kSub; ++n) v = fmaxf(v, fmaxf(z[n][2 * e], z[n][2 * e + 1]));
                high[e] = fmaxf(quad_max(v), top[e]);
                any |= top[e] == -INFINITY ? high[e] > -INFINITY : (high[e] - top[e]) * p.scale_log2 > kRescaleAt;
            }
            if (__any_sync(0xffffffffu, any)) {
                float lower = 1.f;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bool none = top[e] == -INFINITY;
                    const bool moves = none ? high[e] > -INFINITY : (high[e] - top[e]) * p.scale_log2 > kRescaleAt;
                    const float new_bias = moves ? high[e] * p.scale_log2 - kExpOffset : bias[e];
                    float keep = none ? 1.f : exp2_approx(bias[e] - new_bias);
                    if (e == 0) lower = keep; else if (folded) keep = lower;
                    top[e] = moves ? high[e] : top[e];
                    bias[e] = new_bias;
                    sum[e] *= keep;
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) { o[n][2 * e] *= keep; o[n][2 * e + 1] *= keep; }
                }
            }
            // A weight meets its value as the sum of two 16-bit values, which keeps 22 bits of it (16 where they are bf16).  The second
            // ones take a product of their own, or where the tile has no more than eight rows the upper rows of the first.
            unsigned w[kSub][4], rest[kSub][4] = {};
            if (folded) {
#pragma unroll
                for (int n = 0; n < 2 * kSub; ++n) {
                    const float a = exp2_approx(fmaf(z[n][0], p.scale_log2, -bias[0]));
                    const float b = exp2_approx(fmaf(z[n][1], p.scale_log2, -bias[0]));
                    sum[0] += a + b;
                    const uint2 both = Pair16<T>::split(a, b);
                    w[n >> 1][(n & 1) * 2] = both.x;
                    w[n >> 1][(n & 1) * 2 + 1] = both.y;
                }
            } else {
#pragma unroll
                for (int n = 0; n < 2 * kSub; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float a = exp2_approx(fmaf(z[n][2 * e], p.scale_log2, -bias[e]));
                        const float b = exp2_approx(fmaf(z[n][2 * e + 1], p.scale_log2, -bias[e]));
                        sum[e] += a + b;
                        const uint2 both = Pair16<T>::split(a, b);
                        w[n >> 1][(n & 1) * 2 + e] = both.x;
                        rest[n >> 1][(n & 1) * 2 + e] = both.y;
                    }
            }
            // Values behind the last key a row sees may be anything, and a weight of zero must make them zero: what lies
            // behind the last token's is cleared.  Where the tokens see different keys of this unit and a value is not finite,
            // every token's rows take their own product.
            const bool tail = it.keys - key0 < kUnit;
            bool apart = false;
            if (it.tokens > 1 && it.seen + 1 - key0 < kUnit) {
                unsigned acc = 0;                              // two zeros, or NaN where something was not finite
#pragma unroll
                for (int i = 0; i < kStageBytes / 2 / 512; ++i) {
                    const int at = i * 32 + lane, key = (at >> 7) % kSub * 16 + (at >> 3) % 16;        // 16-byte unit, its key
                    const uint4 u = *reinterpret_cast<const uint4*>(ring + s * kStageBytes + kStageBytes / 2 + at * 16);
                    if (key0 + key < it.keys) {
                        acc = Pair16<T>::zero_times(u.x, acc);
                        acc = Pair16<T>::zero_times(u.y, acc);
                        acc = Pair16<T>::zero_times(u.z, acc);
                        acc = Pair16<T>::zero_times(u.w, acc);
                    }
                }
                const float2 end = Pair16<T>::unpack(acc);
                apart = __any_sync(0xffffffffu, end.x != end.x || end.y != end.y);
            }
#pragma unroll 1
            for (int part = folded ? 1 : 0;; ++part) {              // a loop, not twice the code: short calls wait for their instructions
                if (!apart) {
                    product<T, HD, false>(o, w, v_at, tail, it.keys - key0, true, true);
                } else {
                    for (int token = 0; token < min(it.tokens, tile_tokens); ++token)
                        product<T, HD, true>(o, w, v_at, true, it.seen + token + 1 - key0, seen[0] == it.seen + token, seen[1] == it.seen + token);
                }
                if (part == 1) break;
#pragma unroll
                for (int b = 0; b < kSub; ++b)
#pragma unroll
                    for (int c = 0; c < 4; ++c) w[b][c] = rest[b][c];
            }
            __syncwarp();                                       // all lanes have read the stage
            if (i + kStages < units) {
                const int now = next_page;
                next_page = page_of(i + kStages + 1);
                load(i + kStages, now);
            }
        }

        // the four warps' results meet; each lies where its stages were
        if (ok) {
            float* const mine = reinterpret_cast<float*>(ring);
            if (folded) {
#pragma unroll
                for (int n = 0; n < HD / 8; ++n) { o[n][0] += o[n][2]; o[n][1] += o[n][3]; }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = e * 8 + g;
                const float all = quad_sum(sum[e]);
                if (t == 0) stats[warp][row] = make_float2(bias[e], all);
#pragma unroll
                for (int n = 0; n < HD / 8; ++n)
                    *reinterpret_cast<float2*>(mine + row * kPitch + n * 8 + 2 * t) = make_float2(o[n][2 * e], o[n][2 * e + 1]);
            }
        } else {
            stop = 1;
        }
        __syncthreads();
        ok = *static_cast<volatile int*>(&stop) == 0;
        if (!ok) break;
        const float* const rings = reinterpret_cast<const float*>(ring - warp * (kStages * kStageBytes));
        const int rows = p.heads_per_tile * min(it.tokens, tile_tokens);
        for (int x = tid; x < rows * (HD / 4); x += kThreads) {
            const int row = x / (HD / 4), col = x % (HD / 4) * 4;
            float2 st[kWarps];
            float high = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                st[w] = stats[w][row];
                if (st[w].y != 0.f) high = fmaxf(high, st[w].x);
            }
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float all = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                if (st[w].y == 0.f) continue;
                const float f = exp2_approx(st[w].x - high);
                const float4 y = *reinterpret_cast<const float4*>(rings + w * (kStages * kStageBytes / 4) + row * kPitch + col);
                all += st[w].y * f;
                v.x += y.x * f; v.y += y.y * f; v.z += y.z * f; v.w += y.w * f;
            }
            if (it.slot < 0) {
                const float inv = all == 0.f ? 0.f : 1.f / all;
                const int token = row / p.heads_per_tile;
                *reinterpret_cast<uint2*>(p.out + (static_cast<long long>(it.row + token) * p.n_heads + it.head + row % p.heads_per_tile) * HD + col) =
                    make_uint2(Pair16<T>::pack(v.x * inv, v.y * inv), Pair16<T>::pack(v.z * inv, v.w * inv));
            } else {
                float* const piece = p.partial + it.slot * piece_floats(kRows, HD);
                reinterpret_cast<float4*>(piece)[col / 4 * kRows + row] = v;
                if (col == 0) {
                    piece[kRows * HD + row] = all == 0.f ? 0.f : high;
                    piece[kRows * HD + kRows + row] = all;
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the stages are written by TMA again
        __syncthreads();
    }
    if (p.clear_rest) clear_rest<kThreads, HD>(p);
    if (tid == 0 && !cut_written && p.cut_tiles != nullptr) p.cut_tiles[blockIdx.x].of = 0;
    if (!ok) {
        // copies still in flight write shared memory: wait for them before it is given up
        volatile int never = 0;
        for (; used < issued; ++used) warp_wait(smem_u32(&full[warp][used % kStages]), (used / kStages) & 1u, &never);
        if (lane == 0 && p.status != nullptr) atomicExch(p.status, EPTQ_ERR_TIMEOUT);
    }
}

constexpr CutRule kRule = {4, 1, 1, 2};

template <typename T, int HD>
int run(const CUtensorMap& k, const CUtensorMap& v, const AttentionArgs& args, int dev, cudaStream_t stream) {
    static std::once_flag once[64];
    static bool set[64] = {};
    std::call_once(once[dev], [dev]() {
        set[dev] = cudaFuncSetAttribute(attention_rows_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) == cudaSuccess;
    });
    if (!set[dev]) return EPTQ_ERR_LAUNCH;
    return launch_dependent(attention_rows_kernel<T, HD>, dim3(kSms * kBlocksPerSm), kThreads, kSmemBytes, stream, k, v, args, kRule);
}

}  // namespace

AttentionPlan attention_rows_plan(const EptqAttention& a) {
    AttentionPlan plan;
    plan.shares = kSms * kBlocksPerSm;
    plan.tile_rows = kRows;
    plan.may_cut = static_cast<long long>(a.table_width) * a.page_size > static_cast<long long>(kRule.least) * key_block(a.head_dim);
    return plan;
}

int launch_attention_rows(const EptqAttention& a, AttentionArgs& p, int dev, cudaStream_t stream) {
    p.heads_per_tile = heads_in(p.kv_group, kRows);
    p.tokens_per_half = kRows / p.heads_per_tile;
    CUtensorMap k, v;
    if (!encode_page_maps(&k, &v, a, 16)) return EPTQ_ERR_LAUNCH;
    if (a.dtype == EPTQ_FP16) return a.head_dim == 128 ? run<__half, 128>(k, v, p, dev, stream) : run<__half, 64>(k, v, p, dev, stream);
    return a.head_dim == 128 ? run<__nv_bfloat16, 128>(k, v, p, dev, stream) : run<__nv_bfloat16, 64>(k, v, p, dev, stream);
}

}  // namespace eptq
