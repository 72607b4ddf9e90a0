// Causal attention of many rows on the tensor cores (tcgen05 + TMEM + TMA), sm_100a: packed prompts, and chunks of new
// tokens over a paged cache.
//
//   o = softmax(scale q k^T) v, one pass over the keys with the running maximum and sum of each row.
//
// Row tile: two halves of 128 rows.  The query heads that share a key/value head share the tile too (row = token * heads +
// head), so a block of keys is read once for all of them and few tokens fill the rows.  Blocks of 128 keys.
//
//   warp 0      walks this block's share of the work (attention_schedule.cuh), tells the others its items through a small
//               ring, loads Q once per item and K and V by TMA (128-byte swizzle) into a ring of 128-key slots.
//   warp 1      issues the tcgen05.mma: S = Q K^T (M 128, N 128) into TMEM, and O += P V with P read from TMEM where S was
//               and V from shared memory as it lies (keys along K, head columns contiguous).  S of one half is formed while
//               the other half's softmax runs.
//   warps 4-11  softmax, one thread per row and half: S from TMEM, maximum, exp2, P back to TMEM in 16 bits.
//
// Per 128 x 128 half-block the tensor core needs 1024 cycles (head 128) and the exponentials 1024 cycles of the SM's
// special-function units: the two bound the kernel together.  O is rescaled only when a row's maximum has grown by more
// than 2^8, by the softmax thread itself; P then stays below 2^15 because exponents carry an offset of 7, which also
// keeps small weights out of fp16's subnormal range.
//
// Keys behind a request's end are masked by index, whatever is stored there; their values would still meet a weight of
// zero, so the product ends with the last key (in steps of 16, the rest of the last step cleared in shared memory).
//
// TMEM: S/P of half 0 at column 0, of half 1 at 128; O of half 0 at 256, of half 1 at 256 + head_dim.

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "attention_args.cuh"
#include "pair16.cuh"

namespace eptq {
namespace {

constexpr int kThreads = 384;
constexpr int kItems = 4;                      // ring of items
constexpr int kMaxSlots = 10;
constexpr int kKeysSeen = 16;                  // ring of per-block page flags
constexpr unsigned long long kWaitNs = 2000000000ull;
constexpr float kExpOffset = 7.f;
constexpr float kRescaleAt = 8.f;

// Q: two halves of 128 rows; K and V: slots of 128 keys; each in head_dim / 64 boxes of 128-byte rows.
__host__ __device__ constexpr int tile_bytes(int hd) { return 128 * hd * 2; }
__host__ __device__ constexpr int slots(int hd) { return hd == 128 ? 5 : 10; }
__host__ __device__ constexpr int smem_bytes(int hd) { return (2 + slots(hd)) * tile_bytes(hd) + 1024; }
static_assert(slots(64) <= kMaxSlots && slots(128) <= kMaxSlots, "barrier array");

struct Item {
    int row, tokens, head, request;    // first row, tokens that exist, first query head; request < 0: no more items
    int seen;                          // last key that the first token sees
    int keys;                          // keys of the request that the tile's last token sees
    int block, blocks;                 // first block of keys, number of blocks
    int count[2];                      // blocks of either half
    int slot;                          // where its partial result goes, -1: it is the whole tile
    int pad;
};

__device__ __forceinline__ unsigned smem_u32(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(unsigned bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(unsigned bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(unsigned bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
// Bounded by the global timer; a wait that runs out raises `stop`, which ends the other warps' waits as well.
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, volatile int* stop) {
    unsigned long long t0 = 0;
    for (unsigned it = 0;; ++it) {
        unsigned done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
        if ((it & 255u) == 255u) {
            if (*stop) return false;
            unsigned long long now;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (t0 == 0) t0 = now;
            else if (now - t0 > kWaitNs) { *stop = 1; return false; }
        }
    }
}
// The same for a whole warp: all lanes agree on the outcome.
__device__ __forceinline__ bool warp_wait(unsigned bar, unsigned parity, volatile int* stop) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, stop));
}
__device__ __forceinline__ void commit(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Operand tiles in 128-byte swizzle, groups of 8 rows 1024 B apart.  K-major (Q, K): the leading offset is unused.
// MN-major (V: keys along K, 64 head columns in a row): the leading offset leads to the next 64 columns.
__device__ __forceinline__ uint64_t desc_sw128(unsigned addr, unsigned leading) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(leading >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}
// fp32 accumulate, 16-bit operands of one type, M 128.
__host__ __device__ constexpr uint32_t instr_desc(int n, bool bf16, bool b_mn_major, bool negate_a) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (negate_a ? 1u << 13 : 0u) | (b_mn_major ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_smem(unsigned d, uint64_t a, uint64_t b, uint32_t idesc, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_tmem(unsigned d, unsigned a, uint64_t b, uint32_t idesc, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld32(unsigned addr, float* v) {
    unsigned* r = reinterpret_cast<unsigned*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st32(unsigned addr, const unsigned* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        :: "r"(addr),
           "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
           "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
           "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
           "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tma_3d(unsigned dst, const CUtensorMap* map, int x, int y, int z, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_4d(unsigned dst, const CUtensorMap* map, int x, int y, int z, int w, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}

__device__ __forceinline__ Request load_request(const AttentionArgs& p, int b, bool paged) {
    return request_from(__ldg(p.cu_rows + b), __ldg(p.cu_rows + b + 1), p.rows, paged ? __ldg(p.kv_lens + b) : 0, p.table_keys, paged);
}

struct Shared {
    unsigned long long q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2], o_empty[2];
    unsigned long long kv_full[kMaxSlots], kv_empty[kMaxSlots], item_full[kItems], item_empty[kItems];
    Item items[kItems];
    long long scan[kThreads / 32 + 1];
    long long place_before[2];             // blocks before the request that holds the share's begin and end
    int place_request[2];
    unsigned lost[kKeysSeen];              // 16-key groups of a block that are on no page of the cache
    unsigned tmem;
    int stop;
};

template <typename T, int HD, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1)
attention_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttentionArgs p, const CutRule rule) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ Shared sh;
    constexpr int kBoxes = HD / 64;
    constexpr int kTile = tile_bytes(HD), kBox = 128 * 64 * 2, kSlots = slots(HD);
    constexpr bool kBf16 = sizeof(T) == 2 && !__is_same(T, __half);
    unsigned char* const tiles = smem + ((1024u - (smem_u32(smem) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int share_id = blockIdx.x, n_shares = gridDim.x;
    const int tile_tokens = 2 * p.tokens_per_half, groups = p.n_heads / p.heads_per_tile;

    if (tid == 0) {
        for (int h = 0; h < 2; ++h) {
            mbar_init(smem_u32(&sh.q_full[h]), 1);
            mbar_init(smem_u32(&sh.q_empty[h]), 1);
            mbar_init(smem_u32(&sh.s_full[h]), 1);
            mbar_init(smem_u32(&sh.p_full[h]), 4);
            mbar_init(smem_u32(&sh.o_full[h]), 1);
            mbar_init(smem_u32(&sh.o_empty[h]), 4);
        }
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(smem_u32(&sh.kv_full[s]), 1);
            mbar_init(smem_u32(&sh.kv_empty[s]), 1);
        }
        for (int s = 0; s < kItems; ++s) {
            mbar_init(smem_u32(&sh.item_full[s]), 1);
            mbar_init(smem_u32(&sh.item_empty[s]), 9);
        }
        sh.stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(&map_q)) : "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(&map_k)) : "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(&map_v)) : "memory");
    }
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---------------- this block's share: blocks of all requests summed, then the requests that hold its two ends
    long long all = 0, share = 0, mine[2] = {0, 0};
    for (int pass = 0; pass < 2; ++pass) {
        long long before = 0;
        for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
            const int b = b0 + tid;
            long long w = 0;
            if (b < p.batch) {
                const Request r = load_request(p, b, PAGED);
                w = blocks_before(r, tile_tokens, tiles_of(r, tile_tokens)) * groups;
            }
            long long ends = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long up = __shfl_up_sync(0xffffffffu, ends, o);
                if (lane >= o) ends += up;
            }
            __syncthreads();
            if (lane == 31) sh.scan[warp] = ends;
            __syncthreads();
            long long chunk = 0;
#pragma unroll
            for (int i = 0; i < kThreads / 32; ++i) {
                if (i == warp) ends += chunk;
                chunk += sh.scan[i];
            }
            ends += before;
            if (pass == 0 && b0 + kThreads >= p.batch) {          // the sum is known: this chunk may hold the ends already
                all = before + chunk;
                share = share_of(all, n_shares, rule);
                mine[0] = share_id * share;
                mine[1] = share_id + 1 < n_shares ? mine[0] + share : all;
            }
            if (pass == 1 || b0 + kThreads >= p.batch)
                for (int e = 0; e < 2; ++e)
                    if (mine[e] < ends && mine[e] >= ends - w) { sh.place_request[e] = b; sh.place_before[e] = ends - w; }
            before += chunk;
        }
        if (p.batch <= kThreads) break;                           // one chunk: both passes in one
    }
    __syncthreads();
    long long cut[2];
    Place at[2];
    int request0 = 0;
    for (int e = 0; e < 2; ++e) {                                  // every thread alike: the values are needed by all
        cut[e] = all;
        if (mine[e] < all) {
            const int b = sh.place_request[e];
            const Request r = load_request(p, b, PAGED);
            at[e] = place_of(r, tile_tokens, mine[e] - sh.place_before[e]);
            cut[e] = mine[e] + moved(at[e], rule);
            if (e == 0) request0 = b;
        }
    }
    if (cut[0] >= cut[1]) {                                        // nothing left for this block
        if (tid == 0 && p.cut_tiles != nullptr) p.cut_tiles[share_id].of = 0;
        return;
    }

    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&sh.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const unsigned tmem = sh.tmem;
    bool ok = true;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0) {
            // ---------------- items and loads
            int b = request0;
            Request r = load_request(p, b, PAGED);
            Place now = at[0];
            int step = moved(at[0], rule);
            if (step == now.blocks - now.block && step != 0) { now.block = 0; ++now.tile; } else now.block += step;
            long long left = cut[1] - cut[0], flat = cut[0];
            unsigned kv_seq = 0, n_items = 0, q_count[2] = {0, 0}, block_seq = 0;
            bool cut_written = false;
            for (;;) {
                // the next tile that exists
                int row_tiles = tiles_of(r, tile_tokens);
                if (now.tile >= row_tiles) { now.tile = 0; ++now.group; }
                while (left > 0 && (row_tiles == 0 || now.group >= groups)) {
                    r = load_request(p, ++b, PAGED);
                    row_tiles = tiles_of(r, tile_tokens);
                    now.group = now.tile = 0;
                }
                const int ring = n_items % kItems;
                ok = warp_wait(smem_u32(&sh.item_empty[ring]), ((n_items / kItems) & 1u) ^ 1u, &sh.stop);
                if (!ok) break;
                if (left <= 0) {
                    if (lane == 0) {
                        sh.items[ring].request = -1;
                        mbar_arrive(smem_u32(&sh.item_full[ring]));
                    }
                    break;
                }
                const int blocks = blocks_of(r, tile_tokens, now.tile);
                Item it;
                it.request = b;
                it.row = r.first + now.tile * tile_tokens;
                it.tokens = min(tile_tokens, r.n - now.tile * tile_tokens);
                it.head = now.group * p.heads_per_tile;
                it.seen = r.past + now.tile * tile_tokens;
                it.keys = max(0, it.seen + it.tokens);
                it.block = now.block;
                it.blocks = static_cast<int>(min(static_cast<long long>(blocks - now.block), left));
                // half 0 sees fewer keys than half 1; a half without tokens has no blocks
                const int keys0 = it.seen + min(it.tokens, p.tokens_per_half);
                const int need0 = keys0 <= kKeyBlock ? 1 : (keys0 + kKeyBlock - 1) / kKeyBlock;
                it.count[0] = max(0, min(it.blocks, need0 - it.block));
                it.count[1] = it.tokens > p.tokens_per_half ? it.blocks : 0;
                const bool whole = it.blocks == blocks;
                it.slot = whole ? -1 : 2 * share_id + (it.block == 0 ? 1 : 0);
                it.pad = 0;
                if (lane == 0) {
                    sh.items[ring] = it;
                    mbar_arrive(smem_u32(&sh.item_full[ring]));
                    if (!whole && it.block == 0) {
                        CutTile c;
                        c.of = last_share(flat + blocks, share, rule) - share_id + 1;
                        c.row = it.row; c.tokens = it.tokens; c.head = it.head;
                        c.pad[0] = c.pad[1] = c.pad[2] = c.pad[3] = 0;
                        p.cut_tiles[share_id] = c;
                        cut_written = true;
                    }
                }
                ++n_items;
                for (int h = 0; h < 2 && ok; ++h) {
                    if (it.count[h] == 0) continue;
                    ok = warp_wait(smem_u32(&sh.q_empty[h]), (q_count[h] & 1u) ^ 1u, &sh.stop);
                    if (!ok) break;
                    ++q_count[h];
                    if (lane == 0) {
                        const unsigned bar = smem_u32(&sh.q_full[h]);
                        mbar_arrive_expect_tx(bar, p.heads_per_tile * p.tokens_per_half * HD * 2);
                        for (int x = 0; x < kBoxes; ++x)
                            tma_3d(smem_u32(tiles + h * kTile + x * kBox), &map_q, x * 64, it.head, it.row + h * p.tokens_per_half, bar);
                    }
                }
                const int kv_head = it.head / p.kv_group;
                const int last_key = it.keys;
                int table_at = -1, page_id = 0;                    // table columns table_at .. table_at + 31, one per lane
                for (int j = 0; j < it.blocks && ok; ++j) {
                    const int key0 = (it.block + j) * kKeyBlock;
                    int pages = 0, page = 0;
                    unsigned lost = 0;
                    if (PAGED) {
                        // this block's pages: lane i holds page i
                        pages = (max(0, min(kKeyBlock, last_key - key0)) + p.page_size - 1) / p.page_size;
                        const int col = key0 / p.page_size;
                        if (table_at < 0 || col < table_at || col + pages > table_at + 32) {
                            table_at = col;
                            page_id = col + lane < p.table_width ? __ldg(p.tables + b * p.table_stride + col + lane) : -1;
                        }
                        page = __shfl_sync(0xffffffffu, page_id, (col - table_at + lane) & 31);
                        const bool gone = lane < pages && (page < 0 || page >= p.n_pages);
                        if (gone) page = p.n_pages;                // outside: reads as zeros
                        const unsigned bad = __ballot_sync(0xffffffffu, gone);
                        if (bad) {
                            const int per = p.page_size / 16;
                            for (int i = 0; i < 8; ++i)
                                if ((bad >> (i / per)) & 1u) lost |= 1u << i;
                        }
                        if (lane == 0) sh.lost[block_seq % kKeysSeen] = lost;
                        ++block_seq;
                    }
                    for (int kv = 0; kv < 2; ++kv, ++kv_seq) {
                        const int s = kv_seq % kSlots;
                        ok = warp_wait(smem_u32(&sh.kv_empty[s]), ((kv_seq / kSlots) & 1u) ^ 1u, &sh.stop);
                        if (!ok) break;
                        const unsigned bar = smem_u32(&sh.kv_full[s]);
                        const unsigned dst = smem_u32(tiles + (2 + s) * kTile);
                        const CUtensorMap* map = kv ? &map_v : &map_k;
                        if (PAGED) {
                            if (lane == 0) mbar_arrive_expect_tx(bar, pages * p.page_size * HD * 2);
                            __syncwarp();
                            if (lane < pages)
                                for (int x = 0; x < kBoxes; ++x)
                                    tma_4d(dst + x * kBox + lane * p.page_size * 128, map, x * 64, 0, kv_head, page, bar);
                        } else if (lane == 0) {
                            mbar_arrive_expect_tx(bar, kTile);
                            for (int x = 0; x < kBoxes; ++x)
                                tma_3d(dst + x * kBox, map, x * 64, kv_head, r.first + key0, bar);
                        }
                    }
                }
                if (!ok) break;
                left -= it.blocks;
                flat += it.blocks;
                now.block = 0;
                ++now.tile;
            }
            if (lane == 0 && !cut_written && p.cut_tiles != nullptr) p.cut_tiles[share_id].of = 0;
            if (!ok) {
                // copies still in flight write shared memory: wait for them before it is given up
                __syncwarp();
                volatile int never = 0;
                for (int h = 0; h < 2; ++h)
                    if (q_count[h] > 0) mbar_wait(smem_u32(&sh.q_full[h]), (q_count[h] - 1) & 1u, &never);
                for (unsigned i = kv_seq > kSlots ? kv_seq - kSlots : 0; i < kv_seq; ++i)
                    mbar_wait(smem_u32(&sh.kv_full[i % kSlots]), (i / kSlots) & 1u, &never);
            }
        } else if (warp == 1) {
            // ---------------- MMA
            const uint32_t qk = instr_desc(kKeyBlock, kBf16, false, p.negative != 0);
            const uint32_t pv = instr_desc(HD, kBf16, true, false);
            unsigned kv_seq = 0, n_items = 0, q_count[2] = {0, 0}, p_count[2] = {0, 0}, o_count[2] = {0, 0};
            while (ok) {
                const int ring = n_items % kItems;
                ok = warp_wait(smem_u32(&sh.item_full[ring]), (n_items / kItems) & 1u, &sh.stop);
                if (!ok) break;
                const int request = sh.items[ring].request, blocks = sh.items[ring].blocks;
                const int count[2] = {sh.items[ring].count[0], sh.items[ring].count[1]};
                const int keys = sh.items[ring].keys - sh.items[ring].block * kKeyBlock;
                if (request < 0) break;
                ++n_items;
                for (int j = 0; j <= blocks && ok; ++j) {
                    const unsigned k_seq = kv_seq + 2 * j, v_seq = kv_seq + 2 * j - 1;
                    const int k_slot = k_seq % kSlots, v_slot = v_seq % kSlots;
                    bool k_here = false, v_here = false;
                    for (int h = 0; h < 2 && ok; ++h) {
                        const unsigned s_at = tmem + h * 128, o_at = tmem + 256 + h * HD;
                        if (j > 0 && j - 1 < count[h]) {
                            const int live = min(kKeyBlock, max(0, keys - (j - 1) * kKeyBlock));
                            if (!v_here) {
                                ok = warp_wait(smem_u32(&sh.kv_full[v_slot]), (v_seq / kSlots) & 1u, &sh.stop);
                                if (!ok) break;
                                v_here = true;
                                if (live & 15) {                  // clear the rest of the last 16 keys
                                    const int gone = 16 - (live & 15);
                                    unsigned char* const v = tiles + (2 + v_slot) * kTile + live * 128;
                                    for (int i = lane; i < gone * 8 * kBoxes; i += 32)
                                        *reinterpret_cast<uint4*>(v + (i / (gone * 8)) * kBox + (i % (gone * 8)) * 16) = make_uint4(0, 0, 0, 0);
                                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                                    __syncwarp();
                                }
                            }
                            if (j == 1) {                         // the last item's O has been read
                                ok = warp_wait(smem_u32(&sh.o_empty[h]), (o_count[h] & 1u) ^ 1u, &sh.stop);
                                if (!ok) break;
                                ++o_count[h];
                            }
                            ok = warp_wait(smem_u32(&sh.p_full[h]), p_count[h] & 1u, &sh.stop);
                            if (!ok) break;
                            ++p_count[h];
                            fence_after();
                            if (lane == 0) {
                                const uint64_t dv = desc_sw128(smem_u32(tiles + (2 + v_slot) * kTile), kBox);
                                const int steps = (live + 15) >> 4;
                                for (int k = 0; k < steps; ++k)
                                    mma_tmem(o_at, s_at + k * 8, dv + static_cast<uint64_t>((k * 2048) >> 4), pv, j > 1 || k > 0);
                                if (j == count[h]) commit(smem_u32(&sh.o_full[h]));
                            }
                            __syncwarp();
                        }
                        if (j < count[h]) {
                            if (!k_here) {
                                ok = warp_wait(smem_u32(&sh.kv_full[k_slot]), (k_seq / kSlots) & 1u, &sh.stop);
                                if (!ok) break;
                                k_here = true;
                            }
                            if (j == 0) {
                                ok = warp_wait(smem_u32(&sh.q_full[h]), q_count[h] & 1u, &sh.stop);
                                if (!ok) break;
                                ++q_count[h];
                            }
                            fence_after();
                            if (lane == 0) {
                                for (int x = 0; x < kBoxes; ++x) {
                                    const uint64_t dq = desc_sw128(smem_u32(tiles + h * kTile + x * kBox), 16);
                                    const uint64_t dk = desc_sw128(smem_u32(tiles + (2 + k_slot) * kTile + x * kBox), 16);
#pragma unroll
                                    for (int k = 0; k < 4; ++k)
                                        mma_smem(s_at, dq + static_cast<uint64_t>((k * 32) >> 4), dk + static_cast<uint64_t>((k * 32) >> 4), qk, x > 0 || k > 0);
                                }
                                commit(smem_u32(&sh.s_full[h]));
                                if (j == count[h] - 1) commit(smem_u32(&sh.q_empty[h]));
                            }
                            __syncwarp();
                        }
                    }
                    if (!ok) break;
                    if (lane == 0) {
                        if (j > 0) commit(smem_u32(&sh.kv_empty[v_slot]));
                        if (j < blocks) commit(smem_u32(&sh.kv_empty[k_slot]));
                    }
                    __syncwarp();
                }
                kv_seq += 2 * blocks;
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.item_empty[ring]));
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        // ---------------- softmax: thread = row of half h
        const int h = (warp - 4) >> 2;
        const int row = (warp & 3) * 32 + lane;
        const unsigned lanes = static_cast<unsigned>((warp & 3) * 32) << 16;
        const unsigned s_at = tmem + lanes + h * 128, o_at = tmem + lanes + 256 + h * HD;
        const int token = h * p.tokens_per_half + row / p.heads_per_tile, head = row % p.heads_per_tile;
        const bool in_tile = row < p.heads_per_tile * p.tokens_per_half;
        unsigned n_items = 0, s_count = 0, o_count = 0, block_seq = 0;
        while (ok) {
            const int ring = n_items % kItems;
            ok = warp_wait(smem_u32(&sh.item_full[ring]), (n_items / kItems) & 1u, &sh.stop);
            if (!ok) break;
            const Item it = sh.items[ring];
            if (it.request < 0) break;
            ++n_items;
            const int count = it.count[h];
            const bool live_row = in_tile && token < it.tokens;
            const int seen = it.seen + min(token, it.tokens - 1);              // the last key this row sees
            float top = -INFINITY, bias = 0.f, sum = 0.f;                       // maximum of s; exponent = s * scale - bias
            for (int j = 0; j < count && ok; ++j) {
                ok = warp_wait(smem_u32(&sh.s_full[h]), s_count & 1u, &sh.stop);
                if (!ok) break;
                ++s_count;
                fence_after();
                float s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(s_at + c * 32, s + c * 32);
                tmem_wait_ld();
                const int key0 = (it.block + j) * kKeyBlock;
                const int allowed = seen + 1 - key0;
                const unsigned lost = PAGED ? sh.lost[(block_seq + j) % kKeysSeen] : 0u;
                if (__any_sync(0xffffffffu, allowed < kKeyBlock) || (PAGED && lost != 0)) {
#pragma unroll
                    for (int i = 0; i < 128; ++i)
                        if (i >= allowed || (PAGED && ((lost >> (i / 16)) & 1u))) s[i] = -INFINITY;
                }
                float m = top;
#pragma unroll
                for (int i = 0; i < 128; ++i) m = fmaxf(m, s[i]);
                // The exponents' reference moves only when it has to: on the first block that has keys, or by more than 2^8.
                const bool first = top == -INFINITY;
                const bool moves = first ? m > -INFINITY : (m - top) * p.scale_log2 > kRescaleAt;
                if (__any_sync(0xffffffffu, moves)) {
                    const float new_bias = moves ? m * p.scale_log2 - kExpOffset : bias;
                    const float keep = first ? 1.f : exp2_approx(bias - new_bias);
                    top = moves ? m : top;
                    bias = new_bias;
                    sum *= keep;
                    if (j > 0) {
#pragma unroll 1
                        for (int c = 0; c < HD / 32; ++c) {
                            float o[32];
                            tmem_ld32(o_at + c * 32, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] *= keep;
                            tmem_st32(o_at + c * 32, reinterpret_cast<const unsigned*>(o));
                        }
                    }
                }
                float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    unsigned w[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float a = exp2_approx(fmaf(s[c * 64 + 2 * i], p.scale_log2, -bias));
                        const float b = exp2_approx(fmaf(s[c * 64 + 2 * i + 1], p.scale_log2, -bias));
                        part[(2 * i) & 3] += a;
                        part[(2 * i + 1) & 3] += b;
                        w[i] = Pair16<T>::pack(a, b);
                    }
                    tmem_st32(s_at + c * 32, w);
                }
                sum += (part[0] + part[1]) + (part[2] + part[3]);
                tmem_wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[h]));
            }
            block_seq += it.blocks;
            if (!ok) break;
            if (count > 0) {
                ok = warp_wait(smem_u32(&sh.o_full[h]), o_count & 1u, &sh.stop);
                if (!ok) break;
                ++o_count;
                fence_after();
            }
            if (it.slot < 0) {
                if (count > 0) {
                    const float inv = sum > 0.f ? 1.f / sum : 0.f;
                    uint16_t* const dst = p.out + (static_cast<long long>(it.row + token) * p.n_heads + it.head + head) * HD;
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        float o[32];
                        tmem_ld32(o_at + c * 32, o);
                        tmem_wait_ld();
                        if (!live_row) continue;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint4 v;
                            unsigned* const w = reinterpret_cast<unsigned*>(&v);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float a = o[i * 8 + 2 * e], b = o[i * 8 + 2 * e + 1];
                                w[e] = sum == 0.f ? 0u : Pair16<T>::pack(a * inv, b * inv);
                            }
                            *reinterpret_cast<uint4*>(dst + c * 32 + i * 8) = v;
                        }
                    }
                }
            } else if (it.tokens > h * p.tokens_per_half) {
                float* const piece = p.partial + static_cast<long long>(it.slot) * (256 * (HD + 2));
                const int at_row = h * 128 + row;
                piece[256 * HD + at_row] = count > 0 ? bias : 0.f;
                piece[256 * HD + 256 + at_row] = count > 0 ? sum : 0.f;
                if (count > 0) {
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        float o[32];
                        tmem_ld32(o_at + c * 32, o);
                        tmem_wait_ld();
                        if (!live_row) continue;
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            reinterpret_cast<float4*>(piece)[(c * 8 + i) * 256 + at_row] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) {
                if (count > 0) mbar_arrive(smem_u32(&sh.o_empty[h]));
                mbar_arrive(smem_u32(&sh.item_empty[ring]));
            }
        }
    }
    if (!ok) {
        sh.stop = 1;
        if (lane == 0 && p.status != nullptr) atomicExch(p.status, EPTQ_ERR_TIMEOUT);
    }
    fence_before();
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512) : "memory");
}

// ---- joining the pieces of cut tiles -------------------------------------------------------------------
// Block (share, 32 rows of its cut tile), one warp per quarter of the head.  Pieces are added in the order of the keys.
template <typename T, int HD>
__global__ void __launch_bounds__(128) attention_join_kernel(const __grid_constant__ AttentionArgs p) {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const CutTile c = p.cut_tiles[blockIdx.x];
    if (c.of == 0) return;
    const int at_row = blockIdx.y * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
    const int h = at_row >> 7, row = at_row & 127;
    const int token = h * p.tokens_per_half + row / p.heads_per_tile, head = row % p.heads_per_tile;
    if (row >= p.heads_per_tile * p.tokens_per_half || token >= c.tokens) return;
    constexpr int kVec = HD / 16;                                     // float4 of a quarter
    constexpr long long kPiece = 256 * (HD + 2);
    float top = -INFINITY;
    for (int i = 0; i < c.of; ++i) {
        const float* piece = p.partial + (2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * kPiece + 256 * HD + at_row;
        if (__ldcg(piece + 256) > 0.f) top = fmaxf(top, __ldcg(piece));
    }
    float4 o[kVec];
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < kVec; ++v) o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < c.of; ++i) {
        const float* piece = p.partial + (2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * kPiece;
        const float s = __ldcg(piece + 256 * HD + 256 + at_row);
        if (s == 0.f) continue;                                       // no key seen: its o was not written
        const float w = exp2_approx(__ldcg(piece + 256 * HD + at_row) - top);
        sum += s * w;
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(piece) + (part * kVec + v) * 256 + at_row);
            o[v].x += x.x * w; o[v].y += x.y * w; o[v].z += x.z * w; o[v].w += x.w * w;
        }
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    uint16_t* const dst = p.out + (static_cast<long long>(c.row + token) * p.n_heads + c.head + head) * HD + part * (HD / 4);
#pragma unroll
    for (int v = 0; v < kVec; v += 2) {
        uint4 w;
        w.x = Pair16<T>::pack(o[v].x * inv, o[v].y * inv);
        w.y = Pair16<T>::pack(o[v].z * inv, o[v].w * inv);
        w.z = Pair16<T>::pack(o[v + 1].x * inv, o[v + 1].y * inv);
        w.w = Pair16<T>::pack(o[v + 1].z * inv, o[v + 1].w * inv);
        *reinterpret_cast<uint4*>(dst + v * 4) = w;
    }
}

PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
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

// Boxes of 64 columns in 128-byte swizzle; what lies outside reads as zeros.  strides[i] in elements, of dims[i + 1].
bool encode(CUtensorMap* map, const EptqAttention& a, const void* base, int rank, const cuuint64_t* dims, const int64_t* strides, const cuuint32_t* box) {
    cuuint64_t bytes[4];
    const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
    for (int i = 0; i + 1 < rank; ++i) bytes[i] = static_cast<cuuint64_t>(strides[i]) * 2;
    return map_encoder()(map, a.dtype == EPTQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                         const_cast<void*>(base), dims, bytes, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr CutRule kRule = {8, 2, 4};
constexpr size_t kCutTileBytes = (kSms * sizeof(CutTile) + 255) / 256 * 256;

size_t piece_bytes(int hd) { return static_cast<size_t>(256) * (hd + 2) * sizeof(float); }

// Whether any tile may have more blocks than stay uncut, by what the host knows.
bool may_cut(const EptqAttention& a) {
    const long long keys = a.page_size != 0 ? static_cast<long long>(a.table_width) * a.page_size : a.rows;
    return keys > static_cast<long long>(kRule.least) * kKeyBlock;
}

template <typename Args0, typename... Args>
int launch(void (*kernel)(Args0, Args...), dim3 grid, int threads, int smem, cudaStream_t stream, const Args0& a0, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, a0, args...) != cudaSuccess) {
        cudaGetLastError();
        return EPTQ_ERR_LAUNCH;
    }
    return EPTQ_OK;
}

template <typename T, int HD, bool PAGED>
int run(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const AttentionArgs& args, bool join, int dev, cudaStream_t stream) {
    static std::once_flag once[64];
    static bool set[64] = {};
    std::call_once(once[dev], [dev]() {
        set[dev] = cudaFuncSetAttribute(attention_tcgen05_kernel<T, HD, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(HD)) == cudaSuccess;
    });
    if (!set[dev]) return EPTQ_ERR_LAUNCH;
    int st = launch(attention_tcgen05_kernel<T, HD, PAGED>, dim3(kSms), kThreads, smem_bytes(HD), stream, q, k, v, args, kRule);
    if (st != EPTQ_OK) return st;
    count_launch(EPTQ_KERNEL_OTHER);
    if (!join) return EPTQ_OK;
    st = launch(attention_join_kernel<T, HD>, dim3(kSms, 8), 128, 0, stream, args);
    if (st == EPTQ_OK) count_launch(EPTQ_KERNEL_OTHER);
    return st;
}

}  // namespace

size_t attention_tcgen05_bytes(const EptqAttention& a) {
    return may_cut(a) ? kCutTileBytes + 2 * kSms * piece_bytes(a.head_dim) : 0;
}

// Needs keys to exist as memory: a paged call with at least one page.
int launch_attention_tcgen05(const EptqAttention& a, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    if (map_encoder() == nullptr) return EPTQ_ERR_LAUNCH;
    const bool paged = a.page_size != 0, join = may_cut(a);
    if (join && (workspace == nullptr || workspace_bytes < attention_tcgen05_bytes(a))) return EPTQ_ERR_WORKSPACE;
    if (join && (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return EPTQ_ERR_ALIGN;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return EPTQ_ERR_LAUNCH;
    AttentionArgs p = {};
    p.tables = a.tables; p.kv_lens = a.kv_lens; p.cu_rows = a.cu_rows;
    p.out = a.out; p.status = a.status;
    p.cut_tiles = join ? static_cast<CutTile*>(workspace) : nullptr;
    p.partial = join ? reinterpret_cast<float*>(static_cast<char*>(workspace) + kCutTileBytes) : nullptr;
    p.table_stride = a.table_stride;
    p.table_keys = static_cast<long long>(a.table_width) * a.page_size;
    p.rows = a.rows; p.batch = a.batch; p.n_heads = a.n_heads;
    p.kv_group = a.n_heads / a.n_kv_heads;
    p.heads_per_tile = p.kv_group;                       // all heads of a key/value head, or as many of them as fit 128 rows
    while (p.heads_per_tile > 128 || p.kv_group % p.heads_per_tile != 0) --p.heads_per_tile;
    p.tokens_per_half = 128 / p.heads_per_tile;
    p.page_size = a.page_size; p.n_pages = a.n_pages; p.table_width = a.table_width;
    // A scale of zero stays the smallest step above it: masked scores are -infinity and must stay so.
    p.scale_log2 = a.scale == 0.f ? 1e-30f : (a.scale < 0.f ? -a.scale : a.scale) * kLog2e;
    p.negative = a.scale < 0.f;
    CUtensorMap q, k, v;
    const cuuint64_t hd = a.head_dim, nkv = a.n_kv_heads;
    {
        const cuuint64_t dims[3] = {hd, static_cast<cuuint64_t>(a.n_heads), static_cast<cuuint64_t>(a.rows)};
        const int64_t strides[2] = {a.head_dim, a.q_stride};
        const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(p.heads_per_tile), static_cast<cuuint32_t>(p.tokens_per_half)};
        if (!encode(&q, a, a.q, 3, dims, strides, box)) return EPTQ_ERR_LAUNCH;
    }
    bool ok;
    if (paged) {
        const cuuint64_t dims[4] = {hd, static_cast<cuuint64_t>(a.page_size), nkv, static_cast<cuuint64_t>(a.n_pages)};
        const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(a.page_size), 1, 1};
        const int64_t ks[3] = {a.head_dim, static_cast<int64_t>(a.page_size) * a.head_dim, a.k_stride};
        const int64_t vs[3] = {a.head_dim, static_cast<int64_t>(a.page_size) * a.head_dim, a.v_stride};
        ok = encode(&k, a, a.k, 4, dims, ks, box) && encode(&v, a, a.v, 4, dims, vs, box);
    } else {
        const cuuint64_t dims[3] = {hd, nkv, static_cast<cuuint64_t>(a.rows)};
        const cuuint32_t box[3] = {64, 1, kKeyBlock};
        const int64_t ks[2] = {a.head_dim, a.k_stride}, vs[2] = {a.head_dim, a.v_stride};
        ok = encode(&k, a, a.k, 3, dims, ks, box) && encode(&v, a, a.v, 3, dims, vs, box);
    }
    if (!ok) return EPTQ_ERR_LAUNCH;
    if (a.dtype == EPTQ_FP16) {
        if (a.head_dim == 128) return paged ? run<__half, 128, true>(q, k, v, p, join, dev, stream) : run<__half, 128, false>(q, k, v, p, join, dev, stream);
        return paged ? run<__half, 64, true>(q, k, v, p, join, dev, stream) : run<__half, 64, false>(q, k, v, p, join, dev, stream);
    }
    if (a.head_dim == 128) return paged ? run<__nv_bfloat16, 128, true>(q, k, v, p, join, dev, stream) : run<__nv_bfloat16, 128, false>(q, k, v, p, join, dev, stream);
    return paged ? run<__nv_bfloat16, 64, true>(q, k, v, p, join, dev, stream) : run<__nv_bfloat16, 64, false>(q, k, v, p, join, dev, stream);
}

}  // namespace eptq
