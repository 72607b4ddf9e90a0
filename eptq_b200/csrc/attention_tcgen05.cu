// Causal attention of many rows on the tensor cores (tcgen05 + TMEM + TMA), sm_100a: packed prompts, and chunks of new
// tokens over a paged cache.
//
//   o = softmax(scale q k^T) v, one pass over the keys with the running maximum and sum of each row.
//
// Row tile: two halves of 128 rows.  The query heads that share a key/value head share the tile too (row = token * heads +
// head), so a block of keys is read once for all of them and few tokens fill the rows.  Blocks of 128 keys.
//
//   warp 0      walks this block's share of the work (attention_schedule.cuh), tells the others its items through a small
//               ring, loads Q once per item and K by TMA (128-byte swizzle) into a ring of 128-key slots; warp 2 loads V.
//   warp 1      issues the tcgen05.mma: S = Q K^T (M 128, N 128) into TMEM, and O += P V with P read from TMEM where S was
//               and V from shared memory as it lies (keys along K, head columns contiguous).  S of one half is formed while
//               the other half's softmax runs.
//   warps 4-11  softmax, one thread per row and half: S from TMEM, maximum, exp2, P back to TMEM in 16 bits.
//
// Per 128 x 128 half-block (head 128) the tensor cores need 1024 cycles and the exponentials 1024 cycles of the SM's
// special-function units.  What bounds the kernel is the chain of one half: 2100 cycles of softmax, one warp's instructions one
// after the other, then 1200 until the next scores are there; two halves in turn keep the tensor cores busy 60 % of the time.
// O is rescaled only when a row's maximum has grown by more than 2^8, by the softmax thread itself; P then stays below
// 2^15 because exponents carry an offset of 7, which also keeps small weights out of fp16's subnormal range.
//
// Measured on one B200, calls back to back: prompt of 16384 tokens, 32 over 8 heads of 128, 1.73 ms (1270 TFLOP/s); 1024 tokens 26 us.
// Replayed: 8191 tokens, 32 heads, bf16, 510 us (1080 TFLOP/s); 509 rows of 64 over 8 heads on 24001 keys 377 us (1070 TFLOP/s); over
// seconds, under the power cap, 590 and 438 us.
//
// Keys behind a request's end are masked by index, whatever is stored there; their values would still meet a weight of
// zero, so the product ends with the last key (in steps of 16, the rest of the last step cleared in shared memory).  Where a
// block holds keys that some of its rows do not see, its values are looked at: if one is not finite, the softmax threads form
// that block's product themselves, each row over the keys it sees.
//
// TMEM: S/P of half 0 at column 0, of half 1 at 128; O of half 0 at 256, of half 1 at 256 + head_dim.

#include <mutex>
#include <type_traits>

#include "attention_args.cuh"
#include "attention_host.cuh"
#include "pair16.cuh"

namespace eptq {
namespace {

constexpr int kThreads = 384;
constexpr int kKeyBlock = 128;
constexpr int kItems = 4;                      // ring of items
constexpr int kMaxSlots = 5;
constexpr int kKeysSeen = 16;                  // ring of per-block page flags

// Q: two halves of 128 rows; K and V: rings of slots of 128 keys; each in head_dim / 64 boxes of 128-byte rows.
__host__ __device__ constexpr int tile_bytes(int hd) { return 128 * hd * 2; }
__host__ __device__ constexpr int k_slots(int hd) { return hd == 128 ? 3 : 5; }
__host__ __device__ constexpr int v_slots(int hd) { return hd == 128 ? 2 : 5; }
__host__ __device__ constexpr int smem_bytes(int hd) { return (2 + k_slots(hd) + v_slots(hd)) * tile_bytes(hd) + 1024; }

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
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "add.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// The lane whose bit BIT is clear gives b and gets the other's a for it, the other the other way round.
template <int BIT>
__device__ __forceinline__ void swap_units(uint4& a, uint4& b, int lane) {
    const bool upper = lane & BIT;
    uint4 give = upper ? a : b;
    give.x = __shfl_xor_sync(0xffffffffu, give.x, BIT);
    give.y = __shfl_xor_sync(0xffffffffu, give.y, BIT);
    give.z = __shfl_xor_sync(0xffffffffu, give.z, BIT);
    give.w = __shfl_xor_sync(0xffffffffu, give.w, BIT);
    if (upper) a = give; else b = give;
}

// Whether a half whose first row sees the keys up to `seen` does not see all of the block that begins with key0.
__device__ __forceinline__ bool is_edge(int seen, int key0) { return seen + 1 - key0 < kKeyBlock; }

// Whether any of the first `keys` rows of a slot of V holds an infinity or a NaN (0 x value is then a NaN): one warp's part of
// what the 128 threads of a half look at.
template <typename T, int HD>
__device__ __forceinline__ bool any_not_finite(const unsigned char* v, int keys, int row) {
    unsigned acc = 0;                                           // two zeros, or NaN where something was not finite
#pragma unroll
    for (int x = 0; x < HD / 64; ++x)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = i * 128 + row;                       // 16-byte unit of the box, 8 to a key
            if (at >> 3 >= keys) continue;
            const uint4 u = *reinterpret_cast<const uint4*>(v + x * (128 * 128) + at * 16);
            acc = Pair16<T>::zero_times(u.x, acc);
            acc = Pair16<T>::zero_times(u.y, acc);
            acc = Pair16<T>::zero_times(u.z, acc);
            acc = Pair16<T>::zero_times(u.w, acc);
        }
    const float2 end = Pair16<T>::unpack(acc);
    return __any_sync(0xffffffffu, end.x != end.x || end.y != end.y);
}

// o += sum of p_k v_k over the first `keys` keys of a slot of V, by the row's own thread, p read back from tensor memory (o starts
// anew if `fresh`).  Inline and without an array that is indexed at run time: a call, or a stack, in the kernel cost the
// blocks that do not come here 10 %.
template <typename T, int HD>
__device__ __forceinline__ void product_by_hand(unsigned o_at, unsigned p_at, const unsigned char* v, int keys, bool fresh) {
#pragma unroll 1
    for (int c = 0; c < HD / 32; ++c) {
        float o[32];
        tmem_ld32(o_at + c * 32, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = fresh ? 0.f : o[i];
#pragma unroll 1
        for (int k = 0; k < kKeyBlock; ++k) {
            unsigned w2;
            asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(w2) : "r"(p_at + (k >> 1)) : "memory");
            tmem_wait_ld();
            const float2 both = Pair16<T>::unpack(w2);
            const float w = k & 1 ? both.y : both.x;
            const unsigned char* const at = v + (c >> 1) * (128 * 128) + k * 128;
            if (k < keys) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 u = *reinterpret_cast<const uint4*>(at + ((((c & 1) * 4 + i) ^ (k & 7)) << 4));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = Pair16<T>::unpack(e == 0 ? u.x : e == 1 ? u.y : e == 2 ? u.z : u.w);
                        o[i * 8 + 2 * e] = fmaf(w, f.x, o[i * 8 + 2 * e]);
                        o[i * 8 + 2 * e + 1] = fmaf(w, f.y, o[i * 8 + 2 * e + 1]);
                    }
                }
            }
            __syncwarp();
        }
        tmem_st32(o_at + c * 32, reinterpret_cast<const unsigned*>(o));
    }
    tmem_wait_st();
}

// An item and the blocks of keys that either half of its rows sees.
struct HalvedItem {
    Item it;
    int count[2];
    int first;                             // the request's first row
};

// The page table's columns column .. column + 31 of one request, one per lane.
struct PageRow {
    int column, id;

    // Pages of `keys` keys from key0 on: their number, and in lane i the i-th one's id (n_pages where it is outside the cache,
    // which reads as zeros).
    __device__ __forceinline__ int fetch(const AttentionArgs& p, int request, int key0, int keys, int lane, int& page) {
        const int shift = 31 - __clz(p.page_size), at = key0 >> shift, n = (max(0, keys) + p.page_size - 1) >> shift;
        if (column < 0 || at + n > column + 32) {
            column = at;
            id = at + lane < p.table_width ? p.tables[request * p.table_stride + at + lane] : -1;
        }
        page = __shfl_sync(0xffffffffu, id, (at - column + lane) & 31);
        if (page < 0 || page >= p.n_pages) page = p.n_pages;
        return n;
    }
};

// One block of keys or values into a slot, by a whole warp.
template <int HD, bool PAGED>
__device__ __forceinline__ void load_keys(const AttentionArgs& p, const CUtensorMap* map, unsigned dst, unsigned bar, int row, int head, int n_pages, int page) {
    constexpr int kBoxBytes = 128 * 64 * 2;
    if (PAGED) {
        if (elect_one()) mbar_arrive_expect_tx(bar, n_pages * p.page_size * HD * 2);
        for (int i = 0; i < n_pages; ++i) {
            const int id = __shfl_sync(0xffffffffu, page, i);
            if (elect_one()) {
#pragma unroll
                for (int x = 0; x < HD / 64; ++x) tma_4d(dst + x * kBoxBytes + i * p.page_size * 128, map, x * 64, 0, head, id, bar);
            }
        }
    } else if (elect_one()) {
        mbar_arrive_expect_tx(bar, tile_bytes(HD));
#pragma unroll
        for (int x = 0; x < HD / 64; ++x) tma_3d(dst + x * kBoxBytes, map, x * 64, head, row, bar);
    }
    __syncwarp();
}

struct Shared {
    unsigned long long q_full[2], q_empty[2], s_full[2], p_full[2][2], o_full[2], o_empty[2];
    unsigned long long k_full[kMaxSlots], k_empty[kMaxSlots], v_full[kMaxSlots], v_empty[kMaxSlots], item_full[kItems], item_empty[kItems];
    HalvedItem items[kItems];
    ShareScratch<kThreads> share;
    unsigned long long voted[2];
    int votes[2][4];                       // ring: a half's block holds a value that is not finite
    int by_hand[2];                        // the block's product was formed by the softmax threads
    unsigned lost[kKeysSeen];              // 16-key groups of a block that are on no page of the cache
    unsigned tmem;
    int stop;
    unsigned long long drained;
};

template <typename T, int HD, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1)
attention_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttentionArgs p, CutRule rule) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ Shared sh;
    constexpr int kBoxes = HD / 64;
    constexpr int kTile = tile_bytes(HD), kBox = 128 * 64 * 2, kKSlots = k_slots(HD), kVSlots = v_slots(HD);
    constexpr bool kBf16 = sizeof(T) == 2 && !__is_same(T, __half);
    unsigned char* const tiles = smem + ((1024u - (smem_u32(smem) & 1023u)) & 1023u);
    unsigned char* const k_tiles = tiles + 2 * kTile;
    unsigned char* const v_tiles = k_tiles + kKSlots * kTile;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int tile_tokens = 2 * p.tokens_per_half;

    if (tid == 0) {
        for (int h = 0; h < 2; ++h) {
            mbar_init(smem_u32(&sh.q_full[h]), 1);
            mbar_init(smem_u32(&sh.q_empty[h]), 1);
            mbar_init(smem_u32(&sh.s_full[h]), 1);
            mbar_init(smem_u32(&sh.p_full[h][0]), 4);
            mbar_init(smem_u32(&sh.p_full[h][1]), 4);
            mbar_init(smem_u32(&sh.o_full[h]), 1);
            mbar_init(smem_u32(&sh.o_empty[h]), 4);
            mbar_init(smem_u32(&sh.voted[h]), 4);
            for (int i = 0; i < 4; ++i) sh.votes[h][i] = 0;
        }
        for (int s = 0; s < kMaxSlots; ++s) {
            mbar_init(smem_u32(&sh.k_full[s]), 1);
            mbar_init(smem_u32(&sh.k_empty[s]), 1);
            mbar_init(smem_u32(&sh.v_full[s]), 1);
            mbar_init(smem_u32(&sh.v_empty[s]), 1);
        }
        for (int s = 0; s < kItems; ++s) {
            mbar_init(smem_u32(&sh.item_full[s]), 1);
            mbar_init(smem_u32(&sh.item_empty[s]), 10);
        }
        mbar_init(smem_u32(&sh.drained), 1);
        sh.stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(&map_q)) : "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(&map_k)) : "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(&map_v)) : "memory");
    }
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    if (p.clear_rest) clear_rest<kThreads, HD>(p);
    const Share share = find_share<kThreads, 1>(p, tile_tokens, kKeyBlock, rule, sh.share);
    if (share.begin >= share.end) {                                // nothing left for this block
        if (tid == 0 && p.cut_tiles != nullptr) p.cut_tiles[blockIdx.x].of = 0;
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
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            // ---------------- items, Q and K
            ShareWalk walk;
            walk.start(p, share);
            unsigned k_seq = 0, n_items = 0, q_count[2] = {0, 0}, block_seq = 0;
            bool cut_written = false;
            PageRow pages;
            HalvedItem hit;
            Item& it = hit.it;
            bool more = walk.next(p, tile_tokens, kKeyBlock, rule, it);
            for (;;) {
                const int ring = n_items % kItems;
                ok = warp_wait(smem_u32(&sh.item_empty[ring]), ((n_items / kItems) & 1u) ^ 1u, &sh.stop);
                if (!ok) break;
                if (!more) {
                    if (elect_one()) {
                        sh.items[ring].it.request = -1;
                        mbar_arrive(smem_u32(&sh.item_full[ring]));
                    }
                    break;
                }
                half_blocks(it.seen, it.tokens, p.tokens_per_half, kKeyBlock, it.block, it.blocks, hit.count);
                hit.first = walk.r.first;
                if (elect_one()) {
                    sh.items[ring] = hit;
                    mbar_arrive(smem_u32(&sh.item_full[ring]));
                    if (it.of > 0) write_cut_tile(p, it);
                }
                cut_written |= it.of > 0;
                ++n_items;
                const int kv_head = it.head / p.kv_group;
                pages.column = -1;
                auto load_q = [&](int h) {
                    if (hit.count[h] == 0) return true;
                    if (!warp_wait(smem_u32(&sh.q_empty[h]), (q_count[h] & 1u) ^ 1u, &sh.stop)) return false;
                    ++q_count[h];
                    if (elect_one()) {
                        const unsigned bar = smem_u32(&sh.q_full[h]);
                        mbar_arrive_expect_tx(bar, p.heads_per_tile * p.tokens_per_half * HD * 2);
#pragma unroll
                        for (int x = 0; x < kBoxes; ++x)
                            tma_3d(smem_u32(tiles + h * kTile + x * kBox), &map_q, x * 64, it.head, it.row + h * p.tokens_per_half, bar);
                    }
                    __syncwarp();
                    return true;
                };
                ok = load_q(0);
                for (int j = 0; j < it.blocks && ok; ++j) {
                    const int key0 = (it.block + j) * kKeyBlock;
                    int n_pages = 0, page = 0;
                    if (PAGED) {
                        n_pages = pages.fetch(p, it.request, key0, min(kKeyBlock, it.keys - key0), lane, page);
                        const unsigned bad = __ballot_sync(0xffffffffu, lane < n_pages && page == p.n_pages);
                        unsigned lost = 0;
                        if (bad) {
                            const int per = p.page_size / 16;
                            for (int i = 0; i < 8; ++i)
                                if ((bad >> (i / per)) & 1u) lost |= 1u << i;
                        }
                        if (elect_one()) sh.lost[block_seq % kKeysSeen] = lost;
                        ++block_seq;
                    }
                    const int s = k_seq % kKSlots;
                    ok = warp_wait(smem_u32(&sh.k_empty[s]), ((k_seq / kKSlots) & 1u) ^ 1u, &sh.stop);
                    if (!ok) break;
                    ++k_seq;
                    load_keys<HD, PAGED>(p, &map_k, smem_u32(k_tiles + s * kTile), smem_u32(&sh.k_full[s]), hit.first + key0, kv_head, n_pages, page);
                    if (j == 0) ok = load_q(1);
                }
                if (!ok) break;
                more = walk.next(p, tile_tokens, kKeyBlock, rule, it);
            }
            if (lane == 0 && !cut_written && p.cut_tiles != nullptr) p.cut_tiles[blockIdx.x].of = 0;
            if (!ok) {
                // copies still in flight write shared memory: wait for them before it is given up
                volatile int never = 0;
                for (int h = 0; h < 2; ++h)
                    if (q_count[h] > 0) warp_wait(smem_u32(&sh.q_full[h]), (q_count[h] - 1) & 1u, &never);
                for (unsigned i = k_seq > kKSlots ? k_seq - kKSlots : 0; i < k_seq; ++i)
                    warp_wait(smem_u32(&sh.k_full[i % kKSlots]), (i / kKSlots) & 1u, &never);
            }
        } else if (warp == 2) {
            // ---------------- V
            unsigned v_seq = 0, n_items = 0;
            PageRow pages;
            while (ok) {
                const int ring = n_items % kItems;
                ok = warp_wait(smem_u32(&sh.item_full[ring]), (n_items / kItems) & 1u, &sh.stop);
                if (!ok) break;
                const Item it = sh.items[ring].it;
                const int first = sh.items[ring].first;
                if (it.request < 0) break;
                ++n_items;
                const int kv_head = it.head / p.kv_group;
                pages.column = -1;
                for (int j = 0; j < it.blocks && ok; ++j) {
                    const int key0 = (it.block + j) * kKeyBlock;
                    int n_pages = 0, page = 0;
                    if (PAGED) n_pages = pages.fetch(p, it.request, key0, min(kKeyBlock, it.keys - key0), lane, page);
                    const int s = v_seq % kVSlots;
                    ok = warp_wait(smem_u32(&sh.v_empty[s]), ((v_seq / kVSlots) & 1u) ^ 1u, &sh.stop);
                    if (!ok) break;
                    ++v_seq;
                    load_keys<HD, PAGED>(p, &map_v, smem_u32(v_tiles + s * kTile), smem_u32(&sh.v_full[s]), first + key0, kv_head, n_pages, page);
                }
                __syncwarp();
                if (elect_one()) mbar_arrive(smem_u32(&sh.item_empty[ring]));
            }
            if (!ok) {
                volatile int never = 0;
                for (unsigned i = v_seq > kVSlots ? v_seq - kVSlots : 0; i < v_seq; ++i)
                    warp_wait(smem_u32(&sh.v_full[i % kVSlots]), (i / kVSlots) & 1u, &never);
            }
        } else if (warp == 1) {
            // ---------------- MMA.  The whole warp walks, one lane issues: what is the same for all lanes stays in uniform
            // registers, as the instructions want it (one lane walking alone was 15 % slower).
            const uint32_t qk = instr_desc(kKeyBlock, kBf16, false, p.negative != 0);
            constexpr uint32_t pv = instr_desc(HD, kBf16, true, false);
            const uint64_t q_desc = desc_sw128(smem_u32(tiles), 16), k_desc = desc_sw128(smem_u32(k_tiles), 16);
            const uint64_t v_desc = desc_sw128(smem_u32(v_tiles), kBox);
            unsigned k_seq = 0, v_seq = 0, n_items = 0, q_count[2] = {0, 0}, p_count[2] = {0, 0}, o_count[2] = {0, 0};
            while (ok) {
                const int ring = n_items % kItems;
                ok = warp_wait(smem_u32(&sh.item_full[ring]), (n_items / kItems) & 1u, &sh.stop);
                if (!ok) break;
                const HalvedItem& hit = sh.items[ring];
                const int request = hit.it.request, blocks = hit.it.blocks;
                const int count[2] = {hit.count[0], hit.count[1]};
                const int block0 = hit.it.block, keys = hit.it.keys - block0 * kKeyBlock;
                const int seen_first[2] = {hit.it.seen, hit.it.seen + min(p.tokens_per_half, hit.it.tokens - 1)};
                if (request < 0) break;
                ++n_items;
                for (int j = 0; j <= blocks && ok; ++j) {
                    const int k_slot = k_seq % kKSlots, v_slot = v_seq % kVSlots;        // of K(j) and V(j - 1)
                    bool k_here = false, v_here = false;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const unsigned s_at = tmem + h * 128, o_at = tmem + 256 + h * HD;
                        if (j > 0 && j - 1 < count[h]) {
                            if (!v_here) {
                                ok = warp_wait(smem_u32(&sh.v_full[v_slot]), (v_seq / kVSlots) & 1u, &sh.stop);
                                if (!ok) break;
                                v_here = true;
                            }
                            if (j == 1) {                         // the last item's O has been read
                                ok = warp_wait(smem_u32(&sh.o_empty[h]), (o_count[h] & 1u) ^ 1u, &sh.stop);
                                if (!ok) break;
                                ++o_count[h];
                            }
                            const uint64_t dv = v_desc + static_cast<uint64_t>((v_slot * kTile) >> 4);
                            const unsigned more = j > 1;
                            if (!is_edge(seen_first[h], (block0 + j - 1) * kKeyBlock)) {
#pragma unroll
                                for (int part = 0; part < 2; ++part) {  // P comes in two parts of 64 keys
                                    ok = warp_wait(smem_u32(&sh.p_full[h][part]), p_count[h] & 1u, &sh.stop);
                                    if (!ok) break;
                                    fence_after();
                                    if (elect_one()) {
#pragma unroll
                                        for (int k = part * 4; k < part * 4 + 4; ++k)
                                            mma_tmem(o_at, s_at + k * 8, dv + ((k * 2048) >> 4), pv, k > 0 ? 1u : more);
                                        if (part == 1 && j == count[h]) commit(smem_u32(&sh.o_full[h]));
                                    }
                                    __syncwarp();
                                }
                            } else {
                                const int live = min(kKeyBlock, max(0, keys - (j - 1) * kKeyBlock));
                                ok = warp_wait(smem_u32(&sh.p_full[h][0]), p_count[h] & 1u, &sh.stop) && warp_wait(smem_u32(&sh.p_full[h][1]), p_count[h] & 1u, &sh.stop);
                                if (!ok) break;
                                fence_after();
                                const bool by_hand = *static_cast<volatile int*>(&sh.by_hand[h]) != 0;
                                if (elect_one()) {
#pragma unroll 1
                                    for (int k = 0; k * 16 < live && !by_hand; ++k)
                                        mma_tmem(o_at, s_at + k * 8, dv + static_cast<uint64_t>((k * 2048) >> 4), pv, k > 0 ? 1u : more);
                                    if (j == count[h]) commit(smem_u32(&sh.o_full[h]));
                                }
                                __syncwarp();
                            }
                            if (!ok) break;
                            ++p_count[h];
                        }
                        if (j < count[h]) {
                            if (!k_here) {
                                ok = warp_wait(smem_u32(&sh.k_full[k_slot]), (k_seq / kKSlots) & 1u, &sh.stop);
                                if (!ok) break;
                                k_here = true;
                            }
                            if (j == 0) {
                                ok = warp_wait(smem_u32(&sh.q_full[h]), q_count[h] & 1u, &sh.stop);
                                if (!ok) break;
                                ++q_count[h];
                            }
                            fence_after();
                            if (elect_one()) {
                                const uint64_t dq = q_desc + ((h * kTile) >> 4), dk = k_desc + static_cast<uint64_t>((k_slot * kTile) >> 4);
#pragma unroll
                                for (int k = 0; k < HD / 16; ++k) {
                                    const uint64_t at = ((k >> 2) * kBox + (k & 3) * 32) >> 4;
                                    mma_smem(s_at, dq + at, dk + at, qk, k > 0);
                                }
                                commit(smem_u32(&sh.s_full[h]));
                                if (j == count[h] - 1) commit(smem_u32(&sh.q_empty[h]));
                            }
                            __syncwarp();
                        }
                    }
                    if (!ok) break;
                    if (elect_one()) {
                        if (j > 0) commit(smem_u32(&sh.v_empty[v_slot]));
                        if (j < blocks) commit(smem_u32(&sh.k_empty[k_slot]));
                    }
                    __syncwarp();
                    if (j > 0) ++v_seq;
                    if (j < blocks) ++k_seq;
                }
                __syncwarp();
                if (elect_one()) mbar_arrive(smem_u32(&sh.item_empty[ring]));
            }
            if (!ok) {
                // products still in flight read shared memory and write tensor memory: wait for them before both are given up
                volatile int never = 0;
                __syncwarp();
                if (elect_one()) commit(smem_u32(&sh.drained));
                __syncwarp();
                warp_wait(smem_u32(&sh.drained), 0, &never);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ---------------- softmax: thread = row of half h
        const int h = (warp - 4) >> 2;
        const int row = (warp & 3) * 32 + lane;
        const unsigned lanes = static_cast<unsigned>((warp & 3) * 32) << 16;
        const unsigned s_at = tmem + lanes + h * 128, o_at = tmem + lanes + 256 + h * HD;
        const int token = h * p.tokens_per_half + row / p.heads_per_tile, head = row % p.heads_per_tile;
        const bool in_tile = row < p.heads_per_tile * p.tokens_per_half;
        unsigned n_items = 0, s_count = 0, o_count = 0, block_seq = 0, vote = 0;
        bool sat_out = false;                                                   // blocks of the item before
        while (ok) {
            const int ring = n_items % kItems;
            ok = warp_wait(smem_u32(&sh.item_full[ring]), (n_items / kItems) & 1u, &sh.stop);
            if (!ok) break;
            const Item it = sh.items[ring].it;
            const int count = sh.items[ring].count[h];
            if (it.request < 0) break;
            ++n_items;
            const bool live_row = in_tile && token < it.tokens;
            const int seen = it.seen + min(token, it.tokens - 1);              // the last key this row sees
            const int seen_first = it.seen + min(h * p.tokens_per_half, it.tokens - 1);      // and the half's first row
            float top = -INFINITY, bias = 0.f, sum = 0.f;                       // maximum of s; exponent = s * scale - bias
            // One block of keys.  `Edge` where its rows do not all see all of its keys; apart, so that the registers and the schedule of
            // the others, which are nearly all, do not pay for it.
            auto block = [&](auto edge, int j, int key0, unsigned lost, bool by_hand) {
                constexpr bool kEdge = decltype(edge)::value;
                float s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(s_at + c * 32, s + c * 32);
                tmem_wait_ld();
                const int allowed = seen + 1 - key0;
                if constexpr (kEdge) {
#pragma unroll
                    for (int i = 0; i < 128; ++i)
                        if (i >= allowed || (PAGED && ((lost >> (i / 16)) & 1u))) s[i] = -INFINITY;
                }
                float m8[8];                                    // eight chains: one would wait for itself 128 times
#pragma unroll
                for (int i = 0; i < 8; ++i) m8[i] = fmaxf(s[i], s[i + 8]);
#pragma unroll
                for (int i = 16; i < 128; i += 16)
#pragma unroll
                    for (int k = 0; k < 8; ++k) m8[k] = fmaxf(fmaxf(m8[k], s[i + k]), s[i + k + 8]);
                const float m = fmaxf(fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])), fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7]))), top);
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
                if constexpr (kEdge) {
                    if (lane == 0) sh.by_hand[h] = by_hand;
                    __syncwarp();
                }
                const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), bias2 = make_float2(-bias, -bias);
                float2 part[4];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    unsigned w[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float2 e = fma2(make_float2(s[c * 64 + 2 * i], s[c * 64 + 2 * i + 1]), scale2, bias2);
                        e = make_float2(exp2_approx(e.x), exp2_approx(e.y));
                        part[i & 3] = c == 0 && i < 4 ? e : add2(part[i & 3], e);
                        w[i] = Pair16<T>::pack(e.x, e.y);
                    }
                    tmem_st32(s_at + c * 32, w);
                    tmem_wait_st();
                    if constexpr (kEdge) {
                        if (c == 1 && by_hand) product_by_hand<T, HD>(o_at, s_at, v_tiles + (block_seq + j) % kVSlots * kTile, allowed, j == 0);
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[h][c]));
                    if (c == 0) __syncwarp();                       // the next tcgen05.st wants the whole warp
                }
                const float2 all = add2(add2(part[0], part[1]), add2(part[2], part[3]));
                sum += all.x + all.y;
            };
            // (the first block waits for them again, and goes on at once)
            if (scores_before_values(sat_out, count)) ok = warp_wait(smem_u32(&sh.s_full[h]), s_count & 1u, &sh.stop);
            for (int j = 0; j < count && ok; ++j) {
                const int key0 = (it.block + j) * kKeyBlock;
                const bool edge = is_edge(seen_first, key0);
                bool by_hand = false;
                if (edge) {                                    // while the scores are formed: what stands in V behind the keys seen
                    const int slot = (block_seq + j) % kVSlots, rest = it.keys - key0;
                    ok = warp_wait(smem_u32(&sh.v_full[slot]), ((block_seq + j) / kVSlots) & 1u, &sh.stop);
                    if (!ok) break;
                    unsigned char* const v = v_tiles + slot * kTile;
                    if (rest < kKeyBlock && (rest & 15) != 0) {
                        // What lies behind the last key may be anything; its weight is zero, and zero times it must be too.  The
                        // product ends with the last key's 16: clear the rest of those.
                        const int gone = rest > 0 ? 16 - (rest & 15) : 0;
                        for (int i = row; i < gone * 8 * kBoxes; i += 128)
                            *reinterpret_cast<uint4*>(v + rest * 128 + (i / (gone * 8)) * kBox + (i % (gone * 8)) * 16) = make_uint4(0, 0, 0, 0);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    if (seen_first + 1 - key0 < min(rest, kKeyBlock)) {
                        // The half's four warps agree by a bounded wait like all others.  Two entries on, the ring is cleared: whoever is
                        // past the last vote knows that all have read the one before it.
                        const bool bad = any_not_finite<T, HD>(v, rest, row);
                        if (lane == 0) {
                            sh.votes[h][(vote + 2) & 3] = 0;
                            if (bad) sh.votes[h][vote & 3] = 1;
                            mbar_arrive(smem_u32(&sh.voted[h]));
                        }
                        ok = warp_wait(smem_u32(&sh.voted[h]), vote & 1u, &sh.stop);
                        if (!ok) break;
                        by_hand = *static_cast<volatile int*>(&sh.votes[h][vote & 3]) != 0;
                        ++vote;
                    }
                }
                ok = warp_wait(smem_u32(&sh.s_full[h]), s_count & 1u, &sh.stop);
                if (!ok) break;
                ++s_count;
                fence_after();
                const unsigned lost = PAGED ? sh.lost[(block_seq + j) % kKeysSeen] : 0u;
                if (edge || (PAGED && lost != 0)) block(std::true_type{}, j, key0, lost, by_hand);
                else block(std::false_type{}, j, key0, 0u, false);
            }
            block_seq += it.blocks;
            sat_out = count < it.blocks;
            if (!ok) break;
            if (count > 0) {
                ok = warp_wait(smem_u32(&sh.o_full[h]), o_count & 1u, &sh.stop);
                if (!ok) break;
                ++o_count;
                fence_after();
            }
            if (it.slot < 0) {
                if (count > 0) {
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
                    // A lane holds a row; rows are far apart in `out`, and a store that touches 32 of them takes the load/store unit 32
                    // turns (4450 cycles a tile).  So four lanes exchange what they hold, 16 bytes at a time, and write 64
                    // bytes of one row after the other together.
                    const long long mine = live_row ? (static_cast<long long>(it.row + token) * p.n_heads + it.head + head) * HD : -1;
                    long long at[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) at[r] = __shfl_sync(0xffffffffu, mine, (lane & ~3) + r);
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        float o[32];
                        tmem_ld32(o_at + c * 32, o);
                        tmem_wait_ld();
                        uint4 u[4];
                        unsigned* const w = reinterpret_cast<unsigned*>(u);
#pragma unroll
                        for (int i = 0; i < 16; ++i) w[i] = sum == 0.f ? 0u : Pair16<T>::pack(o[2 * i] * inv, o[2 * i + 1] * inv);
                        swap_units<1>(u[0], u[1], lane);
                        swap_units<1>(u[2], u[3], lane);
                        swap_units<2>(u[0], u[2], lane);
                        swap_units<2>(u[1], u[3], lane);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (at[r] >= 0) *reinterpret_cast<uint4*>(p.out + at[r] + c * 32 + (lane & 3) * 8) = u[r];
                        __syncwarp();                               // the next tcgen05.ld wants the whole warp
                    }
                }
            } else if (it.tokens > h * p.tokens_per_half) {
                float* const piece = p.partial + it.slot * piece_floats(256, HD);
                const int at_row = h * 128 + row;
                piece[256 * HD + at_row] = count > 0 ? bias : 0.f;
                piece[256 * HD + 256 + at_row] = count > 0 ? sum : 0.f;
                if (count > 0) {
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        float o[32];
                        tmem_ld32(o_at + c * 32, o);
                        tmem_wait_ld();
                        if (live_row) {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                reinterpret_cast<float4*>(piece)[(c * 8 + i) * 256 + at_row] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        }
                        __syncwarp();                               // the next tcgen05.ld wants the whole warp
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
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512) : "memory");
}

constexpr CutRule kRule = {12, 2, 1, 2};
template <typename T, int HD, bool PAGED>
int run(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const AttentionArgs& args, int dev, cudaStream_t stream) {
    static std::once_flag once[64];
    static bool set[64] = {};
    std::call_once(once[dev], [dev]() {
        set[dev] = cudaFuncSetAttribute(attention_tcgen05_kernel<T, HD, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(HD)) == cudaSuccess;
    });
    if (!set[dev]) return EPTQ_ERR_LAUNCH;
    return launch_dependent(attention_tcgen05_kernel<T, HD, PAGED>, dim3(kSms), kThreads, smem_bytes(HD), stream, q, k, v, args, kRule);
}

}  // namespace

AttentionPlan attention_tcgen05_plan(const EptqAttention& a) {
    AttentionPlan plan;
    plan.shares = kSms;
    plan.tile_rows = 256;
    const long long keys = a.page_size != 0 ? static_cast<long long>(a.table_width) * a.page_size : a.rows;
    plan.may_cut = keys > static_cast<long long>(kRule.least) * kKeyBlock;
    return plan;
}

int launch_attention_tcgen05(const EptqAttention& a, AttentionArgs& p, int dev, cudaStream_t stream) {
    const bool paged = a.page_size != 0;
    p.heads_per_tile = heads_in(p.kv_group, 128);
    p.tokens_per_half = 128 / p.heads_per_tile;
    CUtensorMap q, k, v;
    const cuuint64_t hd = a.head_dim, nkv = a.n_kv_heads;
    {
        const cuuint64_t dims[3] = {hd, static_cast<cuuint64_t>(a.n_heads), static_cast<cuuint64_t>(a.rows)};
        const int64_t strides[2] = {a.head_dim, a.q_stride};
        const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(p.heads_per_tile), static_cast<cuuint32_t>(p.tokens_per_half)};
        if (!encode_map(&q, a.dtype, a.q, 3, dims, strides, box)) return EPTQ_ERR_LAUNCH;
    }
    if (paged) {
        if (!encode_page_maps(&k, &v, a, a.page_size)) return EPTQ_ERR_LAUNCH;
    } else {
        const cuuint64_t dims[3] = {hd, nkv, static_cast<cuuint64_t>(a.rows)};
        const cuuint32_t box[3] = {64, 1, kKeyBlock};
        const int64_t ks[2] = {a.head_dim, a.k_stride}, vs[2] = {a.head_dim, a.v_stride};
        if (!encode_map(&k, a.dtype, a.k, 3, dims, ks, box) || !encode_map(&v, a.dtype, a.v, 3, dims, vs, box)) return EPTQ_ERR_LAUNCH;
    }
    if (a.dtype == EPTQ_FP16) {
        if (a.head_dim == 128) return paged ? run<__half, 128, true>(q, k, v, p, dev, stream) : run<__half, 128, false>(q, k, v, p, dev, stream);
        return paged ? run<__half, 64, true>(q, k, v, p, dev, stream) : run<__half, 64, false>(q, k, v, p, dev, stream);
    }
    if (a.head_dim == 128) return paged ? run<__nv_bfloat16, 128, true>(q, k, v, p, dev, stream) : run<__nv_bfloat16, 128, false>(q, k, v, p, dev, stream);
    return paged ? run<__nv_bfloat16, 64, true>(q, k, v, p, dev, stream) : run<__nv_bfloat16, 64, false>(q, k, v, p, dev, stream);
}

}  // namespace eptq
