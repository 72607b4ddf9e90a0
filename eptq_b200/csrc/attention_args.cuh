// What the kernels of a ragged attention call share: their arguments and the partial results of row tiles that are cut.
#pragma once

#include <cuda.h>

#include "attention_schedule.cuh"
#include "common.cuh"

namespace eptq {

// Descriptor of a tile that share c begins and later shares end; of == 0: there is none.
struct CutTile {
    int of;            // number of pieces: shares c .. c + of - 1
    int row;           // first row of the tile
    int tokens;        // tokens of the tile that exist
    int head;          // first query head
    int pad[4];
};

struct AttentionArgs {
    const int *tables, *kv_lens, *cu_rows;
    uint16_t* out;
    int* status;
    CutTile* cut_tiles;            // [shares]
    float* partial;                // [2 * shares] pieces: share c's first item at 2c, one that others continue at 2c + 1
    const uint16_t* q;
    long long q_stride, table_stride, table_keys;
    int rows, batch, n_heads, kv_group;      // kv_group: query heads per key/value head
    int heads_per_tile, tokens_per_half;     // heads that share a row tile; tokens of one 128-row half, or of a smaller tile
    int tile_rows;                           // 256 in halves of 128, or fewer: row = token * heads_per_tile + head in each
    int page_size, n_pages, table_width;
    float scale_log2;              // |scale| * log2(e)
    int negative;                  // scale is below zero
    int clear_rest;                // rows of no request become zeros
};

// A piece of a cut tile: o [head_dim / 4][tile_rows][4], then the exponent's reference and the sum of each row, fp32.  Rows whose
// sum is zero have no o.
__host__ __device__ constexpr long long piece_floats(int rows, int hd) { return static_cast<long long>(rows) * (hd + 2); }

// Exponents of 2 carry this offset, so that the weights of a row reach 2^7 and not 1: small ones stay out of fp16's
// subnormal range, and the row's maximum may grow by 2^kRescaleAt (to 2^15 of fp16's 2^16) before what is summed is scaled.
constexpr float kExpOffset = 7.f;
constexpr float kRescaleAt = 8.f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr unsigned long long kWaitNs = 2000000000ull;      // limit of one wait

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
// One lane of a converged warp.  Unlike `lane == 0` it tells the compiler that one thread runs what follows, which the
// instructions that take uniform registers (tcgen05.mma, TMA) need: a loop over the active lanes around each of them cost
// 195 cycles an MMA of 64.
__device__ __forceinline__ bool elect_one() {
    unsigned p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
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

// (Plain loads here and wherever a kernel reads what the one before it may have written: it may start before that one has
// ended, and a read-only load may be served from before its own wait.)
__device__ __forceinline__ Request load_request(const AttentionArgs& p, int b) {
    const bool paged = p.page_size != 0;
    return request_from(p.cu_rows[b], p.cu_rows[b + 1], p.rows, paged ? p.kv_lens[b] : 0, p.table_keys, paged);
}

// The rows ahead of the first request and behind the last one become zeros, 16 bytes a thread.  Not inline: the registers it would take
// cost the kernel of few rows 4 % where a call has nothing to clear.
template <int kThreads, int HD>
__device__ __noinline__ void clear_rest(const AttentionArgs& p) {
    const long long row = static_cast<long long>(p.n_heads) * (HD / 8), first = min(max(p.cu_rows[0], 0), p.rows) * row;
    const long long end = min(max(p.cu_rows[p.batch], 0), p.rows) * row, rest = first + p.rows * row - end;
    for (long long i = blockIdx.x * kThreads + threadIdx.x; i < rest; i += gridDim.x * kThreads)
        reinterpret_cast<uint4*>(p.out)[i < first ? i : end + i - first] = make_uint4(0, 0, 0, 0);
}

// The part of the work that falls to one block of the launch.
struct Share {
    long long begin, end;        // in what the sequence counts
    long long size;              // of an uncut share
    int request;                 // that holds the begin
    Request r;                   // its lengths
    Place at;                    // the begin there
};
template <int kThreads>
struct ShareScratch {
    long long sums[kThreads / 32];
    long long before[2];         // blocks before the request that holds the share's begin and its end
    int request[2];
    long long cut[2];
    Request r;
    Place at;
};

// Sums the blocks of all requests, kPer requests a thread at a time, and finds the requests that hold the share's ends.
// All threads of the block call it and get the same answer.
template <int kThreads, int kPer>
__device__ __forceinline__ Share find_share(const AttentionArgs& p, int tile, int kb, CutRule& rule, ShareScratch<kThreads>& sh) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, groups = p.n_heads / p.heads_per_tile;
    long long all = 0, ends[2] = {0, 0};
    Share share = {};
    for (int pass = 0; pass < 2; ++pass) {
        long long before = 0;
        for (int b0 = 0; b0 < p.batch; b0 += kThreads * kPer) {
            long long w[kPer], mine = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int b = b0 + tid * kPer + i;
                w[i] = 0;
                if (b < p.batch) {
                    const Request r = load_request(p, b);
                    w[i] = cost_before(r, tile, kb, rule, tiles_of(r, tile)) * groups;
                }
                mine += w[i];
            }
            long long upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long up = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += up;
            }
            __syncthreads();
            if (lane == 31) sh.sums[warp] = upto;
            __syncthreads();
            long long chunk = 0;
#pragma unroll
            for (int i = 0; i < kThreads / 32; ++i) {
                if (i == warp) upto += chunk;
                chunk += sh.sums[i];
            }
            upto += before - mine;                                  // blocks before this thread's first request
            const bool last = b0 + kThreads * kPer >= p.batch;
            if (pass == 0 && last) {                                // the sum is known: this chunk may hold the ends already
                all = before + chunk;
                share.size = share_of(all, gridDim.x, rule);
                ends[0] = blockIdx.x * share.size;
                ends[1] = blockIdx.x + 1 < gridDim.x ? ends[0] + share.size : all;
            }
            if (pass == 1 || last) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    for (int e = 0; e < 2; ++e)
                        if (ends[e] >= upto && ends[e] < upto + w[i]) { sh.request[e] = b0 + tid * kPer + i; sh.before[e] = upto; }
                    upto += w[i];
                }
            }
            before += chunk;
        }
        if (p.batch <= kThreads * kPer) break;                      // one chunk: both passes in one
    }
    __syncthreads();
    if (warp < 2) {                                                 // one warp for each end
        const long long end = warp == 0 ? ends[0] : ends[1];
        long long cut = all;
        if (end < all) {
            const Request r = load_request(p, sh.request[warp]);
            // 32 tiles looked at in each round: the sums before a tile take a few divisions
            Place at = place_of(r, tile, kb, rule, end - sh.before[warp], [&](int lo, int hi, long long y) {
                while (lo < hi) {
                    const int step = (hi - lo + 31) / 32, i = lo + (lane + 1) * step;
                    const bool begins = i <= hi && cost_before(r, tile, kb, rule, i) <= y;
                    const int n = __popc(__ballot_sync(0xffffffffu, begins));      // beginnings rise: the first n lanes
                    lo += n * step;
                    hi = min(hi, lo + step - 1);
                }
                return lo;
            });
            cut = moved(at, rule, end);
            if (warp == 0 && lane == 0) {
                sh.at = at;
                sh.r = r;
            }
        }
        if (lane == 0) sh.cut[warp] = cut;
    }
    __syncthreads();
    share.request = sh.request[0];
    share.r = sh.r;
    share.at = sh.at;
    share.begin = sh.cut[0];
    share.end = sh.cut[1];
    return share;
}

// One row tile, or the part of it that falls to a share.
struct Item {
    int row, tokens, head, request;    // first row, tokens that exist, first query head; request < 0: no more items
    int seen;                          // last key that the first token sees
    int keys;                          // keys that the last token sees
    int block, blocks;                 // first block of keys, number of blocks
    int slot;                          // where the partial result goes, -1: it is the whole tile
    int of;                            // > 0: the tile's first piece, of that many
};

// Walks the items of a share.
struct ShareWalk {
    Request r;
    int b;
    Place now;
    long long left, flat, size;

    __device__ __forceinline__ void start(const AttentionArgs& p, const Share& s) {
        b = s.request;
        r = s.r;
        now = s.at;
        left = s.end - s.begin;
        flat = s.begin;
        size = s.size;
    }
    __device__ __forceinline__ bool next(const AttentionArgs& p, int tile, int kb, const CutRule& rule, Item& it) {
        const int groups = p.n_heads / p.heads_per_tile;
        if (left <= 0) { it.request = -1; return false; }
        int row_tiles = tiles_of(r, tile);
        if (now.tile >= row_tiles) { now.tile = 0; ++now.group; }
        while (row_tiles == 0 || now.group >= groups) {
            r = load_request(p, ++b);
            row_tiles = tiles_of(r, tile);
            now.group = now.tile = now.block = 0;
        }
        const int blocks = blocks_of(r, tile, kb, now.tile);
        it.request = b;
        it.row = r.first + now.tile * tile;
        it.tokens = min(tile, r.n - now.tile * tile);
        it.head = now.group * p.heads_per_tile;
        it.seen = r.past + now.tile * tile;
        it.keys = max(0, it.seen + it.tokens);
        it.block = now.block;
        const int ahead = now.block == 0 ? rule.tile : 0;
        it.blocks = static_cast<int>(min(static_cast<long long>(blocks - now.block), left - ahead));
        const bool whole = it.blocks == blocks;
        it.slot = whole ? -1 : 2 * static_cast<int>(blockIdx.x) + (it.block == 0 ? 1 : 0);
        it.of = whole || it.block != 0 ? 0 : last_share(flat + ahead + blocks, size, rule) - static_cast<int>(blockIdx.x) + 1;
        left -= ahead + it.blocks;
        flat += ahead + it.blocks;
        now.block = 0;
        ++now.tile;
        return true;
    }
};

__device__ __forceinline__ void write_cut_tile(const AttentionArgs& p, const Item& it) {
    CutTile c;
    c.of = it.of; c.row = it.row; c.tokens = it.tokens; c.head = it.head;
    c.pad[0] = c.pad[1] = c.pad[2] = c.pad[3] = 0;
    p.cut_tiles[blockIdx.x] = c;
}

}  // namespace eptq
