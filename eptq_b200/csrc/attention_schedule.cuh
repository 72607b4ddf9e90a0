// How the work of a ragged attention call is cut into equal shares, one per block of the launch, from lengths that only
// the device knows.
//
// A request with n new rows behind `past` keys has, for every group of `hp` query heads that share their keys, row tiles
// of `tile` tokens; a tile reads the keys its last row sees, in blocks of `kb`.  All blocks of keys of all tiles form one
// sequence -- request, head group, row tile, block -- and launch block c takes the blocks from cut(c) to cut(c + 1).  Cuts
// at equal distances balance requests of any lengths without knowing them on the host; a tile cut in two or more is joined
// from partial results.  Joining costs about as much as a few blocks, so a cut moves to the end of a tile that is short or near.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define EPTQ_HD __host__ __device__ __forceinline__
#else
#define EPTQ_HD inline
#endif

namespace eptq {

struct CutRule {
    int least;     // a tile of at most this many blocks is not cut
    int near;      // a cut this near an end of its tile moves there
    int share;     // least blocks of a share
};

struct Request {
    int first;     // its first row
    int n;         // rows
    int past;      // keys before its first row (negative: that many rows see no key)
};

// Rows outside the call and keys outside the table do not exist, whatever the arrays say.
EPTQ_HD Request request_from(int row0, int row1, int rows, long long kv_len, long long table_keys, bool paged) {
    Request r;
    r.first = row0 < 0 ? 0 : row0 > rows ? rows : row0;
    const int end = row1 < r.first ? r.first : row1 > rows ? rows : row1;
    r.n = end - r.first;
    const long long keys = kv_len < 0 ? 0 : kv_len > table_keys ? table_keys : kv_len;
    r.past = paged ? static_cast<int>(keys - r.n) : 0;
    return r;
}

EPTQ_HD int tiles_of(const Request& r, int tile) { return (r.n + tile - 1) / tile; }

// Blocks of keys that row tile i reads (one at least: rows without keys are written too).
EPTQ_HD int blocks_of(const Request& r, int tile, int kb, int i) {
    const long long rows = static_cast<long long>(i + 1) * tile < r.n ? static_cast<long long>(i + 1) * tile : r.n;
    const long long keys = r.past + rows;
    return keys <= kb ? 1 : static_cast<int>((keys + kb - 1) / kb);
}

// sum of floor((a i + b) / m) for i = 0 .. n-1, a, b >= 0: the usual exchange of the axes under the line
// (Euclid's algorithm on a and m).
EPTQ_HD long long floor_sum(unsigned n, unsigned m, unsigned a, unsigned b) {
    long long sum = 0;
    while (n > 0) {
        sum += static_cast<long long>(n) * (n - 1) / 2 * (a / m) + static_cast<long long>(n) * (b / m);
        a %= m;
        b %= m;
        const unsigned long long top = static_cast<unsigned long long>(a) * n + b;
        if (top < m) break;
        n = static_cast<unsigned>(top / m);
        b = static_cast<unsigned>(top % m);
        const unsigned t = m; m = a; a = t;
    }
    return sum;
}

// Blocks of the row tiles before tile i, i <= tiles_of.
EPTQ_HD long long blocks_before(const Request& r, int tile, int kb, int i) {
    if (i <= 0) return 0;
    const int full = static_cast<long long>(i) * tile <= r.n ? i : i - 1;        // tiles that are not cut off by the request's end
    int z = r.past < 0 ? -r.past / tile : 0;                                      // tiles without keys: one block each
    if (z > full) z = full;
    long long sum = z;
    if (full > z)
        sum += floor_sum(static_cast<unsigned>(full - z), kb, static_cast<unsigned>(tile),
                         static_cast<unsigned>(r.past + static_cast<long long>(z + 1) * tile + kb - 1));
    if (i > full) sum += blocks_of(r, tile, kb, i - 1);
    return sum;
}

// A place in the sequence inside one request.
struct Place {
    int group, tile, block;    // head group, row tile, block of keys
    int blocks;                // of that row tile
};

// x = blocks of the request before the place, 0 <= x < groups * blocks_before(all tiles).
EPTQ_HD Place place_of(const Request& r, int tile, int kb, long long x) {
    const int tiles = tiles_of(r, tile);
    const long long per_group = blocks_before(r, tile, kb, tiles);
    Place p;
    p.group = static_cast<int>(x / per_group);
    const long long y = x - p.group * per_group;
    int lo = 0, hi = tiles - 1;                       // the last tile that begins at or before y
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (blocks_before(r, tile, kb, mid) <= y) lo = mid; else hi = mid - 1;
    }
    p.tile = lo;
    p.block = static_cast<int>(y - blocks_before(r, tile, kb, lo));
    p.blocks = blocks_of(r, tile, kb, lo);
    return p;
}

EPTQ_HD long long share_of(long long all_blocks, int n_shares, const CutRule& rule) {
    const long long u = (all_blocks + n_shares - 1) / n_shares;
    return u < rule.share ? rule.share : u;
}

// How far a cut at place p moves.
EPTQ_HD int moved(const Place& p, const CutRule& rule) {
    if (p.block == 0) return 0;
    if (p.blocks <= rule.least) return 2 * p.block < p.blocks ? -p.block : p.blocks - p.block;
    if (p.block <= rule.near) return -p.block;
    if (p.blocks - p.block <= rule.near) return p.blocks - p.block;
    return 0;
}

// The last share that holds blocks of a cut tile which ends at `tile_end` in the sequence.
EPTQ_HD int last_share(long long tile_end, long long share, const CutRule& rule) {
    return static_cast<int>((tile_end - rule.near + share - 1) / share) - 1;
}

}  // namespace eptq
