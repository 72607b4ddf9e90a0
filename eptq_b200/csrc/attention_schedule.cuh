// How the work of a ragged attention call is cut into equal shares, one per block of the launch, from lengths that only
// the device knows.
//
// A request with n new rows behind `past` keys has, for every group of `hp` query heads that share their keys, row tiles
// of `tile` tokens; a tile reads the keys its last row sees, in blocks of `kb`.  All blocks of keys of all tiles form one
// sequence -- request, head group, row tile, block -- and launch block c takes the blocks from cut(c) to cut(c + 1).  Cuts
// at equal distances balance requests of any lengths without knowing them on the host; a tile cut in two or more is joined
// from partial results.  Joining costs about as much as a few blocks, so a cut moves to the end of a tile that is short or near.
// Beginning and ending a tile costs time too: each counts as rule.tile blocks more, ahead of its first one.
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
    int near;      // a cut this near an end of its tile moves there, where that is at most an eighth of a share
    int share;     // least blocks of a share
    int tile;      // blocks that a tile's beginning and end count as
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

// (One tile is the common case of running requests, and a division is a hundred cycles of a small call: here and below.)
EPTQ_HD int tiles_of(const Request& r, int tile) { return r.n <= tile ? (r.n > 0 ? 1 : 0) : (r.n + tile - 1) / tile; }

// Blocks of keys that row tile i reads (one at least: rows without keys are written too).
EPTQ_HD int blocks_of(const Request& r, int tile, int kb, int i) {
    const long long rows = static_cast<long long>(i + 1) * tile < r.n ? static_cast<long long>(i + 1) * tile : r.n;
    const long long keys = r.past + rows;
    return keys <= kb ? 1 : static_cast<int>((keys + kb - 1) / kb);
}

EPTQ_HD int log2_of(unsigned power) {
#ifdef __CUDA_ARCH__
    return 31 - __clz(power);
#else
    return 31 - __builtin_clz(power);
#endif
}

// sum of floor((a i + b) / m) for i = 0 .. n-1, b >= 0, a and m powers of two: shifts, no division.
EPTQ_HD long long floor_sum_powers(unsigned n, unsigned m, unsigned a, unsigned b) {
    const int am = log2_of(a), mm = log2_of(m);
    if (am >= mm) return (static_cast<long long>(n) * (n - 1) / 2 << (am - mm)) + static_cast<long long>(n) * (b >> mm);
    // floor((a i + b) / m) = floor((i + c) / d), c = floor(b / a), d = m / a: whole runs of d, then the rest of one
    const int d = mm - am;
    const unsigned c = b >> am, top = c + n;
    const long long qt = top >> d, qc = c >> d;
    const long long upto_top = (qt * (qt - 1) / 2 << d) + qt * (top & ((1u << d) - 1));
    const long long upto_c = (qc * (qc - 1) / 2 << d) + qc * (c & ((1u << d) - 1));
    return upto_top - upto_c;
}

// sum of floor((a i + b) / m) for i = 0 .. n-1, a, b >= 0: the usual exchange of the axes under the line (Euclid's
// algorithm on a and m).  Needs a n + b < 2^32 once a and b are reduced by m, which holds here: a is at most the tokens of a
// tile, n the tiles of a request.
EPTQ_HD long long floor_sum(unsigned n, unsigned m, unsigned a, unsigned b) {
    // the first step apart: its m is a constant power of two of the caller, and where it divides a the sum is done
    long long sum = static_cast<long long>(n) * (n - 1) / 2 * (a / m) + static_cast<long long>(n) * (b / m);
    a %= m;
    b %= m;
    const unsigned top0 = a * n + b;
    if (n == 0 || top0 < m) return sum;
    n = top0 / m;
    b = top0 % m;
    {
        const unsigned t = m; m = a; a = t;
    }
    while (n > 0) {
        sum += static_cast<long long>(n) * (n - 1) / 2 * (a / m) + static_cast<long long>(n) * (b / m);
        a %= m;
        b %= m;
        const unsigned top = a * n + b;
        if (top < m) break;
        n = top / m;
        b = top % m;
        const unsigned t = m; m = a; a = t;
    }
    return sum;
}

// 64-bit division is a long routine on the device; nearly all quotients here are of 32-bit values.
EPTQ_HD long long quotient(long long x, long long y) {
    if (((x | y) >> 32) == 0) return static_cast<unsigned>(x) / static_cast<unsigned>(y);
    return x / y;
}

// Blocks of the row tiles before tile i, i <= tiles_of.
EPTQ_HD long long blocks_before(const Request& r, int tile, int kb, int i) {
    if (i <= 0) return 0;
    if (r.n <= tile) return blocks_of(r, tile, kb, 0);
    const int full = static_cast<long long>(i) * tile <= r.n ? i : i - 1;        // tiles that are not cut off by the request's end
    int z = r.past < 0 ? -r.past / tile : 0;                                      // tiles without keys: one block each
    if (z > full) z = full;
    long long sum = z;
    if (full > z) {
        const unsigned n = static_cast<unsigned>(full - z), b = static_cast<unsigned>(r.past + static_cast<long long>(z + 1) * tile + kb - 1);
        sum += (tile & (tile - 1)) == 0 ? floor_sum_powers(n, kb, tile, b) : floor_sum(n, kb, tile, b);
    }
    if (i > full) sum += blocks_of(r, tile, kb, i - 1);
    return sum;
}

// What the row tiles before tile i count.
EPTQ_HD long long cost_before(const Request& r, int tile, int kb, const CutRule& rule, int i) {
    return blocks_before(r, tile, kb, i) + static_cast<long long>(i) * rule.tile;
}

// A place in the sequence inside one request.
struct Place {
    int group, tile, block;    // head group, row tile, block of keys
    int blocks;                // of that row tile
    int ahead;                 // what the place counts ahead of the tile's first block (then block is 0)
};

// x = what the request counts before the place, 0 <= x < groups * cost_before(all tiles).  `last_tile_at(lo, hi, y)` gives the
// last tile of lo .. hi that begins at or before y.
template <typename Search>
EPTQ_HD Place place_of(const Request& r, int tile, int kb, const CutRule& rule, long long x, const Search& last_tile_at) {
    const int tiles = tiles_of(r, tile);
    const long long per_group = cost_before(r, tile, kb, rule, tiles);
    Place p;
    p.group = static_cast<int>(quotient(x, per_group));
    const long long y = x - p.group * per_group;
    p.tile = tiles == 1 ? 0 : last_tile_at(0, tiles - 1, y);
    const int u = static_cast<int>(y - cost_before(r, tile, kb, rule, p.tile));
    p.block = u > rule.tile ? u - rule.tile : 0;
    p.ahead = u < rule.tile ? rule.tile - u : 0;
    p.blocks = blocks_of(r, tile, kb, p.tile);
    return p;
}

EPTQ_HD long long share_of(long long all_blocks, int n_shares, CutRule& rule) {
    const long long u = quotient(all_blocks + n_shares - 1, n_shares), size = u < rule.share ? rule.share : u;
    if (size < 8 * rule.near) rule.near = static_cast<int>(size / 8);
    return size;
}

// How far a cut at place p moves, from there: to the tile's own begin, to its end, or not.  Returns what the place counts then.
EPTQ_HD long long moved(Place& p, const CutRule& rule, long long x) {
    if (p.block == 0) {                                                           // to the tile's begin
        x -= rule.tile - p.ahead;
    } else if (p.blocks <= rule.least ? 2 * p.block < p.blocks : p.block <= rule.near) {
        x -= p.block + rule.tile;
        p.block = 0;
    } else if (p.blocks <= rule.least || p.blocks - p.block <= rule.near) {
        x += p.blocks - p.block;
        p.block = 0;
        ++p.tile;
    }
    p.ahead = rule.tile;
    return x;
}

// The last share that holds blocks of a cut tile which ends at `tile_end` in the sequence.
EPTQ_HD int last_share(long long tile_end, long long share, const CutRule& rule) {
    return static_cast<int>(quotient(tile_end - rule.near + share - 1, share)) - 1;
}

// ---- a row tile in two halves of tokens, which take turns ----

// Blocks of an item (the tile's blocks `block` .. block + blocks - 1) that each half takes part in, from the first on: half 0 sees
// fewer keys than half 1, and a half without tokens has no blocks.
EPTQ_HD void half_blocks(int seen, int tokens, int tokens_per_half, int kb, int block, int blocks, int (&count)[2]) {
    const int keys0 = seen + (tokens < tokens_per_half ? tokens : tokens_per_half);
    const int need0 = keys0 <= kb ? 1 : (keys0 + kb - 1) / kb, left0 = need0 - block;
    count[0] = left0 < 0 ? 0 : left0 < blocks ? left0 : blocks;
    count[1] = tokens > tokens_per_half ? blocks : 0;
}

// Whether a half that takes part in `count` blocks of an item waits for the scores of the first before it waits for any values.  A wait by
// parity tells only neighbouring fills of a ring's slot apart, so whoever waits for a fill has to know that the one before it has
// landed.  A half that took part in the block before knows it of all values but that block's: its last scores were formed behind them.  One
// that sat out blocks of the item before (all of them, where it has no tokens) may be any number of fills behind, and knows it only
// from the scores of its own next block, which are formed behind all earlier values.
EPTQ_HD bool scores_before_values(bool sat_out, int count) { return sat_out && count > 0; }

}  // namespace eptq
