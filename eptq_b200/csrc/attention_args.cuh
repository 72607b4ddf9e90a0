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
    long long table_stride, table_keys;
    int rows, batch, n_heads, kv_group;      // kv_group: query heads per key/value head
    int heads_per_tile, tokens_per_half;     // heads that share a row tile; tokens of one 128-row half (or of the tile)
    int page_size, n_pages, table_width;
    float scale_log2;              // |scale| * log2(e)
    int negative;                  // scale is below zero
};

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace eptq
