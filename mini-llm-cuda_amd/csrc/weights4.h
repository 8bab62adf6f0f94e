// Matrices of 4-bit codes (mlh_weights4): where their bytes lie.
//
// 16 rows x 128 columns are a tile, the tiles of 16 rows lie one behind the other.  A tile is what 64 lanes load as 16 bytes each: lane l holds row l % 16, and of each
// of the tile's four steps of 32 columns the eight from 8 * (l / 16) on, one word a step.  Column 2j of the eight stands in bits 4j + 3 to 4j + 6
// of the word and column 2j + 1 sixteen bits higher (bits behind the last go on at bit 0), so that one mask takes a pair of neighbours to the two halves of a word, where the matrix instructions want
// them, and to the place in a half that w4_pair needs.  Behind the 1024 bytes of codes stand 16 rows of
// 128 / group (minimum, scale) pairs.  Rows behind N and columns behind K are zero.
#pragma once
#include "kv_cache.h"

#define W4_ROWS 16
#define W4_COLS 128
#define W4_CODES (W4_ROWS * W4_COLS / 2)
__host__ __device__ constexpr int w4_groups(int group) { return W4_COLS / group; } // of a tile
__host__ __device__ constexpr int w4_tile(int group) { return W4_CODES + W4_ROWS * w4_groups(group) * 4; } // bytes of it
__host__ __device__ constexpr int w4_tiles(int K) { return (K + W4_COLS - 1) / W4_COLS; } // of a row
// eight codes in the order of their columns, a nibble each, <-> that word
__host__ __device__ inline uint32_t w4_spread(uint32_t x) {
    uint32_t y = 0;
    for (int j = 0; j < 4; j++) y |= (x >> (8 * j) & 15u) << (4 * j) | (x >> (8 * j + 4) & 15u) << (4 * j + 16);
    return y << 3 | y >> 29;
}
__host__ __device__ inline uint32_t w4_gather(uint32_t y) {
    uint32_t x = 0;
    y = y >> 3 | y << 29;
    for (int j = 0; j < 4; j++) x |= (y >> (4 * j) & 15u) << (8 * j) | (y >> (4 * j + 16) & 15u) << (8 * j + 4);
    return x;
}
