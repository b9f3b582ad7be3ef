// What the kernels of the requests' adapters share.
//
// Rows go by tiles: `tiles[t]` = (adapter, place, count) names `count` rows of one adapter, those at
// order[place], order[place + 1], ...; adapter `n` stands for "none", an adapter of -1 for no tile.
#pragma once

#include "common.cuh"

namespace adapters {

struct Tile {
    int adapter, place, count;
};

__device__ __forceinline__ Tile load_tile(const int* __restrict__ tiles, int t) {
    return Tile{tiles[3 * t], tiles[3 * t + 1], tiles[3 * t + 2]};
}

constexpr int MAX_PARTS = 8;

// The projection's columns by parts, each with an A of its own: parts side by side (part s is columns
// [end[s - 1], end[s])), or two parts woven (column 2 j + s is column j of part s).
struct Parts {
    int n, woven;
    int end[MAX_PARTS];
    __host__ __device__ __forceinline__ int part_of(int col) const {
        if (woven) return col & 1;
        int s = 0;
        while (s + 1 < n && col >= end[s]) ++s;
        return s;
    }
};

// The arguments of out = base + scale_a B_a (A_a x), rows' adapters from the tiles.
struct Args {
    const void* base;      // [R, N], rows ld_base apart
    void* out;             // [R, N], rows ld_out apart; may be `base`
    const void* x;         // [R, K], rows ld_x apart
    const void* a;         // [n, parts, rank, lda]
    const void* b;         // [n, N, rank]
    const float* scale;    // [n]
    const int* ranks;      // [n]: rank rows that are not zero, or null: all
    const int* order;      // [R]
    const int* tiles;      // [max_tiles][3]
    float* low;            // scratch
    long long ld_base, ld_out, ld_x;
    int n, R, K, lda, N, rank, max_tiles, tile;
    Parts parts;
    __device__ __forceinline__ int rank_of(int adapter) const {
        return ranks ? max(0, min(rank, ranks[adapter])) : rank;
    }
};

// tiles of 16 rows, bfloat16 (adapters_step.cu)
bool step_takes(const Args& p);
int step_form(const Args& p, int dt_out, cudaStream_t s);
// tiles of 128 rows, bfloat16 (adapters_prompt.cu)
bool prompt_takes(const Args& p, int dt_out);
long long prompt_low_floats(int R, int W);
int prompt_form(const Args& p, int dt_out, int* err, cudaStream_t s);

}  // namespace adapters
