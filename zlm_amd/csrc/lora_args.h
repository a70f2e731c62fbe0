// lora_args.h -- the argument block of the adapter kernels (zlm_lora.hip), shared with the
// host library that fills it.
#pragma once
#include <stdint.h>

namespace zlm {

constexpr uint32_t kLoraAdapters = 4096;  // of one pool (the grouping counts their tokens in LDS)
constexpr uint32_t kLoraRank = 256;
constexpr uint32_t kLoraOwn = 256;        // tokens that a workgroup groups by itself
constexpr uint32_t kLoraTiles[2] = {32, 16};  // tokens of a tile, of many tokens and of few
// Waves of the first product's workgroups, and runs of 32 of k that each has in flight (at
// most), with tiles of 16 tokens and of 32.
constexpr uint32_t kLoraWaves[2] = {8, 4}, kLoraRuns[2] = {4, 2};

// Tokens order[first .. first + n) have one adapter (kLoraAdapters and above: none).
struct LoraTile {
    uint32_t adapter, first, n;
};

struct LoraArgs {
    const void* a;  // n_adapters x rank x k
    const void* b;  // n_adapters x rows x rank
    const int32_t* adapter;  // of each token
    const int32_t* ranks;    // null: all `rank`
    const float* scales;     // null: 1
    const float* x;
    const float* res;        // null: 0
    float* y;
    uint64_t x_stride, y_stride;
    uint32_t n_adapters, rank, rows, k, n_tokens;
    uint32_t tiles;   // of the grid: a bound of their number
    uint32_t per_tile;  // tokens, of kLoraTiles
    uint32_t splits;  // of k over workgroups
    uint32_t wave_rows;  // of y, that a wave of the second product takes
    uint32_t in_place, vectors;  // y is res; rows of y and res go by 16 bytes
    float* part;      // splits x tiles x tokens of a tile x rank: A x
    uint32_t* order;  // what the grouping leaves (more than kLoraOwn tokens)
    LoraTile* tile;
    uint32_t* n_tiles;
};

}  // namespace zlm
