// Attention over the paged cache: what its two kernels share.
#pragma once
#include "paged.cuh"

namespace nats {

struct PagedAttnParams {
    PagedKv kv;
    const __nv_bfloat16* q;
    long long q_slot, q_head, q_token;           // strides in elements
    void* o;
    long long o_slot, o_head, o_token;
    int o_f32;
    const int32_t* n_new;                        // [S] or nullptr: N everywhere
    int N, G;
    int splits;                                  // of the pages of a row
    int split_pages;                             // pages per split (rows kernel)
    int row_tiles;                               // tiles of query rows per (slot, kv-head)
    float scale_log2;
    int32_t* tickets;
    int32_t* counter;                            // next work item (tile kernel)
    float* partials;
    int32_t* status;
};

// Tile kernel: query rows of a tile are 128 / G tokens with their G heads each
inline int tile_tokens(int G) { return kTile / G; }
constexpr int kTileMaxPages = 4096;              // pages that a work item looks at
int launch_paged_tiles(const PagedAttnParams& p, cudaStream_t st);
size_t paged_tile_partial_floats(int S, int Hq, int N, int D, int splits);

}  // namespace nats
