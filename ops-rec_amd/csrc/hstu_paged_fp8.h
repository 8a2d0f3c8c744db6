// Argument blocks and constants of the kernels of the 8-bit paged cache, shared with the host side (no device code here).
#pragma once
#include <stdint.h>

namespace hstu {

constexpr int kFp8Block = 32;         // tokens that share a scale, and keys of one step of the attention kernel
constexpr int kFp8MostKeys = 1 << 24; // rows of a sequence in the cache, at most (what places are found by is exact up to there)
constexpr int kFp8MostSlots = 1 << 22;  // workgroups of an attention launch, of up to 512 threads: a grid has less than 2^32 threads
// Of partial sums of weights in the workspace of a call, at most.  Where a row tile's take more than half of it a launch takes one tile, which
// keeps none; the parts of its keys are still those for all tiles at once.
constexpr int64_t kFp8WeightBytes = int64_t{512} << 20;
constexpr int kFp8JoinEnough = 1024;  // workgroups of the joins that fill the machine
constexpr int kFp8AppendThreads = 128;
constexpr int kFp8SelectKeys = 32768;   // scores that the selecting kernel holds in LDS
constexpr int kFp8SelectFew = 1024;     // longest sequence of its variant with few threads

// The cache of one layer, and whose pages are whose.
struct Fp8Cache {
    uint8_t* k;       // [num_pages][n_heads][blocks_per_page][32][dim]
    uint8_t* v;       // [num_pages][n_heads][blocks_per_page][dim][32]
    float* k_scale;   // [num_pages][n_heads][blocks_per_page], powers of two
    float* v_scale;
    float* weights;   // [num_pages][n_heads][blocks_per_page * 32], or null
    const void* cache_len;     // [n_batch]
    const void* page_offsets;  // [n_batch + 1]
    const void* page_ids;      // [n_page_ids]
    int n_batch;
    int n_heads;
    int dim;
    int blocks_per_page;
    int num_pages;
    int n_page_ids;
    int idx64;
};

struct Fp8AttendArgs {
    Fp8Cache c;
    const void* q;
    const void* offs_q;
    const void* num_target;  // or null
    void* out;
    float* partial;         // [total_parts * n_heads][row_tiles][rows of a tile][dim], where there are parts
    int2* joins;            // [n_batch * n_heads][row_tiles] how many parts a tile was done in, and the first of them; where there are parts
    float* weight_partial;  // [n_batch * n_heads][row_tiles][max_blocks * 32], for weights over more than one row tile
    int64_t total_q;
    int n_heads_q;
    int ratio;  // query heads per key / value head
    int max_q;
    int max_k;
    int group;
    int window;  // 0: none
    int sinks;
    int row_tiles;    // of a (sequence, key head) pair that the launch takes, at most
    int tile_first;   // the first of them
    int total_parts;  // the keys of the sequences are dealt to so many parts in all; 0: a sequence is one part
    int parts;        // of each sequence, where they are not dealt by length (more than 64 sequences)
    int chunk;        // blocks of a part: at least (dealt by length), or exactly
    int most_blocks;  // that a row tile sweeps, but for targets behind a window, which may see more (the last part of a tile takes what is left)
    int max_blocks;  // pitch of weight_partial, in blocks
    float c_exp;     // -alpha * log2(e): silu(alpha s) = alpha * s / (1 + 2^(c_exp s))
    float c_out;     // alpha * silu_scale
};

struct Fp8AppendArgs {
    Fp8Cache c;
    const void* k;
    const void* v;
    const void* offs;
    int64_t total;
    int64_t k_row, k_head, v_row, v_head;  // strides, in elements
    int max_rows;
};

struct Fp8EvictArgs {
    Fp8Cache c;
    const void* new_page_offsets;
    const void* new_page_ids;
    void* new_len;    // [n_batch], of the index type
    void* kept;       // [n_batch][keep], of the index type
    uint32_t* keys;   // workspace [n_batch][key_pitch], for more scores than fit LDS: in an order that compares as integers
    int64_t key_pitch;
    int n_new_page_ids;
    int max_k;
    int keep;
    int sinks;
    int recent;
};

}  // namespace hstu
