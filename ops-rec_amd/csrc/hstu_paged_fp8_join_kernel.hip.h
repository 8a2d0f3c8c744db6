// What follows a launch of the attention kernel over the 8-bit paged cache whose workgroups shared the keys of a tile, or the rows of a
// sequence: partial outputs, and partial sums of weights, added in a fixed order.
#pragma once
#include "hstu_paged_fp8_attend_kernel.hip.h"

namespace hstu {

// Adds the parts of tiles whose keys were dealt to several workgroups, in their order.  Four values of a row per thread; a workgroup
// per (256 of them, row tile, pair).
template <typename Tag>
__global__ __launch_bounds__(256) void hstu_paged_fp8_join_kernel(const Fp8AttendArgs a, int tile_rows)
{
    const Fp8Cache& c = a.c;
    const int pair = static_cast<int>(blockIdx.z), tile = static_cast<int>(blockIdx.y);
    const int b = uniform(pair / c.n_heads), g = pair - b * c.n_heads;
    const bool by_length = c.n_batch <= 64;
    Fp8DealLanes lanes = {a.chunk, 0, 0};
    int all_parts = a.parts, rank = 0;
    if (by_length) {
        lanes = fp8_deal_lanes(a);
        all_parts = __builtin_amdgcn_readlane(lanes.parts, b);
        rank = __builtin_amdgcn_readlane(lanes.rank, b);
    }
    const Fp8Item item = fp8_item(a, b);
    const int n_rows = item.n_rows * a.ratio;  // (row, head) pairs
    const int m0 = tile * tile_rows, m1 = m0 + tile_rows < n_rows ? m0 + tile_rows : n_rows;
    if (m0 >= m1 || all_parts == 1) {
        return;
    }
    const int n_blocks = fp8_runs(item.mask, div_small(m0, a.ratio), div_small(m1 - 1, a.ratio) + 1).count();
    int parts = uniform((n_blocks + lanes.chunk - 1) / lanes.chunk);
    parts = parts < all_parts ? parts : all_parts;
    if (parts <= 1) {
        return;  // (the one part has written the rows)
    }
    const int dim = c.dim, pieces = dim >> 2, x = static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x);
    const bool here = x < (m1 - m0) * pieces;  // (every lane takes part in finding the parts)
    const int64_t tile_words = static_cast<int64_t>(tile_rows) * dim, pitch = static_cast<int64_t>(c.n_heads) * a.row_tiles * tile_words;
    const float* const from = a.partial + (static_cast<int64_t>(g) * a.row_tiles + tile) * tile_words + (here ? 4 * x : 0);
    f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
    int before = 0;  // parts of all sequences ahead of the p-th ones
    for (int p0 = 0; p0 < parts; p0 += 8) {
        f32x4_t v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int p = p0 + i;
            const int slot = by_length ? before + rank : b * a.parts + p;
            before += by_length ? lanes.count(p) : 0;
            v[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (p < parts) {
                v[i] = *reinterpret_cast<const f32x4_t*>(from + slot * pitch);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sum += v[i];
        }
    }
    if (!here) {
        return;
    }
    const int r = div_small(x, pieces), d = 4 * (x - r * pieces), m = m0 + r, i = div_small(m, a.ratio);
    const int64_t at = ((item.q0 + i) * a.n_heads_q + g * a.ratio + (m - i * a.ratio)) * static_cast<int64_t>(dim) + d;
    u32x2_t w;
    w[0] = pack2<Tag>(sum[0] * a.c_out, sum[1] * a.c_out);
    w[1] = pack2<Tag>(sum[2] * a.c_out, sum[3] * a.c_out);
    *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(a.out) + at) = w;
}

// Adds the sums of |P| of several row tiles to the weights, in the order of the tiles.  A workgroup per (eight blocks, pair); a tile
// has left sums for the blocks that its rows see.
__global__ __launch_bounds__(256) void hstu_paged_fp8_weights_kernel(const Fp8AttendArgs a, int tile_rows, int tiles)
{
    const Fp8Cache& c = a.c;
    const int pair = static_cast<int>(blockIdx.y), blk = static_cast<int>(blockIdx.x) * 8 + static_cast<int>(threadIdx.x >> 5);
    const int b = pair / c.n_heads, g = pair - b * c.n_heads, key = threadIdx.x & 31;
    const Fp8Item item = fp8_item(a, b);
    const int n_pairs_rows = item.n_rows * a.ratio;
    if (blk * kFp8Block >= item.seq.len) {
        return;
    }
    float sum = 0.0f;
    for (int t = 0; t < tiles && t * tile_rows < n_pairs_rows; ++t) {
        const int m0 = t * tile_rows, m1 = m0 + tile_rows < n_pairs_rows ? m0 + tile_rows : n_pairs_rows;
        const Fp8Runs r = fp8_runs(item.mask, div_small(m0, a.ratio), div_small(m1 - 1, a.ratio) + 1);
        if (blk < r.n_a || (blk >= r.b0 && blk < r.b0 + r.n_b) || (blk >= r.c0 && blk < r.c0 + r.n_c)) {
            sum += a.weight_partial[((static_cast<int64_t>(pair) * tiles + t) * a.max_blocks + blk) * kFp8Block + key];
        }
    }
    const int lin = fp8_block(c, c.page_ids, item.seq.first, g, blk);
    if (lin >= 0) {
        unsafeAtomicAdd(c.weights + static_cast<int64_t>(lin) * kFp8Block + key, sum);  // (a page may be in two sequences)
    }
}

}  // namespace hstu
