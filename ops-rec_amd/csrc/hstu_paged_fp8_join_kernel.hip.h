// What follows a launch of the attention kernel over the 8-bit paged cache whose workgroups shared the keys of a tile, or the rows of a
// sequence: partial outputs, and partial sums of weights, added in a fixed order.
#pragma once
#include "hstu_paged_fp8_attend_kernel.hip.h"

namespace hstu {

// Adds the parts of tiles whose keys were dealt to several workgroups, in their order.  A workgroup per (pair, row tile).
template <typename Tag>
__global__ __launch_bounds__(256) void hstu_paged_fp8_join_kernel(const Fp8AttendArgs a, int tile_rows)
{
    const Fp8Cache& c = a.c;
    const int pair = static_cast<int>(blockIdx.x), tile = static_cast<int>(blockIdx.y);
    const int b = pair / c.n_heads, g = pair - b * c.n_heads;
    const Fp8Item item = fp8_item(a, b);
    const int64_t q0 = item.q0;
    const int n_pairs_rows = item.n_rows * a.ratio;
    const int m0 = tile * tile_rows, m1 = m0 + tile_rows < n_pairs_rows ? m0 + tile_rows : n_pairs_rows;
    if (m0 >= m1) {
        return;
    }
    const int n_blocks = fp8_runs(item.mask, div_small(m0, a.ratio), div_small(m1 - 1, a.ratio) + 1).count();
    int parts = (n_blocks + a.chunk - 1) / a.chunk;
    if (parts <= 1) {
        return;  // the one part has written the rows
    }
    parts = parts < a.parts ? parts : a.parts;
    const int dim = c.dim;
    const int64_t pitch = static_cast<int64_t>(tile_rows) * dim;
    const float* const from = a.partial + static_cast<int64_t>(pair * a.row_tiles + tile) * a.parts * pitch;
    uint16_t* const out = static_cast<uint16_t*>(a.out);
    const int pieces = dim >> 2;
    for (int x = threadIdx.x; x < (m1 - m0) * pieces; x += 256) {
        const int r = div_small(x, pieces), d = 4 * (x - r * pieces);
        f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int p = 0; p < parts; ++p) {
            sum += *reinterpret_cast<const f32x4_t*>(from + p * pitch + static_cast<int64_t>(r) * dim + d);
        }
        const int m = m0 + r, i = div_small(m, a.ratio);
        const int64_t at = ((q0 + i) * a.n_heads_q + g * a.ratio + (m - i * a.ratio)) * static_cast<int64_t>(dim) + d;
        u32x2_t w;
        w[0] = pack2<Tag>(sum[0] * a.c_out, sum[1] * a.c_out);
        w[1] = pack2<Tag>(sum[2] * a.c_out, sum[3] * a.c_out);
        *reinterpret_cast<u32x2_t*>(out + at) = w;
    }
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
