// What follows a launch of the attention kernel over the 8-bit paged cache whose workgroups shared the keys of a tile, or the rows of a
// sequence: partial outputs, and partial sums of weights, added in a fixed order.
#pragma once
#include "hstu_paged_fp8_attend_kernel.hip.h"

namespace hstu {

// Adds the parts of tiles whose keys were dealt to several workgroups, in a fixed order.  Four values of a row per lane, a workgroup
// for every gridDim.x-th so many of a (row tile, pair).  Where a value has many parts, which is where there are few values, the four
// wavefronts take a quarter of the parts each.  Bound by the latency of two loads, the record that the attention kernel has left of a
// tile's parts and the parts, so there are hardly more workgroups than run at once: 64 pairs of 8 tiles of 128 x 128, the half of them in
// two parts, 11 us, and 22 in 8192 workgroups that found the parts for themselves; 128 pairs of one tile 6, and 9 in twice as many.
template <typename Tag>
__global__ __launch_bounds__(256) void hstu_paged_fp8_join_kernel(const Fp8AttendArgs a, int tile_rows)
{
    __shared__ f32x4_t s_sum[3][64];
    const Fp8Cache& c = a.c;
    const int pair = static_cast<int>(blockIdx.z), tile = static_cast<int>(blockIdx.y);
    const int b = uniform(pair / c.n_heads), g = pair - b * c.n_heads;
    const int2 join = a.joins[pair * a.row_tiles + tile];
    const Fp8Item item = fp8_item(a, b);
    const int n_rows = item.n_rows * a.ratio;  // (row, head) pairs
    const int m0 = (a.tile_first + tile) * tile_rows, m1 = m0 + tile_rows < n_rows ? m0 + tile_rows : n_rows, parts = uniform(join.x);
    if (m0 >= m1 || parts <= 1) {
        return;  // (no rows, of which nothing stands in joins, or the one part has written them)
    }
    const int dim = c.dim, pieces = dim >> 2, n_pieces = (m1 - m0) * pieces;
    const bool quarters = parts > 4;
    const int wave = uniform(static_cast<int>(threadIdx.x) >> 6), lane = threadIdx.x & 63;
    const int share = quarters ? (parts + 3) >> 2 : parts, first = quarters ? wave * share : 0;
    const int last = first + share < parts ? first + share : parts;
    const int step = quarters ? 64 : 256, mine = quarters ? lane : static_cast<int>(threadIdx.x);
    const int64_t tile_words = static_cast<int64_t>(tile_rows) * dim, pitch = static_cast<int64_t>(c.n_heads) * a.row_tiles * tile_words;
    const float* const tile_at = a.partial + uniform(join.y) * pitch + (static_cast<int64_t>(g) * a.row_tiles + tile) * tile_words;
    for (int x0 = static_cast<int>(blockIdx.x) * step; x0 < n_pieces; x0 += static_cast<int>(gridDim.x) * step) {
        const int x = x0 + mine;
        const bool here = x < n_pieces;
        const float* const from = tile_at + (here ? 4 * x : 0);
        f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int p0 = first; p0 < last; p0 += 8) {
            f32x4_t v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int p = p0 + i;
                v[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
                if (p < last) {
                    v[i] = *reinterpret_cast<const f32x4_t*>(from + p * pitch);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum += v[i];
            }
        }
        if (quarters) {
            __syncthreads();  // (read by the first wavefront in the turn before)
            if (wave > 0) {
                s_sum[wave - 1][lane] = sum;
            }
            __syncthreads();
            if (wave == 0) {
                sum = ((sum + s_sum[0][lane]) + s_sum[1][lane]) + s_sum[2][lane];
            }
        }
        if (here && (wave == 0 || !quarters)) {
            const int r = div_small(x, pieces), d = 4 * (x - r * pieces), m = m0 + r, i = div_small(m, a.ratio);
            const int64_t at = ((item.q0 + i) * a.n_heads_q + g * a.ratio + (m - i * a.ratio)) * static_cast<int64_t>(dim) + d;
            u32x2_t w;
            w[0] = pack2<Tag>(sum[0] * a.c_out, sum[1] * a.c_out);
            w[1] = pack2<Tag>(sum[2] * a.c_out, sum[3] * a.c_out);
            *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(a.out) + at) = w;
        }
    }
}

// Adds the sums of |P| of the launch's row tiles, of 32 rows each, to the weights, in the order of the tiles.  A workgroup per (eight
// blocks, pair); a tile has left sums for the blocks that its rows see.
__global__ __launch_bounds__(256) void hstu_paged_fp8_weights_kernel(const Fp8AttendArgs a)
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
    for (int t = 0; t < a.row_tiles && (a.tile_first + t) * kFp8KeysRows < n_pairs_rows; ++t) {
        const int m0 = (a.tile_first + t) * kFp8KeysRows, m1 = m0 + kFp8KeysRows < n_pairs_rows ? m0 + kFp8KeysRows : n_pairs_rows;
        const Fp8Runs r = fp8_runs(item.mask, div_small(m0, a.ratio), div_small(m1 - 1, a.ratio) + 1);
        if (blk < r.n_a || (blk >= r.b0 && blk < r.b0 + r.n_b) || (blk >= r.c0 && blk < r.c0 + r.n_c)) {
            sum += a.weight_partial[((static_cast<int64_t>(pair) * a.row_tiles + t) * a.max_blocks + blk) * kFp8Block + key];
        }
    }
    const int lin = fp8_block(c, c.page_ids, item.seq.first, g, blk);
    if (lin >= 0) {
        unsafeAtomicAdd(c.weights + static_cast<int64_t>(lin) * kFp8Block + key, sum);  // (a page may be in two sequences)
    }
}

}  // namespace hstu
