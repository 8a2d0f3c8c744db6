// New key and value rows written into the 8-bit paged cache (gfx950).
//
// One workgroup per (block of 32 tokens that the call touches, key head, K or V, sequence).  It reads the
// new rows of its block and, in the first block of a sequence, the rows that are there already (decoded with the block's old
// scale); the largest finite magnitude of all of them gives the block's scale, a power of two, so that dividing by it rounds
// nothing, live rows move to a larger scale by a change of exponent alone (only what falls below the smallest normal code
// rounds), and writing the same rows again changes nothing.  The whole block is written: rows behind the new end are cleared.
//   K: 16 bytes of a row per lane, 8 codes out, at the row's place.
//   V: the block is stored with the tokens innermost (what the attention kernel's matrix instruction reads); a lane takes two
//      dims of 16 tokens, 4 bytes a load -- a wavefront's lanes read 256 bytes of a row together -- and has 16 bytes of each dim
//      to store, without an exchange between lanes.
// Bound by the bytes of the rows and codes.
#pragma once
#include "hstu_paged_fp8_common.hip.h"

namespace hstu {

template <typename Tag, int DS>
__global__ __launch_bounds__(kFp8AppendThreads) void hstu_paged_fp8_append_kernel(const Fp8AppendArgs a)
{
    constexpr int T = kFp8AppendThreads;
    constexpr int KP = kFp8Block * DS / 8 / T;     // 8-dim pieces per lane
    constexpr int VP = DS / T > 0 ? DS / T : 1;  // (dim pair, 16 tokens) units per lane
    __shared__ uint32_t s_top[kFp8AppendThreads / 64];

    const Fp8Cache& c = a.c;
    const int b = static_cast<int>(blockIdx.z), g = static_cast<int>(blockIdx.y >> 1);
    const Fp8Sequence seq = fp8_sequence(c, b);
    int64_t r0 = load_index_uniform(a.offs, b, c.idx64), r1 = load_index_uniform(a.offs, b + 1, c.idx64);
    r0 = r0 < 0 ? 0 : r0;
    r1 = r1 > a.total ? a.total : r1;
    r1 = r1 > r0 + a.max_rows ? r0 + a.max_rows : r1;
    const int room = fp8_room(c, seq.n_pages) - seq.len;
    int n_new = static_cast<int>(r1 > r0 ? r1 - r0 : 0);
    n_new = n_new < room ? n_new : room;
    const int blk = seq.len / kFp8Block + static_cast<int>(blockIdx.x);
    const int start = blk * kFp8Block, end = seq.len + n_new;
    if (n_new <= 0 || start >= end) {
        return;
    }
    const int lin = uniform(fp8_block(c, c.page_ids, seq.first, g, blk));
    if (lin < 0) {
        return;  // no such page: the rows have no place
    }
    const int live = seq.len > start ? seq.len - start : 0;            // rows of the block that are there already
    const int fill = end - start < kFp8Block ? end - start : kFp8Block;  // ... and that are there after the call
    const int64_t row0 = r0 + start - seq.len;                          // input row of the block's row 0 (only rows from `live` on exist)
    const int t = threadIdx.x;
    const int dim = c.dim;
    const int64_t codes_at = static_cast<int64_t>(lin) * kFp8Block * dim;

    if ((blockIdx.y & 1) == 0) {
        const uint16_t* const src = static_cast<const uint16_t*>(a.k) + static_cast<int64_t>(g) * a.k_head;
        uint8_t* const dst = c.k + codes_at;
        const float old_scale = live > 0 ? c.k_scale[lin] : 0.0f;
        const int cpr = dim >> 3, pieces = kFp8Block * cpr;
        float x[KP][8];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int p = t + i * T, row = div_small(p, cpr), col = (p - row * cpr) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[i][j] = 0.0f;
            }
            if (p < pieces && row >= live && row < fill) {
                const u32x4_t w = *reinterpret_cast<const u32x4_t*>(src + (row0 + row) * a.k_row + col);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[i][2 * j] = lo_to_float<Tag>(w[j]);
                    x[i][2 * j + 1] = hi_to_float<Tag>(w[j]);
                }
            } else if (p < pieces && row < live) {
                const u32x2_t w = *reinterpret_cast<const u32x2_t*>(dst + row * dim + col);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const f32x2_t lo = fp8_values2<false>(w[j]), hi = fp8_values2<true>(w[j]);
                    x[i][4 * j] = lo[0] * old_scale;
                    x[i][4 * j + 1] = lo[1] * old_scale;
                    x[i][4 * j + 2] = hi[0] * old_scale;
                    x[i][4 * j + 3] = hi[1] * old_scale;
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t m = finite_bits(x[i][j]);
                top = m > top ? m : top;
            }
        }
        const uint32_t field = fp8_scale_field(block_top<T / 64>(top, s_top));
        const float inverse = fp8_inverse_of(field);
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int p = t + i * T, row = div_small(p, cpr), col = (p - row * cpr) * 8;
            u32x2_t w;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t codes = fp8_codes2<false>(x[i][4 * j], x[i][4 * j + 1], inverse, 0u);
                w[j] = fp8_codes2<true>(x[i][4 * j + 2], x[i][4 * j + 3], inverse, codes);
            }
            if (p < pieces) {
                *reinterpret_cast<u32x2_t*>(dst + row * dim + col) = w;
            }
        }
        if (t == 0) {
            c.k_scale[lin] = fp8_scale_of(field);
        }
        if (c.weights != nullptr && t >= live && t < kFp8Block) {
            c.weights[static_cast<int64_t>(lin) * kFp8Block + t] = 0.0f;
        }
    } else {
        const uint16_t* const src = static_cast<const uint16_t*>(a.v) + static_cast<int64_t>(g) * a.v_head;
        uint8_t* const dst = c.v + codes_at;
        const float old_scale = live > 0 ? c.v_scale[lin] : 0.0f;
        const int pairs = dim >> 1;
        float x[VP][2][16];  // [unit][dim of the pair][token]
        uint32_t top = 0;
#pragma unroll
        for (int u = 0; u < VP; ++u) {
            const int n = t + u * T, half = n >= pairs ? 1 : 0, d = 2 * (n - half * pairs);
            const bool mine = n < 2 * pairs;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int row = 16 * half + i;
                x[u][0][i] = x[u][1][i] = 0.0f;
                if (mine && row >= live && row < fill) {
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(src + (row0 + row) * a.v_row + d);
                    x[u][0][i] = lo_to_float<Tag>(w);
                    x[u][1][i] = hi_to_float<Tag>(w);
                }
            }
            if (live > 16 * half && mine) {  // (the first block of a sequence only)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const u32x4_t w = *reinterpret_cast<const u32x4_t*>(dst + (d + e) * kFp8Block + 16 * half);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const f32x2_t lo = fp8_values2<false>(w[j]), hi = fp8_values2<true>(w[j]);
                        const float old[4] = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            x[u][e][4 * j + i] = 16 * half + 4 * j + i < live ? old[i] * old_scale : x[u][e][4 * j + i];
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t m0 = finite_bits(x[u][0][i]), m1 = finite_bits(x[u][1][i]);
                top = m0 > top ? m0 : top;
                top = m1 > top ? m1 : top;
            }
        }
        const uint32_t field = fp8_scale_field(block_top<T / 64>(top, s_top));
        const float inverse = fp8_inverse_of(field);
#pragma unroll
        for (int u = 0; u < VP; ++u) {
            const int n = t + u * T, half = n >= pairs ? 1 : 0, d = 2 * (n - half * pairs);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                u32x4_t w;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t codes = fp8_codes2<false>(x[u][e][4 * j], x[u][e][4 * j + 1], inverse, 0u);
                    w[j] = fp8_codes2<true>(x[u][e][4 * j + 2], x[u][e][4 * j + 3], inverse, codes);
                }
                if (n < 2 * pairs) {
                    *reinterpret_cast<u32x4_t*>(dst + (d + e) * kFp8Block + 16 * half) = w;
                }
            }
        }
        if (t == 0) {
            c.v_scale[lin] = fp8_scale_of(field);
        }
    }
}

}  // namespace hstu
