// New key and value rows written into the 8-bit paged cache (gfx950).
//
// One workgroup per (block of 32 tokens that the call touches, key head, K or V, sequence).  It reads the new rows of the block and, in
// the first block of a sequence, the rows that are there already (decoded with the block's old scale); the largest finite magnitude of
// all of them gives the block's scale, a power of two, so that dividing by it rounds nothing, live rows move to a larger scale by a
// change of exponent alone (only what falls below the smallest normal code rounds), and writing the same rows again changes nothing.
// The whole block is written: rows behind the new end are cleared.
//   K: 16 bytes of a row per lane, 8 codes out, at the row's place.
//   V: the block is stored with the tokens innermost (what the attention kernel's matrix instruction reads); a lane takes two
//      dims of 16 tokens, 4 bytes a load -- a wavefront's lanes read 256 bytes of a row together -- and has 16 bytes of each dim
//      to store, without an exchange between lanes.
// Blocks without older rows stay 16-bit words: an instruction converts two values and divides by the scale, two more find the largest
// of two; blocks with them are added up in fp32.  Bound by the bytes of the rows and codes (72000 f16 rows, 8 key heads, 128 dims: 446 MB in
// 86 us; 136 when all values went through fp32; two to four blocks a workgroup, the next one's rows on their way, 90 to 95).
#pragma once
#include "hstu_paged_fp8_common.hip.h"

namespace hstu {

// a row of a block that the call brings rows [live, fill) of
__device__ __forceinline__ int clamp_row(int row, int live, int fill) { return row < live ? live : (row < fill ? row : fill - 1); }

template <typename Tag, int DS>
__global__ __launch_bounds__(kFp8AppendThreads) void hstu_paged_fp8_append_kernel(const Fp8AppendArgs a)
{
    constexpr int T = kFp8AppendThreads;
    constexpr int KP = kFp8Block * DS / 8 / T;     // 8-dim pieces per lane
    constexpr int VP = DS / T > 0 ? DS / T : 1;  // (dim pair, 16 tokens) units per lane
    __shared__ uint32_t s_top[T / 64];

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
    const int blk = seq.len / kFp8Block + static_cast<int>(blockIdx.x), start = blk * kFp8Block, end = seq.len + n_new;
    if (n_new <= 0 || start >= end) {
        return;
    }
    const int t = threadIdx.x, dim = c.dim;
    // the block's rows that are there before and after the call, and the input row of its row 0
    const int live = seq.len > start ? seq.len - start : 0, fill = end - start < kFp8Block ? end - start : kFp8Block;
    const int64_t row0 = r0 + start - seq.len;
    const int lin = uniform(fp8_block(c, c.page_ids, seq.first, g, blk));
    const bool old = live > 0 && lin >= 0;

    if ((blockIdx.y & 1) == 0) {
        const uint16_t* const src = static_cast<const uint16_t*>(a.k) + static_cast<int64_t>(g) * a.k_head;
        const int cpr = dim >> 3, pieces = kFp8Block * cpr;
        int rows[KP], cols[KP];
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int p = t + i * T, row = div_small(p, cpr);
            rows[i] = p < pieces ? row : kFp8Block;  // (of no block)
            cols[i] = (p - row * cpr) * 8;
        }
        uint8_t* const dst = c.k + static_cast<int64_t>(lin < 0 ? 0 : lin) * kFp8Block * dim;
        u32x4_t raw[KP];
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            raw[i] = *reinterpret_cast<const u32x4_t*>(src + (row0 + clamp_row(rows[i], live, fill)) * a.k_row + cols[i]);
            if (fill < kFp8Block && rows[i] >= fill) {
                raw[i] = u32x4_t{0u};
            }
        }
        u32x2_t was[KP];
        float old_scale = 0.0f;
        if (old) {
            old_scale = c.k_scale[lin];
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                was[i] = *reinterpret_cast<const u32x2_t*>(dst + (rows[i] < live ? rows[i] * dim + cols[i] : 0));
            }
        }
        u32x2_t w[KP];
        uint32_t field;
        if (old) {  // with the rows that are there, in fp32
            float x[KP][8];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < KP; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[i][2 * j] = lo_to_float<Tag>(raw[i][j]);
                    x[i][2 * j + 1] = hi_to_float<Tag>(raw[i][j]);
                }
                if (rows[i] < live) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const f32x2_t lo = fp8_values2<false>(was[i][j]), hi = fp8_values2<true>(was[i][j]);
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
            field = fp8_scale_field(block_top<T / 64>(top, s_top));
            const float inverse = fp8_inverse_of(field);
#pragma unroll
            for (int i = 0; i < KP; ++i) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t codes = fp8_codes2<false>(x[i][4 * j], x[i][4 * j + 1], inverse, 0u);
                    w[i][j] = fp8_codes2<true>(x[i][4 * j + 2], x[i][4 * j + 3], inverse, codes);
                }
            }
        } else {
            FiniteTop<Tag> top;
#pragma unroll
            for (int i = 0; i < KP; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t word = raw[i][j];
                    top.take(word);
                }
            }
            field = fp8_scale_field(block_top<T / 64>(top.bits(), s_top));
            const float scale = fp8_scale_of(field);
#pragma unroll
            for (int i = 0; i < KP; ++i) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t a0 = raw[i][2 * j], a1 = raw[i][2 * j + 1];
                    w[i][j] = fp8_codes2<Tag, true>(a1, scale, fp8_codes2<Tag, false>(a0, scale, 0u));
                }
            }
        }
        if (field == kFp8TopField) {
#pragma unroll
            for (int i = 0; i < KP; ++i) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    w[i][j] = fp8_below_infinity(w[i][j]);
                }
            }
        }
        if (lin >= 0) {  // (otherwise there is no such page: the rows have no place)
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                if (rows[i] < kFp8Block) {
                    *reinterpret_cast<u32x2_t*>(dst + rows[i] * dim + cols[i]) = w[i];
                }
            }
            if (t == 0) {
                c.k_scale[lin] = fp8_scale_of(field);
            }
            if (c.weights != nullptr && t >= live && t < kFp8Block) {
                c.weights[static_cast<int64_t>(lin) * kFp8Block + t] = 0.0f;
            }
        }
    } else {
        const uint16_t* const src = static_cast<const uint16_t*>(a.v) + static_cast<int64_t>(g) * a.v_head;
        const int pairs = dim >> 1;
        int halves[VP], dims[VP];
#pragma unroll
        for (int u = 0; u < VP; ++u) {
            const int m = t + u * T;
            halves[u] = m >= pairs ? (m < 2 * pairs ? 16 : 2 * kFp8Block) : 0;  // first of the 16 tokens
            dims[u] = m >= 2 * pairs ? 0 : 2 * (m >= pairs ? m - pairs : m);
        }
        uint8_t* const dst = c.v + static_cast<int64_t>(lin < 0 ? 0 : lin) * kFp8Block * dim;
        uint32_t raw[VP][16];
#pragma unroll
        for (int u = 0; u < VP; ++u) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int row = halves[u] + i;
                raw[u][i] = *reinterpret_cast<const uint32_t*>(src + (row0 + clamp_row(row, live, fill)) * a.v_row + dims[u]);
                if (fill < kFp8Block && row >= fill) {
                    raw[u][i] = 0u;
                }
            }
        }
        u32x4_t was[VP][2];
        float old_scale = 0.0f;
        if (old) {
            old_scale = c.v_scale[lin];
#pragma unroll
            for (int u = 0; u < VP; ++u) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    was[u][e] = *reinterpret_cast<const u32x4_t*>(dst + (dims[u] + e) * kFp8Block + (halves[u] & 16));
                }
            }
        }
        u32x4_t w[VP][2];
        uint32_t field;
        if (old) {
            float x[VP][2][16];  // [unit][dim of the pair][token]
            uint32_t top = 0;
#pragma unroll
            for (int u = 0; u < VP; ++u) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    x[u][0][i] = lo_to_float<Tag>(raw[u][i]);
                    x[u][1][i] = hi_to_float<Tag>(raw[u][i]);
                }
                if (halves[u] < live) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const f32x2_t lo = fp8_values2<false>(was[u][e][j]), hi = fp8_values2<true>(was[u][e][j]);
                            const float had[4] = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                x[u][e][4 * j + i] = halves[u] + 4 * j + i < live ? had[i] * old_scale : x[u][e][4 * j + i];
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
            field = fp8_scale_field(block_top<T / 64>(top, s_top));
            const float inverse = fp8_inverse_of(field);
#pragma unroll
            for (int u = 0; u < VP; ++u) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t codes = fp8_codes2<false>(x[u][e][4 * j], x[u][e][4 * j + 1], inverse, 0u);
                        w[u][e][j] = fp8_codes2<true>(x[u][e][4 * j + 2], x[u][e][4 * j + 3], inverse, codes);
                    }
                }
            }
        } else {
            FiniteTop<Tag> top;
#pragma unroll
            for (int u = 0; u < VP; ++u) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    top.take(raw[u][i]);
                }
            }
            field = fp8_scale_field(block_top<T / 64>(top.bits(), s_top));
            const float scale = fp8_scale_of(field);
#pragma unroll
            for (int u = 0; u < VP; ++u) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // four tokens: codes of both dims of two and two, then of one dim of all four
                    const uint32_t ab = fp8_codes2<Tag, true>(raw[u][4 * j + 1], scale, fp8_codes2<Tag, false>(raw[u][4 * j], scale, 0u));
                    const uint32_t cd = fp8_codes2<Tag, true>(raw[u][4 * j + 3], scale, fp8_codes2<Tag, false>(raw[u][4 * j + 2], scale, 0u));
                    w[u][0][j] = __builtin_amdgcn_perm(cd, ab, 0x06040200u);
                    w[u][1][j] = __builtin_amdgcn_perm(cd, ab, 0x07050301u);
                }
            }
        }
        if (field == kFp8TopField) {
#pragma unroll
            for (int u = 0; u < VP; ++u) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        w[u][e][j] = fp8_below_infinity(w[u][e][j]);
                    }
                }
            }
        }
        if (lin >= 0) {
#pragma unroll
            for (int u = 0; u < VP; ++u) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (halves[u] < kFp8Block) {
                        *reinterpret_cast<u32x4_t*>(dst + (dims[u] + e) * kFp8Block + halves[u]) = w[u][e];
                    }
                }
            }
            if (t == 0) {
                c.v_scale[lin] = fp8_scale_of(field);
            }
        }
    }
}

}  // namespace hstu
