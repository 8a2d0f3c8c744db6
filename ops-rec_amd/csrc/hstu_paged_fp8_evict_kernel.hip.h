// Eviction from the 8-bit paged cache by accumulated attention weights (gfx950): which rows of a sequence stay, and their move to
// other pages.
#pragma once
#include "hstu_paged_fp8_common.hip.h"

namespace hstu {

// A score as an integer that compares as the score does (larger is larger): NaN below everything, the two zeros the same.
__device__ __forceinline__ uint32_t score_key(float s)
{
    if (s != s) {
        return 0u;
    }
    const uint32_t bits = __builtin_bit_cast(uint32_t, s + 0.0f);
    return (bits & 0x80000000u) != 0 ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ void store_index(void* p, int64_t i, int64_t value, int idx64)
{
    if (idx64) {
        static_cast<int64_t*>(p)[i] = value;
    } else {
        static_cast<int32_t*>(p)[i] = static_cast<int32_t>(value);
    }
}

// How many rows of a sequence stay, and how many of them stay whatever their score.
struct Fp8Budget {
    int len, keep, sinks, recent;
};
__device__ __forceinline__ Fp8Budget fp8_budget(const Fp8EvictArgs& a, const Fp8Sequence& seq, int new_pages)
{
    Fp8Budget r;
    r.len = seq.len < a.max_k ? seq.len : a.max_k;
    const int room = fp8_room(a.c, new_pages);
    int n = r.len < a.keep ? r.len : a.keep;
    r.keep = n < room ? n : room;
    r.sinks = r.keep < a.sinks ? r.keep : a.sinks;
    const int rest = r.keep - r.sinks;
    r.recent = rest < a.recent ? rest : a.recent;
    return r;
}

// One workgroup per sequence.  A row's score is the sum of its weights over the key heads, in their order, in fp32.  The keep-th
// largest among the rows that are not kept anyway is found by its bits, eight at a time from the top (four histograms in LDS
// over the scores, which stay where the first pass left them); rows above it stay, and of those equal to it the first few.  The
// kept rows' indices are written in order.
__global__ __launch_bounds__(kFp8SelectThreads) void hstu_paged_fp8_select_kernel(const Fp8EvictArgs a)
{
    constexpr int T = kFp8SelectThreads, WAVES = T / 64;
    __shared__ uint32_t s_hist[256];
    __shared__ uint32_t s_above[2][WAVES], s_equal[2][WAVES];
    __shared__ uint32_t s_pick[2];

    const Fp8Cache& c = a.c;
    const int b = static_cast<int>(blockIdx.x), tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63;
    const Fp8Sequence seq = fp8_sequence(c, b);
    const Fp8Sequence to = fp8_pages(a.new_page_offsets, a.n_new_page_ids, c.idx64, b);
    const Fp8Budget n = fp8_budget(a, seq, to.n_pages);
    const int64_t kept = static_cast<int64_t>(b) * a.keep;
    if (tid == 0) {
        store_index(a.new_len, b, n.keep, c.idx64);
    }
    for (int i = n.keep + tid; i < a.keep; i += T) {
        store_index(a.kept, kept + i, -1, c.idx64);
    }
    if (n.keep == n.len) {
        for (int i = tid; i < n.keep; i += T) {
            store_index(a.kept, kept + i, i, c.idx64);
        }
        return;
    }
    // rows [sinks, len - recent) compete for the places left; there are fewer places than rows
    const int lo = n.sinks, hi = n.len - n.recent;
    const int places = n.keep - n.sinks - n.recent;
    uint32_t* const keys = a.keys + static_cast<int64_t>(b) * a.max_k;
    const int64_t head_pitch = static_cast<int64_t>(c.blocks_per_page) * kFp8Block;
    for (int j = lo + tid; j < hi; j += T) {
        const int lin = fp8_block(c, c.page_ids, seq.first, 0, j / kFp8Block);
        float score = 0.0f;
        if (lin >= 0) {
            const float* const w = c.weights + static_cast<int64_t>(lin) * kFp8Block + (j & (kFp8Block - 1));
            score = w[0];
            for (int h = 1; h < c.n_heads; ++h) {
                score += w[h * head_pitch];
            }
        }
        keys[j] = score_key(score);
    }
    uint32_t prefix = 0, left = static_cast<uint32_t>(places);  // of the rows whose top bits are `prefix`, `left` stay
    if (places > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += T) {
                s_hist[i] = 0;
            }
            __syncthreads();
            for (int j = lo + tid; j < hi; j += T) {
                const uint32_t k = keys[j];
                if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) {
                    atomicAdd(&s_hist[(k >> shift) & 255u], 1u);
                }
            }
            __syncthreads();
            if (wave == 0) {
                // lane l has the digits 255 - 4 l .. 252 - 4 l: counts from the top
                uint32_t mine[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    mine[i] = s_hist[255 - 4 * lane - i];
                    sum += mine[i];
                }
                uint32_t before = sum;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const uint32_t up = static_cast<uint32_t>(__shfl_up(static_cast<int>(before), d, 64));
                    before += lane >= d ? up : 0u;
                }
                before -= sum;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (before < left && before + mine[i] >= left) {  // (true for one digit of one lane)
                        s_pick[0] = static_cast<uint32_t>(255 - 4 * lane - i);
                        s_pick[1] = left - before;
                    }
                    before += mine[i];
                }
            }
            __syncthreads();
            prefix |= s_pick[0] << shift;
            left = s_pick[1];
        }
    }
    // rows above `prefix` stay, and the first `left` of those equal to it; none where there are no places
    const uint32_t none = places > 0 ? 0u : 1u;
    uint32_t n_kept = static_cast<uint32_t>(n.sinks), n_equal = 0;
    for (int i = tid; i < n.sinks; i += T) {
        store_index(a.kept, kept + i, i, c.idx64);
    }
    int turn = 0;
    for (int base = lo; base < hi && none == 0; base += T, turn ^= 1) {
        const int j = base + tid;
        const uint32_t k = j < hi ? keys[j] : 0u;
        const bool above = j < hi && k > prefix, equal = j < hi && k == prefix;
        const uint64_t m_above = __ballot(above), m_equal = __ballot(equal);
        if (lane == 0) {
            s_above[turn][wave] = static_cast<uint32_t>(__popcll(m_above));
            s_equal[turn][wave] = static_cast<uint32_t>(__popcll(m_equal));
        }
        __syncthreads();
        uint32_t a_before = 0, e_before = 0, a_all = 0, e_all = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            a_before += w < wave ? s_above[turn][w] : 0u;
            e_before += w < wave ? s_equal[turn][w] : 0u;
            a_all += s_above[turn][w];
            e_all += s_equal[turn][w];
        }
        const uint64_t below = (uint64_t{1} << lane) - 1;
        const uint32_t a_rank = a_before + static_cast<uint32_t>(__popcll(m_above & below));
        const uint32_t e_rank = n_equal + e_before + static_cast<uint32_t>(__popcll(m_equal & below));
        const uint32_t e_kept = (e_rank < left ? e_rank : left) - (n_equal < left ? n_equal : left);  // equal rows of this turn that stay, before mine
        if (above || (equal && e_rank < left)) {
            store_index(a.kept, kept + n_kept + a_rank + e_kept, j, c.idx64);
        }
        const uint32_t e_after = n_equal + e_all;
        n_kept += a_all + (e_after < left ? e_after : left) - (n_equal < left ? n_equal : left);
        n_equal = e_after;
    }
    for (int i = tid; i < n.recent; i += T) {
        store_index(a.kept, kept + n.keep - n.recent + i, hi + i, c.idx64);
    }
}

// The kept rows to the new pages: a workgroup per (block of the new pages, key head and K or V, sequence), which gathers the
// block's 32 rows, gives them the block's own scale and writes codes in whole blocks.
template <int DS>
__global__ __launch_bounds__(kFp8AppendThreads) void hstu_paged_fp8_move_kernel(const Fp8EvictArgs a)
{
    constexpr int T = kFp8AppendThreads;
    constexpr int KP = kFp8Block * DS / 8 / T;
    constexpr int VP = DS / T > 0 ? DS / T : 1;
    __shared__ uint32_t s_top[T / 64];
    __shared__ int s_block[kFp8Block];  // where a row of the new block comes from: the block's number, and its place in it
    __shared__ int s_slot[kFp8Block];
    __shared__ float s_scale[kFp8Block];

    const Fp8Cache& c = a.c;
    const int b = static_cast<int>(blockIdx.z), g = static_cast<int>(blockIdx.y >> 1), blk = static_cast<int>(blockIdx.x);
    const bool is_v = (blockIdx.y & 1) != 0;
    const Fp8Sequence seq = fp8_sequence(c, b);
    const Fp8Sequence to = fp8_pages(a.new_page_offsets, a.n_new_page_ids, c.idx64, b);
    const Fp8Budget n = fp8_budget(a, seq, to.n_pages);
    const int start = blk * kFp8Block;
    if (start >= n.keep) {
        return;
    }
    const int lin = uniform(fp8_block(c, a.new_page_ids, to.first, g, blk));
    if (lin < 0) {
        return;
    }
    const int t = threadIdx.x, dim = c.dim;
    if (t < kFp8Block) {
        int from = -1, slot = 0;
        if (start + t < n.keep) {
            const int64_t j = load_index(a.kept, static_cast<int64_t>(b) * a.keep + start + t, c.idx64);
            from = fp8_block(c, c.page_ids, seq.first, g, static_cast<int>(j) / kFp8Block);
            slot = static_cast<int>(j) & (kFp8Block - 1);
        }
        s_block[t] = from;
        s_slot[t] = slot;
        s_scale[t] = from >= 0 ? (is_v ? c.v_scale : c.k_scale)[from] : 0.0f;
        if (c.weights != nullptr && !is_v) {
            c.weights[static_cast<int64_t>(lin) * kFp8Block + t] = from >= 0 ? c.weights[static_cast<int64_t>(from) * kFp8Block + slot] : 0.0f;
        }
    }
    __syncthreads();
    const int64_t pitch = static_cast<int64_t>(kFp8Block) * dim;
    if (!is_v) {
        uint8_t* const dst = c.k + lin * pitch;
        const int cpr = dim >> 3, pieces = kFp8Block * cpr;
        float x[KP][8];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int p = t + i * T, row = div_small(p, cpr), col = (p - row * cpr) * 8;
            const int from = p < pieces ? s_block[row] : -1;
            u32x2_t w = {0u, 0u};
            float scale = 0.0f;
            if (from >= 0) {
                w = *reinterpret_cast<const u32x2_t*>(c.k + from * pitch + s_slot[row] * dim + col);
                scale = s_scale[row];
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const f32x2_t lo = fp8_values2<false>(w[j]), hi = fp8_values2<true>(w[j]);
                x[i][4 * j] = lo[0] * scale;
                x[i][4 * j + 1] = lo[1] * scale;
                x[i][4 * j + 2] = hi[0] * scale;
                x[i][4 * j + 3] = hi[1] * scale;
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
                const uint32_t codes = fp8_codes2<false>(x[i][4 * j], x[i][4 * j + 1], inverse, 0u);
                w[j] = fp8_codes2<true>(x[i][4 * j + 2], x[i][4 * j + 3], inverse, codes);
            }
            if (p < pieces) {
                *reinterpret_cast<u32x2_t*>(dst + row * dim + col) = w;
            }
        }
        if (t == 0) {
            c.k_scale[lin] = fp8_scale_of(field);
        }
    } else {
        uint8_t* const dst = c.v + lin * pitch;
        const int pairs = dim >> 1;
        float x[VP][2][16];
        uint32_t top = 0;
#pragma unroll
        for (int u = 0; u < VP; ++u) {
            const int m = t + u * T, half = m >= pairs ? 1 : 0, d = 2 * (m - half * pairs);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int row = 16 * half + i, from = m < 2 * pairs ? s_block[row] : -1;
                x[u][0][i] = x[u][1][i] = 0.0f;
                if (from >= 0) {
                    const uint8_t* const src = c.v + from * pitch + d * kFp8Block + s_slot[row];
                    const f32x2_t two = fp8_values2<false>(static_cast<uint32_t>(src[0]) | static_cast<uint32_t>(src[kFp8Block]) << 8);
                    x[u][0][i] = two[0] * s_scale[row];
                    x[u][1][i] = two[1] * s_scale[row];
                }
                const uint32_t m0 = finite_bits(x[u][0][i]), m1 = finite_bits(x[u][1][i]);
                top = m0 > top ? m0 : top;
                top = m1 > top ? m1 : top;
            }
        }
        const uint32_t field = fp8_scale_field(block_top<T / 64>(top, s_top));
        const float inverse = fp8_inverse_of(field);
#pragma unroll
        for (int u = 0; u < VP; ++u) {
            const int m = t + u * T, half = m >= pairs ? 1 : 0, d = 2 * (m - half * pairs);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                u32x4_t w;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t codes = fp8_codes2<false>(x[u][e][4 * j], x[u][e][4 * j + 1], inverse, 0u);
                    w[j] = fp8_codes2<true>(x[u][e][4 * j + 2], x[u][e][4 * j + 3], inverse, codes);
                }
                if (m < 2 * pairs) {
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
