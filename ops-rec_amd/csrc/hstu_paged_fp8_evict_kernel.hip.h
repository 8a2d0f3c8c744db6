// Eviction from the 8-bit paged cache by accumulated attention weights (gfx950): which rows of a sequence stay, and their move to
// other pages.
#pragma once
#include "hstu_paged_fp8_common.hip.h"

namespace hstu {

// A score as an integer that compares as the score does (larger is larger): NaN as -infinity, the two zeros the same.
__device__ __forceinline__ uint32_t score_key(float s)
{
    const uint32_t bits = __builtin_bit_cast(uint32_t, s == s ? s + 0.0f : -__builtin_inff());
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

typedef __attribute__((ext_vector_type(4))) float f32x4_t;

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

// Adds `x` over the lanes and wavefronts ahead of this one: the sum before it, and that of all in `all`.  `s` has a word per wavefront.
template <int WAVES>
__device__ __forceinline__ uint32_t sum_before(uint32_t x, uint32_t (&s)[WAVES], uint32_t& all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t until = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t below = static_cast<uint32_t>(__shfl_up(static_cast<int>(until), d, 64));
        until += lane >= d ? below : 0u;
    }
    __syncthreads();  // (s of an earlier sum has been read)
    if (lane == 63) {
        s[wave] = until;
    }
    __syncthreads();
    uint32_t before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        before += w < wave ? s[w] : 0u;
        all += s[w];
    }
    return before + until - x;
}

// One workgroup per sequence.  A row's score is the sum of its weights over the key heads, in their order, in fp32.  The last of the
// places that are left beside the rows kept anyway goes to the k-th largest score, which is found by its bits, eleven, eleven and
// ten at a time from the top: histograms in LDS (2048 bins: with the eight bits of sign and exponent alone most scores of a sequence
// fall into a few, whose additions then wait for each other) over the scores, in LDS too up to kFp8SelectKeys of them, else
// where the first pass left them.  Rows above it stay, and of those equal to it the first few: every thread counts those of a
// stretch of rows, one sum over the workgroup says where its indices go.
// Bound by the latency of its passes: 32 sequences of 4096 .. 16384 rows and 4 key heads 22 us, with scores in memory 76.
// T threads and KEYS scores in LDS: 1024 and kFp8SelectKeys, or for short sequences few (16 sequences, with the move: of 500 rows 12.4 us
// with 256 threads and 13.5 with 1024, of 1000 13.3 and 14.3, of 2000 17.1 and 16.5).
template <int T, int KEYS>
__global__ __launch_bounds__(T) void hstu_paged_fp8_select_kernel(const Fp8EvictArgs a)
{
    constexpr int WAVES = T / 64, BINS = 2048, OWN = BINS / T;
    __shared__ __attribute__((aligned(16))) uint32_t s_keys[KEYS];
    __shared__ uint32_t s_hist[BINS];
    __shared__ uint32_t s_sum[WAVES];
    __shared__ uint32_t s_pick[2];

    const Fp8Cache& c = a.c;
    const int b = static_cast<int>(blockIdx.x), tid = threadIdx.x;
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
    // rows [lo, hi) compete for the places that are left; the others stay
    const int lo = n.sinks, hi = n.len - n.recent;
    const int places = n.keep - n.sinks - n.recent;
    const bool all_stay = n.keep == n.len;
    for (int i = tid; i < (all_stay ? n.keep : n.sinks); i += T) {
        store_index(a.kept, kept + i, i, c.idx64);
    }
    if (all_stay) {
        return;
    }
    for (int i = tid; i < n.recent; i += T) {
        store_index(a.kept, kept + n.keep - n.recent + i, hi + i, c.idx64);
    }
    if (places == 0) {
        return;
    }
    // scores of four rows at a time (of one block: lo is rounded down to a multiple of four, what lies ahead of it scores nothing)
    const int first = lo & ~3, rows = (hi - first + 3) & ~3;
    const bool in_lds = rows <= KEYS;
    uint32_t* const far = a.keys + static_cast<int64_t>(b) * a.key_pitch;
    const int64_t head_pitch = static_cast<int64_t>(c.blocks_per_page) * kFp8Block;
    for (int r = 4 * tid; r < rows; r += 4 * T) {
        const int j = first + r, lin = fp8_block(c, c.page_ids, seq.first, 0, j / kFp8Block);
        f32x4_t score = {0.0f, 0.0f, 0.0f, 0.0f};
        if (lin >= 0) {
            const float* const w = c.weights + static_cast<int64_t>(lin) * kFp8Block + (j & (kFp8Block - 1));
            for (int h0 = 0; h0 < c.n_heads; h0 += 4) {  // (four heads on their way together)
                f32x4_t v[4];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    v[h] = *reinterpret_cast<const f32x4_t*>(w + (h0 + h < c.n_heads ? h0 + h : h0) * head_pitch);
                }
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    if (h0 + h < c.n_heads) {
                        score = h0 + h == 0 ? v[0] : score + v[h];
                    }
                }
            }
        }
        u32x4_t k;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float s = score[i];
            k[i] = score_key(s);
        }
        *reinterpret_cast<u32x4_t*>((in_lds ? s_keys : far) + r) = k;
    }
    const auto keys_of = [&](int r) { return *reinterpret_cast<const u32x4_t*>((in_lds ? s_keys : far) + r); };  // four, r a multiple of four
    const auto competes = [&](int r) { return first + r >= lo && first + r < hi; };
    __syncthreads();
    uint32_t prefix = 0, left = static_cast<uint32_t>(places);  // of the rows whose top bits are `prefix`, `left` stay
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < BINS; i += T) {
            s_hist[i] = 0;
        }
        __syncthreads();
        for (int r = 4 * tid; r < rows; r += 4 * T) {
            const u32x4_t four = keys_of(r);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t k = four[i];
                if (competes(r + i) && (pass == 0 || (k >> (shift + bits)) == (prefix >> (shift + bits)))) {
                    atomicAdd(&s_hist[(k >> shift) & ((1u << bits) - 1u)], 1u);
                }
            }
        }
        __syncthreads();
        // thread t has OWN digits from BINS - 1 - OWN t down: counts from the top
        uint32_t count[OWN], sum = 0, all;
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
            count[i] = s_hist[BINS - 1 - OWN * tid - i];
            sum += count[i];
        }
        uint32_t before = sum_before<WAVES>(sum, s_sum, all);
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
            if (before < left && before + count[i] >= left) {  // (true for one digit of one thread)
                s_pick[0] = static_cast<uint32_t>(BINS - 1 - OWN * tid - i);
                s_pick[1] = left - before;
            }
            before += count[i];
        }
        __syncthreads();
        prefix |= s_pick[0] << shift;
        left = s_pick[1];
    }
    // rows above `prefix` stay, and the first `left` of those equal to it
    const int stretch = ((rows + T - 1) / T + 3) & ~3, r0 = tid * stretch < rows ? tid * stretch : rows, r1 = r0 + stretch < rows ? r0 + stretch : rows;
    uint32_t above = 0, equal = 0;
    for (int r = r0; r < r1; r += 4) {
        const u32x4_t four = keys_of(r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            above += competes(r + i) && four[i] > prefix ? 1u : 0u;
            equal += competes(r + i) && four[i] == prefix ? 1u : 0u;
        }
    }
    uint32_t all;
    uint32_t ties = sum_before<WAVES>(equal, s_sum, all);
    uint32_t at = sum_before<WAVES>(above, s_sum, all) + (ties < left ? ties : left) + static_cast<uint32_t>(n.sinks);
    for (int r = r0; r < r1; r += 4) {
        const u32x4_t four = keys_of(r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool tied = competes(r + i) && four[i] == prefix;
            if (competes(r + i) && (four[i] > prefix || (tied && ties < left))) {
                store_index(a.kept, kept + at++, first + r + i, c.idx64);
            }
            ties += tied ? 1u : 0u;
        }
    }
}

// The kept rows to the new pages: a workgroup per (block of the new pages, key head and K or V, sequence), which gathers the
// block's 32 rows, gives them the block's own scale and writes codes in whole blocks.  Bound by the lines it touches: a token of V is a
// byte in each line of its block, so that where one row in five stays all of V is read (2048 rows of 4096 .. 16384 of 32 sequences, 4 key
// heads of 128 dims: 235 MB read for 67 MB kept, 69 us, 4.4 TB/s with what is written).
template <int DS>
__global__ __launch_bounds__(kFp8AppendThreads) void hstu_paged_fp8_move_kernel(const Fp8EvictArgs a)
{
    constexpr int T = kFp8AppendThreads;
    constexpr int KP = kFp8Block * DS / 8 / T;
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
        // a lane has a row of the new block, and of its dims a quarter: a load takes a byte of 32 rows, which came from few blocks, for two
        // dims, so that its lanes meet in few lines (two dims of 64 lanes' own, a row at a time: 64 lines a load, 106 us where this takes 69)
        uint8_t* const dst = c.v + lin * pitch;
        const int quarter = dim >> 2, row = t & 31, d0 = (t >> 5) * quarter;
        const int from = s_block[row];
        const float scale = s_scale[row];
        const uint8_t* const src = c.v + (from >= 0 ? from : 0) * pitch + d0 * kFp8Block + s_slot[row];
        uint32_t byte[DS / 4];
#pragma unroll
        for (int i = 0; i < DS / 4; ++i) {
            byte[i] = 0u;
            if (from >= 0 && i < quarter) {
                byte[i] = src[i * kFp8Block];
            }
        }
        uint32_t top = 0;
        float x[DS / 4];
#pragma unroll
        for (int i = 0; i < DS / 4; ++i) {
            const f32x2_t two = fp8_values2<false>(byte[i]);
            x[i] = two[0] * scale;
            const uint32_t m = finite_bits(x[i]);
            top = m > top ? m : top;
        }
        const uint32_t field = fp8_scale_field(block_top<T / 64>(top, s_top));
        const float inverse = fp8_inverse_of(field);
#pragma unroll
        for (int i = 0; i < DS / 4; i += 4) {
            // four dims of this row, and of the rows of four lanes one dim each
            uint32_t mine = fp8_codes2<false>(x[i], x[i + 1], inverse, 0u);
            mine = fp8_codes2<true>(x[i + 2], x[i + 3], inverse, mine);
            uint32_t w = 0;
#pragma unroll
            for (int l = 0; l < 4; ++l) {
                const uint32_t theirs = static_cast<uint32_t>(__shfl(static_cast<int>(mine), (t & 60) + l, 64));
                w |= (theirs >> (8 * (t & 3)) & 0xffu) << (8 * l);
            }
            if (i < quarter) {
                *reinterpret_cast<uint32_t*>(dst + (d0 + i + (t & 3)) * kFp8Block + (row & ~3)) = w;
            }
        }
        if (t == 0) {
            c.v_scale[lin] = fp8_scale_of(field);
        }
    }
}

}  // namespace hstu
