// HSTU attention over the 8-bit paged cache for tiles of many rows (gfx950): the arithmetic of hstu_paged_fp8_attend_kernel.hip.h with the
// codes converted once per workgroup.
//
// A 32 x 32 block of scores costs 16 matrix instructions (248 ns on a SIMD alone) and, in the vector unit, 32 transcendental
// instructions and some 60 others (230 ns; both together, from two wavefronts, 300 ns), and 64 conversions of codes (150 ns) in a
// kernel whose wavefronts work alone.  Here four wavefronts, 32 rows each, bring the same blocks in together, each a part of the
// chunks: codes two steps ahead in registers, converted (v_cvt_scalef32_pk) and left in LDS in the order of the matrix operands, 16
// bytes per lane, so that reads have no bank conflicts; two buffers for K and three for V, one barrier a step.  The products of K(t)
// and of V(t - 1) go together, a chain of eight that wait for each other between four pairs that do not.  Three workgroups fit a CU,
// and what one leaves of a SIMD's units another, which is nowhere in step with it, takes.  Bound by the vector and the matrix unit, which
// overlap little: 16 x 4 key heads of 1024 rows on 2048 .. 8192 keys, d 128, 237 us (770 TFLOP/s; fp16, with its units, 252), 64 such sequences
// of 5120 keys 850 TFLOP/s.  P is rounded to the type of q, once, as in the 16-bit forward kernels: outputs are 1.4 times as far off as their
// own rounding leaves them (0.0023 of their size in bf16; 0.0020 from the other kernel, which calls of fewer rows take).  A product for what that
// rounding leaves of half the keys makes this 272 us, which is what the other kernel, with such a product, takes.  (Eight wavefronts half a step
// apart, one half multiplying while the other weighs, changing places at every barrier, took 10 % longer; two shares of the keys for tiles of 64 rows
// lost to wavefronts alone.)
//   step t : S = K(t) Q and O += V(t - 1) P; convert K, V (t + 1) to LDS, request those of t + 3; P = silu(S) masked
#pragma once
#include "hstu_paged_fp8_attend_kernel.hip.h"

namespace hstu {

template <typename Tag, int NC>
__global__ __launch_bounds__(kFp8TileThreads) __attribute__((amdgpu_waves_per_eu(3, 3))) void hstu_paged_fp8_tile_kernel(const Fp8AttendArgs a)
{
    constexpr int T = kFp8TileThreads, RG = T / 64, TILE = kFp8TileRows;
    constexpr bool F16 = __is_same(Tag, f16_tag);
    constexpr int CHUNKS = (2 * NC + RG - 1) / RG;  // chunks of 1 KiB of codes that a wavefront brings in per block
    constexpr int FRAG = 64 * 16;                   // bytes of an operand: 16 per lane
    constexpr int BUFFER = 2 * NC * FRAG;           // K or V of a block, 16 bits a value
    constexpr int BUFFERS = 5 * BUFFER;             // two of K, three of V
    constexpr int SUMS = RG * 1024 * 4;             // a group of 32 dims of all wavefronts
    constexpr int LDS = BUFFERS > 2 * SUMS ? BUFFERS : 2 * SUMS;
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[LDS];

    const Fp8Cache& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, rg = uniform(tid >> 6);
    const int col = lane & 31, half = lane >> 5;

    int g, tile;
    const Fp8Deal deal = fp8_slot(a, g, tile);
    if (deal.b < 0) {
        return;
    }
    const int b = deal.b, part = deal.part, pair = b * c.n_heads + g;
    const Fp8Item item = fp8_item(a, b);
    const Fp8Sequence& seq = item.seq;
    const Fp8Mask& mask = item.mask;
    const int dim = c.dim;
    uint16_t* const out = static_cast<uint16_t*>(a.out);
    if (a.tile_first + tile == 0 && part == 0) {
        fp8_clear_rows<T>(a, item, b, g, out);
    }
    const int n_rows = item.n_rows * a.ratio;  // (row, head) pairs
    const int t0 = (a.tile_first + tile) * TILE, t1 = t0 + TILE < n_rows ? t0 + TILE : n_rows;
    if (t0 >= t1) {
        return;
    }
    // the tile's blocks, and the bounds inside which a block needs no mask for the tile, and for this wavefront's rows
    const int ti0 = uniform(div_small(t0, a.ratio)), ti1 = uniform(div_small(t1 - 1, a.ratio));
    Fp8Runs runs = fp8_runs(mask, ti0, ti1 + 1);
    runs = {uniform(runs.n_a), uniform(runs.n_b), uniform(runs.n_c), uniform(runs.b0), uniform(runs.c0)};
    const int n_blocks = runs.count();
    const int parts_used = deal.parts == 1 ? 1 : uniform((n_blocks + deal.chunk - 1) / deal.chunk);
    if (part > 0 && part >= parts_used) {
        return;
    }
    if (part == 0 && a.joins != nullptr && threadIdx.x == 0) {
        a.joins[pair * a.row_tiles + tile] = int2{parts_used < deal.parts ? parts_used : deal.parts, deal.slot};
    }
    const int n_begin = deal.parts == 1 ? 0 : part * deal.chunk;
    const int n_end = part == deal.parts - 1 || n_blocks - n_begin < deal.chunk ? n_blocks : n_begin + deal.chunk;
    const int m0 = t0 + 32 * rg;
    const bool rows_here = m0 < n_rows;
    const int m1 = m0 + 32 < n_rows ? m0 + 32 : n_rows;
    const int i_first = rows_here ? uniform(div_small(m0, a.ratio)) : ti0, i_last = rows_here ? uniform(div_small(m1 - 1, a.ratio)) : ti0;
    const Fp8Whole whole = fp8_whole(mask, i_first, i_last), tile_whole = fp8_whole(mask, ti0, ti1);

    // this lane's row of q
    u32x4_t q[NC][2];
    const int m = m0 + col, i_row = div_small(m < n_rows ? m : 0, a.ratio);
    const int lim = m < n_rows ? mask.lim(i_row) : 0, hole = mask.hole(i_row), low = mask.low(i_row);
    {
        const uint32_t bytes = static_cast<uint32_t>(item.n_rows) * static_cast<uint32_t>(a.n_heads_q) * dim * 2u;
        const __amdgpu_buffer_rsrc_t rsrc =
            make_rsrc(static_cast<const uint16_t*>(a.q) + item.q0 * a.n_heads_q * static_cast<int64_t>(dim), bytes);
        const uint32_t at = (static_cast<uint32_t>(i_row) * a.n_heads_q + g * a.ratio + (m - i_row * a.ratio)) * dim * 2u;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int d = 32 * n + 16 * half + 8 * u;
                q[n][u] = load_codes(rsrc, m < n_rows && d < dim ? at + d * 2u : kOutOfRange);
            }
        }
    }
    const auto sees_key = [&](int j) {
        return static_cast<bool>((j < lim) & ((j < mask.first_key) | (j >= hole)) & ((j >= low) | (j < mask.sinks)));
    };

    // the chunks this wavefront brings in: number rg + RG i of the block's 2 NC, K first
    const int pi = 16 * ((col >> 2) & 1) + 4 * (col >> 3) + (col & 3);
    const uint32_t block_bytes = static_cast<uint32_t>(kFp8Block) * dim;
    uint32_t code_at[CHUNKS];
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        const int n = rg + RG * i, d = 32 * n + 16 * half, dv = 32 * (n - NC) + pi;
        const uint32_t k_at = d < dim ? static_cast<uint32_t>(pi) * dim + d : kOutOfRange;
        const uint32_t v_at = dv < dim ? static_cast<uint32_t>(dv) * kFp8Block + 16 * half : kOutOfRange;
        code_at[i] = n < NC ? k_at : (n < 2 * NC ? v_at : kOutOfRange);
    }

    // a step is a block; an even number of steps, the last perhaps without one (requests then stand in one order at the loop's head, and
    // a wait is for a block's own).  Places and scales of 64 steps, and of the 64 behind them, a step per lane; looked up and handed
    // out with every lane active.
    const int mine = n_end - n_begin > 0 ? n_end - n_begin : 0, n_steps = (mine + 1) / 2 * 2;
    const auto block_of = [&](int s) { return runs.block(n_begin + s); };
    int lin_a = -1, lin_b = -1;
    float ks_a = 1.0f, ks_b = 1.0f, vs_a = 1.0f, vs_b = 1.0f;
    int base = 0;
    const auto look_up = [&](int first, int& lin, float& ks, float& vs) {
        lin = -1;
        if (first < mine) {
            const int s = first + lane < mine ? first + lane : mine - 1;
            const int at = fp8_block(c, c.page_ids, seq.first, g, block_of(s));
            const float k_at = c.k_scale[at >= 0 ? at : 0], v_at = c.v_scale[at >= 0 ? at : 0];
            ks = at >= 0 ? k_at : 1.0f;  // (a page that is none: zeros, see the other kernel)
            vs = at >= 0 ? v_at : 1.0f;
            lin = first + lane < mine ? at : -1;
        }
    };
    // lane s mod 64 of the first or the second of these: steps base .. base + 127
    const auto pick = [&](int x_a, int x_b, int s) {
        const int l_a = __builtin_amdgcn_readlane(x_a, s & 63), l_b = __builtin_amdgcn_readlane(x_b, s & 63);
        return s < base + 64 ? l_a : l_b;
    };
    const auto lin_of = [&](int s) { return pick(lin_a, lin_b, s); };
    const auto scale_of = [&](float x_a, float x_b, int s) {
        return __builtin_bit_cast(float, pick(__builtin_bit_cast(int, x_a), __builtin_bit_cast(int, x_b), s));
    };

    u32x4_t raw[2][CHUNKS];
    const auto request = [&](u32x4_t (&to)[CHUNKS], int t) {
        const int lin = lin_of(t);
        const int64_t at = static_cast<int64_t>(lin < 0 ? 0 : lin) * block_bytes;
        const __amdgpu_buffer_rsrc_t kr = make_rsrc(c.k + at, lin < 0 ? 0u : block_bytes), vr = make_rsrc(c.v + at, lin < 0 ? 0u : block_bytes);
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            if (rg + RG * i < NC) {
                to[i] = load_codes(kr, code_at[i]);
            } else {
                to[i] = load_codes(vr, code_at[i]);
            }
        }
    };
    bool poisoned = false;
    const auto convert = [&](u32x4_t (&from)[CHUNKS], int t, uint8_t* to_k, uint8_t* to_v) {
        const int blk = block_of(t);
        const float ks = scale_of(ks_a, ks_b, t), vs = scale_of(vs_a, vs_b, t);
        if (t < mine && !tile_whole.has(blk)) {
            // codes behind the last row may be anything; NaN that some rows do not see: see the other kernel
            const int left = seq.len - blk * kFp8Block - 16 * half;
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) {
                if (rg + RG * i >= NC) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int k = left - 4 * j;
                        const uint32_t live = from[i][j] & (k >= 4 ? 0xffffffffu : (k <= 0 ? 0u : (1u << (8 * k)) - 1u));
                        const uint32_t bits = nan_codes(live);
                        any |= bits;
                        from[i][j] = live & ~((bits >> 7) * 0xffu);
                    }
                }
            }
            poisoned = poisoned || __any(any != 0);
        }
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const int n = rg + RG * i;
            if (n < 2 * NC) {
                const Fp8Pair x = fp8_widen<Tag>(from[i], F16 ? 1.0f : (n < NC ? ks : vs));
                uint8_t* const to = (n < NC ? to_k + 2 * n * FRAG : to_v + 2 * (n - NC) * FRAG) + lane * 16;
                *reinterpret_cast<u32x4_t*>(to) = x.lo;
                *reinterpret_cast<u32x4_t*>(to + FRAG) = x.hi;
            }
        }
    };

    f32x16_t acc[NC], sc;
    u32x4_t p[2] = {u32x4_t{0u}, u32x4_t{0u}};
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        acc[n] = f32x16_t{0.0f};
    }
    const auto operand = [&](const uint8_t* from, int n) { return *reinterpret_cast<const u32x4_t*>(from + n * FRAG + lane * 16); };
    // There is no branch around a product: ahead of the first step and behind the last they run on weights and values of zero.
    const auto multiply = [&](const uint8_t* k, const uint8_t* v) {
        sc = f32x16_t{0.0f};
#pragma unroll
        for (int n = 0; n < NC; ++n) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                sc = mfma32<Tag>(operand(k, 2 * n + u), q[n][u], sc);
                acc[n] = mfma32<Tag>(operand(v, 2 * n + u), p[u], acc[n]);
            }
        }
        // operands are read six ahead of their products (left to itself the compiler reads each into the same registers and waits
        // for it: 16 times the LDS's latency)
        constexpr int N = 4 * NC, AHEAD = N < 6 ? N : 6;
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);  // LDS reads
#pragma unroll
        for (int i = 0; i < N; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction
            if (i + AHEAD < N) {
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    Fp8Unit unit(q, dim);  // (fp16)
    const int most_scale = fp8_most_scale(a.c_exp);
    const auto weigh = [&](int t) {
        const int blk = block_of(t), c0 = blk * kFp8Block;
        float w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float x = sc[i];
            w[i] = F16 ? x : x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * a.c_exp));
        }
        bool sees = true;  // (this lane's row, a key of the block)
        if (t >= mine || !whole.has(blk)) {
            const int end = t < mine ? lim : 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int j = c0 + 16 * half + i;
                w[i] = ((j < end) & ((j < mask.first_key) | (j >= hole)) & ((j >= low) | (j < mask.sinks))) ? w[i] : 0.0f;
            }
            sees = F16 && fp8_some_score(w);
        }
        if constexpr (F16) {
            const int k = Fp8Unit::exponent(scale_of(ks_a, ks_b, t)), v = Fp8Unit::exponent(scale_of(vs_a, vs_b, t));
            unit.fit<NC>(acc, k + v, sees);  // (the sums are of the blocks before this one)
            fp8_weights_in_units(w, a.c_exp, k, most_scale, unit.denominator(k + v));
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[u][i] = pack2<Tag>(w[8 * u + 2 * i], w[8 * u + 2 * i + 1]);
            }
        }
    };

    uint8_t *v_last = s_mem + 4 * BUFFER, *v_now = s_mem + 2 * BUFFER, *v_next = s_mem + 3 * BUFFER;  // V of t - 1, t, t + 1
    const auto step = [&](u32x4_t (&next)[CHUNKS], int t, int turn) {
        multiply(s_mem + turn * BUFFER, v_last);
        convert(next, t + 1, s_mem + (turn ^ 1) * BUFFER, v_next);
        request(next, t + 3);
        weigh(t);
        __syncthreads();
        uint8_t* const free = v_last;
        v_last = v_now;
        v_now = v_next;
        v_next = free;
    };
    for (int x = rg; x < 2 * NC; x += RG) {
        *reinterpret_cast<u32x4_t*>(v_last + x * FRAG + lane * 16) = u32x4_t{0u};
    }
    look_up(0, lin_a, ks_a, vs_a);
    look_up(64, lin_b, ks_b, vs_b);
    request(raw[0], 0);
    request(raw[1], 1);
    convert(raw[0], 0, s_mem, v_now);
    request(raw[0], 2);
    __syncthreads();
    for (int t = 0; t < n_steps; t += 2) {
        if (t >= base + 64) {
            base += 64;
            lin_a = lin_b;
            ks_a = ks_b;
            vs_a = vs_b;
            look_up(base + 64, lin_b, ks_b, vs_b);
            // (waited for here, every 64 steps: where paths meet, the compiler would wait for these loads, and so for the codes asked
            // for before them, in every step)
            __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
        }
        step(raw[1], t, 0);
        step(raw[0], t + 1, 1);
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        acc[n] = mfma32<Tag>(operand(v_last, 2 * n), p[0], acc[n]);
        acc[n] = mfma32<Tag>(operand(v_last, 2 * n + 1), p[1], acc[n]);
    }
    // (a flag where K and V were)
    int* const s_poison = reinterpret_cast<int*>(s_mem);
    __syncthreads();
    if (rg == 0 && lane_here() == 0) {
        *s_poison = 0;
    }
    __syncthreads();
    if (poisoned) {
        *s_poison = 1;
    }
    __syncthreads();
    const bool any_poison = *s_poison != 0;
    __syncthreads();  // (the sums go there next)
    if (any_poison) {
        const int lane_p = lane_here(), col_p = lane_p & 31, half_p = lane_p >> 5, pi_p = 16 * ((col_p >> 2) & 1) + 4 * (col_p >> 3) + (col_p & 3);
        const uint32_t v_at = static_cast<uint32_t>(pi_p) * kFp8Block + 16 * half_p;
        for (int s = 0; s < mine; ++s) {
            const int blk = block_of(s);
            if (!tile_whole.has(blk)) {
                fp8_poison<Tag, NC>(acc, c, uniform(fp8_block(c, c.page_ids, seq.first, g, blk)), v_at, blk * kFp8Block + 16 * half_p, seq.len, sees_key);
            }
        }
    }

    if constexpr (F16) {
        unit.undo<NC>(acc);
    }
    // ---- the store ----
    const int lane_e = lane_here(), tid_e = 64 * rg + lane_e, half_e = lane_e >> 5, ratio = here(a.ratio);
    const bool partial = parts_used > 1 && deal.parts > 1;
    float* const to_partial = a.partial + (static_cast<int64_t>(deal.slot * c.n_heads + g) * a.row_tiles + tile) * TILE * dim;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        float* const s = reinterpret_cast<float*>(s_mem) + (n & 1) * (SUMS / 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // (16 bytes at a time, their places exchanged so that neither side has bank conflicts)
            const f32x4_t x = {acc[n][4 * i], acc[n][4 * i + 1], acc[n][4 * i + 2], acc[n][4 * i + 3]};
            *reinterpret_cast<f32x4_t*>(s + rg * 1024 + 4 * (i * 64 + (lane_e ^ (2 * i + 8 * half_e)))) = x;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r) {  // four dims per lane, eight lanes together the 32 of a row
            const int word = tid_e + r * T, i = word & 3, h = (word >> 2) & 1, row_in = word >> 3;
            const float* const from = s + (row_in >> 5) * 1024 + 4 * (i * 64 + ((32 * h + (row_in & 31)) ^ (2 * i + 8 * h)));
            const f32x4_t x = *reinterpret_cast<const f32x4_t*>(from);
            const int row = t0 + row_in, d = 32 * n + 16 * h + 4 * i;
            if (row < n_rows && d < dim) {
                if (partial) {
                    *reinterpret_cast<f32x4_t*>(to_partial + static_cast<int64_t>(row_in) * dim + d) = x;
                } else {
                    const int ir = div_small(row, ratio);
                    const int64_t at = ((item.q0 + ir) * a.n_heads_q + g * ratio + (row - ir * ratio)) * static_cast<int64_t>(dim) + d;
                    *reinterpret_cast<u32x2_t*>(out + at) = u32x2_t{pack2<Tag>(x[0] * a.c_out, x[1] * a.c_out), pack2<Tag>(x[2] * a.c_out, x[3] * a.c_out)};
                }
            }
        }
    }
}

}  // namespace hstu
