// Rotary positions on jagged q and k, gfx950.
//
//   angle = position * frequency_j;  (a, b) -> magnitude * (a cos - b sin, b cos + a sin) for every pair j of every head
//
// The angle is formed in 64 bits and cut to a fraction of a turn before it goes to 32: at position 10^6 an angle of 32 bits is off by 0.06.
//
// Bound by HBM: every value is read and written once.  A thread has 8 pairs of a row (two 16-byte pieces of a head, whichever layout)
// and turns them in several heads of q and k, so that a sine and a cosine serve them all; short batches give each thread fewer heads, down
// to one, and pay the sines again for more threads.  Values of a head past its pairs are copied by threads of their own, 8 each.  Pieces start
// anywhere (16-byte accesses need no alignment here); a part-filled last piece goes value by value.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "layer_norm_kernel.hip.h"

namespace hstu {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryAtOnce = 4;  // heads whose loads are in flight together

__device__ __forceinline__ int64_t rotary_index(const void* p, int64_t i, int idx64)
{
    return idx64 ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}

// The last of n offsets (not decreasing) that is at most `row`, -1 if none is: eight ways at a time, whose loads go together.
__device__ __forceinline__ int rotary_sequence(const void* offsets, int n, int idx64, int64_t row)
{
    if (rotary_index(offsets, 0, idx64) > row) {
        return -1;
    }
    int lo = 0, left = n;
    while (left > 1) {
        const int step = (left + 7) >> 3;
        int below = 0;
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            const int at = i * step;
            below += at < left && rotary_index(offsets, lo + min(at, left - 1), idx64) <= row ? 1 : 0;
        }
        lo += below * step;
        left = min(step, left - below * step);
    }
    return lo;
}

// cos and sin of `turns` full turns, |turns| <= 1/2: the hardware's instructions take turns, and are exact enough for results of
// 16 bits; fp32 results go through the library
template <typename T>
__device__ __forceinline__ void rotary_turn(float turns, float& c, float& s)
{
    if constexpr (ln_traits<T>::kPerChunk == 4) {
        sincospif(2.0f * turns, &s, &c);
    } else {
        c = __builtin_amdgcn_cosf(turns);
        s = __builtin_amdgcn_sinf(turns);
    }
}

template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const RotaryArgs a)
{
    using E = typename ln_traits<T>::elem_t;
    const uint32_t id = blockIdx.x * static_cast<uint32_t>(kRotaryThreads) + threadIdx.x;
    const uint32_t rest = id / static_cast<uint32_t>(a.items);
    const int item = static_cast<int>(id - rest * static_cast<uint32_t>(a.items));
    const uint32_t row = rest / static_cast<uint32_t>(a.head_blocks);
    if (row >= a.rows) {
        return;
    }
    const int first = static_cast<int>(rest - row * static_cast<uint32_t>(a.head_blocks)) * a.heads_each;
    const int last = min(first + a.heads_each, a.heads);

    bool inside = true;
    double position = 0.0;
    if (a.positions != nullptr) {
        position = static_cast<double>(rotary_index(a.positions, row, a.positions64));
    } else {
        const int64_t at = a.row0 + row;
        const int b = rotary_sequence(a.seq_offset, a.n_offsets, a.offsets64, at);
        inside = b >= 0 && b < a.n_offsets - 1;
        if (inside) {
            int64_t p = at - rotary_index(a.seq_offset, b, a.offsets64);
            if (a.start != nullptr) {
                p += rotary_index(a.start, b, a.start64);
            }
            position = static_cast<double>(p);
        }
    }
    const auto from = [&](int h) -> const E* {
        return h < a.heads_q ? static_cast<const E*>(a.q) + row * a.q_stride_row + h * a.q_stride_head
                             : static_cast<const E*>(a.k) + row * a.k_stride_row + (h - a.heads_q) * a.k_stride_head;
    };
    const auto to = [&](int h) -> E* {
        return h < a.heads_q ? static_cast<E*>(a.q_out) + (static_cast<int64_t>(row) * a.heads_q + h) * a.dim
                             : static_cast<E*>(a.k_out) + (static_cast<int64_t>(row) * (a.heads - a.heads_q) + (h - a.heads_q)) * a.dim;
    };

    if (item >= a.turned) {  // values that are not turned
        const int c = item - a.turned, begin = 2 * a.pairs, n = a.dim - begin;
        for (int h0 = first; h0 < last; h0 += kRotaryAtOnce) {
            norm_piece<T> p[kRotaryAtOnce];
#pragma unroll
            for (int i = 0; i < kRotaryAtOnce; ++i) {
                if (h0 + i < last) {
                    p[i] = norm_load<T>(from(h0 + i) + begin, c, n);
                }
            }
#pragma unroll
            for (int i = 0; i < kRotaryAtOnce; ++i) {
                if (h0 + i < last) {
                    float f[8];
                    norm_unpack<T>(p[i], f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        f[j] = inside ? f[j] : 0.0f;
                    }
                    norm_store<T>(to(h0 + i) + begin, c, n, f);
                }
            }
        }
        return;
    }

    float cs[8], sn[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int pair = min(8 * item + j, a.pairs - 1);
        double turns = position * a.frequencies[pair] * 0.15915494309189533577;  // 1 / (2 pi)
        turns -= rint(turns);
        rotary_turn<T>(static_cast<float>(turns), cs[j], sn[j]);
        cs[j] = inside ? cs[j] * a.magnitude : 0.0f;
        sn[j] = inside ? sn[j] * a.magnitude * a.sign : 0.0f;
    }
    // side by side: 16 values from 16 item on, as two pieces; halves: piece `item` of each
    constexpr int kSecond = INTERLEAVED ? 1 : 0;
    const int n = INTERLEAVED ? 2 * a.pairs : a.pairs;
    const int c0 = INTERLEAVED ? 2 * item : item, c1 = c0 + kSecond;
    const int half = INTERLEAVED ? 0 : a.pairs;
    const bool two = 8 * c1 < n;
    for (int h0 = first; h0 < last; h0 += kRotaryAtOnce) {
        norm_piece<T> lo[kRotaryAtOnce], hi[kRotaryAtOnce];
#pragma unroll
        for (int i = 0; i < kRotaryAtOnce; ++i) {
            if (h0 + i < last) {
                const E* const p = from(h0 + i);
                lo[i] = norm_load<T>(p, c0, n);
                hi[i] = norm_load<T>(p + half, c1, n);
            }
        }
#pragma unroll
        for (int i = 0; i < kRotaryAtOnce; ++i) {
            if (h0 + i < last) {
                float u[8], v[8];
                norm_unpack<T>(lo[i], u);
                norm_unpack<T>(hi[i], v);
                if constexpr (INTERLEAVED) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float a0 = u[2 * j], b0 = u[2 * j + 1], a1 = v[2 * j], b1 = v[2 * j + 1];
                        u[2 * j] = a0 * cs[j] - b0 * sn[j];
                        u[2 * j + 1] = b0 * cs[j] + a0 * sn[j];
                        v[2 * j] = a1 * cs[4 + j] - b1 * sn[4 + j];
                        v[2 * j + 1] = b1 * cs[4 + j] + a1 * sn[4 + j];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float a0 = u[j], b0 = v[j];
                        u[j] = a0 * cs[j] - b0 * sn[j];
                        v[j] = b0 * cs[j] + a0 * sn[j];
                    }
                }
                if (!inside) {  // (zeros, whatever the values: a product with 0 would keep NaN)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        u[j] = 0.0f;
                        v[j] = 0.0f;
                    }
                }
                E* const p = to(h0 + i);
                norm_store<T>(p, c0, n, u);
                if (two) {
                    norm_store<T>(p + half, c1, n, v);
                }
            }
        }
    }
}

}  // namespace hstu
