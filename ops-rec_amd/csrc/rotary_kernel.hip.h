// Rotary positions on jagged q and k, gfx950.
//
//   angle = position * frequency_j;  (a, b) -> magnitude * (a cos - b sin, b cos + a sin) for every pair j of every head
//
// The angle is formed in 64 bits and cut to a fraction of a turn before it goes to 32: at position 10^6 an angle of 32 bits is off by 0.06.
//
// Bound by HBM: every value is read and written once.  A thread has two 16-byte pieces of a head -- the same piece of both halves, or two
// pieces of pairs that lie side by side, half of the turned values apart, so that neighbouring threads have neighbouring pieces either way -- and turns them in
// several heads of q and k: a sine and a cosine serve them all.  Short batches give each thread fewer heads, down to one, and pay the sines again for more
// threads.  Values of a head past its pairs are copied by threads of their own, two pieces each.  Pieces start anywhere (16-byte accesses need no
// alignment here); a last piece that is not whole starts earlier.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "layer_norm_kernel.hip.h"

namespace hstu {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryHeads = 8;  // heads of a thread, at most: their loads are all in flight while the row's place and its sines are worked out

// Stores that fill whole 128-byte lines go past the caches (kRotaryLines), others do not: there a line's parts meet before it is written (65536 rows of 8 + 8
// heads of 96 values, 64 of them turned, bf16: 135 us past the caches, 103 through them; 20292 rows of 4 + 4 heads, halves of 64 values, 18.3 and 20.2).
// Heads with runs of fewer values than a piece have (kRotaryShort) ask for them one by one.
constexpr int kRotaryLines = 0, kRotaryPieces = 1, kRotaryShort = 2;

// ---- 16 bytes of a run of n values, from `first` on; of a shorter run those that are there, the others undefined ----
template <typename Tag, int KIND>
struct rotary_piece {
    typedef uint32_t words_t __attribute__((ext_vector_type(4), aligned(2)));
    static constexpr int kValues = ln_traits<Tag>::kPerChunk;
    using elem_t = typename ln_traits<Tag>::elem_t;
    words_t w;

    // where piece c starts: the last, where it is not whole, is the row's last values, some of which the piece before has too (the same bits twice), and
    // a piece past the row is that one again
    static __device__ __forceinline__ bool whole(int n) { return KIND != kRotaryShort || n >= kValues; }
    static __device__ __forceinline__ int place(int c, int n) { return whole(n) ? min(c * kValues, n - kValues) : c * kValues; }
    // `at`: where the piece starts in the head
    __device__ __forceinline__ void load(const elem_t* head, int at, int first, int n)
    {
        if (whole(n)) {
            w = __builtin_nontemporal_load(reinterpret_cast<const words_t*>(head + at));
        } else {
            elem_t e[kValues];
#pragma unroll
            for (int i = 0; i < kValues; ++i) {
                e[i] = first + i < n ? head[at + i] : static_cast<elem_t>(0.0f);
            }
            __builtin_memcpy(&w, e, sizeof w);
        }
    }
    __device__ __forceinline__ void unpack(float (&f)[kValues]) const { ln_traits<Tag>::unpack(w, f); }
    static __device__ __forceinline__ void store(elem_t* head, int at, int first, int n, const float (&f)[kValues])
    {
        if (whole(n)) {
            const words_t packed = ln_traits<Tag>::pack(f);
            if constexpr (KIND == kRotaryLines) {
                __builtin_nontemporal_store(packed, reinterpret_cast<words_t*>(head + at));
            } else {
                *reinterpret_cast<words_t*>(head + at) = packed;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kValues; ++i) {
                if (first + i < n) {
                    head[at + i] = static_cast<elem_t>(f[i]);
                }
            }
        }
    }
};

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
// 16 bits; fp32 results go through the library, and are turned on by what the 32 bits of its argument leave of the angle (up to 2^-26 of a turn, which would be
// more than the rounding of the results)
template <typename T>
__device__ __forceinline__ void rotary_turn(double turns, float& c, float& s)
{
    const float most = static_cast<float>(turns);
    if constexpr (ln_traits<T>::kPerChunk == 4) {
        float c0, s0;
        sincospif(2.0f * most, &s0, &c0);
        const float rest = static_cast<float>(turns - most) * 6.2831853f;
        c = __builtin_fmaf(-rest, s0, c0);
        s = __builtin_fmaf(rest, c0, s0);
    } else {
        c = __builtin_amdgcn_cosf(most);
        s = __builtin_amdgcn_sinf(most);
    }
}

template <typename T, bool INTERLEAVED, int KIND>
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

    const auto from = [&](int h) -> const E* {
        return h < a.heads_q ? static_cast<const E*>(a.q) + row * a.q_stride_row + h * a.q_stride_head
                             : static_cast<const E*>(a.k) + row * a.k_stride_row + (h - a.heads_q) * a.k_stride_head;
    };
    const auto to = [&](int h) -> E* {
        return h < a.heads_q ? static_cast<E*>(a.q_out) + (static_cast<int64_t>(row) * a.heads_q + h) * a.dim
                             : static_cast<E*>(a.k_out) + (static_cast<int64_t>(row) * (a.heads - a.heads_q) + (h - a.heads_q)) * a.dim;
    };

    using Piece = rotary_piece<T, KIND>;
    constexpr int kValues = Piece::kValues;
    // turned values: side by side pieces `item` and `item + turned` of all of them, halves piece `item` of each; copied values: two pieces of the rest
    const bool copied = item >= a.turned;
    const int rest0 = item - a.turned;
    const int begin = copied ? 2 * a.pairs : 0, n = copied ? a.dim - begin : INTERLEAVED ? 2 * a.pairs : a.pairs;
    const int c0 = Piece::place(copied ? rest0 : item, n);
    const int c1 = Piece::place(copied ? rest0 + a.items - a.turned : INTERLEAVED ? item + a.turned : item, n);
    const int at0 = begin + c0, at1 = begin + c1 + (copied || INTERLEAVED ? 0 : a.pairs);
    Piece lo[kRotaryHeads], hi[kRotaryHeads];
#pragma unroll
    for (int i = 0; i < kRotaryHeads; ++i) {
        if (first + i < last) {
            const E* const p = from(first + i);
            lo[i].load(p, at0, c0, n);
            hi[i].load(p, at1, c1, n);
        }
    }
    __builtin_amdgcn_sched_barrier(0);

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
    float cs[kValues], sn[kValues];
    if (!copied) {
#pragma unroll
        for (int j = 0; j < kValues; ++j) {
            const int at = INTERLEAVED ? (j < kValues / 2 ? c0 : c1) / 2 + j % (kValues / 2) : c0 + j;
            double turns = position * a.frequencies[min(at, a.pairs - 1)] * 0.15915494309189533577;  // 1 / (2 pi)
            turns -= rint(turns);
            rotary_turn<T>(turns, cs[j], sn[j]);
            cs[j] *= a.magnitude;
            sn[j] *= a.magnitude * a.sign;
        }
    }
#pragma unroll
    for (int i = 0; i < kRotaryHeads; ++i) {
        if (first + i < last) {
            float u[kValues], v[kValues];
            lo[i].unpack(u);
            hi[i].unpack(v);
            if (!copied) {
                if constexpr (INTERLEAVED) {
                    constexpr int kPairs = kValues / 2;
#pragma unroll
                    for (int j = 0; j < kPairs; ++j) {
                        const float a0 = u[2 * j], b0 = u[2 * j + 1], a1 = v[2 * j], b1 = v[2 * j + 1];
                        u[2 * j] = a0 * cs[j] - b0 * sn[j];
                        u[2 * j + 1] = b0 * cs[j] + a0 * sn[j];
                        v[2 * j] = a1 * cs[kPairs + j] - b1 * sn[kPairs + j];
                        v[2 * j + 1] = b1 * cs[kPairs + j] + a1 * sn[kPairs + j];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < kValues; ++j) {
                        const float a0 = u[j], b0 = v[j];
                        u[j] = a0 * cs[j] - b0 * sn[j];
                        v[j] = b0 * cs[j] + a0 * sn[j];
                    }
                }
            }
            if (!inside) {  // (zeros, whatever the values: a product with 0 would keep NaN)
#pragma unroll
                for (int j = 0; j < kValues; ++j) {
                    u[j] = 0.0f;
                    v[j] = 0.0f;
                }
            }
            E* const p = to(first + i);
            Piece::store(p, at0, c0, n, u);
            Piece::store(p, at1, c1, n, v);
        }
    }
}

}  // namespace hstu
