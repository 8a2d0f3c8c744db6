// The gated projections for few rows, gfx950: hidden = act(x Wg^T + bg) * (x Wu^T + bu) for single tokens and small batches.
//
// Bound by the bytes of the weight, each read once, and for small layers by latency.  A workgroup has C columns of
// hidden: C rows of the gate's weight and the C of the other projection, straight from memory into v_mfma_f32_16x16x32 operands (a lane's 16
// bytes are 8 values of one weight row; nothing of the weight is read twice, so LDS would only add a trip).  Its eight wavefronts share
// the depth: each takes every eighth run of 64 values, whose loads are all in flight before the first product, and the partial sums meet in LDS.
// C is 8 (gate and other projection are the two halves of one operand) where 16 would leave compute units without a workgroup.
#pragma once
#include "gated_linear_gemm.hip.h"

namespace hstu {

constexpr int kFewWaves = 8;
constexpr int kFewThreads = 64 * kFewWaves;
constexpr int kFewStep = 64;  // values of the depth a wavefront takes at a time: two operands' worth, a whole 128-byte line of a weight row
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

template <typename Tag>
__device__ __forceinline__ f32x4_t gated_mfma16(u32x4_t a, u32x4_t b, f32x4_t c)
{
    if constexpr (std::is_same_v<Tag, bf16_tag>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
}

// MB = blocks of 16 rows, C = columns of hidden per workgroup (8 or 16)
template <typename Tag, int MB, int C>
__global__ __launch_bounds__(kFewThreads) void gated_few_rows_kernel(const GatedFewRowsArgs a)
{
    constexpr int AB = C == 16 ? 2 : 1;  // 16-row weight operands
    constexpr int kRows = 16 * MB;
    // partial sums of half the wavefronts [wavefront][operand][row of x][16 weight rows], rows padded by 4 so that 16 rows at 16 bytes spread over
    // the banks.  (Of all of them, 64 rows would leave room for one workgroup to a compute unit: 48 rows, 2048 -> 5632, 22 us.)
    constexpr int kPitch = 16 + 4, kHalf = kFewWaves / 2;
    __shared__ __attribute__((aligned(16))) float s_part[kHalf * AB * kRows * kPitch];

    const int lane = threadIdx.x & 63;
    const int wave = uniform(threadIdx.x >> 6);
    const int n0 = static_cast<int>(blockIdx.x) * C;
    const int rows = static_cast<int>(a.rows);  // (at most kRows)
    const int cols = min(C, a.inner - n0);
    const uint32_t row_bytes = static_cast<uint32_t>(a.depth) * 2u;
    // rows past the end read as zeros
    const __amdgpu_buffer_rsrc_t g_rsrc = make_rsrc(static_cast<const uint8_t*>(a.weight) + static_cast<int64_t>(n0) * row_bytes, static_cast<uint32_t>(cols) * row_bytes);
    const __amdgpu_buffer_rsrc_t u_rsrc =
        make_rsrc(static_cast<const uint8_t*>(a.weight) + (static_cast<int64_t>(a.inner) + n0) * row_bytes, static_cast<uint32_t>(cols) * row_bytes);
    const __amdgpu_buffer_rsrc_t x_rsrc = make_rsrc(a.x, static_cast<uint32_t>(rows) * row_bytes);

    const int r = lane & 15, quarter = lane >> 4;
    auto offset = [&](int row, int d) -> int {
        return static_cast<int>(d < a.depth ? static_cast<uint32_t>(row) * row_bytes + static_cast<uint32_t>(d) * 2u : kOutOfRange);
    };
    // (the weight is read once: non-temporal, so that x stays in the caches)
    auto load_weight = [&](__amdgpu_buffer_rsrc_t rsrc, int row, int d) -> u32x4_t { return __builtin_amdgcn_raw_buffer_load_b128(rsrc, offset(row, d), 0, 2); };
    f32x4_t acc[AB][MB];
#pragma unroll
    for (int i = 0; i < AB; ++i) {
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    constexpr int kUnroll = MB <= 2 ? 4 : 2;
    for (int d0 = wave * kFewStep; d0 < a.depth; d0 += kFewWaves * kFewStep * kUnroll) {
        u32x4_t w[kUnroll][2][AB], x[kUnroll][2][MB];
#pragma unroll
        for (int s = 0; s < kUnroll; ++s) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int d = d0 + s * kFewWaves * kFewStep + 32 * k + 8 * quarter;
                if constexpr (C == 16) {
                    w[s][k][0] = load_weight(g_rsrc, r, d);
                    w[s][k][1] = load_weight(u_rsrc, r, d);
                } else {
                    // (rows 0 .. 7 the gate's, 8 .. 15 the other projection's, by lane)
                    const uint32_t in_row = d < a.depth && (r & 7) < cols ? static_cast<uint32_t>(d) * 2u : kOutOfRange;
                    const int64_t row = static_cast<int64_t>(n0) + (r & 7) + (r >= 8 ? a.inner : 0);
                    u32x4_t v = {0u, 0u, 0u, 0u};
                    if (in_row != kOutOfRange) {
                        v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(static_cast<const uint8_t*>(a.weight) + row * row_bytes + in_row));
                    }
                    w[s][k][0] = v;
                }
#pragma unroll
                for (int j = 0; j < MB; ++j) {
                    x[s][k][j] = __builtin_amdgcn_raw_buffer_load_b128(x_rsrc, offset(16 * j + r, d), 0, 0);
                }
            }
        }
#pragma unroll
        for (int s = 0; s < kUnroll; ++s) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int i = 0; i < AB; ++i) {
#pragma unroll
                    for (int j = 0; j < MB; ++j) {
                        acc[i][j] = gated_mfma16<Tag>(w[s][k][i], x[s][k][j], acc[i][j]);
                    }
                }
            }
        }
    }
    // a lane has weight rows 4 quarter .. + 3 of row r of x; the second half of the wavefronts hands its sums to the first
    auto place = [&](int w, int i, int j) { return reinterpret_cast<f32x4_t*>(s_part + ((w * AB + i) * kRows + 16 * j + r) * kPitch + 4 * quarter); };
    if (wave >= kHalf) {
#pragma unroll
        for (int i = 0; i < AB; ++i) {
#pragma unroll
            for (int j = 0; j < MB; ++j) {
                *place(wave - kHalf, i, j) = acc[i][j];
            }
        }
    }
    __syncthreads();
    if (wave < kHalf) {
#pragma unroll
        for (int i = 0; i < AB; ++i) {
#pragma unroll
            for (int j = 0; j < MB; ++j) {
                *place(wave, i, j) += acc[i][j];
            }
        }
    }
    __syncthreads();
    for (int at = threadIdx.x; at < kRows * C; at += kFewThreads) {
        const int row = at / C, c = at % C;
        if (row >= rows || c >= cols) {
            continue;
        }
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
            for (int w = 0; w < kHalf; ++w) {
                const int i = C == 16 ? p : 0, col = C == 16 ? c : c + 8 * p;
                sum[p] += s_part[((w * AB + i) * kRows + row) * kPitch + col];
            }
            if (a.bias != nullptr) {
                const uint32_t b = static_cast<const uint16_t*>(a.bias)[static_cast<int64_t>(p) * a.inner + n0 + c];
                sum[p] += lo_to_float<Tag>(b);
            }
        }
        const int64_t to = row;
        if (a.hidden != nullptr) {
            float act = 0.0f;
            with_activation(a.activation, [&](auto chosen) { act = gated_act<decltype(chosen)::value>(sum[0]); });
            static_cast<uint16_t*>(a.hidden)[to * a.inner + n0 + c] = static_cast<uint16_t>(pack2<Tag>(act * sum[1], 0.0f));
        }
        if (a.mixed != nullptr) {
            uint16_t* const m = static_cast<uint16_t*>(a.mixed) + to * 2 * a.inner + n0 + c;
            m[0] = static_cast<uint16_t>(pack2<Tag>(sum[0], 0.0f));
            m[a.inner] = static_cast<uint16_t>(pack2<Tag>(sum[1], 0.0f));
        }
    }
}

}  // namespace hstu
