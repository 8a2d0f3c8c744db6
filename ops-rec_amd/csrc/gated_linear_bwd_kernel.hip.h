// The element-wise stage of the gated projections' backward, and the sums of what is computed in parts, for gfx950.
//
//   mixed = (g, u), grad = gradient of hidden:   d g = grad * u * act'(g),   d u = grad * act(g),   d mixed = (d g, d u)
//   d bias = column sums of d mixed, taken of the values before they are rounded
//
// Bound by HBM: 8 bytes read and 4 written per column of hidden.  (d mixed is rounded to the type of x, half a step of it: what the matrix instructions of
// the products behind it multiply; in fp16 it is scaled ahead of that, kGatedScaled.)  A thread has 8 columns and walks over the rows of its slice; its
// sums stay in registers, those of a workgroup's eight rows of threads meet in LDS, and a row of partial sums per workgroup goes to the workspace.
#pragma once
#include "gated_linear_gemm.hip.h"

namespace hstu {

constexpr int kStageThreads = 256;
constexpr int kStageCols = 256;  // columns of hidden per workgroup: 32 threads of 8
constexpr int kStageRows = kStageThreads / (kStageCols / 8);

template <typename Tag>
__global__ __launch_bounds__(kStageThreads) void gated_stage_kernel(const GatedStageArgs a)
{
    __shared__ float s_sums[kStageRows][2][kStageCols];
    const int sub = threadIdx.x / (kStageCols / 8), c = threadIdx.x % (kStageCols / 8);
    const uint32_t blocks = static_cast<uint32_t>((a.inner + kStageCols - 1) / kStageCols);
    const uint32_t slice = blockIdx.x / blocks;
    const int col = static_cast<int>(blockIdx.x - slice * blocks) * kStageCols + 8 * c;
    const bool have = col < a.inner;
    float scale = kGatedScale, largest = 0.0f;
    if constexpr (kGatedScaled<Tag>) {
        if (a.scale != nullptr) {
            scale = *a.scale;
            if (scale == kGatedScale) {  // the first pass was enough
                return;
            }
        }
    }
    const auto pack = [&](float x, float y) {
        if constexpr (kGatedScaled<Tag>) {
            largest = gated_larger(gated_larger(largest, x), y);
            x *= scale;
            y *= scale;
        }
        return pack2<Tag>(x, y);
    };
    float dg[8], du[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        dg[e] = du[e] = 0.0f;
    }
    const int64_t step = static_cast<int64_t>(a.slices) * kStageRows;
    if (have) {
        with_activation(a.activation, [&](auto chosen) {
            constexpr int kind = decltype(chosen)::value;
            for (int64_t row = static_cast<int64_t>(slice) * kStageRows + sub; row < a.rows; row += step) {
                const u32x4_t d4 = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.grad) + row * a.inner + col));
                const uint16_t* const m = static_cast<const uint16_t*>(a.mixed) + row * 3 * a.inner + col;
                const u32x4_t g4 = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(m));
                const u32x4_t u4 = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(m + a.inner));
                const u32x4_t low = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(m + 2 * a.inner));
                u32x4_t og, ou;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float d[2], x[2], y[2];
                    ils_unpack2<Tag>(d4[e], d[0], d[1]);
                    const uint32_t gl = low[e / 2], ul = low[2 + e / 2];
                    const float g[2] = {e % 2 == 0 ? kept_value<0, 0>(g4[e], gl) : kept_value<0, 2>(g4[e], gl),
                                        e % 2 == 0 ? kept_value<1, 1>(g4[e], gl) : kept_value<1, 3>(g4[e], gl)};
                    const float u[2] = {e % 2 == 0 ? kept_value<0, 0>(u4[e], ul) : kept_value<0, 2>(u4[e], ul),
                                        e % 2 == 0 ? kept_value<1, 1>(u4[e], ul) : kept_value<1, 3>(u4[e], ul)};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float act, slope;
                        gated_act_slope<kind>(g[h], act, slope);
                        x[h] = d[h] * u[h] * slope;
                        y[h] = d[h] * act;
                        dg[2 * e + h] += x[h];
                        du[2 * e + h] += y[h];
                    }
                    og[e] = pack(x[0], x[1]);
                    ou[e] = pack(y[0], y[1]);
                }
                uint16_t* const to = static_cast<uint16_t*>(a.d_mixed) + row * 2 * a.inner + col;
                *reinterpret_cast<u32x4_t*>(to) = og;
                *reinterpret_cast<u32x4_t*>(to + a.inner) = ou;
            }
        });
    }
    if constexpr (kGatedScaled<Tag>) {
        if (a.range != nullptr) {
            gated_note_range(largest, a.range + static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 64);
        }
    }
    if (a.partial == nullptr) {
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        s_sums[sub][0][8 * c + e] = dg[e];
        s_sums[sub][1][8 * c + e] = du[e];
    }
    __syncthreads();
    const int first = static_cast<int>(blockIdx.x - slice * blocks) * kStageCols;
    for (int at = threadIdx.x; at < 2 * kStageCols; at += kStageThreads) {
        const int p = at / kStageCols, i = at % kStageCols;
        if (first + i < a.inner) {
            float t = 0.0f;
#pragma unroll
            for (int s = 0; s < kStageRows; ++s) {
                t += s_sums[s][p][i];
            }
            a.partial[(static_cast<int64_t>(slice) * 2 + p) * a.inner + first + i] = t;
        }
    }
}

// The weight gradient's partial outputs, added chunk by chunk in one order and rounded once.
template <typename Tag>
__global__ __launch_bounds__(256) void gated_sum_kernel(const GatedSumArgs a)
{
    const int64_t pieces = a.n / 8;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < pieces; i += static_cast<int64_t>(gridDim.x) * 256) {
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            t[e] = 0.0f;
        }
#pragma unroll 4
        for (int c = 0; c < a.chunks; ++c) {
            const float4* const from = reinterpret_cast<const float4*>(a.partial + static_cast<int64_t>(c) * a.n) + 2 * i;
            const float4 lo = from[0], hi = from[1];
            t[0] += lo.x, t[1] += lo.y, t[2] += lo.z, t[3] += lo.w;
            t[4] += hi.x, t[5] += hi.y, t[6] += hi.z, t[7] += hi.w;
        }
        if constexpr (kGatedScaled<Tag>) {
            const float back = a.scale[1];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                t[e] *= back;
            }
        }
        const u32x4_t w = {pack2<Tag>(t[0], t[1]), pack2<Tag>(t[2], t[3]), pack2<Tag>(t[4], t[5]), pack2<Tag>(t[6], t[7])};
        reinterpret_cast<u32x4_t*>(a.out)[i] = w;
    }
}

}  // namespace hstu
