// Norms around a block of a layer, forward and backward, gfx950.
//
//   in front of a block:  s = residual + scale * x;  r = s rounded to the stream's type;  y = norm(s) * gamma + beta
//   behind a block:       m = norm(x) * gamma + beta per part of a row;  out = [residual + residual_scale *] m * act(gate)
//   norm(s) = (s - mean) * rstd, or s * rstd (root mean square);  rstd = 1 / sqrt(mean of the squares + eps)
//
// y is the norm of the sum before it is rounded, and the backward starts from what has all its bits: from the stream that was
// written where that is fp32, from x and the residual that went in where it is 16-bit.  (From the rounded sum the gradients of
// gamma and scale, fp32 sums over all rows, would be off by 2^-9 each row.)  Nothing is saved per row: a row is in registers in the
// backward as well, where its mean and rstd cost two reductions and no memory.
//
//   backward, with n = norm(s), g = (gradient of m or y) * gamma, means over the part of a row:
//     d s = rstd * (g - mean(g) - n * mean(g * n))       (root mean square: without mean(g))
//     d gamma = sum over rows of (gradient of m or y) * n,  d beta = sum of it,  d scale = sum of d s * x
//     d gate = d m * m * act'(gate)
//
// A dozen flops per value: bound by HBM.  A row (or part) belongs to G lanes -- a slice of a wavefront, a wavefront or a workgroup --
// which hold it in registers as NV pieces of 8 values per lane; all loads of a row are in flight before the first use, and sums
// over a wavefront go through DPP and lane swaps (10 instructions, no LDS).  Pieces start anywhere: the 16-byte accesses of this
// machine need no alignment, so odd widths and strides take the same path, and a row's last piece, where it is not whole, is its last 8 values (norm_base).
//
// The backward is persistent: a workgroup keeps one part of the columns and walks over rows, its lanes adding up the gradients of
// gamma, beta and scale in registers; the sums of a workgroup's lane groups meet in LDS, one row of partial sums per workgroup goes to the
// workspace, and a second kernel adds those in a fixed order: the same bits every launch.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lane_sums.hip.h"
#include "layer_args.h"
#include "ln_mul_kernel.hip.h"

namespace hstu {

constexpr int kNormFront = 0, kNormBehind = 1;

constexpr int norm_fwd_threads(int g) { return g > 256 ? g : 256; }
constexpr int norm_bwd_threads(int g) { return g > 64 ? g : 512; }  // (barriers inside a row: one row at a time)

// a lane's group within its workgroup: where a group is whole wavefronts, it and all that follows from it (rows, addresses) is the same in all lanes
// and kept in scalar registers
template <int G>
__device__ __forceinline__ int norm_sub()
{
    const int sub = threadIdx.x / G;
    return G >= 64 ? __builtin_amdgcn_readfirstlane(sub) : sub;
}

// ---- 8 values of a row, as they lie in memory ----
template <typename Tag>
struct norm_piece {
    typedef uint32_t words_t __attribute__((ext_vector_type(4), aligned(2)));
    words_t w[ln_traits<Tag>::kPerChunk == 8 ? 1 : 2];
};

// Piece c of a row of n values is columns 8 c .. + 7; the row's last piece, where it is not whole, is its last 8 columns, some of which the piece before has
// too: every lane's access is one of 16 bytes, and what two lanes hold is stored twice, the same bits, and counted once (norm_own).  (A last
// piece taken value by value cost rows of 1002 columns a quarter of the bandwidth.)  Rows of fewer than 8 values (SHORT) are such a piece that
// starts ahead of the row, and do go value by value, in kernels of their own: with the choice at each load 8192 x 4096 took 46 us, 40 so.  Pieces
// past the row repeat its last one, and count nowhere.
__device__ __forceinline__ int norm_base(int c, int n) { return 8 * c + 8 <= n ? 8 * c : n - 8; }
// the first of a piece's values that is its own: 0 of a whole piece, 8 of a piece past the row
__device__ __forceinline__ int norm_own(int c, int n)
{
    const int left = n - 8 * c;
    return left >= 8 ? 0 : 8 - (left > 0 ? left : 0);
}

template <typename Tag, bool SHORT>
__device__ __forceinline__ norm_piece<Tag> norm_load(const typename ln_traits<Tag>::elem_t* row, int c, int n)
{
    using E = typename ln_traits<Tag>::elem_t;
    norm_piece<Tag> p;
    if constexpr (!SHORT) {
        const typename norm_piece<Tag>::words_t* at = reinterpret_cast<const typename norm_piece<Tag>::words_t*>(row + norm_base(c, n));
        p.w[0] = __builtin_nontemporal_load(at);
        if constexpr (sizeof(E) == 4) {
            p.w[1] = __builtin_nontemporal_load(at + 1);
        }
    } else {
        E e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            e[i] = i >= 8 - n ? row[i - (8 - n)] : static_cast<E>(0.0f);
        }
        __builtin_memcpy(&p, e, sizeof e);
    }
    return p;
}

template <typename Tag>
__device__ __forceinline__ void norm_unpack(const norm_piece<Tag>& p, float (&f)[8])
{
    using T = ln_traits<Tag>;
#pragma unroll
    for (int i = 0; i < 8 / T::kPerChunk; ++i) {
        T::unpack(p.w[i], f + T::kPerChunk * i);
    }
}

template <typename Tag, bool SHORT>
__device__ __forceinline__ void norm_store(typename ln_traits<Tag>::elem_t* row, int c, int n, const float (&f)[8])
{
    using T = ln_traits<Tag>;
    using E = typename T::elem_t;
    if (8 * c >= n) {
        return;
    }
    if constexpr (!SHORT) {
        typename norm_piece<Tag>::words_t* at = reinterpret_cast<typename norm_piece<Tag>::words_t*>(row + norm_base(c, n));
#pragma unroll
        for (int i = 0; i < 8 / T::kPerChunk; ++i) {
            const typename norm_piece<Tag>::words_t w = T::pack(f + T::kPerChunk * i);
            __builtin_nontemporal_store(w, at + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >= 8 - n) {
                row[i - (8 - n)] = static_cast<E>(f[i]);
            }
        }
    }
}

// 8 values per column (gamma, beta, scale)
template <typename Tag, bool SHORT>
__device__ __forceinline__ void norm_columns(const void* p, bool f32, int64_t offset, int c, int n, float (&f)[8])
{
    if (f32) {
        norm_unpack<ln_f32_tag>(norm_load<ln_f32_tag, SHORT>(static_cast<const float*>(p) + offset, c, n), f);
    } else {
        norm_unpack<Tag>(norm_load<Tag, SHORT>(static_cast<const typename ln_traits<Tag>::elem_t*>(p) + offset, c, n), f);
    }
}

// ---- sums over the G lanes of a row ----
// K sums at once.  G > 64: through LDS, a slot of K * 16 floats per call, two slots in turn: a wavefront writes a slot again only
// past the barrier of the call between, which every wavefront reaches after it has read the slot.
constexpr int kNormSlots = 2;
template <int G, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float* s_part, int& slot)
{
#pragma unroll
    for (int k = 0; k < K; ++k) {
        v[k] = wave_sum<G>(v[k]);
    }
    if constexpr (G > 64) {
        constexpr int kWaves = G / 64;
        float* const part = s_part + slot * 2 * 16;
        slot ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                part[16 * k + (threadIdx.x % G) / 64] = v[k];
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float t = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                t += part[16 * k + w];
            }
            v[k] = t;
        }
    }
}

// ---- act(z) and its slope: the hardware's exp2 and reciprocal where the result is rounded to 16 bits, library functions for fp32 ----
template <typename Tag>
__device__ __forceinline__ float norm_sigmoid(float z)
{
    if constexpr (ln_traits<Tag>::kPerChunk == 4) {
        return 1.0f / (1.0f + expf(-z));
    } else {
        return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
    }
}

// s (a lane's NV pieces) -> norm(s) in place; returns rstd.  Two passes over registers; the mean's own rounding is taken out by the sum of the centred
// values, which is 0 for an exact mean.  `full`: rows that fill the lanes, whose values are all their own.
template <int G, int NV>
__device__ __forceinline__ float normalise(float (&s)[NV][8], const int (&own)[NV], bool full, int len, bool rms, float epsilon, float* s_part, int& slot)
{
    const float inv_n = 1.0f / static_cast<float>(len);
    const auto each = [&](auto&& f) {  // over the values that are the lane's own
        if (full) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    f(s[i][j]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    f(j >= own[i] ? s[i][j] : 0.0f);
                }
            }
        }
    };
    if (!rms) {
        float sum[1] = {0.0f};
        each([&](float v) { sum[0] += v; });
        row_sums<G>(sum, s_part, slot);
        const float mean = sum[0] * inv_n;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s[i][j] -= mean;
            }
        }
    }
    float sq[2] = {0.0f, 0.0f};
    each([&](float v) {
        sq[0] = __builtin_fmaf(v, v, sq[0]);
        sq[1] += v;
    });
    row_sums<G>(sq, s_part, slot);
    const float shift = rms ? 0.0f : sq[1] * inv_n;
    const float size = sq[0] * inv_n - shift * shift;
    const float rstd = 1.0f / sqrtf((size < 0.0f ? 0.0f : size) + epsilon);  // (NaN stays: a row with one has no root mean square)
    const float away = -shift * rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            s[i][j] = __builtin_fmaf(s[i][j], rstd, away);
        }
    }
    return rstd;
}

// T = type of x (and of y, gate), R = type of the stream; U = parts of rows whose loads are in flight together.  Lanes stay with their columns: from part to
// part they move on by the lanes of the whole grid, a multiple of the parts of a row, and hold gamma, beta and scale in registers.  (Loaded for every row
// again they were half of the kernel's requests: 65536 x 1024 with a gate 99 us, 76 so.)
template <typename T, typename R, int MODE, int G, int NV, int U, bool SHORT>
__global__ __launch_bounds__(norm_fwd_threads(G)) void norm_fwd_kernel(const NormArgs a)
{
    static_assert(G <= 64 || U == 1, "lanes that share barriers have one row");
    using TE = typename ln_traits<T>::elem_t;
    using RE = typename ln_traits<R>::elem_t;
    constexpr uint32_t kPerWg = norm_fwd_threads(G) / G;
    __shared__ float s_part[G > 64 ? kNormSlots * 2 * 16 : 1];
    const int lane = threadIdx.x % G;
    const int len = a.len;
    const bool full = len == 8 * G * NV;
    int own[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        own[i] = norm_own(lane + i * G, len);
    }
    const bool f32 = a.affine_f32 != 0;
    const uint32_t first = blockIdx.x * kPerWg + norm_sub<G>(), step = gridDim.x * kPerWg;
    const uint32_t groups = static_cast<uint32_t>(a.groups);
    const int64_t col0 = groups == 1 ? 0 : static_cast<int64_t>(first % groups) * len;
    int slot = 0;

    float gamma[NV][8], beta[NV][8], scale[NV][8];
    const auto hold = [&] {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = lane + i * G;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                beta[i][j] = 0.0f;
                scale[i][j] = 1.0f;
            }
            norm_columns<T, SHORT>(a.gamma, f32, col0, c, len, gamma[i]);
            if (a.beta != nullptr) {
                norm_columns<T, SHORT>(a.beta, f32, col0, c, len, beta[i]);
            }
            if (MODE == kNormFront && a.scale != nullptr) {
                norm_columns<T, SHORT>(a.scale, f32, col0, c, len, scale[i]);
            }
        }
    };

    bool held = false;
    for (uint64_t unit0 = first; unit0 < a.units; unit0 += static_cast<uint64_t>(step) * U) {  // (G > 64: all of a workgroup's lanes go round as often)
        norm_piece<T> xp[U][NV], gp[U][NV];
        norm_piece<R> rp[U][NV];
        int64_t dense[U];
#pragma unroll
        for (int t = 0; t < U; ++t) {
            const uint64_t unit = unit0 + static_cast<uint64_t>(t) * step;
            dense[t] = -1;
            if (unit < a.units) {
                const uint32_t row = groups == 1 ? static_cast<uint32_t>(unit) : static_cast<uint32_t>(unit) / groups;
                dense[t] = static_cast<int64_t>(row) * len * a.groups + col0;
                const TE* const x = static_cast<const TE*>(a.x) + static_cast<int64_t>(row) * a.x_stride + col0;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    xp[t][i] = norm_load<T, SHORT>(x, lane + i * G, len);
                }
                if (MODE == kNormFront || a.residual != nullptr) {
                    const RE* const res = static_cast<const RE*>(a.residual) + static_cast<int64_t>(row) * a.residual_stride + col0;
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        rp[t][i] = norm_load<R, SHORT>(res, lane + i * G, len);
                    }
                }
                if (MODE == kNormBehind && a.gate != nullptr) {
                    const TE* const gate = static_cast<const TE*>(a.gate) + static_cast<int64_t>(row) * a.gate_stride + col0;
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        gp[t][i] = norm_load<T, SHORT>(gate, lane + i * G, len);
                    }
                }
            }
        }
        if (!held) {  // (behind the first rows' loads)
            held = true;
            hold();
        }
#pragma unroll
        for (int t = 0; t < U; ++t) {
            if (dense[t] < 0) {
                continue;
            }
            float s[NV][8];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                norm_unpack<T>(xp[t][i], s[i]);
            }
            if constexpr (MODE == kNormFront) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    float f[8];
                    norm_unpack<R>(rp[t][i], f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        s[i][j] = __builtin_fmaf(scale[i][j], s[i][j], f[j]);
                    }
                    norm_store<R, SHORT>(static_cast<RE*>(a.sum) + dense[t], lane + i * G, len, s[i]);
                }
            }
            normalise<G, NV>(s, own, full, len, a.rms != 0, a.epsilon, s_part, slot);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    y[j] = __builtin_fmaf(s[i][j], gamma[i][j], beta[i][j]);
                }
                if constexpr (MODE == kNormBehind) {
                    if (a.gate != nullptr) {
                        float u[8];
                        norm_unpack<T>(gp[t][i], u);
                        if (a.silu) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                y[j] *= u[j] * norm_sigmoid<T>(u[j]);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                y[j] *= u[j];
                            }
                        }
                    }
                    if (a.residual != nullptr) {
                        float f[8];
                        norm_unpack<R>(rp[t][i], f);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            y[j] = __builtin_fmaf(a.residual_scale, y[j], f[j]);
                        }
                    }
                    norm_store<R, SHORT>(static_cast<RE*>(a.out) + dense[t], lane + i * G, len, y);
                } else {
                    norm_store<T, SHORT>(static_cast<TE*>(a.out) + dense[t], lane + i * G, len, y);
                }
            }
        }
    }
}

template <typename T, typename R, int MODE, int G, int NV, bool SHORT>
__global__ __launch_bounds__(norm_bwd_threads(G)) void norm_bwd_kernel(const NormBwdArgs a)
{
    using TE = typename ln_traits<T>::elem_t;
    using RE = typename ln_traits<R>::elem_t;
    constexpr int kThreads = norm_bwd_threads(G);
    constexpr int kRows = kThreads / G;                          // rows of a workgroup at a time
    constexpr bool kFromSum = MODE == kNormFront && ln_traits<R>::kPerChunk == 4;
    constexpr bool kGradR = MODE == kNormBehind;                 // the gradient of the result has the stream's type
    __shared__ float s_part[G > 64 ? kNormSlots * 2 * 16 : 1];
    __shared__ __attribute__((aligned(16))) float s_sums[kRows > 1 ? kThreads * NV * 8 : 1];
    const NormArgs& f = a.f;
    const int sub = norm_sub<G>(), lane = threadIdx.x % G;
    const int part = static_cast<int>(blockIdx.x % static_cast<uint32_t>(f.groups));
    const uint32_t slice = blockIdx.x / static_cast<uint32_t>(f.groups);
    const int len = f.len, cols = f.len * f.groups;
    const bool full = len == 8 * G * NV;
    int own[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        own[i] = norm_own(lane + i * G, len);
    }
    const int64_t col0 = static_cast<int64_t>(part) * len;
    const uint32_t rows = f.units / static_cast<uint32_t>(f.groups);
    const bool f32 = f.affine_f32 != 0;
    const bool need_x = !kFromSum || f.scale != nullptr;
    int slot = 0;

    // The longest rows (2048 pieces) have no registers for gamma, beta and scale, which are loaded for every row, nor for the sums of gamma's and beta's
    // gradients, which are kept in LDS, a lane's own in its own place.  (All in registers, which spill: 2048 x 16384 228 us with a gate, 230 in
    // front; 150 and 127 so.)
    constexpr bool kHold = NV * G < 2048;
    __shared__ float4 s_acc[kHold ? 1 : 2 * NV * 2 * kThreads];
    const auto acc_at = [&](int kind, int i, int h) { return s_acc + ((kind * NV + i) * 2 + h) * kThreads + threadIdx.x; };
    const auto add = [&](float (&sums)[NV][8], int kind, int i, const float (&v)[8]) {
        if constexpr (kHold) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sums[i][j] += v[j];
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float4 t = *acc_at(kind, i, h);
                t.x += v[4 * h], t.y += v[4 * h + 1], t.z += v[4 * h + 2], t.w += v[4 * h + 3];
                *acc_at(kind, i, h) = t;
            }
        }
    };
    float gamma[NV][8], beta[NV][8], scale[NV][8];
    float d_gamma[NV][8], d_beta[NV][8], d_scale[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            d_gamma[i][j] = d_beta[i][j] = d_scale[i][j] = 0.0f;
        }
        if constexpr (!kHold) {
#pragma unroll
            for (int at = 0; at < 4; ++at) {
                *acc_at(at / 2, i, at % 2) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
    }
    const auto hold = [&](int i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            beta[i][j] = 0.0f;
        }
        norm_columns<T, SHORT>(f.gamma, f32, col0, lane + i * G, len, gamma[i]);
        if (MODE == kNormBehind && f.beta != nullptr) {
            norm_columns<T, SHORT>(f.beta, f32, col0, lane + i * G, len, beta[i]);
        }
    };
    const auto hold_scale = [&](int i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            scale[i][j] = 1.0f;
        }
        if (MODE == kNormFront && f.scale != nullptr) {
            norm_columns<T, SHORT>(f.scale, f32, col0, lane + i * G, len, scale[i]);
        }
    };
    if constexpr (kHold) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            hold(i);
            hold_scale(i);
        }
    }

    // a row's values as they lie in memory; those of the next row are on their way while one is worked on
    struct Row {
        norm_piece<T> x[NV], y[NV], gate[NV];
        norm_piece<R> s[NV], d[NV];
    };
    const auto load = [&](uint32_t row, Row& w) {
        const int64_t dense = static_cast<int64_t>(row) * cols + col0;
        if (need_x) {
            const TE* const x = static_cast<const TE*>(f.x) + static_cast<int64_t>(row) * f.x_stride + col0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                w.x[i] = norm_load<T, SHORT>(x, lane + i * G, len);
            }
        }
        if constexpr (MODE == kNormFront) {
            const RE* const from = kFromSum ? static_cast<const RE*>(a.sum) + dense
                                            : static_cast<const RE*>(f.residual) + static_cast<int64_t>(row) * f.residual_stride + col0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                w.s[i] = norm_load<R, SHORT>(from, lane + i * G, len);
            }
            if (a.sum_grad != nullptr) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    w.d[i] = norm_load<R, SHORT>(static_cast<const RE*>(a.sum_grad) + dense, lane + i * G, len);
                }
            }
            if (a.grad != nullptr) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    w.y[i] = norm_load<T, SHORT>(static_cast<const TE*>(a.grad) + dense, lane + i * G, len);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                w.d[i] = norm_load<R, SHORT>(static_cast<const RE*>(a.grad) + dense, lane + i * G, len);
            }
            if (f.gate != nullptr) {
                const TE* const gate = static_cast<const TE*>(f.gate) + static_cast<int64_t>(row) * f.gate_stride + col0;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    w.gate[i] = norm_load<T, SHORT>(gate, lane + i * G, len);
                }
            }
        }
    };
    constexpr bool kAhead = G < 1024;
    Row next;
    if (kAhead && slice * kRows + sub < rows) {
        load(slice * kRows + sub, next);
    }
    for (uint64_t row0 = static_cast<uint64_t>(slice) * kRows; row0 < rows; row0 += static_cast<uint64_t>(a.slices) * kRows) {
        const uint64_t row = row0 + sub, after = row + static_cast<uint64_t>(a.slices) * kRows;
        if (kRows > 1 && row >= rows) {  // (the lanes of a row leave together; no barrier in this loop for G <= 64)
            break;
        }
        const int64_t dense = static_cast<int64_t>(row) * cols + col0;
        Row now;
        if constexpr (kAhead) {
            now = next;
            if (after < rows) {
                load(static_cast<uint32_t>(after), next);
            }
        } else {
            load(static_cast<uint32_t>(row), now);
        }
        float n[NV][8];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (MODE == kNormFront) {
                norm_unpack<R>(now.s[i], n[i]);
                if constexpr (!kFromSum) {
                    if constexpr (!kHold) {
                        hold_scale(i);
                    }
                    float v[8];
                    norm_unpack<T>(now.x[i], v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        n[i][j] = __builtin_fmaf(scale[i][j], v[j], n[i][j]);
                    }
                }
            } else {
                norm_unpack<T>(now.x[i], n[i]);
            }
        }
        const float rstd = normalise<G, NV>(n, own, full, len, f.rms != 0, f.epsilon, s_part, slot);

        // g = (gradient of m or y) * gamma; the gradient itself goes into the sums
        float g[NV][8];
        float means[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float d[8];
            if constexpr (!kHold) {
                hold(i);
            }
            if constexpr (kGradR) {
                norm_unpack<R>(now.d[i], d);
                float u[8], dg[8];
                if (f.gate != nullptr) {
                    norm_unpack<T>(now.gate[i], u);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float dz = d[j] * f.residual_scale;
                    float act = 1.0f, slope = 1.0f;
                    if (f.gate != nullptr) {
                        act = u[j];
                        if (f.silu) {
                            const float sg = norm_sigmoid<T>(u[j]);
                            act = u[j] * sg;
                            slope = sg * __builtin_fmaf(u[j], 1.0f - sg, 1.0f);
                        }
                    }
                    dg[j] = dz * __builtin_fmaf(n[i][j], gamma[i][j], beta[i][j]) * slope;
                    d[j] = dz * act;
                }
                if (f.gate != nullptr && a.gate_grad != nullptr) {
                    norm_store<T, SHORT>(static_cast<TE*>(a.gate_grad) + dense, lane + i * G, len, dg);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    d[j] = 0.0f;
                }
                if (a.grad != nullptr) {
                    norm_unpack<T>(now.y[i], d);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                g[i][j] = d[j] * gamma[i][j];
            }
            // (sums take a lane's own values: what another lane has too, or lies past the row, must not reach them, NaN least of all)
            float dn[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                dn[j] = d[j] * n[i][j];
            }
            add(d_gamma, 0, i, dn);
            add(d_beta, 1, i, d);
            if (full) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    means[0] = __builtin_fmaf(g[i][j], n[i][j], means[0]);
                    means[1] += g[i][j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const bool mine = j >= own[i];
                    means[0] += mine ? g[i][j] * n[i][j] : 0.0f;
                    means[1] += mine ? g[i][j] : 0.0f;
                }
            }
        }
        row_sums<G>(means, s_part, slot);
        const float inv_n = 1.0f / static_cast<float>(len);
        const float along = means[0] * inv_n, level = f.rms ? 0.0f : means[1] * inv_n;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float d[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                d[j] = rstd * (g[i][j] - __builtin_fmaf(n[i][j], along, level));
            }
            if constexpr (MODE == kNormFront) {
                if (a.sum_grad != nullptr) {
                    float v[8];
                    norm_unpack<R>(now.d[i], v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        d[j] += v[j];
                    }
                }
                norm_store<R, SHORT>(static_cast<RE*>(a.residual_grad) + dense, lane + i * G, len, d);
                if (a.want_scale) {
                    float v[8];
                    norm_unpack<T>(now.x[i], v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        d_scale[i][j] = __builtin_fmaf(d[j], v[j], d_scale[i][j]);
                    }
                }
                if (a.x_grad != nullptr) {
                    if constexpr (!kHold) {
                        hold_scale(i);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        d[j] *= scale[i][j];
                    }
                    norm_store<T, SHORT>(static_cast<TE*>(a.x_grad) + dense, lane + i * G, len, d);
                }
            } else if (a.x_grad != nullptr) {
                norm_store<T, SHORT>(static_cast<TE*>(a.x_grad) + dense, lane + i * G, len, d);
            }
        }
    }

    // the sums over this workgroup's rows, kind by kind: a column from the lane whose own it is
    if constexpr (!kHold) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 g4 = *acc_at(0, i, h), b4 = *acc_at(1, i, h);
                d_gamma[i][4 * h] = g4.x, d_gamma[i][4 * h + 1] = g4.y, d_gamma[i][4 * h + 2] = g4.z, d_gamma[i][4 * h + 3] = g4.w;
                d_beta[i][4 * h] = b4.x, d_beta[i][4 * h + 1] = b4.y, d_beta[i][4 * h + 2] = b4.z, d_beta[i][4 * h + 3] = b4.w;
            }
        }
    }
    const auto put = [&](const float (&v)[NV][8], int kind) {
        float* const out = a.partial + (static_cast<int64_t>(kind) * a.slices + slice) * cols + col0;
        if constexpr (kRows > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int base = norm_base(lane + i * G, len);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (j >= own[i]) {
                        s_sums[sub * NV * G * 8 + base + j] = v[i][j];
                    }
                }
            }
            __syncthreads();
            for (int c = threadIdx.x; c < len; c += kThreads) {
                float t = 0.0f;
#pragma unroll
                for (int s = 0; s < kRows; ++s) {
                    t += s_sums[s * NV * G * 8 + c];
                }
                out[c] = t;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int base = norm_base(lane + i * G, len);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (j >= own[i]) {
                        out[base + j] = v[i][j];
                    }
                }
            }
        }
    };
    put(d_gamma, 0);
    if (a.want_beta) {
        put(d_beta, 1);
    }
    if (MODE == kNormFront && a.want_scale) {
        put(d_scale, 1 + a.want_beta);
    }
}

}  // namespace hstu
