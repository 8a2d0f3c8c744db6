// The gated projections for few rows, gfx950: hidden = act(x Wg^T + bg) * (x Wu^T + bu) for single tokens and small batches.
//
// Bound by the bytes of the weight, each read once, by those of x, which every workgroup reads, and for small layers by latency.  A workgroup has C columns
// of hidden: C rows of the gate's weight, the C of the other projection, and all rows of x.  Its eight wavefronts share the depth: each takes every eighth
// run of 64 values, brings in the run's whole 128-byte lines of all these rows by direct-to-LDS requests, reads them back as v_mfma_f32_16x16x32 operands (16-byte
// chunks XOR-ed with (row / 2) % 8), and the partial sums meet in LDS.  (Operands straight from memory take half a line of 16 rows an instruction, and a compute unit
// has only so many requests under way: 48 rows, 2048 -> 5632, 18.6 us, 12.7 so, of 9.3 that the bytes would take; one row, 4096 -> 11264, 39.7 and 30.0.)
// C is 8, 16, 24 or 32, whichever leaves the fullest compute unit the least to read: rounds of workgroups times 2 C + rows.  (48 rows,
// 2048 -> 5632, straight from memory: 352 workgroups of 16 columns, two on some compute units, took 25 us; 235 of 24, one on each, 18.6.)  Two to four runs of a
// wavefront under way instead of one, in as much more LDS, are level or slower.
#pragma once
#include "gated_linear_gemm.hip.h"

namespace hstu {

constexpr int kFewWaves = 8;
constexpr int kFewThreads = 64 * kFewWaves;
constexpr int kFewStep = 64;  // values of the depth a wavefront takes at a time: two operands' worth, a whole 128-byte line of a row
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

// MB = blocks of 16 rows, AB = blocks of 16 weight rows (C = 8 AB)
template <typename Tag, int MB, int AB>
__global__ __launch_bounds__(kFewThreads) void gated_few_rows_kernel(const GatedFewRowsArgs a)
{
    constexpr int C = 8 * AB;
    constexpr int kRows = 16 * MB;
    // partial sums of half the wavefronts [wavefront][operand][row of x][16 weight rows], rows padded by 4 so that 16 rows at 16 bytes spread over
    // the banks
    constexpr int kPitch = 16 + 4, kHalf = kFewWaves / 2;
    // a wavefront's run on its way to the operands: rows of x, then of the weight
    constexpr int kRun = (kRows + 16 * AB) * kFewStep;  // values
    constexpr int kPart = kHalf * AB * kRows * kPitch * 4, kRuns = kFewWaves * kRun * 2;
    __shared__ __attribute__((aligned(1024))) uint8_t s_all[kPart > kRuns ? kPart : kRuns];
    float* const s_part = reinterpret_cast<float*>(s_all);

    const int lane = threadIdx.x & 63;
    const int wave = uniform(threadIdx.x >> 6);
    const int n0 = static_cast<int>(blockIdx.x) * C;
    const int rows = static_cast<int>(a.rows);  // (at most kRows)
    const int cols = min(C, a.inner - n0);
    const uint32_t row_bytes = static_cast<uint32_t>(a.depth) * 2u;
    // rows and columns past the end read as zeros
    const __amdgpu_buffer_rsrc_t w_rsrc = make_rsrc(a.weight, static_cast<uint32_t>(2 * a.inner) * row_bytes);
    const __amdgpu_buffer_rsrc_t x_rsrc = make_rsrc(a.x, static_cast<uint32_t>(rows) * row_bytes);

    const int r = lane & 15, quarter = lane >> 4;
    // the lane's weight rows, the gate's C ahead of the other projection's
    uint32_t w_row[2 * AB];
#pragma unroll
    for (int g = 0; g < 2 * AB; ++g) {
        const int at = 8 * g + (lane >> 3), c = at < C ? at : at - C;
        w_row[g] = c < cols ? static_cast<uint32_t>((at < C ? 0 : a.inner) + n0 + c) * row_bytes : kOutOfRange;
    }
    f32x4_t acc[AB][MB];
#pragma unroll
    for (int i = 0; i < AB; ++i) {
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    // Workgroups begin at different runs of the depth: rows a multiple of 4 KB apart lie in one channel of the L2, which all would ask at once.
    const int runs = (a.depth + kFewStep - 1) / kFewStep, turn = static_cast<int>(blockIdx.x * 5u % static_cast<uint32_t>(runs));
    uint16_t* const s_x = reinterpret_cast<uint16_t*>(s_all) + wave * kRun;
    uint16_t* const s_w = s_x + kRows * kFewStep;
    typedef __attribute__((address_space(3))) void lds_t;
    const auto operand = [&](const uint16_t* rows_at, int block, int k) {
        return *reinterpret_cast<const u32x4_t*>(rows_at + (16 * block + r) * kFewStep + 8 * ((4 * k + quarter) ^ ((r >> 1) & 7)));
    };
    for (int run0 = wave; run0 < runs; run0 += kFewWaves) {
        const int run = run0 + turn, d0 = (run < runs ? run : run - runs) * kFewStep;
        // 8 rows a request, a whole line each
        const auto along = [&](int row) { return d0 + 8 * ((lane & 7) ^ ((row >> 1) & 7)); };
#pragma unroll
        for (int g = 0; g < 2 * AB; ++g) {  // (the weight is read once: non-temporal, so that x stays in the caches)
            const int d = along(8 * g + (lane >> 3));
            const uint32_t off = d < a.depth && w_row[g] != kOutOfRange ? w_row[g] + static_cast<uint32_t>(d) * 2u : kOutOfRange;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(w_rsrc, (lds_t*)(s_w + 8 * g * kFewStep), 16, static_cast<int>(off), 0, 0, 2);
        }
#pragma unroll
        for (int g = 0; g < 2 * MB; ++g) {
            const int row = 8 * g + (lane >> 3), d = along(row);
            const uint32_t off = d < a.depth ? static_cast<uint32_t>(row) * row_bytes + static_cast<uint32_t>(d) * 2u : kOutOfRange;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(x_rsrc, (lds_t*)(s_x + 8 * g * kFewStep), 16, static_cast<int>(off), 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(gemm_wait(0, 15));
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int i = 0; i < AB; ++i) {
                const u32x4_t w = operand(s_w, i, k);
#pragma unroll
                for (int j = 0; j < MB; ++j) {
                    acc[i][j] = gated_mfma16<Tag>(w, operand(s_x, j, k), acc[i][j]);
                }
            }
        }
        __builtin_amdgcn_s_waitcnt(gemm_wait(63, 0));  // (a run is read before the next is written)
        __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();  // (sums go where other wavefronts' x was)
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
    for (int one = threadIdx.x; one < kRows * C; one += kFewThreads) {
        const int row = one / C, c = one % C;
        if (row >= rows || c >= cols) {
            continue;
        }
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
            for (int w = 0; w < kHalf; ++w) {
                const int at = c + p * C;
                sum[p] += s_part[((w * AB + at / 16) * kRows + row) * kPitch + at % 16];
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
            uint16_t* const m = static_cast<uint16_t*>(a.mixed) + to * 3 * a.inner;
            uint8_t* const low = reinterpret_cast<uint8_t*>(m + 2 * a.inner) + 16 * ((n0 + c) / 8) + (n0 + c) % 8;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const uint32_t bits = __builtin_bit_cast(uint32_t, sum[p]);
                m[p * a.inner + n0 + c] = static_cast<uint16_t>(bits >> 16);
                low[8 * p] = static_cast<uint8_t>(bits >> 8);
            }
        }
    }
}

}  // namespace hstu
