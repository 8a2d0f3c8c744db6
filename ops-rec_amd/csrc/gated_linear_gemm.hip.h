// The matrix products of the gated projections for gfx950: one tile kernel for the forward and both products of the backward.
//
//   forward          mixed = x W^T + b = (g, u);  hidden = act(g) * u          depth = columns of x
//   x gradient       d x = d_mixed W                                           depth = 2 inner
//   weight gradient  d W = d_mixed^T x                                         depth = rows, in chunks
//
// Bound by the matrix units (and in the forward up to a depth of a few hundred by its stores).  A workgroup of four wavefronts has a tile of BM
// rows by BN columns of the output, each wavefront a quarter of it in v_mfma_f32_32x32x16 blocks; the columns' side is the A operand, so that a lane
// has outputs of one row, and its columns are placed in a permuted order that gives it runs of 8 consecutive ones: 16-byte pieces.
// The depth goes by in steps of 32 through a ring of STAGES tiles in LDS, filled by direct-to-LDS loads and read while later ones are under way.
// In the forward the BN columns are BN / 2 of the gate and the same BN / 2 of the other projection, dealt so that a wavefront has both
// halves of a column in the same lane: activation and product never leave registers.
//
// A side whose rows run along the depth is kept in LDS by rows of 64 bytes (chunk index XOR-ed with (row / 4) % 4) and read as 16-byte operands;
// a side that is stored the other way -- the weight for d x, both sides of d W -- is kept as it lies, 32 rows of the tile's width, and read
// back with the transposing LDS read (64-byte groups XOR-ed with row % 4): no operand is transposed through memory.
//
// Tiles are dealt to the XCDs in equal runs of a list that goes through the rows in bands of eight tiles, the eight first: the
// 64 workgroups of an XCD work on 8 x 8 tiles at a time, whose operands its L2 holds.
#pragma once
#include "gated_linear_args.h"
#include "in_linear_silu_kernel.hip.h"

namespace hstu {

constexpr int kGemmThreads = 256;
constexpr int kGemmStep = 32;  // of the depth
constexpr int kGemmForward = 0, kGemmXGrad = 1, kGemmWeightGrad = 2;
constexpr int kGemmBand = 8;  // row tiles of a band

__device__ __forceinline__ float gated_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f)); }

// act(z): silu, gelu by its tanh form -- z * sigmoid(2 sqrt(2 / pi) (z + 0.044715 z^3)) --, or the sigmoid.  (hardware exp2 and reciprocal, 1 ulp
// each: the results are rounded to 8 or 11 bits.  Past |z| = 30 gelu's cube could make infinity times 0: its argument is bounded there, where the
// sigmoid is 0 or 1 to all bits.)
template <int ACT>
__device__ __forceinline__ float gated_act(float z)
{
    if constexpr (ACT == kActSilu) {
        return z * gated_sigmoid(z);
    } else if constexpr (ACT == kActGelu) {
        const float t = fminf(fmaxf(z, -30.0f), 30.0f);
        return z * gated_sigmoid(1.5957691216057308f * t * __builtin_fmaf(0.044715f * t, t, 1.0f));
    } else {
        return gated_sigmoid(z);
    }
}

// `f` called with the activation as a constant: one choice for all of a kernel's values (a branch at each made 5000 instructions of an epilogue)
template <typename F>
__device__ __forceinline__ void with_activation(int kind, const F& f)
{
    if (kind == kActSilu) {
        f(std::integral_constant<int, kActSilu>{});
    } else if (kind == kActGelu) {
        f(std::integral_constant<int, kActGelu>{});
    } else {
        f(std::integral_constant<int, kActSigmoid>{});
    }
}

template <int ACT>
__device__ __forceinline__ void gated_act_slope(float z, float& act, float& slope)
{
    if constexpr (ACT == kActSilu) {
        const float s = gated_sigmoid(z);
        act = z * s;
        slope = s * __builtin_fmaf(z, 1.0f - s, 1.0f);
    } else if constexpr (ACT == kActGelu) {
        const float t = fminf(fmaxf(z, -30.0f), 30.0f);
        const float s = gated_sigmoid(1.5957691216057308f * t * __builtin_fmaf(0.044715f * t, t, 1.0f));
        act = z * s;
        slope = s * __builtin_fmaf(t * (1.0f - s), 1.5957691216057308f * __builtin_fmaf(0.134145f * t, t, 1.0f), 1.0f);
    } else {
        act = gated_sigmoid(z);
        slope = act * (1.0f - act);
    }
}

// MFMA row -> column of the transposing read: within 16 lanes the second and third group of four change places, which puts the
// columns into the order of ils_column_of_mfma_row
__device__ __forceinline__ int gemm_tr_col(int lane) { return 16 * ((lane >> 4) & 1) + 4 * (((lane & 1) << 1) | ((lane >> 1) & 1)); }

constexpr int gemm_workgroups_per_cu(int bn, int bm) { return bn * bm >= 256 * 128 ? 2 : (bn * bm >= 128 * 128 ? 3 : 4); }

template <typename Tag, int MODE, int BN, int BM, int STAGES>
__global__ __launch_bounds__(kGemmThreads, gemm_workgroups_per_cu(BN, BM)) void gated_gemm_kernel(const GatedGemmArgs a)
{
    constexpr bool NT = MODE != kGemmForward;     // the columns' side is read transposed
    constexpr bool MT = MODE == kGemmWeightGrad;  // the rows' side is
    constexpr int kReqsN = BN / 64, kReqsM = BM / 64, kReqs = kReqsN + kReqsM;  // direct-to-LDS instructions per wavefront and stage
    constexpr int kNElems = BN * kGemmStep, kStage = (BN + BM) * kGemmStep;
    constexpr int NB = BN / 64, MB = BM / 64;  // 32 x 32 blocks of a wavefront
    constexpr int kEpiRow = 64 + 8;            // staged rows of 64 columns
    constexpr int kEpiPlanes = MODE == kGemmForward ? 3 : 1;
    constexpr int kEpiWave = kEpiPlanes * 32 * kEpiRow;
    constexpr int kLds = STAGES * kStage > 4 * kEpiWave ? STAGES * kStage : 4 * kEpiWave;
    __shared__ __attribute__((aligned(1024))) uint16_t s_tiles[kLds];

    const int lane = threadIdx.x & 63;
    const int wave = uniform(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;

    // ---- the workgroup's tile
    const uint32_t tiles = static_cast<uint32_t>(a.tiles_m) * static_cast<uint32_t>(a.tiles_n);
    const uint32_t all = tiles * static_cast<uint32_t>(a.chunks);
    const uint32_t each = (all + 7u) >> 3;
    const uint32_t place = (blockIdx.x & 7u) * each + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= each || place >= all) {
        return;
    }
    const uint32_t part = place / tiles, tile = place - part * tiles;
    const uint32_t in_band = static_cast<uint32_t>(kGemmBand) * static_cast<uint32_t>(a.tiles_n);
    const uint32_t band = tile / in_band, at = tile - band * in_band;
    const uint32_t high = min(static_cast<uint32_t>(kGemmBand), static_cast<uint32_t>(a.tiles_m) - band * kGemmBand);
    const int tile_n = static_cast<int>(at / high), tile_m = static_cast<int>(band * kGemmBand + at % high);

    const int64_t m0 = static_cast<int64_t>(tile_m) * BM;
    constexpr int kOutCols = MODE == kGemmForward ? BN / 2 : BN;
    const int n0 = tile_n * kOutCols;
    const int64_t depth0 = static_cast<int64_t>(part) * a.chunk;
    const int depth = static_cast<int>(min(a.chunk, a.depth - depth0));  // of this workgroup

    // ---- sources.  Rows and depth past the end read as zeros on both sides (out-of-range bytes of a descriptor)
    const uint32_t n_row_bytes = static_cast<uint32_t>(NT ? a.cols : static_cast<int>(a.depth)) * 2u;
    const uint32_t m_row_bytes = MT ? static_cast<uint32_t>(a.rows) * 2u : static_cast<uint32_t>(a.depth) * 2u;
    __amdgpu_buffer_rsrc_t n_rsrc, u_rsrc, m_rsrc;
    if constexpr (NT) {
        n_rsrc = make_rsrc(static_cast<const uint8_t*>(a.n_side) + depth0 * n_row_bytes, static_cast<uint32_t>(depth) * n_row_bytes);
        u_rsrc = n_rsrc;
    } else {
        const int rows_w = min(kOutCols, a.cols - n0);
        const uint8_t* const w = static_cast<const uint8_t*>(a.n_side);
        n_rsrc = make_rsrc(w + static_cast<int64_t>(n0) * n_row_bytes, static_cast<uint32_t>(rows_w) * n_row_bytes);
        u_rsrc = make_rsrc(w + (static_cast<int64_t>(a.cols) + n0) * n_row_bytes, static_cast<uint32_t>(rows_w) * n_row_bytes);
    }
    if constexpr (MT) {
        m_rsrc = make_rsrc(static_cast<const uint8_t*>(a.m_side) + depth0 * m_row_bytes, static_cast<uint32_t>(depth) * m_row_bytes);
    } else {
        const int rows_m = a.rows - m0 < BM ? static_cast<int>(a.rows - m0) : BM;
        const uint32_t skipped = static_cast<uint32_t>(depth0) * 2u;
        m_rsrc = make_rsrc(static_cast<const uint8_t*>(a.m_side) + m0 * m_row_bytes + skipped, static_cast<uint32_t>(rows_m) * m_row_bytes - skipped);
    }

    // ---- requests: byte offset of the lane's 16 bytes at depth 0, and (row-wise sides) where in the step they are
    uint32_t req_off[kReqs];
    int req_depth[kReqs];
#pragma unroll
    for (int i = 0; i < kReqs; ++i) {
        const bool n_part = i < kReqsN;
        const int q = wave + 4 * (n_part ? i : i - kReqsN);  // instruction of the side
        if (n_part ? NT : MT) {
            const int width = n_part ? BN : BM;
            const int per_row = width / 8;  // 16-byte pieces
            const int row = q * (64 / per_row) + lane / per_row;
            const int piece = n_part ? v_chunk_swizzle<BN>(row, lane % per_row) : v_chunk_swizzle<BM>(row, lane % per_row);
            const int64_t col = (n_part ? static_cast<int64_t>(n0) : m0) + 8 * piece;
            // (columns past the end of a row are the next row's: outputs that are not stored; past the matrix they read as zeros)
            req_off[i] = static_cast<uint32_t>(row) * (n_part ? n_row_bytes : m_row_bytes) + static_cast<uint32_t>(col) * 2u;
            req_depth[i] = row;
        } else {
            const int lds_row = 16 * q + (lane >> 2);
            const int chunk = (lane & 3) ^ ((lds_row >> 2) & 3);
            int row = lds_row;
            if (n_part) {
                // a wavefront's BN / 2 rows: BN / 4 of the gate, BN / 4 of the other projection
                const int w = lds_row / (BN / 2), r = lds_row % (BN / 2) % (BN / 4);
                row = w * (BN / 4) + (r & ~31) + ils_column_of_mfma_row(r & 31);
            }
            req_off[i] = static_cast<uint32_t>(row) * (n_part ? n_row_bytes : m_row_bytes) + chunk * 16u;
            req_depth[i] = 8 * chunk;
        }
    }
    auto request = [&](int stage, int step) {
        uint16_t* const base = s_tiles + stage * kStage;
        const int d0 = step * kGemmStep;
#pragma unroll
        for (int i = 0; i < kReqs; ++i) {
            const bool n_part = i < kReqsN;
            const int q = wave + 4 * (n_part ? i : i - kReqsN);
            const bool across = n_part ? NT : MT;
            const uint32_t along = across ? static_cast<uint32_t>(d0) * (n_part ? n_row_bytes : m_row_bytes) : static_cast<uint32_t>(d0) * 2u;
            const uint32_t off = d0 + req_depth[i] < depth ? req_off[i] + along : kOutOfRange;
            // (forward: 16 LDS rows of one projection per instruction)
            const bool upper = MODE == kGemmForward && n_part && (16 * q) % (BN / 2) >= BN / 4;
            load_to_lds_b128(n_part ? (upper ? u_rsrc : n_rsrc) : m_rsrc, base + (n_part ? 0 : kNElems) + q * 512, off);
        }
    };

    // ---- operand reads: wavefront (wm, wn) has rows BM / 2 wm .. and columns BN / 2 wn .. of the tile
    int n_off[NB], m_off[MB];
    const int r = lane & 31, half = lane >> 5;
    const int swz = (r >> 2) & 3;
    const int tr_row = 8 * half + ((lane & 15) >> 2);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        if constexpr (NT) {
            const int c = BN / 2 * wn + 32 * i + gemm_tr_col(lane);
            n_off[i] = tr_row * BN + v_chunk_swizzle<BN>(tr_row, c >> 3) * 8 + (c & 7);
        } else {
            n_off[i] = (BN / 2 * wn + 32 * i + r) * kGemmStep;
        }
    }
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        if constexpr (MT) {
            const int c = BM / 2 * wm + 32 * j + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
            m_off[j] = kNElems + tr_row * BM + v_chunk_swizzle<BM>(tr_row, c >> 3) * 8 + (c & 7);
        } else {
            m_off[j] = kNElems + (BM / 2 * wm + 32 * j + r) * kGemmStep;
        }
    }
    auto read_across = [&](const uint16_t* p, int width) -> u32x4_t {
        const u32x2_t lo = lds_read_tr16_b64(p);
        const u32x2_t hi = lds_read_tr16_b64(p + 4 * width);
        const u32x4_t v = {lo[0], lo[1], hi[0], hi[1]};
        return v;
    };

    f32x16_t acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int j = 0; j < MB; ++j) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                acc[i][j][e] = 0.0f;
            }
        }
    }

    const int n_steps = (depth + kGemmStep - 1) / kGemmStep;
    constexpr int kAhead = STAGES - 1;
    for (int s = 0; s < kAhead && s < n_steps; ++s) {
        request(s, s);
    }
    constexpr int kWait0 = 0 | (7 << 4) | (15 << 8);
    constexpr int kWait1 = kReqs | (7 << 4) | (15 << 8);
    static_assert(STAGES <= 3 && kReqs <= 15, "the count must fit the low bits of the wait instruction");
    for (int t = 0; t < n_steps; ++t) {
        // requests issued after step t's own: those of step t + 1 with three stages
        __builtin_amdgcn_sched_barrier(0);
        if (STAGES == 3 && t + 1 < n_steps) {
            __builtin_amdgcn_s_waitcnt(kWait1);
        } else {
            __builtin_amdgcn_s_waitcnt(kWait0);
        }
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        // every wavefront is past step t - 1: its stage may be overwritten
        if (t + kAhead < n_steps) {
            request((t + kAhead) % STAGES, t + kAhead);
        }
        const uint16_t* const st = s_tiles + (t % STAGES) * kStage;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int chunk = ((2 * kk + half) ^ swz) * 8;
            u32x4_t nv[NB], mv[MB];
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                if constexpr (NT) {
                    nv[i] = read_across(st + n_off[i] + 16 * kk * BN, BN);
                } else {
                    nv[i] = *reinterpret_cast<const u32x4_t*>(st + n_off[i] + chunk);
                }
            }
#pragma unroll
            for (int j = 0; j < MB; ++j) {
                if constexpr (MT) {
                    mv[j] = read_across(st + m_off[j] + 16 * kk * BM, BM);
                } else {
                    mv[j] = *reinterpret_cast<const u32x4_t*>(st + m_off[j] + chunk);
                }
            }
#pragma unroll
            for (int i = 0; i < NB; ++i) {
#pragma unroll
                for (int j = 0; j < MB; ++j) {
                    acc[i][j] = mfma32<Tag>(nv[i], mv[j], acc[i][j]);
                }
            }
        }
    }

    // ---- gradients in chunks of the depth: fp32 partial outputs, runs of 8 columns
    const int64_t row_of_lane = m0 + BM / 2 * wm + r;
    if (MODE != kGemmForward && a.partial != nullptr) {
        float* const out = a.partial + static_cast<int64_t>(part) * a.rows * a.cols;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int j = 0; j < MB; ++j) {
                const int64_t row = row_of_lane + 32 * j;
#pragma unroll
                for (int run = 0; run < 2; ++run) {
                    const int col = n0 + BN / 2 * wn + 32 * i + 16 * run + 8 * half;
                    if (row < a.rows && col < a.cols) {
                        float4* const to = reinterpret_cast<float4*>(out + row * a.cols + col);
                        to[0] = make_float4(acc[i][j][8 * run], acc[i][j][8 * run + 1], acc[i][j][8 * run + 2], acc[i][j][8 * run + 3]);
                        to[1] = make_float4(acc[i][j][8 * run + 4], acc[i][j][8 * run + 5], acc[i][j][8 * run + 6], acc[i][j][8 * run + 7]);
                    }
                }
            }
        }
        return;
    }

    // ---- 16-bit outputs, through LDS in pieces of 32 rows by 64 columns per wavefront, so that every store writes whole 128-byte runs
    __builtin_amdgcn_s_barrier();  // every wavefront is done reading the last stage
    uint16_t* const staged = s_tiles + wave * kEpiWave;
    const int out_row = lane >> 3, out_chunk = lane & 7;
    auto settle = [] {  // (a wavefront's own LDS accesses stay in order; the compiler must keep them so)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    if constexpr (MODE == kGemmForward) {
        constexpr int kRound = BN / 4 < 64 ? BN / 4 : 64;  // columns of both projections a wavefront has: BN / 4, by up to 64
        static_assert(BN / 4 == kRound, "one round");
        constexpr int HB = NB / 2;  // blocks of each projection
        const int col0 = n0 + BN / 4 * wn;
        float bias[2][HB][2][8];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
            for (int i = 0; i < HB; ++i) {
#pragma unroll
                for (int run = 0; run < 2; ++run) {
                    const int col = col0 + 32 * i + 16 * run + 8 * half;
                    u32x4_t w = {0u, 0u, 0u, 0u};
                    if (a.bias != nullptr && col < a.cols) {
                        w = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.bias) + static_cast<int64_t>(p) * a.cols + col);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        ils_unpack2<Tag>(w[e], bias[p][i][run][2 * e], bias[p][i][run][2 * e + 1]);
                    }
                }
            }
        }
        with_activation(a.activation, [&](auto chosen) {
            constexpr int kind = decltype(chosen)::value;
#pragma unroll
            for (int j = 0; j < MB; ++j) {
#pragma unroll
                for (int i = 0; i < HB; ++i) {
#pragma unroll
                    for (int run = 0; run < 2; ++run) {
                        u32x4_t hw, gw, uw;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float g0 = acc[i][j][8 * run + 2 * e] + bias[0][i][run][2 * e], g1 = acc[i][j][8 * run + 2 * e + 1] + bias[0][i][run][2 * e + 1];
                            const float u0 = acc[HB + i][j][8 * run + 2 * e] + bias[1][i][run][2 * e],
                                        u1 = acc[HB + i][j][8 * run + 2 * e + 1] + bias[1][i][run][2 * e + 1];
                            // (hidden is taken of the sums as they are, before mixed is rounded for the backward)
                            hw[e] = pack2<Tag>(gated_act<kind>(g0) * u0, gated_act<kind>(g1) * u1);
                            gw[e] = pack2<Tag>(g0, g1);
                            uw[e] = pack2<Tag>(u0, u1);
                        }
                        uint16_t* const to = staged + r * kEpiRow + 32 * i + 16 * run + 8 * half;
                        *reinterpret_cast<u32x4_t*>(to) = hw;
                        *reinterpret_cast<u32x4_t*>(to + 32 * kEpiRow) = gw;
                        *reinterpret_cast<u32x4_t*>(to + 64 * kEpiRow) = uw;
                    }
                }
                settle();
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int in_block = 8 * q + out_row;
                    const int64_t row = m0 + BM / 2 * wm + 32 * j + in_block;
                    const int col = col0 + 8 * out_chunk;
                    const uint16_t* const from = staged + in_block * kEpiRow + 8 * out_chunk;
                    if (row < a.rows && 8 * out_chunk < kRound && col < a.cols) {
                        if (a.out != nullptr) {
                            __builtin_nontemporal_store(*reinterpret_cast<const u32x4_t*>(from),
                                                        reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(a.out) + row * a.cols + col));
                        }
                        if (a.mixed != nullptr) {
                            uint16_t* const to = static_cast<uint16_t*>(a.mixed) + row * 2 * a.cols + col;
                            __builtin_nontemporal_store(*reinterpret_cast<const u32x4_t*>(from + 32 * kEpiRow), reinterpret_cast<u32x4_t*>(to));
                            __builtin_nontemporal_store(*reinterpret_cast<const u32x4_t*>(from + 64 * kEpiRow), reinterpret_cast<u32x4_t*>(to + a.cols));
                        }
                    }
                }
                settle();
            }
        });
    } else {
        static_assert(MODE == kGemmForward || NB % 2 == 0, "rounds of 64 columns");
#pragma unroll
        for (int j = 0; j < MB; ++j) {
#pragma unroll
            for (int c = 0; c < NB / 2; ++c) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int run = 0; run < 2; ++run) {
                        u32x4_t w;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            w[e] = pack2<Tag>(acc[2 * c + i][j][8 * run + 2 * e], acc[2 * c + i][j][8 * run + 2 * e + 1]);
                        }
                        *reinterpret_cast<u32x4_t*>(staged + r * kEpiRow + 32 * i + 16 * run + 8 * half) = w;
                    }
                }
                settle();
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int in_block = 8 * q + out_row;
                    const int64_t row = m0 + BM / 2 * wm + 32 * j + in_block;
                    const int col = n0 + BN / 2 * wn + 64 * c + 8 * out_chunk;
                    if (row < a.rows && col < a.cols) {
                        __builtin_nontemporal_store(*reinterpret_cast<const u32x4_t*>(staged + in_block * kEpiRow + 8 * out_chunk),
                                                    reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(a.out) + row * a.cols + col));
                    }
                }
                settle();
            }
        }
    }
}

}  // namespace hstu
