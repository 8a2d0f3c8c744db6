// The matrix products of the gated projections for gfx950: one tile kernel for the forward and both products of the backward.
//
//   forward          mixed = x W^T + b = (g, u);  hidden = act(g) * u          depth = columns of x
//   d_mixed          (grad u act'(g), grad act(g)) of (g, u) multiplied again     depth = columns of x
//   x gradient       d x = d_mixed W                                           depth = 2 inner
//   weight gradient  d W = d_mixed^T x                                         depth = rows, in chunks
//
// Bound by the matrix units (and in the forward up to a depth of a few hundred by its stores).  A workgroup of four wavefronts has a tile of BM
// rows by BN columns of the output, each wavefront a quarter of it in v_mfma_f32_32x32x16 blocks; the columns' side is the A operand, so that a lane
// has outputs of one row, and its columns are placed in a permuted order that gives it runs of 8 consecutive ones: 16-byte pieces.
// The depth goes by in steps of 32, or 64 where a tile has the LDS to itself, through a ring of STAGES tiles in LDS, filled by direct-to-LDS loads and read
// while later ones are under way.  (Steps of 64 ask for whole 128-byte lines: 8191 x 2048 -> 5632 357 us in four stages of 32, 343 in two of 64.)
// In the forward the BN columns are BN / 2 of the gate and the same BN / 2 of the other projection, dealt so that a wavefront has both
// halves of a column in the same lane: activation and product never leave registers.
//
// A side whose rows run along the depth is kept in LDS by rows of 64 or 128 bytes (chunk index XOR-ed with (row / 4) % 4 or (row / 2) % 8) and read as 16-byte operands;
// a side that is stored the other way -- the weight for d x, both sides of d W -- is kept as it lies, 32 rows of the tile's width, and read
// back with the transposing LDS read (64-byte groups XOR-ed with row % 4): no operand is transposed through memory.
//
// Tiles are dealt to the XCDs in equal runs of a list that goes through the rows in bands of eight tiles, the eight first: the
// 64 workgroups of an XCD work on 8 x 8 tiles at a time, whose operands its L2 holds.
#pragma once
#include "gated_linear_args.h"
#include "in_linear_silu_kernel.hip.h"
#include "lane_sums.hip.h"

namespace hstu {

constexpr int kGemmThreads = 256;
constexpr int kGemmStep = 32;  // of the depth, where not 64
constexpr int kGemmForward = 0, kGemmXGrad = 1, kGemmWeightGrad = 2, kGemmMixedGrad = 3;
constexpr int kGemmBand = 8;  // row tiles of a band

__device__ __forceinline__ float gated_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f)); }

// z, at most 30 from zero; NaN stays NaN (which the minimum of a maximum would make -30)
__device__ __forceinline__ float gated_bounded(float z) { return z > 30.0f ? 30.0f : z < -30.0f ? -30.0f : z; }

// act(z): silu, gelu by its tanh form -- z * sigmoid(2 sqrt(2 / pi) (z + 0.044715 z^3)) --, or the sigmoid.  (hardware exp2 and reciprocal, 1 ulp
// each: the results are rounded to 8 or 11 bits.  Past |z| = 30 gelu's cube could make infinity times 0: its argument is bounded there, where the
// sigmoid is 0 or 1 to all bits.)
template <int ACT>
__device__ __forceinline__ float gated_act(float z)
{
    if constexpr (ACT == kActSilu) {
        return z * gated_sigmoid(z);
    } else if constexpr (ACT == kActGelu) {
        const float t = gated_bounded(z);
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

// What a backward needs of g and u, "mixed": the upper 24 bits of their fp32 sums, 2^-15 of them at most cut off, whatever the type of x.  Rounded to that type they
// would add to the gradients as much as the rounding of d_mixed and that of the gradients themselves do; the third byte costs 17 us of writing and as much of
// reading at 20292 rows of 2 x 2048.  A row is [g's upper 16 bits][u's upper 16 bits][for every 8 columns: g's 8 third bytes, u's 8].
__device__ __forceinline__ uint32_t kept_high(float a, float b)
{
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302);
}
__device__ __forceinline__ uint32_t kept_low(float a, float b, float c, float d)
{
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x0c0c0501) |
           __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, d), __builtin_bit_cast(uint32_t, c), 0x05010c0c);
}
// value H of the pair `high`, its third byte at K of `low`
template <int H, int K>
__device__ __forceinline__ float kept_value(uint32_t high, uint32_t low)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_perm(high, low, (H == 0 ? 0x0504000cu : 0x0706000cu) | (K << 8)));
}

template <int ACT>
__device__ __forceinline__ void gated_act_slope(float z, float& act, float& slope)
{
    if constexpr (ACT == kActSilu) {
        const float s = gated_sigmoid(z);
        act = z * s;
        slope = s * __builtin_fmaf(z, 1.0f - s, 1.0f);
    } else if constexpr (ACT == kActGelu) {
        const float t = gated_bounded(z);
        const float s = gated_sigmoid(1.5957691216057308f * t * __builtin_fmaf(0.044715f * t, t, 1.0f));
        act = z * s;
        slope = s * __builtin_fmaf(t * (1.0f - s), 1.5957691216057308f * __builtin_fmaf(0.134145f * t, t, 1.0f), 1.0f);
    } else {
        act = gated_sigmoid(z);
        slope = act * (1.0f - act);
    }
}

// d_mixed in fp16 is a power of two times its values, the same for all of a call, which the products' results are divided by again: fp16 ends at 65504 and has
// steps of 2^-24 from zero, where sums over many rows may have more of either side.  The first pass multiplies by kGatedScale and notes the largest value;
// where that does not fit, or leaves a step more than 2^-22 of the largest, a second pass takes a power of two that does.  (Its launch, and the one that
// looks, are 5 us where nothing is left for them to do, 8 behind the largest stages: 64 rows, 512 -> 2048, kept, 20.3 -> 25.2 us, 20292 rows 260 -> 268.)
template <typename Tag>
constexpr bool kGatedScaled = std::is_same_v<Tag, f16_tag>;

// the largest of the magnitudes so far and of v, where it is finite: what is not stays so at any scale
__device__ __forceinline__ float gated_larger(float largest, float v)
{
    const float m = __builtin_fabsf(v);
    return m > largest && m < __builtin_inff() ? m : largest;
}
__device__ __forceinline__ void gated_note_range(float largest, float* to)
{
#pragma unroll
    for (int i = 32; i > 0; i /= 2) {
        largest = fmaxf(largest, __shfl_xor(largest, i));
    }
    if ((threadIdx.x & 63) == 0) {
        *to = largest;
    }
}

// MFMA row -> column of the transposing read: within 16 lanes the second and third group of four change places, which puts the
// columns into the order of ils_column_of_mfma_row
__device__ __forceinline__ int gemm_tr_col(int lane) { return 16 * ((lane >> 4) & 1) + 4 * (((lane & 1) << 1) | ((lane >> 1) & 1)); }

// A direct-to-LDS request: each lane's 16 bytes land at lds_byte_address + 16 * lane; out-of-range sources write zeros.  In assembly, and waited for by
// count: behind the builtin the compiler lets no transposing LDS read pass before every request under way has arrived.
__device__ __forceinline__ void gemm_request(uint32_t lds_byte_address, uint32_t voffset, u32x4_t rsrc, uint32_t soffset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(lds_byte_address), "v"(voffset), "s"(rsrc), "s"(soffset)
                 : "memory", "m0");
}
__device__ __forceinline__ u32x4_t gemm_rsrc(const void* base, uint32_t bytes)
{
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    const u32x4_t r = {static_cast<uint32_t>(at), static_cast<uint32_t>(at >> 32) & 0xffffu, bytes, kBufferFlags};
    return r;
}

// s_waitcnt: at most `vm` memory requests and `lgkm` LDS accesses under way
constexpr int gemm_wait(int vm, int lgkm) { return (vm & 15) | (7 << 4) | (lgkm << 8) | ((vm >> 4) << 14); }

// WM x WN wavefronts, each with MB x NB blocks of 32 x 32; STAGES tiles of LDS, STEP of the depth each
template <typename Tag, int MODE, int WM, int WN, int MB, int NB, int STAGES, int PER_CU, int STEP>
__global__ __launch_bounds__(kGemmThreads, PER_CU) void gated_gemm_kernel(const GatedGemmArgs a)
{
    static_assert(WM * WN == 4, "four wavefronts");
    constexpr int BM = 32 * WM * MB, BN = 32 * WN * NB;  // of the tile
    constexpr int kWaveN = 32 * NB, kWaveM = 32 * MB;
    constexpr bool kBoth = MODE == kGemmForward || MODE == kGemmMixedGrad;  // the tile has both projections
    constexpr bool NT = !kBoth;                   // the columns' side is read transposed
    constexpr bool MT = MODE == kGemmWeightGrad;  // the rows' side is
    static_assert(STEP == 32 || (STEP == 64 && kBoth), "sides stored across the depth go by steps of 32");
    constexpr int kReqsN = BN * STEP / 2048, kReqsM = BM * STEP / 2048, kReqs = kReqsN + kReqsM;  // direct-to-LDS instructions per wavefront and stage
    static_assert(BM % 64 == 0 && BN % 64 == 0, "a stage's instructions are dealt evenly");
    constexpr int kNElems = BN * STEP, kStage = (BN + BM) * STEP;
    constexpr int kEpiRow = kBoth ? kWaveN / 2 : 64 + 8;  // staged rows of up to 64 columns
    constexpr int kEpiPlanes = MODE == kGemmForward ? 4 : kBoth ? 2 : 1;
    // (a second piece where the stages' LDS has room for it)
    constexpr int kEpiPieces = kBoth && 2 * 4 * kEpiPlanes * 32 * kEpiRow <= STAGES * kStage ? 2 : 1;
    constexpr int kEpiWave = kEpiPieces * kEpiPlanes * 32 * kEpiRow;
    constexpr int kLds = STAGES * kStage > 4 * kEpiWave ? STAGES * kStage : 4 * kEpiWave;
    __shared__ __attribute__((aligned(1024))) uint16_t s_tiles[kLds];

    const int lane = threadIdx.x & 63;
    const int wave = uniform(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;

    // ---- the workgroup's tile
    const uint32_t tiles = static_cast<uint32_t>(a.tiles_m) * static_cast<uint32_t>(a.tiles_n);
    const uint32_t each = (a.count + 7u) >> 3, in_launch = (blockIdx.x & 7u) * each + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= each || in_launch >= a.count) {
        return;
    }
    const uint32_t place = a.first + in_launch;
    float scale = kGatedScale;
    if constexpr (MODE == kGemmMixedGrad && kGatedScaled<Tag>) {
        if (a.scale != nullptr) {
            scale = *a.scale;
            if (scale == kGatedScale) {  // the first pass was enough
                return;
            }
        }
    }
    const uint32_t part = place / tiles, tile = place - part * tiles;
    const uint32_t in_band = static_cast<uint32_t>(kGemmBand) * static_cast<uint32_t>(a.tiles_n);
    const uint32_t band = tile / in_band, at = tile - band * in_band;
    const uint32_t high = min(static_cast<uint32_t>(kGemmBand), static_cast<uint32_t>(a.tiles_m) - band * kGemmBand);
    const int tile_n = static_cast<int>(at / high), tile_m = static_cast<int>(band * kGemmBand + at % high);

    const int64_t m0 = static_cast<int64_t>(tile_m) * BM;
    constexpr int kOutCols = kBoth ? BN / 2 : BN;
    const int n0 = tile_n * kOutCols;
    const int64_t depth0 = static_cast<int64_t>(part) * a.chunk;
    const int depth = static_cast<int>(min(a.chunk, a.depth - depth0));  // of this workgroup

    // ---- sources.  Rows and depth past the end read as zeros on both sides (out-of-range bytes of a descriptor)
    const uint32_t n_row_bytes = static_cast<uint32_t>(NT ? a.cols : static_cast<int>(a.depth)) * 2u;
    const uint32_t m_row_bytes = MT ? static_cast<uint32_t>(a.rows) * 2u : static_cast<uint32_t>(a.depth) * 2u;
    u32x4_t n_rsrc, u_rsrc, m_rsrc;
    if constexpr (NT) {
        n_rsrc = gemm_rsrc(static_cast<const uint8_t*>(a.n_side) + depth0 * n_row_bytes, static_cast<uint32_t>(depth) * n_row_bytes);
        u_rsrc = n_rsrc;
    } else {
        const int rows_w = min(kOutCols, a.cols - n0);
        const uint8_t* const w = static_cast<const uint8_t*>(a.n_side);
        n_rsrc = gemm_rsrc(w + static_cast<int64_t>(n0) * n_row_bytes, static_cast<uint32_t>(rows_w) * n_row_bytes);
        u_rsrc = gemm_rsrc(w + (static_cast<int64_t>(a.cols) + n0) * n_row_bytes, static_cast<uint32_t>(rows_w) * n_row_bytes);
    }
    if constexpr (MT) {
        m_rsrc = gemm_rsrc(static_cast<const uint8_t*>(a.m_side) + depth0 * m_row_bytes, static_cast<uint32_t>(depth) * m_row_bytes);
    } else {
        const int rows_m = a.rows - m0 < BM ? static_cast<int>(a.rows - m0) : BM;
        const uint32_t skipped = static_cast<uint32_t>(depth0) * 2u;
        m_rsrc = gemm_rsrc(static_cast<const uint8_t*>(a.m_side) + m0 * m_row_bytes + skipped, static_cast<uint32_t>(rows_m) * m_row_bytes - skipped);
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
            const int lds_row = 512 / STEP * q + lane / (STEP / 8);
            const int chunk = (lane % (STEP / 8)) ^ (STEP == 32 ? (lds_row >> 2) & 3 : (lds_row >> 1) & 7);
            int row = lds_row;
            if (n_part) {
                // a wavefront's rows: half of the gate, half of the other projection
                const int w = lds_row / kWaveN, r = lds_row % kWaveN % (kWaveN / 2);
                row = w * (kWaveN / 2) + (r & ~31) + ils_column_of_mfma_row(r & 31);
            }
            req_off[i] = static_cast<uint32_t>(row) * (n_part ? n_row_bytes : m_row_bytes) + chunk * 16u;
            req_depth[i] = 8 * chunk;
        }
    }
    // A whole step's addresses are the lane's at depth 0 and a scalar; the depth's last, part-filled step and those past it are checked lane by
    // lane (a scalar past a descriptor's end would not be).
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint16_t*)s_tiles));
    auto request = [&](int stage, int step) {
        const int d0 = step * STEP;
        const auto each = [&](auto&& f) {
#pragma unroll
            for (int i = 0; i < kReqs; ++i) {
                const bool n_part = i < kReqsN;
                const int q = wave + 4 * (n_part ? i : i - kReqsN);
                const uint32_t along = static_cast<uint32_t>(d0) * ((n_part ? NT : MT) ? (n_part ? n_row_bytes : m_row_bytes) : 2u);
                // (forward: 16 LDS rows of one projection per instruction)
                const bool upper = kBoth && n_part && (512 / STEP * q) % kWaveN >= kWaveN / 2;
                f(i, lds0 + static_cast<uint32_t>(2 * (stage * kStage + (n_part ? 0 : kNElems) + q * 512)), n_part ? (upper ? u_rsrc : n_rsrc) : m_rsrc, along);
            }
        };
        if (d0 + STEP <= depth) {
            each([&](int i, uint32_t to, u32x4_t rsrc, uint32_t along) { gemm_request(to, req_off[i], rsrc, along); });
        } else {
            each([&](int i, uint32_t to, u32x4_t rsrc, uint32_t along) {
                gemm_request(to, d0 + req_depth[i] < depth ? req_off[i] + along : kOutOfRange, rsrc, 0u);
            });
        }
    };

    // ---- operand reads: wavefront (wm, wn) has rows kWaveM wm .. and columns kWaveN wn .. of the tile.  Addresses within a stage: of a row-wise side,
    // block 0 for each half of the step (further blocks are constants away); of the other, each block (whose 64-byte groups are XOR-ed)
    const int r = lane & 31, half = lane >> 5;
    const int swz = STEP == 32 ? (r >> 2) & 3 : (r >> 1) & 7;
    constexpr int kParts = STEP / 16;  // of a step, as deep as an instruction
    const int tr_row = 8 * half + ((lane & 15) >> 2);
    int n_at[NT ? NB : kParts], m_at[MT ? MB : kParts];
    if constexpr (NT) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int c = kWaveN * wn + 32 * i + gemm_tr_col(lane);
            n_at[i] = tr_row * BN + v_chunk_swizzle<BN>(tr_row, c >> 3) * 8 + (c & 7);
        }
    } else {
#pragma unroll
        for (int kk = 0; kk < kParts; ++kk) {
            n_at[kk] = (kWaveN * wn + r) * STEP + ((2 * kk + half) ^ swz) * 8;
        }
    }
    if constexpr (MT) {
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            const int c = kWaveM * wm + 32 * j + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
            m_at[j] = kNElems + tr_row * BM + v_chunk_swizzle<BM>(tr_row, c >> 3) * 8 + (c & 7);
        }
    } else {
#pragma unroll
        for (int kk = 0; kk < kParts; ++kk) {
            m_at[kk] = kNElems + (kWaveM * wm + r) * STEP + ((2 * kk + half) ^ swz) * 8;
        }
    }
    auto read_across = [&](const uint16_t* p, int width) -> u32x4_t {
        const u32x2_t lo = lds_read_tr16_b64(p);
        const u32x2_t hi = lds_read_tr16_b64(p + 4 * width);
        const u32x4_t v = {lo[0], lo[1], hi[0], hi[1]};
        return v;
    };

    // d_mixed: the gradient's values of the lane's columns and rows, asked for ahead of everything else where there are registers to hold them
    constexpr bool kGradsAhead = MB * NB < 8;
    u32x4_t grads[MODE == kGemmMixedGrad ? MB : 1][NB / 2][2];
    const auto ask_for_grads = [&](int j) {
        const int64_t row = m0 + kWaveM * wm + 32 * j + r;
        const uint16_t* const from = static_cast<const uint16_t*>(a.grad) + row * a.cols + n0 + kWaveN / 2 * wn + 8 * half;
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) {
#pragma unroll
            for (int run = 0; run < 2; ++run) {
                const int along = 32 * i + 16 * run;
                grads[j][i][run] = u32x4_t{0u, 0u, 0u, 0u};
                if (row < a.rows && n0 + kWaveN / 2 * wn + 8 * half + along < a.cols) {
                    grads[j][i][run] = *reinterpret_cast<const u32x4_t*>(from + along);
                }
            }
        }
    };
    if constexpr (MODE == kGemmMixedGrad && kGradsAhead) {
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            ask_for_grads(j);
        }
    }

    // the sums start from the bias: nothing is left to add behind the products
    f32x16_t acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        float first[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            first[e] = 0.0f;
        }
        if constexpr (kBoth) {
            if (a.bias != nullptr) {
#pragma unroll
                for (int run = 0; run < 2; ++run) {
                    const int upper = i / (NB / 2), col = n0 + kWaveN / 2 * wn + 32 * (i % (NB / 2)) + 16 * run + 8 * half;
                    u32x4_t w = {0u, 0u, 0u, 0u};
                    if (col < a.cols) {
                        w = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.bias) + static_cast<int64_t>(upper) * a.cols + col);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        ils_unpack2<Tag>(w[e], first[8 * run + 2 * e], first[8 * run + 2 * e + 1]);
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < MB; ++j) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                acc[i][j][e] = first[e];
            }
        }
    }

    // A step is two or four parts of 16.  While the products of one part run, the operands of the next are read, so that the matrix pipe finds them
    // there; the barrier that hands a stage over stands ahead of the last part's products, when every wavefront has read all of the step:
    // its stage is free and is asked for again at once, STAGES steps ahead.  (Past the end the requests go on, out of range, so that their count
    // stays what the wait expects.)
    const int n_steps = (depth + STEP - 1) / STEP;
    u32x4_t nv[2][NB], mv[2][MB];
    auto read = [&](int set, const uint16_t* st, int kk) {
        const uint16_t* const n_from = st + n_at[NT ? 0 : kk];
        const uint16_t* const m_from = st + m_at[MT ? 0 : kk];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if constexpr (NT) {
                nv[set][i] = read_across(st + n_at[i] + 16 * kk * BN, BN);
            } else {
                nv[set][i] = *reinterpret_cast<const u32x4_t*>(n_from + 32 * i * STEP);
            }
        }
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            if constexpr (MT) {
                mv[set][j] = read_across(st + m_at[j] + 16 * kk * BM, BM);
            } else {
                mv[set][j] = *reinterpret_cast<const u32x4_t*>(m_from + 32 * j * STEP);
            }
        }
    };
    auto multiply = [&](int set) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int j = 0; j < MB; ++j) {
                acc[i][j] = mfma32<Tag>(nv[set][i], mv[set][j], acc[i][j]);
            }
        }
    };
    // the order asked of the scheduler: a read of the next operands behind each of the first products
    constexpr int kReads = NB * (NT ? 2 : 1) + MB * (MT ? 2 : 1);
    auto order = [] {
        constexpr int kProducts = NB * MB, kEach = (kReads + kProducts - 1) / kProducts;
#pragma unroll
        for (int u = 0; u < kProducts; ++u) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);      // an MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);  // LDS reads
        }
    };
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
        request(s, s);
    }
    __builtin_amdgcn_s_waitcnt(gemm_wait((STAGES - 1) * kReqs, 15));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    read(0, s_tiles, 0);
    int stage = 0;
    for (int t = 0; t < n_steps; ++t) {
        __builtin_amdgcn_sched_barrier(0);
        const uint16_t* const st = s_tiles + stage * kStage;
#pragma unroll
        for (int h = 0; h + 1 < kParts; ++h) {
            read((h + 1) & 1, st, h + 1);
            multiply(h & 1);
            order();
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_waitcnt(gemm_wait((STAGES - 2) * kReqs, 0));
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        request(stage, t + STAGES);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        read(0, s_tiles + stage * kStage, 0);
        multiply(1);
        order();
    }
    __builtin_amdgcn_s_waitcnt(gemm_wait(0, 0));  // (the last requests write LDS that is used otherwise below)

    // ---- gradients in chunks of the depth: fp32 partial outputs, runs of 8 columns
    const int64_t row_of_lane = m0 + kWaveM * wm + r;
    if (!kBoth && a.partial != nullptr) {
        float* const out = a.partial + static_cast<int64_t>(part) * a.rows * a.cols;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int j = 0; j < MB; ++j) {
                const int64_t row = row_of_lane + 32 * j;
#pragma unroll
                for (int run = 0; run < 2; ++run) {
                    const int col = n0 + kWaveN * wn + 32 * i + 16 * run + 8 * half;
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

    // ---- 16-bit outputs, through LDS in pieces of 32 rows by up to 64 columns per wavefront, so that every store writes whole 128-byte runs.  Pieces
    // alternate between two places: the values of the next are worked out while the last goes out.
    __builtin_amdgcn_s_barrier();  // every wavefront is done reading the last stage
    auto settle = [] {  // (a wavefront's own LDS accesses stay in order; the compiler must keep them so)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    if constexpr (kBoth) {
        constexpr int kRound = kWaveN / 2;  // columns of both projections a wavefront has
        static_assert(kRound <= 64 && NB % 2 == 0, "one round");
        constexpr int HB = NB / 2;  // blocks of each projection
        constexpr int kPerRow = kRound / 8, kRowsAtOnce = 64 / kPerRow;  // lanes to a row of 16-byte pieces, rows of a store
        const int col = n0 + kRound * wn + 8 * (lane % kPerRow);
        // where a row's 16 bytes lie: rows are not padded, and the rows that share 256 bytes of banks take turns over the whole of them
        const auto at = [](int row, int chunk) { return row * kRound + 8 * (chunk ^ (row / (128 / kRound) % kPerRow)); };
        if constexpr (MODE == kGemmMixedGrad) {
            constexpr int kPlane = 32 * kRound;
            uint16_t* const mine = s_tiles + wave * kEpiWave;
            const auto pack = [&](float x, float y) {
                if constexpr (kGatedScaled<Tag>) {
                    x *= scale;
                    y *= scale;
                }
                return pack2<Tag>(x, y);
            };
            with_activation(a.activation, [&](auto chosen) {
                constexpr int kind = decltype(chosen)::value;
#pragma unroll
                for (int j = 0; j < MB; ++j) {
                    uint16_t* const piece = mine + (j % kEpiPieces) * kEpiPlanes * kPlane;
                    const bool there = row_of_lane + 32 * j < a.rows;
                    if constexpr (!kGradsAhead) {
                        ask_for_grads(j);
                    }
#pragma unroll
                    for (int i = 0; i < HB; ++i) {
#pragma unroll
                        for (int run = 0; run < 2; ++run) {
                            u32x4_t gw, uw;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float d[2];
                                const uint32_t pair = grads[j][i][run][e];
                                ils_unpack2<Tag>(pair, d[0], d[1]);
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const int at_e = 8 * run + 2 * e + h;
                                    float act, slope;
                                    gated_act_slope<kind>(acc[i][j][at_e], act, slope);
                                    // (rows past the end count for nothing, whatever the bias makes of them)
                                    const float x = there ? d[h] * acc[HB + i][j][at_e] * slope : 0.0f, y = there ? d[h] * act : 0.0f;
                                    acc[i][j][at_e] = x;
                                    acc[HB + i][j][at_e] = y;
                                }
                                gw[e] = pack(acc[i][j][8 * run + 2 * e], acc[i][j][8 * run + 2 * e + 1]);
                                uw[e] = pack(acc[HB + i][j][8 * run + 2 * e], acc[HB + i][j][8 * run + 2 * e + 1]);
                            }
                            uint16_t* const to = piece + at(r, 4 * i + 2 * run + half);
                            *reinterpret_cast<u32x4_t*>(to) = gw;
                            *reinterpret_cast<u32x4_t*>(to + kPlane) = uw;
                        }
                    }
                    settle();
#pragma unroll
                    for (int q = 0; q < 32 / kRowsAtOnce; ++q) {
                        const int in_block = kRowsAtOnce * q + lane / kPerRow;
                        const int64_t row = m0 + kWaveM * wm + 32 * j + in_block;
                        const uint16_t* const from = piece + at(in_block, lane % kPerRow);
                        if (row < a.rows && col < a.cols) {
                            uint16_t* const to = static_cast<uint16_t*>(a.out) + row * 2 * a.cols + col;
                            *reinterpret_cast<u32x4_t*>(to) = *reinterpret_cast<const u32x4_t*>(from);
                            *reinterpret_cast<u32x4_t*>(to + a.cols) = *reinterpret_cast<const u32x4_t*>(from + kPlane);
                        }
                    }
                    if constexpr (kEpiPieces == 1) {
                        settle();
                    }
                }
            });
            if constexpr (kGatedScaled<Tag>) {
                if (a.range != nullptr) {
                    float largest = 0.0f;
#pragma unroll
                    for (int i = 0; i < NB; ++i) {
#pragma unroll
                        for (int j = 0; j < MB; ++j) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                largest = gated_larger(largest, acc[i][j][e]);
                            }
                        }
                    }
                    gated_note_range(largest, a.range + static_cast<int64_t>(place) * 4 + wave);
                }
            }
            if (a.partial != nullptr) {  // column sums of the values before they are rounded, a row of them for each wavefront's rows
                float* const out = a.partial + (static_cast<int64_t>(tile_m) * WM + wm) * 2 * a.cols;
#pragma unroll
                for (int i = 0; i < NB; ++i) {
#pragma unroll
                    for (int run = 0; run < 2; ++run) {
                        float t[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            t[e] = acc[i][0][8 * run + e];
#pragma unroll
                            for (int j = 1; j < MB; ++j) {
                                t[e] += acc[i][j][8 * run + e];
                            }
                            t[e] = wave_sum<32>(t[e]);
                        }
                        const int c = n0 + kRound * wn + 32 * (i % HB) + 16 * run + 8 * half;
                        if (r == 0 && c < a.cols) {
                            float4* const to = reinterpret_cast<float4*>(out + static_cast<int64_t>(i / HB) * a.cols + c);
                            to[0] = make_float4(t[0], t[1], t[2], t[3]);
                            to[1] = make_float4(t[4], t[5], t[6], t[7]);
                        }
                    }
                }
            }
        } else {
            const auto finish = [&](auto chosen, auto kept) {
                constexpr int kind = decltype(chosen)::value;
                constexpr bool keep = decltype(kept)::value;
                constexpr int kPlane = 32 * kRound, kPlanes = keep ? kEpiPlanes : 1;
                constexpr int kPieces = 2 * 4 * kPlanes * kPlane <= kLds ? 2 : 1;
                uint16_t* const mine = s_tiles + wave * kPieces * kPlanes * kPlane;
#pragma unroll
                for (int j = 0; j < MB; ++j) {
                    uint16_t* const piece = mine + (j % kPieces) * kPlanes * kPlane;
#pragma unroll
                    for (int i = 0; i < HB; ++i) {
#pragma unroll
                        for (int run = 0; run < 2; ++run) {
                            u32x4_t hw, gw, uw, low;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float g0 = acc[i][j][8 * run + 2 * e], g1 = acc[i][j][8 * run + 2 * e + 1];
                                const float u0 = acc[HB + i][j][8 * run + 2 * e], u1 = acc[HB + i][j][8 * run + 2 * e + 1];
                                // (hidden is taken of the sums as they are)
                                hw[e] = pack2<Tag>(gated_act<kind>(g0) * u0, gated_act<kind>(g1) * u1);
                                if constexpr (keep) {
                                    gw[e] = kept_high(g0, g1);
                                    uw[e] = kept_high(u0, u1);
                                }
                            }
                            uint16_t* const to = piece + at(r, 4 * i + 2 * run + half);
                            *reinterpret_cast<u32x4_t*>(to) = hw;
                            if constexpr (keep) {
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    low[e] = kept_low(acc[i][j][8 * run + 4 * e], acc[i][j][8 * run + 4 * e + 1], acc[i][j][8 * run + 4 * e + 2], acc[i][j][8 * run + 4 * e + 3]);
                                    low[2 + e] = kept_low(acc[HB + i][j][8 * run + 4 * e], acc[HB + i][j][8 * run + 4 * e + 1], acc[HB + i][j][8 * run + 4 * e + 2],
                                                          acc[HB + i][j][8 * run + 4 * e + 3]);
                                }
                                *reinterpret_cast<u32x4_t*>(to + kPlane) = gw;
                                *reinterpret_cast<u32x4_t*>(to + 2 * kPlane) = uw;
                                *reinterpret_cast<u32x4_t*>(to + 3 * kPlane) = low;
                            }
                        }
                    }
                    settle();
#pragma unroll
                    for (int q = 0; q < 32 / kRowsAtOnce; ++q) {
                        const int in_block = kRowsAtOnce * q + lane / kPerRow;
                        const int64_t row = m0 + kWaveM * wm + 32 * j + in_block;
                        const uint16_t* const from = piece + at(in_block, lane % kPerRow);
                        if (row < a.rows && col < a.cols) {
                            if (!keep || a.out != nullptr) {
                                __builtin_nontemporal_store(*reinterpret_cast<const u32x4_t*>(from),
                                                            reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(a.out) + row * a.cols + col));
                            }
                            if constexpr (keep) {
                                uint16_t* const to = static_cast<uint16_t*>(a.mixed) + row * 3 * a.cols + col;
#pragma unroll
                                for (int p = 0; p < 3; ++p) {
                                    __builtin_nontemporal_store(*reinterpret_cast<const u32x4_t*>(from + (1 + p) * kPlane), reinterpret_cast<u32x4_t*>(to + p * a.cols));
                                }
                            }
                        }
                    }
                    if constexpr (kPieces == 1) {
                        settle();
                    }
                }
            };
            with_activation(a.activation, [&](auto chosen) {
                if (a.mixed != nullptr) {
                    finish(chosen, std::true_type{});
                } else {
                    finish(chosen, std::false_type{});
                }
            });
        }
    } else {
        static_assert(kBoth || NB % 2 == 0, "rounds of 64 columns");
        uint16_t* const staged = s_tiles + wave * kEpiWave;
        const int out_row = lane >> 3, out_chunk = lane & 7;
        const float back = kGatedScaled<Tag> ? a.scale[1] : 1.0f;
        const auto pack = [&](float x, float y) {
            if constexpr (kGatedScaled<Tag>) {
                x *= back;
                y *= back;
            }
            return pack2<Tag>(x, y);
        };
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
                            w[e] = pack(acc[2 * c + i][j][8 * run + 2 * e], acc[2 * c + i][j][8 * run + 2 * e + 1]);
                        }
                        *reinterpret_cast<u32x4_t*>(staged + r * kEpiRow + 32 * i + 16 * run + 8 * half) = w;
                    }
                }
                settle();
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int in_block = 8 * q + out_row;
                    const int64_t row = m0 + kWaveM * wm + 32 * j + in_block;
                    const int col = n0 + kWaveN * wn + 64 * c + 8 * out_chunk;
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
