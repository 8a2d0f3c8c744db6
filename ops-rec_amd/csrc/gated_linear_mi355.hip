// C ABI of gated_linear, forward and backward: argument checks, choice of kernels, launches.
#include "../../include/ops_rec_layer_mi355.h"

#include <hip/hip_runtime.h>

#include "gated_linear_variants.h"
#include "hstu_error.h"
#include "layer_args.h"

namespace hstu {

// The largest of n magnitudes of d_mixed -> the power of two it is multiplied by in fp16, and the inverse.  kGatedScale stays where the largest fits, and where a
// step of fp16 from zero (2^-24) is 2^-22 of it at most; otherwise the largest comes to lie in [2^14, 2^15).
constexpr int kRangeThreads = 1024;
__global__ __launch_bounds__(kRangeThreads) void gated_range_kernel(const float* range, int64_t n, float* scale)
{
    __shared__ float s_largest[kRangeThreads / 64];
    float largest = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += kRangeThreads) {
        largest = fmaxf(largest, range[i]);
    }
#pragma unroll
    for (int i = 32; i > 0; i /= 2) {
        largest = fmaxf(largest, __shfl_xor(largest, i));
    }
    if (threadIdx.x % 64 == 0) {
        s_largest[threadIdx.x / 64] = largest;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kRangeThreads / 64; ++i) {
            largest = fmaxf(largest, s_largest[i]);
        }
        float by = kGatedScale;
        if (largest > 0.0f && (largest * by > 65504.0f || largest * by < 0.125f)) {
            int exponent = 0;
            frexpf(largest, &exponent);  // largest < 2^exponent
            by = ldexpf(1.0f, min(15 - exponent, 100));
        }
        scale[0] = by;
        scale[1] = 1.0f / by;
    }
}

}  // namespace hstu

namespace {

using hstu::GatedGemmArgs;
using hstu::GatedTile;
using hstu::set_error;

static_assert(OPS_REC_ACT_SILU == hstu::kActSilu && OPS_REC_ACT_GELU == hstu::kActGelu && OPS_REC_ACT_SIGMOID == hstu::kActSigmoid, "one numbering");

constexpr int64_t kStep = 32;          // of a product's depth
constexpr int64_t kFewRows = 96;       // of a workgroup of the kernel for few rows
constexpr int64_t kMostCols = 1 << 21; // (256 rows of twice as many columns lie behind one descriptor of 2^31 bytes)
constexpr int64_t kMostBytes = int64_t{1} << 31;  // behind one descriptor
constexpr int64_t kMostWorkgroups = (1 << 24) - 8;  // of a launch, which has less than 2^32 threads; whole eights

const hstu::GatedKernels& kernels_of(int dtype) { return dtype == HSTU_DT_BF16 ? hstu::gated_kernels_bf16() : hstu::gated_kernels_f16(); }

int compute_units_or_256()  // (a size asked for where there is no device)
{
    int cus = 0;
    return hstu::compute_units(&cus) == HSTU_OK ? cus : 256;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

int validate(const gated_linear_params* p)
{
    if (p->struct_size != sizeof(gated_linear_params)) {
        return set_error(HSTU_ERR_INVALID, "struct_size %u does not match this library (%zu)", p->struct_size, sizeof(gated_linear_params));
    }
    if (p->x == nullptr || p->weight == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "x and weight must be given");
    }
    if (p->dtype != HSTU_DT_BF16 && p->dtype != HSTU_DT_FP16) {
        return set_error(HSTU_ERR_INVALID, "dtype %d is not one of bf16, fp16", p->dtype);
    }
    if (p->activation < 0 || p->activation > OPS_REC_ACT_SIGMOID) {
        return set_error(HSTU_ERR_INVALID, "activation %d is none", p->activation);
    }
    if (p->rows < 1 || p->rows > 0x7fffffff) {
        return set_error(HSTU_ERR_INVALID, "rows must be in [1, 2^31) (got %lld)", static_cast<long long>(p->rows));
    }
    if (p->cols < 8 || p->cols % 8 != 0 || p->inner < 8 || p->inner % 8 != 0 || p->cols > kMostCols || p->inner > kMostCols ||
        p->inner * p->cols >= (int64_t{1} << 29)) {
        return set_error(HSTU_ERR_INVALID, "the columns of x and hidden must be multiples of 8, at most 2^21, with a product below 2^29 (got %lld and %lld)",
                         static_cast<long long>(p->cols), static_cast<long long>(p->inner));
    }
    for (const void* t : {p->x, p->weight, p->bias, static_cast<const void*>(p->hidden), static_cast<const void*>(p->mixed)}) {
        if (!aligned16(t)) {
            return set_error(HSTU_ERR_INVALID, "tensors must be 16-byte aligned");
        }
    }
    return HSTU_OK;
}

int launched(const char* what)
{
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? HSTU_OK : set_error(HSTU_ERR_RUNTIME, "launch of %s failed: %s", what, hipGetErrorString(err));
}

// The kernel for few rows: its columns of hidden per workgroup, in eights -- the fullest compute unit's weight rows and rows of x are what it waits for.
int64_t few_rows_read(const gated_linear_params* p, int wide)
{
    return ceil_div(ceil_div(p->inner, 8 * wide), compute_units_or_256()) * (16 * wide + p->rows);
}
int few_rows_columns(const gated_linear_params* p)
{
    int best = 1;
    for (int wide = 2; wide <= 4; ++wide) {
        best = few_rows_read(p, wide) < few_rows_read(p, best) ? wide : best;
    }
    return best;
}

// What a product is estimated to take, in us: rounds of workgroups, one per compute unit each, and with several chunks of the depth the traffic of
// their fp32 partial outputs and the launch that adds them.
double cost_of(const GatedTile& t, int64_t rows, int64_t cols, int64_t depth, int64_t chunks)
{
    const int64_t all = ceil_div(rows, t.rows) * ceil_div(cols, t.cols) * chunks, rounds = ceil_div(all, compute_units_or_256());
    const double steps = static_cast<double>(ceil_div(ceil_div(depth, chunks), kStep));
    const double products = static_cast<double>(rounds) * (steps * (rounds == 1 ? t.alone : t.step) + t.fixed);
    return chunks == 1 ? products : products + 4.0 + static_cast<double>(rows) * static_cast<double>(cols) * static_cast<double>(chunks) * 1.1e-6;
}

const GatedTile& best_of(const GatedTile* tiles, int n, const gated_linear_params* p)
{
    const GatedTile* best = &tiles[0];
    for (int i = 1; i < n; ++i) {
        if (cost_of(tiles[i], p->rows, p->inner, p->cols, 1) < cost_of(*best, p->rows, p->inner, p->cols, 1)) {
            best = &tiles[i];
        }
    }
    return *best;
}
const GatedTile& forward_tile(const gated_linear_params* p) { return best_of(kernels_of(p->dtype).forward, hstu::kGatedForwardTiles, p); }
const GatedTile& mixed_tile(const gated_linear_params* p) { return best_of(kernels_of(p->dtype).mixed_grad, hstu::kGatedMixedTiles, p); }

// Up to 96 rows the kernel that streams the weight, unless the tiles are estimated faster: a compute unit reads 45 GB/s there (48 and 64 rows of 2048 x 5632
// and 4096 x 11264), and both take some 4 us besides.
bool few_rows(const gated_linear_params* p)
{
    if (p->rows > kFewRows) {
        return false;
    }
    const double read = static_cast<double>(few_rows_read(p, few_rows_columns(p))) * static_cast<double>(p->cols) * 2.0 / 45e3;
    return read <= 1.25 * cost_of(forward_tile(p), p->rows, p->inner, p->cols, 1);  // (whose steps were measured with weights in the caches)
}

int launch_tiles(const GatedTile& t, GatedGemmArgs a, void* stream, const char* what)
{
    a.tiles_m = static_cast<int>(ceil_div(a.rows, t.rows));
    a.tiles_n = static_cast<int>(ceil_div(a.cols, t.cols));
    const int64_t all = static_cast<int64_t>(a.tiles_m) * a.tiles_n * a.chunks;
    if (all > 0x70000000) {
        return set_error(HSTU_ERR_INVALID, "%s would take %lld workgroups", what, static_cast<long long>(all));
    }
    for (int64_t first = 0; first < all; first += kMostWorkgroups) {
        const int64_t count = all - first < kMostWorkgroups ? all - first : kMostWorkgroups;
        a.first = static_cast<uint32_t>(first);
        a.count = static_cast<uint32_t>(count);
        hipLaunchKernelGGL(t.kernel, dim3(static_cast<uint32_t>(ceil_div(count, 8) * 8)), dim3(256), 0, static_cast<hipStream_t>(stream), a);
        if (const int rc = launched(what); rc != HSTU_OK) {
            return rc;
        }
    }
    return HSTU_OK;
}

// A gradient's product: its tile, and the chunks its depth is cut into where the tiles are too few for the machine -- one or two workgroups to a compute
// unit then, of 256 values of the depth at least.
struct Product {
    const GatedTile* tile;
    int64_t chunk;
    int64_t chunks;
};
Product plan(const GatedTile* tiles, int n, int64_t rows, int64_t cols, int64_t depth, int64_t depth_row_bytes)
{
    const int64_t cus = compute_units_or_256(), fit = ceil_div(depth * depth_row_bytes, kMostBytes - kStep * depth_row_bytes);  // (a chunk lies behind one descriptor)
    const GatedTile* tile = nullptr;
    int64_t chunks = 0;
    double cost = 0.0;
    for (int i = 0; i < n; ++i) {
        const int64_t count = ceil_div(rows, tiles[i].rows) * ceil_div(cols, tiles[i].cols);
        for (const int64_t wanted : {int64_t{1}, cus / count, 2 * cus / count}) {
            int64_t c = wanted < ceil_div(depth, 256) ? wanted : ceil_div(depth, 256);
            c = c > fit ? c : fit;
            const double each = cost_of(tiles[i], rows, cols, depth, c);
            if (tile == nullptr || each < cost) {
                tile = &tiles[i], chunks = c, cost = each;
            }
        }
    }
    Product p{tile, ceil_div(ceil_div(depth, chunks), kStep) * kStep, 0};
    p.chunks = ceil_div(depth, p.chunk);
    return p;
}

uint64_t rounded(uint64_t bytes) { return (bytes + 255u) & ~uint64_t{255}; }

struct BackwardPlan {
    Product x, w;
    int slices;
    int64_t ranges;  // fp16: magnitudes that the pass of d_mixed notes, four a workgroup
    uint64_t d_mixed, sums, range, x_partial, w_partial;  // bytes, in this order
    uint64_t total() const { return d_mixed + sums + range + (x_partial > w_partial ? x_partial : w_partial); }
};

BackwardPlan plan_backward(const gated_linear_bwd_params* p)
{
    const gated_linear_params& f = p->fwd;
    const hstu::GatedKernels& k = kernels_of(f.dtype);
    BackwardPlan b{};
    // workgroups of the element-wise stage: eight per compute unit over all column blocks, a slice of at least 32 rows each
    const int64_t blocks = ceil_div(f.inner, 256), places = 8 * static_cast<int64_t>(compute_units_or_256()) / blocks, useful = ceil_div(f.rows, 32);
    const int64_t most = places > 1 ? places : 1;
    // (multiplied again, d_mixed has a row of column sums for each half of a tile)
    b.slices = static_cast<int>(f.mixed == nullptr ? 2 * ceil_div(f.rows, mixed_tile(&f).rows) : useful < most ? useful : most);
    b.d_mixed = rounded(static_cast<uint64_t>(f.rows) * static_cast<uint64_t>(f.inner) * 4u);
    b.sums = p->bias_grad != nullptr ? rounded(static_cast<uint64_t>(b.slices) * static_cast<uint64_t>(f.inner) * 8u) : 0;
    if (f.dtype == HSTU_DT_FP16) {  // (two floats of scale ahead of them)
        const GatedTile& t = mixed_tile(&f);
        b.ranges = 4 * (f.mixed == nullptr ? ceil_div(f.rows, t.rows) * ceil_div(f.inner, t.cols) : b.slices * blocks);
        b.range = rounded(static_cast<uint64_t>(b.ranges + 2) * 4u);
    }
    if (p->x_grad != nullptr) {
        b.x = plan(k.x_grad, hstu::kGatedXGradTiles, f.rows, f.cols, 2 * f.inner, f.cols * 2);
        b.x_partial = b.x.chunks > 1 ? static_cast<uint64_t>(b.x.chunks) * static_cast<uint64_t>(f.rows) * static_cast<uint64_t>(f.cols) * 4u : 0;
    }
    if (p->weight_grad != nullptr) {
        b.w = plan(k.weight_grad, hstu::kGatedWeightTiles, 2 * f.inner, f.cols, f.rows, (2 * f.inner > f.cols ? 2 * f.inner : f.cols) * 2);
        b.w_partial = b.w.chunks > 1 ? static_cast<uint64_t>(b.w.chunks) * static_cast<uint64_t>(2 * f.inner) * static_cast<uint64_t>(f.cols) * 4u : 0;
    }
    return b;
}

int validate(const gated_linear_bwd_params* p)
{
    if (p == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "params is NULL");
    }
    if (p->struct_size != sizeof(gated_linear_bwd_params)) {
        return set_error(HSTU_ERR_INVALID, "struct_size %u does not match this library (%zu)", p->struct_size, sizeof(gated_linear_bwd_params));
    }
    const int rc = validate(&p->fwd);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (p->grad == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "grad must be given");
    }
    for (const void* t : {p->grad, static_cast<const void*>(p->x_grad), static_cast<const void*>(p->weight_grad), static_cast<const void*>(p->bias_grad)}) {
        if (!aligned16(t)) {
            return set_error(HSTU_ERR_INVALID, "tensors must be 16-byte aligned");
        }
    }
    return HSTU_OK;
}

int launch_product(const hstu::GatedKernels& k, const Product& plan, GatedGemmArgs a, float* partial, void* stream, const char* what)
{
    a.chunk = plan.chunk;
    a.chunks = static_cast<int>(plan.chunks);
    a.partial = plan.chunks > 1 ? partial : nullptr;
    const int rc = launch_tiles(*plan.tile, a, stream, what);
    if (rc != HSTU_OK || a.partial == nullptr) {
        return rc;
    }
    hstu::GatedSumArgs s{};
    s.partial = partial;
    s.scale = a.scale;
    s.out = a.out;
    s.n = a.rows * a.cols;
    s.chunks = a.chunks;
    const int64_t blocks = ceil_div(s.n / 8, 256), most = 16 * static_cast<int64_t>(compute_units_or_256());
    hipLaunchKernelGGL(k.sum, dim3(static_cast<uint32_t>(blocks < most ? blocks : most)), dim3(256), 0, static_cast<hipStream_t>(stream), s);
    return launched("gated_sum_kernel");
}

}  // namespace

extern "C" {

HSTU_API const char* gated_linear_fwd_kernel_name(const gated_linear_params* p)
{
    if (p == nullptr || validate(p) != HSTU_OK) {
        return nullptr;
    }
    return few_rows(p) ? "gated_few_rows" : forward_tile(p).name;
}

HSTU_API int gated_linear_fwd(const gated_linear_params* p, void* stream)
{
    if (p == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "params is NULL");
    }
    const int rc = validate(p);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (p->hidden == nullptr && p->mixed == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "hidden or mixed must be given");
    }
    const hstu::GatedKernels& k = kernels_of(p->dtype);
    if (few_rows(p)) {
        hstu::GatedFewRowsArgs a{};
        a.x = p->x;
        a.weight = p->weight;
        a.bias = p->bias;
        a.hidden = p->hidden;
        a.mixed = p->mixed;
        a.rows = p->rows;
        a.depth = static_cast<int>(p->cols);
        a.inner = static_cast<int>(p->inner);
        a.activation = p->activation;
        const int blocks = static_cast<int>(ceil_div(p->rows, 16)), wide = few_rows_columns(p);
        hipLaunchKernelGGL(k.few_rows[blocks - 1][wide - 1], dim3(static_cast<uint32_t>(ceil_div(p->inner, 8 * wide))), dim3(512), 0,
                           static_cast<hipStream_t>(stream), a);
        return launched("gated_few_rows_kernel");
    }
    GatedGemmArgs a{};
    a.n_side = p->weight;
    a.m_side = p->x;
    a.bias = p->bias;
    a.out = p->hidden;
    a.mixed = p->mixed;
    a.rows = p->rows;
    a.depth = a.chunk = p->cols;
    a.cols = static_cast<int>(p->inner);
    a.chunks = 1;
    a.activation = p->activation;
    return launch_tiles(forward_tile(p), a, stream, "gated_gemm_kernel (forward)");
}

HSTU_API const char* gated_linear_bwd_kernel_name(const gated_linear_bwd_params* p, int part, int64_t* chunks)
{
    if (validate(p) != HSTU_OK) {
        return nullptr;
    }
    const BackwardPlan b = plan_backward(p);
    const Product* product = part == OPS_REC_GATED_X_GRAD ? &b.x : part == OPS_REC_GATED_WEIGHT_GRAD ? &b.w : nullptr;
    if (product != nullptr ? product->tile == nullptr : part != OPS_REC_GATED_MIXED_GRAD) {
        set_error(HSTU_ERR_INVALID, "the call has no part %d", part);
        return nullptr;
    }
    if (chunks != nullptr) {
        *chunks = product != nullptr ? product->chunks : 1;
    }
    return product != nullptr ? product->tile->name : p->fwd.mixed != nullptr ? "gated_stage" : mixed_tile(&p->fwd).name;
}

HSTU_API int gated_linear_bwd_workspace_size(const gated_linear_bwd_params* p, uint64_t* workspace_bytes)
{
    const int rc = validate(p);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (workspace_bytes == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "workspace_bytes is NULL");
    }
    *workspace_bytes = plan_backward(p).total();
    return HSTU_OK;
}

HSTU_API int gated_linear_bwd(const gated_linear_bwd_params* p, void* workspace, uint64_t workspace_bytes, void* stream)
{
    int rc = validate(p);
    if (rc != HSTU_OK) {
        return rc;
    }
    const BackwardPlan b = plan_backward(p);
    if (workspace == nullptr || workspace_bytes < b.total() || !aligned16(workspace)) {
        return set_error(HSTU_ERR_WORKSPACE, "gated_linear_bwd needs %llu bytes of workspace, 16-byte aligned (got %llu)", static_cast<unsigned long long>(b.total()),
                         static_cast<unsigned long long>(workspace_bytes));
    }
    const gated_linear_params& f = p->fwd;
    const hstu::GatedKernels& k = kernels_of(f.dtype);
    uint8_t* const ws = static_cast<uint8_t*>(workspace);
    float* const scale = b.range != 0 ? reinterpret_cast<float*>(ws + b.d_mixed + b.sums) : nullptr;
    float* const partial = reinterpret_cast<float*>(ws + b.d_mixed + b.sums + b.range);

    float* const sums = p->bias_grad != nullptr ? reinterpret_cast<float*>(ws + b.d_mixed) : nullptr;
    // d_mixed: one pass, and in fp16 another that starts only where the first one's scale does not do (every launch is made: the host does not wait to see)
    const auto in_range = [&](auto&& pass) {
        int code = pass(scale == nullptr ? nullptr : scale + 2, nullptr);
        if (code != HSTU_OK || scale == nullptr) {
            return code;
        }
        hipLaunchKernelGGL(hstu::gated_range_kernel, dim3(1), dim3(hstu::kRangeThreads), 0, static_cast<hipStream_t>(stream), scale + 2, b.ranges, scale);
        code = launched("gated_range_kernel");
        return code != HSTU_OK ? code : pass(nullptr, scale);
    };
    if (f.mixed == nullptr) {
        GatedGemmArgs a{};
        a.n_side = f.weight;
        a.m_side = f.x;
        a.bias = f.bias;
        a.grad = p->grad;
        a.out = ws;
        a.rows = f.rows;
        a.depth = a.chunk = f.cols;
        a.cols = static_cast<int>(f.inner);
        a.chunks = 1;
        a.activation = f.activation;
        rc = in_range([&](float* range, const float* by) {
            a.range = range;
            a.scale = by;
            a.partial = by == nullptr ? sums : nullptr;
            return launch_tiles(mixed_tile(&f), a, stream, "gated_gemm_kernel (d_mixed)");
        });
    } else {
        hstu::GatedStageArgs s{};
        s.grad = p->grad;
        s.mixed = f.mixed;
        s.d_mixed = ws;
        s.rows = f.rows;
        s.inner = static_cast<int>(f.inner);
        s.slices = b.slices;
        s.activation = f.activation;
        rc = in_range([&](float* range, const float* by) {
            s.range = range;
            s.scale = by;
            s.partial = by == nullptr ? sums : nullptr;
            hipLaunchKernelGGL(k.stage, dim3(static_cast<uint32_t>(b.slices * ceil_div(f.inner, 256))), dim3(256), 0, static_cast<hipStream_t>(stream), s);
            return launched("gated_stage_kernel");
        });
    }
    if (rc == HSTU_OK && p->bias_grad != nullptr) {
        hstu::NormSumsArgs n{};
        n.partial = sums;
        n.out[0] = p->bias_grad;
        n.kinds = 1;
        n.slices = b.slices;
        n.cols = static_cast<int>(2 * f.inner);
        n.out_dtype = f.dtype;
        rc = hstu::launch_column_sums(n, stream);
    }
    if (rc == HSTU_OK && p->x_grad != nullptr) {
        GatedGemmArgs a{};
        a.n_side = f.weight;
        a.m_side = ws;
        a.scale = scale;
        a.out = p->x_grad;
        a.rows = f.rows;
        a.depth = 2 * f.inner;
        a.cols = static_cast<int>(f.cols);
        rc = launch_product(k, b.x, a, partial, stream, "gated_gemm_kernel (x gradient)");
    }
    if (rc == HSTU_OK && p->weight_grad != nullptr) {
        GatedGemmArgs a{};
        a.n_side = f.x;
        a.m_side = ws;
        a.scale = scale;
        a.out = p->weight_grad;
        a.rows = 2 * f.inner;
        a.depth = f.rows;
        a.cols = static_cast<int>(f.cols);
        rc = launch_product(k, b.w, a, partial, stream, "gated_gemm_kernel (weight gradient)");
    }
    return rc;
}

}  // extern "C"
