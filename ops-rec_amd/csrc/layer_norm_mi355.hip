// C ABI of residual_norm and norm_gate, forward and backward: argument checks, choice of the kernel variant, launches; and the kernel
// that adds the partial sums of the parameters' gradients.
#include "../../include/ops_rec_layer_mi355.h"

#include <hip/hip_runtime.h>

#include "hstu_error.h"
#include "layer_norm_kernel.hip.h"
#include "layer_norm_variants.h"

namespace hstu {

// Partial sums [kinds][slices][cols] -> gradients: a workgroup has 16 columns of one kind, its 64 rows of lanes every 64th slice each, added
// in a fixed order.  (All of it at one lane per column would leave 24 workgroups with 512 additions in a row: 30 us against 4.)
constexpr int kNormSumThreads = 1024, kNormSumCols = 16, kNormSumParts = kNormSumThreads / kNormSumCols;
__global__ __launch_bounds__(kNormSumThreads) void norm_sums_kernel(const NormSumsArgs a)
{
    __shared__ float s_part[kNormSumParts][kNormSumCols];
    const int part = threadIdx.x / kNormSumCols, at = threadIdx.x % kNormSumCols;
    const int col = static_cast<int>(blockIdx.x) * kNormSumCols + at, kind = blockIdx.y;
    const float* const from = a.partial + static_cast<int64_t>(kind) * a.slices * a.cols;
    float t = 0.0f;
    if (col < a.cols) {
#pragma unroll 8
        for (int s = part; s < a.slices; s += kNormSumParts) {
            t += from[static_cast<int64_t>(s) * a.cols + col];
        }
    }
    s_part[part][at] = t;
    __syncthreads();
    for (int n = kNormSumParts / 2; n > 0; n /= 2) {
        if (part < n) {
            s_part[part][at] += s_part[part + n][at];
        }
        __syncthreads();
    }
    if (part == 0 && col < a.cols) {
        const float v = s_part[0][at];
        if (a.out_dtype == HSTU_DT_FP32) {
            ln_traits<ln_f32_tag>::store(a.out[kind], col, v);
        } else if (a.out_dtype == HSTU_DT_BF16) {
            ln_traits<ln_bf16_tag>::store(a.out[kind], col, v);
        } else {
            ln_traits<ln_f16_tag>::store(a.out[kind], col, v);
        }
    }
}

int launch_column_sums(const NormSumsArgs& a, void* stream)
{
    hipLaunchKernelGGL(norm_sums_kernel, dim3((a.cols + kNormSumCols - 1) / kNormSumCols, a.kinds), dim3(kNormSumThreads), 0, static_cast<hipStream_t>(stream), a);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? HSTU_OK : set_error(HSTU_ERR_RUNTIME, "launch of norm_sums_kernel failed: %s", hipGetErrorString(err));
}

}  // namespace hstu

namespace {

using hstu::NormArgs;
using hstu::NormBwdArgs;
using hstu::NormVariant;
using hstu::set_error;

const NormVariant* variant_for(int dtype, int stream_dtype, int64_t len)
{
    const bool f32 = stream_dtype == HSTU_DT_FP32;
    const NormVariant* v = dtype == HSTU_DT_FP32 ? hstu::norm_variants_f32() : dtype == HSTU_DT_BF16 ? hstu::norm_variants_bf16(f32) : hstu::norm_variants_f16(f32);
    while (len > v->capacity) {  // (len is at most the last one's)
        ++v;
    }
    return v;
}

constexpr int64_t kMostCols = 1 << 20;  // (a launch has less than 2^32 threads: a workgroup per part of a row, or per 16 columns of the sums)

int check_common(int64_t rows, int64_t cols, int64_t groups, int dtype, int stream_dtype, int affine_dtype, float epsilon)
{
    if (rows < 1 || cols < 1) {
        return set_error(HSTU_ERR_INVALID, "x must not be empty (got [%lld, %lld])", static_cast<long long>(rows), static_cast<long long>(cols));
    }
    if (dtype != HSTU_DT_FP32 && dtype != HSTU_DT_BF16 && dtype != HSTU_DT_FP16) {
        return set_error(HSTU_ERR_INVALID, "dtype %d is not one of fp32, bf16, fp16", dtype);
    }
    if (stream_dtype != dtype && stream_dtype != HSTU_DT_FP32) {
        return set_error(HSTU_ERR_INVALID, "the residual must be fp32 or of the type of x (got %d for %d)", stream_dtype, dtype);
    }
    if (affine_dtype != dtype && affine_dtype != HSTU_DT_FP32) {
        return set_error(HSTU_ERR_INVALID, "gamma, beta and scale must be fp32 or of the type of x (got %d for %d)", affine_dtype, dtype);
    }
    if (groups < 1 || cols % groups != 0) {
        return set_error(HSTU_ERR_INVALID, "the columns (%lld) must be a multiple of groups (%lld)", static_cast<long long>(cols), static_cast<long long>(groups));
    }
    if (cols / groups > hstu::kNormMaxLen) {
        return set_error(HSTU_ERR_INVALID, "at most %d columns share a mean (got %lld)", hstu::kNormMaxLen, static_cast<long long>(cols / groups));
    }
    if (cols > kMostCols || rows > 0x7fffffff / groups) {
        return set_error(HSTU_ERR_INVALID, "at most 2^20 columns, and rows * groups below 2^31 (got %lld, and %lld rows)", static_cast<long long>(cols),
                         static_cast<long long>(rows));
    }
    if (!(epsilon >= 0.0f)) {
        return set_error(HSTU_ERR_INVALID, "epsilon must not be negative");
    }
    return HSTU_OK;
}

int check_stride(int64_t stride, const char* what)
{
    return stride < 0 ? set_error(HSTU_ERR_INVALID, "the stride of %s must not be negative", what) : HSTU_OK;
}

int finish(hipError_t err, const char* what)
{
    return err == hipSuccess ? HSTU_OK : set_error(HSTU_ERR_RUNTIME, "launch of %s failed: %s", what, hipGetErrorString(err));
}

int describe(const residual_norm_params* p, NormArgs* a)
{
    if (p->struct_size != sizeof(residual_norm_params)) {
        return set_error(HSTU_ERR_INVALID, "struct_size %u does not match this library (%zu)", p->struct_size, sizeof(residual_norm_params));
    }
    int rc = check_common(p->rows, p->cols, 1, p->dtype, p->stream_dtype, p->affine_dtype, p->epsilon);
    rc = rc != HSTU_OK ? rc : check_stride(p->x_stride, "x");
    rc = rc != HSTU_OK ? rc : check_stride(p->residual_stride, "the residual");
    if (rc != HSTU_OK) {
        return rc;
    }
    *a = NormArgs{};
    a->x = p->x;
    a->residual = p->residual;
    a->gamma = p->gamma;
    a->beta = p->beta;
    a->scale = p->scale;
    a->out = p->y;
    a->sum = p->sum;
    a->x_stride = p->x_stride;
    a->residual_stride = p->residual_stride;
    a->units = static_cast<uint32_t>(p->rows);
    a->groups = 1;
    a->len = static_cast<int>(p->cols);
    a->epsilon = p->epsilon;
    a->residual_scale = 1.0f;
    a->affine_f32 = p->affine_dtype == HSTU_DT_FP32;
    a->rms = p->rms != 0;
    return HSTU_OK;
}

int describe(const norm_gate_params* p, NormArgs* a)
{
    if (p->struct_size != sizeof(norm_gate_params)) {
        return set_error(HSTU_ERR_INVALID, "struct_size %u does not match this library (%zu)", p->struct_size, sizeof(norm_gate_params));
    }
    int rc = check_common(p->rows, p->cols, p->groups, p->dtype, p->stream_dtype, p->affine_dtype, p->epsilon);
    rc = rc != HSTU_OK ? rc : check_stride(p->x_stride, "x");
    rc = rc != HSTU_OK ? rc : check_stride(p->gate_stride, "the gate");
    rc = rc != HSTU_OK ? rc : check_stride(p->residual_stride, "the residual");
    if (rc != HSTU_OK) {
        return rc;
    }
    if (p->residual == nullptr && p->stream_dtype != p->dtype) {
        return set_error(HSTU_ERR_INVALID, "without a residual the result has the type of x (got %d for %d)", p->stream_dtype, p->dtype);
    }
    *a = NormArgs{};
    a->x = p->x;
    a->residual = p->residual;
    a->gate = p->gate;
    a->gamma = p->gamma;
    a->beta = p->beta;
    a->out = p->out;
    a->x_stride = p->x_stride;
    a->residual_stride = p->residual_stride;
    a->gate_stride = p->gate_stride;
    a->units = static_cast<uint32_t>(p->rows * p->groups);
    a->groups = p->groups;
    a->len = static_cast<int>(p->cols / p->groups);
    a->epsilon = p->epsilon;
    a->residual_scale = p->residual != nullptr ? p->residual_scale : 1.0f;
    a->affine_f32 = p->affine_dtype == HSTU_DT_FP32;
    a->rms = p->rms != 0;
    a->silu = p->silu != 0;
    return HSTU_OK;
}

int launch_fwd(const NormArgs& a, int dtype, int stream_dtype, int mode, void* stream, const char* what)
{
    const NormVariant* v = variant_for(dtype, stream_dtype, a.len);
    int cus = 0;
    if (const int rc = hstu::compute_units(&cus); rc != HSTU_OK) {
        return rc;
    }
    // workgroups for eight wavefronts per SIMD at most, as many as have equal shares, and a multiple of the parts of a row (lanes keep their columns)
    const int64_t per_wg = v->fwd_threads / v->lanes, wanted = (static_cast<int64_t>(a.units) + per_wg - 1) / per_wg;
    const int64_t places = static_cast<int64_t>(cus) * (2048 / v->fwd_threads), rounds = (wanted + places - 1) / places;
    const int64_t even = (wanted + rounds - 1) / rounds, grid = (even + a.groups - 1) / a.groups * a.groups;
    hipLaunchKernelGGL(v->fwd[mode], dim3(static_cast<uint32_t>(grid)), dim3(v->fwd_threads), 0, static_cast<hipStream_t>(stream), a);
    return finish(hipGetLastError(), what);
}

// Workgroups of a backward launch that share a part of the columns: one, two or four workgroups of 1024, 512 or 256 lanes per compute unit over
// all parts, and no more than there are rows for.  (1: asked for where there is no device)
int slices_of(const NormArgs& a, const NormVariant* v)
{
    int cus = 0;
    if (hstu::compute_units(&cus) != HSTU_OK) {
        cus = 256;
    }
    const int64_t per_wg = v->bwd_threads / v->lanes, rows = a.units / static_cast<uint32_t>(a.groups);
    const int64_t useful = (rows + per_wg - 1) / per_wg, places = static_cast<int64_t>(cus) * (v->lanes > 64 ? (512 / v->bwd_threads > 1 ? 512 / v->bwd_threads : 1) : 1024 / v->bwd_threads) / a.groups;
    const int64_t most = places > 1 ? places : 1;
    return static_cast<int>(useful < most ? useful : most);
}

int kinds_of(bool beta, bool scale) { return 1 + (beta ? 1 : 0) + (scale ? 1 : 0); }

uint64_t partial_bytes(const NormArgs& a, const NormVariant* v, int kinds)
{
    return static_cast<uint64_t>(kinds) * static_cast<uint64_t>(slices_of(a, v)) * static_cast<uint64_t>(a.len) * static_cast<uint64_t>(a.groups) * 4u;
}

int launch_bwd(NormBwdArgs& b, const NormVariant* v, int mode, int affine_dtype, void* const (&outs)[3], void* workspace, uint64_t workspace_bytes,
               void* stream, const char* what)
{
    const int kinds = kinds_of(outs[1] != nullptr, outs[2] != nullptr);
    if (workspace == nullptr || workspace_bytes < partial_bytes(b.f, v, kinds)) {
        return set_error(HSTU_ERR_WORKSPACE, "%s needs %llu bytes of workspace (got %llu)", what,
                         static_cast<unsigned long long>(partial_bytes(b.f, v, kinds)), static_cast<unsigned long long>(workspace_bytes));
    }
    b.partial = static_cast<float*>(workspace);
    b.slices = slices_of(b.f, v);
    b.want_beta = outs[1] != nullptr;
    b.want_scale = outs[2] != nullptr;
    hipLaunchKernelGGL(v->bwd[mode], dim3(static_cast<uint32_t>(b.slices) * static_cast<uint32_t>(b.f.groups)), dim3(v->bwd_threads), 0,
                       static_cast<hipStream_t>(stream), b);
    int rc = finish(hipGetLastError(), what);
    if (rc != HSTU_OK) {
        return rc;
    }
    hstu::NormSumsArgs s{};
    s.partial = b.partial;
    for (int i = 0; i < 3; ++i) {
        if (outs[i] != nullptr) {
            s.out[s.kinds++] = outs[i];
        }
    }
    s.slices = b.slices;
    s.cols = b.f.len * b.f.groups;
    s.out_dtype = affine_dtype;
    return hstu::launch_column_sums(s, stream);
}

int describe(const residual_norm_bwd_params* p, NormBwdArgs* b)
{
    if (p == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "params is NULL");
    }
    if (p->struct_size != sizeof(residual_norm_bwd_params)) {
        return set_error(HSTU_ERR_INVALID, "struct_size %u does not match this library (%zu)", p->struct_size, sizeof(residual_norm_bwd_params));
    }
    *b = NormBwdArgs{};
    const int rc = describe(&p->fwd, &b->f);
    if (rc != HSTU_OK) {
        return rc;
    }
    const bool f32 = p->fwd.stream_dtype == HSTU_DT_FP32;
    if ((f32 ? p->sum == nullptr : p->fwd.residual == nullptr) || ((!f32 || p->fwd.scale != nullptr) && p->fwd.x == nullptr)) {
        return set_error(HSTU_ERR_NULLPTR, "an fp32 stream needs sum, another residual and x, scale needs x");
    }
    if (p->fwd.gamma == nullptr || p->residual_grad == nullptr || p->gamma_grad == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "gamma, residual_grad and gamma_grad must be given");
    }
    if ((p->scale_grad != nullptr && p->fwd.scale == nullptr) ||
        (p->x_grad == nullptr && (p->fwd.scale != nullptr || p->fwd.stream_dtype != p->fwd.dtype))) {
        return set_error(HSTU_ERR_INVALID, "scale_grad needs scale; x_grad may be NULL only without scale and in one type");
    }
    b->sum = f32 ? p->sum : nullptr;
    b->grad = p->y_grad;
    b->sum_grad = p->sum_grad;
    b->x_grad = p->x_grad;
    b->residual_grad = p->residual_grad;
    return HSTU_OK;
}

int describe(const norm_gate_bwd_params* p, NormBwdArgs* b)
{
    if (p == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "params is NULL");
    }
    if (p->struct_size != sizeof(norm_gate_bwd_params)) {
        return set_error(HSTU_ERR_INVALID, "struct_size %u does not match this library (%zu)", p->struct_size, sizeof(norm_gate_bwd_params));
    }
    *b = NormBwdArgs{};
    const int rc = describe(&p->fwd, &b->f);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (p->fwd.x == nullptr || p->fwd.gamma == nullptr || p->out_grad == nullptr || p->x_grad == nullptr || p->gamma_grad == nullptr ||
        (p->fwd.gate != nullptr) != (p->gate_grad != nullptr)) {
        return set_error(HSTU_ERR_NULLPTR, "x, gamma, out_grad, x_grad and gamma_grad must be given, and gate_grad where there is a gate");
    }
    b->grad = p->out_grad;
    b->x_grad = p->x_grad;
    b->gate_grad = p->gate_grad;
    return HSTU_OK;
}

}  // namespace

extern "C" {

HSTU_API int residual_norm_fwd(const residual_norm_params* p, void* stream)
{
    if (p == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "params is NULL");
    }
    NormArgs a;
    const int rc = describe(p, &a);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (p->x == nullptr || p->residual == nullptr || p->gamma == nullptr || p->y == nullptr || p->sum == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "x, residual, gamma, y and sum must be given");
    }
    return launch_fwd(a, p->dtype, p->stream_dtype, hstu::kNormFront, stream, "residual_norm");
}

HSTU_API int residual_norm_bwd_workspace_size(const residual_norm_bwd_params* p, uint64_t* workspace_bytes)
{
    NormBwdArgs b;
    const int rc = describe(p, &b);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (workspace_bytes == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "workspace_bytes is NULL");
    }
    *workspace_bytes = partial_bytes(b.f, variant_for(p->fwd.dtype, p->fwd.stream_dtype, b.f.len), kinds_of(p->beta_grad != nullptr, p->scale_grad != nullptr));
    return HSTU_OK;
}

HSTU_API int residual_norm_bwd(const residual_norm_bwd_params* p, void* workspace, uint64_t workspace_bytes, void* stream)
{
    NormBwdArgs b;
    const int rc = describe(p, &b);
    if (rc != HSTU_OK) {
        return rc;
    }
    void* const outs[3] = {p->gamma_grad, p->beta_grad, p->scale_grad};
    return launch_bwd(b, variant_for(p->fwd.dtype, p->fwd.stream_dtype, b.f.len), hstu::kNormFront, p->fwd.affine_dtype, outs, workspace, workspace_bytes,
                      stream, "residual_norm_bwd");
}

HSTU_API int norm_gate_fwd(const norm_gate_params* p, void* stream)
{
    if (p == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "params is NULL");
    }
    NormArgs a;
    const int rc = describe(p, &a);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (p->x == nullptr || p->gamma == nullptr || p->out == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "x, gamma and out must be given");
    }
    return launch_fwd(a, p->dtype, p->stream_dtype, hstu::kNormBehind, stream, "norm_gate");
}

HSTU_API int norm_gate_bwd_workspace_size(const norm_gate_bwd_params* p, uint64_t* workspace_bytes)
{
    NormBwdArgs b;
    const int rc = describe(p, &b);
    if (rc != HSTU_OK) {
        return rc;
    }
    if (workspace_bytes == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "workspace_bytes is NULL");
    }
    *workspace_bytes = partial_bytes(b.f, variant_for(p->fwd.dtype, p->fwd.stream_dtype, b.f.len), kinds_of(p->beta_grad != nullptr, false));
    return HSTU_OK;
}

HSTU_API int norm_gate_bwd(const norm_gate_bwd_params* p, void* workspace, uint64_t workspace_bytes, void* stream)
{
    NormBwdArgs b;
    const int rc = describe(p, &b);
    if (rc != HSTU_OK) {
        return rc;
    }
    void* const outs[3] = {p->gamma_grad, p->beta_grad, nullptr};
    return launch_bwd(b, variant_for(p->fwd.dtype, p->fwd.stream_dtype, b.f.len), hstu::kNormBehind, p->fwd.affine_dtype, outs, workspace, workspace_bytes,
                      stream, "norm_gate_bwd");
}

}  // extern "C"
