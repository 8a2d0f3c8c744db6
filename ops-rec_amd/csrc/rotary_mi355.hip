// C ABI of rotary: argument checks, how the work is dealt, launch.
#include "../../include/ops_rec_layer_mi355.h"

#include <hip/hip_runtime.h>

#include "hstu_error.h"
#include "rotary_kernel.hip.h"

namespace {

using hstu::RotaryArgs;
using hstu::set_error;

typedef void (*kernel_t)(const RotaryArgs);

template <typename T>
kernel_t kernel_for(bool interleaved, int kind)
{
    using namespace hstu;
    static const kernel_t table[2][3] = {{rotary_kernel<T, false, kRotaryLines>, rotary_kernel<T, false, kRotaryPieces>, rotary_kernel<T, false, kRotaryShort>},
                                         {rotary_kernel<T, true, kRotaryLines>, rotary_kernel<T, true, kRotaryPieces>, rotary_kernel<T, true, kRotaryShort>}};
    return table[interleaved ? 1 : 0][kind];
}

kernel_t kernel_for(int dtype, bool interleaved, int kind)
{
    return dtype == HSTU_DT_FP32   ? kernel_for<hstu::ln_f32_tag>(interleaved, kind)
           : dtype == HSTU_DT_BF16 ? kernel_for<hstu::ln_bf16_tag>(interleaved, kind)
                                   : kernel_for<hstu::ln_f16_tag>(interleaved, kind);
}

int validate(const rotary_params* p)
{
    if (p == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "params is NULL");
    }
    if (p->struct_size != sizeof(rotary_params)) {
        return set_error(HSTU_ERR_INVALID, "struct_size %u does not match this library (%zu)", p->struct_size, sizeof(rotary_params));
    }
    if (p->q == nullptr || p->k == nullptr || p->q_out == nullptr || p->k_out == nullptr || p->frequencies == nullptr) {
        return set_error(HSTU_ERR_NULLPTR, "q, k, q_out, k_out and frequencies must be given");
    }
    if ((p->positions == nullptr) == (p->seq_offset == nullptr) || (p->positions != nullptr && p->start != nullptr)) {
        return set_error(HSTU_ERR_INVALID, "positions or seq_offset must be given, and start only with seq_offset");
    }
    if (p->dtype != HSTU_DT_FP32 && p->dtype != HSTU_DT_BF16 && p->dtype != HSTU_DT_FP16) {
        return set_error(HSTU_ERR_INVALID, "dtype %d is not one of fp32, bf16, fp16", p->dtype);
    }
    if (p->rows < 1 || p->heads_q < 1 || p->heads_k < 1 || p->heads_q > 65536 || p->heads_k > 65536) {
        return set_error(HSTU_ERR_INVALID, "rows must be positive and the heads of q and k in [1, 65536] (got %lld, %lld, %lld)", static_cast<long long>(p->rows),
                         static_cast<long long>(p->heads_q), static_cast<long long>(p->heads_k));
    }
    if (p->dim < 2 || p->dim > 65536 || p->pairs < 1 || 2 * p->pairs > p->dim) {
        return set_error(HSTU_ERR_INVALID, "dim must be in [2, 65536] and hold the pairs (got %lld and %lld)", static_cast<long long>(p->dim),
                         static_cast<long long>(p->pairs));
    }
    if (p->seq_offset != nullptr && (p->n_offsets < 2 || p->n_offsets > 0x7fffffff)) {
        return set_error(HSTU_ERR_INVALID, "seq_offset must have at least two elements (got %lld)", static_cast<long long>(p->n_offsets));
    }
    if (p->q_stride_row < 0 || p->q_stride_head < 0 || p->k_stride_row < 0 || p->k_stride_head < 0) {
        return set_error(HSTU_ERR_INVALID, "strides must not be negative");
    }
    for (const int32_t t : {p->positions_dtype, p->seq_offset_dtype, p->start_dtype}) {
        if (t != HSTU_IDX_I32 && t != HSTU_IDX_I64) {
            return set_error(HSTU_ERR_INVALID, "index dtype %d is not one of int32, int64", t);
        }
    }
    return HSTU_OK;
}

const void* shifted(const void* p, int64_t bytes) { return p == nullptr ? nullptr : static_cast<const uint8_t*>(p) + bytes; }

}  // namespace

extern "C" HSTU_API int rotary_fwd(const rotary_params* p, void* stream)
{
    const int rc = validate(p);
    if (rc != HSTU_OK) {
        return rc;
    }
    int cus = 0;
    if (const int code = hstu::compute_units(&cus); code != HSTU_OK) {
        return code;
    }
    const int64_t size = p->dtype == HSTU_DT_FP32 ? 4 : 2;
    const int heads = static_cast<int>(p->heads_q + p->heads_k);
    RotaryArgs a{};
    a.frequencies = p->frequencies;
    a.seq_offset = p->seq_offset;
    a.start = p->start;
    a.q_stride_row = p->q_stride_row;
    a.q_stride_head = p->q_stride_head;
    a.k_stride_row = p->k_stride_row;
    a.k_stride_head = p->k_stride_head;
    a.heads_q = static_cast<int>(p->heads_q);
    a.heads = heads;
    a.dim = static_cast<int>(p->dim);
    a.pairs = static_cast<int>(p->pairs);
    a.n_offsets = static_cast<int>(p->n_offsets);
    // threads of a head: two 16-byte pieces each.  Halves have their own last pieces; pairs that lie side by side fill theirs together
    const int values = static_cast<int>(16 / size);
    a.turned = p->interleaved ? ((2 * a.pairs + values - 1) / values + 1) / 2 : (a.pairs + values - 1) / values;
    a.items = a.turned + ((a.dim - 2 * a.pairs + values - 1) / values + 1) / 2;
    a.positions64 = p->positions_dtype == HSTU_IDX_I64;
    a.offsets64 = p->seq_offset_dtype == HSTU_IDX_I64;
    a.start64 = p->start_dtype == HSTU_IDX_I64;
    a.magnitude = static_cast<float>(p->magnitude);
    a.sign = p->inverse ? -1.0f : 1.0f;
    // Threads that share a row's pairs, each with as many heads as the others, at most 8; more of them until they give every SIMD two wavefronts (with four, 20292
    // rows of 4 + 4 heads of 128 took 22 us, 18 with two: the sines are paid for again)
    a.head_blocks = (heads + hstu::kRotaryHeads - 1) / hstu::kRotaryHeads;
    while (a.head_blocks < heads && p->rows * a.items * a.head_blocks < static_cast<int64_t>(cus) * 512) {
        ++a.head_blocks;
    }
    a.heads_each = (heads + a.head_blocks - 1) / a.head_blocks;
    a.head_blocks = (heads + a.heads_each - 1) / a.heads_each;
    // runs of values that are turned, and those that are copied; whether all stores of 16 bytes fill whole lines
    const int64_t turned = p->interleaved ? 2 * p->pairs : p->pairs, copied = p->dim - 2 * p->pairs;
    const int64_t run = p->interleaved ? static_cast<int64_t>(a.turned) * 16 : turned * size;
    const bool lines = run % 128 == 0 && a.dim * size % 128 == 0 && reinterpret_cast<uintptr_t>(p->q_out) % 128 == 0 && reinterpret_cast<uintptr_t>(p->k_out) % 128 == 0;
    const bool shorter = turned < values || (copied > 0 && copied < values);
    const kernel_t kernel = kernel_for(p->dtype, p->interleaved != 0, shorter ? hstu::kRotaryShort : lines ? hstu::kRotaryLines : hstu::kRotaryPieces);
    // (a launch numbers its threads in 32 bits)
    const int64_t most = (int64_t{1} << 31) / (static_cast<int64_t>(a.items) * a.head_blocks);
    for (int64_t row0 = 0; row0 < p->rows; row0 += most) {
        const int64_t rows = p->rows - row0 < most ? p->rows - row0 : most;
        a.row0 = row0;
        a.rows = static_cast<uint32_t>(rows);
        a.q = shifted(p->q, row0 * p->q_stride_row * size);
        a.k = shifted(p->k, row0 * p->k_stride_row * size);
        a.q_out = const_cast<void*>(shifted(p->q_out, row0 * p->heads_q * p->dim * size));
        a.k_out = const_cast<void*>(shifted(p->k_out, row0 * p->heads_k * p->dim * size));
        a.positions = shifted(p->positions, row0 * (a.positions64 ? 8 : 4));
        const int64_t threads = rows * a.items * a.head_blocks;
        hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>((threads + hstu::kRotaryThreads - 1) / hstu::kRotaryThreads)), dim3(hstu::kRotaryThreads), 0,
                           static_cast<hipStream_t>(stream), a);
        if (const hipError_t err = hipGetLastError(); err != hipSuccess) {
            return set_error(HSTU_ERR_RUNTIME, "launch of rotary failed: %s", hipGetErrorString(err));
        }
    }
    return HSTU_OK;
}
