// residual_norm, norm_gate, gated_linear and rotary as native dispatcher kernels (device key CUDA = HIP tensors, and AutogradCUDA): a call in
// canonical form is described to the C ABI (include/ops_rec_layer_mi355.h) and launched without entering Python, every other goes to the
// Python implementation (ops_rec/_layer.py), which holds the checks, their messages and the conversions.  The autograd nodes hold the formulas that are
// registered there from Python.
#include "torch_binding.h"

#include "../../include/ops_rec_layer_mi355.h"

namespace {

using namespace ops_rec_binding;

// set once by set_layer_fallbacks(), with them kept_columns; never released (calls may come during interpreter exit)
struct Fallbacks {
    PyObject* residual_norm = nullptr;
    PyObject* residual_norm_backward = nullptr;
    PyObject* norm_gate = nullptr;
    PyObject* norm_gate_backward = nullptr;
    PyObject* rotary = nullptr;
    PyObject* gated_linear = nullptr;
    PyObject* gated_linear_backward = nullptr;
} fallbacks;

int64_t kept_columns = 0;  // _layer.KEPT_COLUMNS: up to so many columns of x nothing is kept for gated_linear's backward

bool is_float(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }

// [rows, cols] with the values of a row side by side
bool plane(const Tensor& t, int64_t rows, int64_t cols, at::ScalarType dtype, const at::Device& device)
{
    return t.defined() && t.dim() == 2 && t.size(0) == rows && t.size(1) == cols && t.scalar_type() == dtype && t.device() == device && t.stride(1) == 1;
}

bool columns(const Tensor& t, int64_t cols, at::ScalarType dtype, const at::Device& device)
{
    return t.defined() && t.dim() == 1 && t.size(0) == cols && t.scalar_type() == dtype && t.device() == device && t.is_contiguous();
}

bool columns(const OptTensor& t, int64_t cols, at::ScalarType dtype, const at::Device& device) { return !is_set(t) || columns(*t, cols, dtype, device); }

// what is allocated and launched for a call; false where the library refuses the description (the Python implementation then says so in its words)
template <typename P>
bool run_with_workspace(int (*size)(const P*, uint64_t*), int (*call)(const P*, void*, uint64_t, void*), const P& p, const Tensor& like, const char* name)
{
    uint64_t bytes = 0;
    if (size(&p, &bytes) != HSTU_OK) {
        return false;
    }
    const Tensor ws = bytes != 0 ? empty({static_cast<int64_t>(bytes)}, at::kByte, like.device()) : Tensor();
    const int rc = call(&p, ptr(ws), bytes, stream_of(like));
    TORCH_CHECK(rc == HSTU_OK, name, " failed (", rc, "): ", hstu_last_error());
    return true;
}

using Pair = std::tuple<Tensor, Tensor>;

// ------------------------------------------------------------------------------------------------------ residual_norm ----

Pair residual_norm(const Tensor& x, const Tensor& residual, const Tensor& gamma, const OptTensor& beta, const OptTensor& scale, double epsilon, bool rms)
{
    const at::ScalarType dtype = x.scalar_type(), stream = residual.scalar_type(), affine = gamma.scalar_type();
    const at::Device device = x.device();
    if (device.is_cuda() && x.dim() == 2 && x.numel() != 0 && is_float(dtype) && (stream == dtype || stream == at::kFloat) &&
        (affine == dtype || affine == at::kFloat) && plane(x, x.size(0), x.size(1), dtype, device) && plane(residual, x.size(0), x.size(1), stream, device) &&
        columns(gamma, x.size(1), affine, device) && columns(beta, x.size(1), affine, device) && columns(scale, x.size(1), affine, device) &&
        x.size(1) <= OPS_REC_NORM_MAX_LEN && epsilon >= 0.0) {
        const c10::DeviceGuard guard(device);
        Tensor y = empty(x.sizes(), dtype, device), sum = empty(x.sizes(), stream, device);
        residual_norm_params p;
        std::memset(&p, 0, sizeof p);
        p.struct_size = sizeof p;
        p.rms = rms;
        p.x = x.data_ptr();
        p.residual = residual.data_ptr();
        p.gamma = gamma.data_ptr();
        p.beta = ptr(beta);
        p.scale = ptr(scale);
        p.y = y.data_ptr();
        p.sum = sum.data_ptr();
        p.rows = x.size(0);
        p.cols = x.size(1);
        p.x_stride = x.stride(0);
        p.residual_stride = residual.stride(0);
        p.dtype = dtype_code(dtype);
        p.stream_dtype = dtype_code(stream);
        p.affine_dtype = dtype_code(affine);
        p.epsilon = static_cast<float>(epsilon);
        const int rc = residual_norm_fwd(&p, stream_of(x));
        TORCH_CHECK(rc == HSTU_OK, "residual_norm failed (", rc, "): ", hstu_last_error());
        return {y, sum};
    }
    return in_python<Pair>(fallbacks.residual_norm, x, residual, gamma, beta, scale, epsilon, rms);
}

using Five = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

bool dense_or_absent(const OptTensor& t, const Tensor& like, at::ScalarType dtype)
{
    return !is_set(t) || (t->sizes() == like.sizes() && t->scalar_type() == dtype && t->device() == like.device() && t->is_contiguous());
}

Five residual_norm_backward(const OptTensor& y_grad_in, const OptTensor& sum_grad_in, const OptTensor& x, const OptTensor& residual, const OptTensor& sum,
                            const Tensor& gamma, const OptTensor& scale, bool has_beta, at::ScalarType dtype, double epsilon, bool rms)
{
    const auto dense = [](const OptTensor& t) { return is_set(t) ? OptTensor(contiguous(*t)) : std::nullopt; };
    const OptTensor y_grad = dense(y_grad_in), sum_grad = dense(sum_grad_in);
    const bool wide = is_set(sum);
    if (wide || is_set(residual)) {
        const Tensor& given = wide ? *sum : *residual;
        const at::ScalarType stream = given.scalar_type(), affine = gamma.scalar_type();
        const at::Device device = given.device();
        if (device.is_cuda() && given.dim() == 2 && given.numel() != 0 && is_float(dtype) && wide == (stream == at::kFloat) && (wide || stream == dtype) &&
            (affine == dtype || affine == at::kFloat) && plane(given, given.size(0), given.size(1), stream, device) && (!wide || given.is_contiguous()) &&
            (is_set(x) || (wide && !is_set(scale))) && (!is_set(x) || plane(*x, given.size(0), given.size(1), dtype, device)) &&
            dense_or_absent(y_grad, given, dtype) && dense_or_absent(sum_grad, given, stream) && columns(gamma, given.size(1), affine, device) &&
            columns(scale, given.size(1), affine, device) && given.size(1) <= OPS_REC_NORM_MAX_LEN && epsilon >= 0.0) {
            const c10::DeviceGuard guard(device);
            const int64_t cols = given.size(1);
            const bool apart = is_set(scale) || stream != dtype;
            Tensor x_grad = apart ? empty(given.sizes(), dtype, device) : empty({0}, dtype, device), residual_grad = empty(given.sizes(), stream, device);
            Tensor gamma_grad = empty({cols}, affine, device), beta_grad = empty({has_beta ? cols : 0}, affine, device),
                   scale_grad = empty({is_set(scale) ? cols : 0}, affine, device);
            residual_norm_bwd_params p;
            std::memset(&p, 0, sizeof p);
            p.struct_size = sizeof p;
            residual_norm_params& f = p.fwd;
            f.struct_size = sizeof f;
            f.rms = rms;
            f.x = ptr(x);
            f.residual = wide ? nullptr : given.data_ptr();
            f.gamma = gamma.data_ptr();
            f.scale = ptr(scale);
            f.rows = given.size(0);
            f.cols = cols;
            f.x_stride = is_set(x) ? x->stride(0) : 0;
            f.residual_stride = wide ? 0 : given.stride(0);
            f.dtype = dtype_code(dtype);
            f.stream_dtype = dtype_code(stream);
            f.affine_dtype = dtype_code(affine);
            f.epsilon = static_cast<float>(epsilon);
            p.sum = wide ? given.data_ptr() : nullptr;
            p.y_grad = ptr(y_grad);
            p.sum_grad = ptr(sum_grad);
            p.x_grad = ptr(x_grad);
            p.residual_grad = residual_grad.data_ptr();
            p.gamma_grad = gamma_grad.data_ptr();
            p.beta_grad = ptr(beta_grad);
            p.scale_grad = ptr(scale_grad);
            if (run_with_workspace(residual_norm_bwd_workspace_size, residual_norm_bwd, p, given, "residual_norm_backward")) {
                return {x_grad, residual_grad, gamma_grad, beta_grad, scale_grad};
            }
        }
    }
    py::gil_scoped_acquire gil;
    return in_python<Five>(fallbacks.residual_norm_backward, y_grad, sum_grad, x, residual, sum, gamma, scale, has_beta, dtype, epsilon, rms);
}

struct ResidualNormFunction : torch::autograd::Function<ResidualNormFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const Tensor& gamma, const OptTensor& beta,
                                 const OptTensor& scale, double epsilon, bool rms)
    {
        static const auto op = operator_handle<decltype(residual_norm)>("ops_rec::residual_norm", "");
        const at::AutoDispatchBelowADInplaceOrView below;
        const auto [y, sum] = op.call(x, residual, gamma, beta, scale, epsilon, rms);
        const bool wide = sum.scalar_type() == at::kFloat;
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({is_set(scale) || !wide ? x : Tensor(), wide ? Tensor() : residual, wide ? sum : Tensor(), gamma, unwrap(scale)});
        ctx->saved_data["beta"] = is_set(beta);
        ctx->saved_data["dtype"] = static_cast<int64_t>(x.scalar_type());
        ctx->saved_data["epsilon"] = epsilon;
        ctx->saved_data["rms"] = rms;
        return {y, sum};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        variable_list out(7);
        if (grads[0].defined() || grads[1].defined()) {
            static const auto op = operator_handle<decltype(residual_norm_backward)>("ops_rec::residual_norm_backward", "");
            const variable_list s = ctx->get_saved_variables();
            const auto dtype = static_cast<at::ScalarType>(ctx->saved_data["dtype"].toInt());
            const bool beta = ctx->saved_data["beta"].toBool();
            const auto [dx, dr, dg, db, ds] = op.call(wrap(grads[0]), wrap(grads[1]), wrap(s[0]), wrap(s[1]), wrap(s[2]), s[3], wrap(s[4]), beta, dtype,
                                                      ctx->saved_data["epsilon"].toDouble(), ctx->saved_data["rms"].toBool());
            out[0] = s[4].defined() || dr.scalar_type() != dtype ? dx : dr;
            out[1] = dr;
            out[2] = dg;
            out[3] = beta ? db : Tensor();
            out[4] = s[4].defined() ? ds : Tensor();
        }
        return out;
    }
};

Pair residual_norm_autograd(const Tensor& x, const Tensor& residual, const Tensor& gamma, const OptTensor& beta, const OptTensor& scale, double epsilon,
                            bool rms)
{
    refuse_tangents("residual_norm", x, residual, gamma, beta, scale);
    if (!at::GradMode::is_enabled() || !(needs_grad(x) || needs_grad(residual) || needs_grad(gamma) || needs_grad(beta) || needs_grad(scale))) {
        static const auto op = operator_handle<decltype(residual_norm)>("ops_rec::residual_norm", "");
        const at::AutoDispatchBelowADInplaceOrView below;
        return op.call(x, residual, gamma, beta, scale, epsilon, rms);
    }
    const variable_list out = ResidualNormFunction::apply(x, residual, gamma, beta, scale, epsilon, rms);
    return {out[0], out[1]};
}

// ---------------------------------------------------------------------------------------------------------- norm_gate ----

// all of the description but the residual and the output; false when the call is not in canonical form
bool describe_norm_gate(const Tensor& x, const OptTensor& gate, const Tensor& gamma, const OptTensor& beta, at::ScalarType stream, double residual_scale,
                        int64_t groups, double epsilon, bool rms, bool silu, norm_gate_params& p)
{
    const at::ScalarType dtype = x.scalar_type(), affine = gamma.scalar_type();
    const at::Device device = x.device();
    if (!device.is_cuda() || x.dim() != 2 || x.numel() == 0 || !is_float(dtype) || (affine != dtype && affine != at::kFloat) ||
        !plane(x, x.size(0), x.size(1), dtype, device) || (is_set(gate) && !plane(*gate, x.size(0), x.size(1), dtype, device)) ||
        !columns(gamma, x.size(1), affine, device) || !columns(beta, x.size(1), affine, device) || groups < 1 || x.size(1) % groups != 0 ||
        x.size(1) / groups > OPS_REC_NORM_MAX_LEN || !(epsilon >= 0.0) || (stream != dtype && stream != at::kFloat)) {
        return false;
    }
    std::memset(&p, 0, sizeof p);
    p.struct_size = sizeof p;
    p.rms = rms;
    p.x = x.data_ptr();
    p.gate = ptr(gate);
    p.gamma = gamma.data_ptr();
    p.beta = ptr(beta);
    p.rows = x.size(0);
    p.cols = x.size(1);
    p.x_stride = x.stride(0);
    p.gate_stride = is_set(gate) ? gate->stride(0) : 0;
    p.groups = static_cast<int32_t>(groups);
    p.silu = silu;
    p.dtype = dtype_code(dtype);
    p.stream_dtype = dtype_code(stream);
    p.affine_dtype = dtype_code(affine);
    p.epsilon = static_cast<float>(epsilon);
    p.residual_scale = static_cast<float>(residual_scale);
    return true;
}

Tensor norm_gate(const Tensor& x, const OptTensor& gate, const Tensor& gamma, const OptTensor& beta, const OptTensor& residual, double residual_scale,
                 int64_t groups, double epsilon, bool rms, bool silu)
{
    norm_gate_params p;
    const at::ScalarType stream = is_set(residual) ? residual->scalar_type() : x.scalar_type();
    if (describe_norm_gate(x, gate, gamma, beta, stream, residual_scale, groups, epsilon, rms, silu, p) &&
        (!is_set(residual) || plane(*residual, x.size(0), x.size(1), stream, x.device()))) {
        const c10::DeviceGuard guard(x.device());
        Tensor out = empty(x.sizes(), stream, x.device());
        p.residual = ptr(residual);
        p.residual_stride = is_set(residual) ? residual->stride(0) : 0;
        p.out = out.data_ptr();
        const int rc = norm_gate_fwd(&p, stream_of(x));
        TORCH_CHECK(rc == HSTU_OK, "norm_gate failed (", rc, "): ", hstu_last_error());
        return out;
    }
    return in_python<Tensor>(fallbacks.norm_gate, x, gate, gamma, beta, residual, residual_scale, groups, epsilon, rms, silu);
}

using Four = std::tuple<Tensor, Tensor, Tensor, Tensor>;

Four norm_gate_backward(const Tensor& grad_in, const Tensor& x, const OptTensor& gate, const Tensor& gamma, const OptTensor& beta, bool has_residual,
                        double residual_scale, int64_t groups, double epsilon, bool rms, bool silu)
{
    const Tensor grad = contiguous(grad_in);
    norm_gate_bwd_params p;
    if (describe_norm_gate(x, gate, gamma, beta, grad.scalar_type(), residual_scale, groups, epsilon, rms, silu, p.fwd) &&
        plane(grad, x.size(0), x.size(1), grad.scalar_type(), x.device()) && (has_residual || grad.scalar_type() == x.scalar_type())) {
        const c10::DeviceGuard guard(x.device());
        const at::ScalarType dtype = x.scalar_type(), affine = gamma.scalar_type();
        Tensor x_grad = empty(x.sizes(), dtype, x.device()), gate_grad = is_set(gate) ? empty(x.sizes(), dtype, x.device()) : empty({0}, dtype, x.device());
        Tensor gamma_grad = empty({x.size(1)}, affine, x.device()), beta_grad = empty({is_set(beta) ? x.size(1) : 0}, affine, x.device());
        p.struct_size = sizeof p;
        p.reserved0 = 0;
        p.fwd.residual = has_residual ? grad.data_ptr() : nullptr;  // (says that there is one)
        p.out_grad = grad.data_ptr();
        p.x_grad = x_grad.data_ptr();
        p.gate_grad = ptr(gate_grad);
        p.gamma_grad = gamma_grad.data_ptr();
        p.beta_grad = ptr(beta_grad);
        if (run_with_workspace(norm_gate_bwd_workspace_size, norm_gate_bwd, p, x, "norm_gate_backward")) {
            return {x_grad, gate_grad, gamma_grad, beta_grad};
        }
    }
    return in_python<Four>(fallbacks.norm_gate_backward, grad, x, gate, gamma, beta, has_residual, residual_scale, groups, epsilon, rms, silu);
}

struct NormGateFunction : torch::autograd::Function<NormGateFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& gate, const Tensor& gamma, const OptTensor& beta,
                          const OptTensor& residual, double residual_scale, int64_t groups, double epsilon, bool rms, bool silu)
    {
        static const auto op = operator_handle<decltype(norm_gate)>("ops_rec::norm_gate", "");
        const at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({x, unwrap(gate), gamma, unwrap(beta)});
        ctx->saved_data["reals"] = std::vector<double>{residual_scale, epsilon};
        ctx->saved_data["ints"] = std::vector<int64_t>{groups, is_set(residual) ? 1 : 0, rms ? 1 : 0, silu ? 1 : 0};
        return op.call(x, gate, gamma, beta, residual, residual_scale, groups, epsilon, rms, silu);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        static const auto op = operator_handle<decltype(norm_gate_backward)>("ops_rec::norm_gate_backward", "");
        const variable_list s = ctx->get_saved_variables();
        const auto reals = ctx->saved_data["reals"].toDoubleVector();
        const auto ints = ctx->saved_data["ints"].toIntVector();
        const auto [dx, du, dg, db] = op.call(grads[0], s[0], wrap(s[1]), s[2], wrap(s[3]), ints[1] != 0, reals[0], ints[0], reals[1], ints[2] != 0, ints[3] != 0);
        return {dx, s[1].defined() ? du : Tensor(), dg, s[3].defined() ? db : Tensor(), ints[1] != 0 ? grads[0] : Tensor(), Tensor(), Tensor(), Tensor(), Tensor(),
                Tensor()};
    }
};

Tensor norm_gate_autograd(const Tensor& x, const OptTensor& gate, const Tensor& gamma, const OptTensor& beta, const OptTensor& residual,
                          double residual_scale, int64_t groups, double epsilon, bool rms, bool silu)
{
    refuse_tangents("norm_gate", x, gate, gamma, beta, residual);
    if (!at::GradMode::is_enabled() || !(needs_grad(x) || needs_grad(gate) || needs_grad(gamma) || needs_grad(beta) || needs_grad(residual))) {
        static const auto op = operator_handle<decltype(norm_gate)>("ops_rec::norm_gate", "");
        const at::AutoDispatchBelowADInplaceOrView below;
        return op.call(x, gate, gamma, beta, residual, residual_scale, groups, epsilon, rms, silu);
    }
    return NormGateFunction::apply(x, gate, gamma, beta, residual, residual_scale, groups, epsilon, rms, silu);
}

// ------------------------------------------------------------------------------------------------------------- rotary ----

bool is_index(const OptTensor& t, int64_t n, const at::Device& device)
{
    return !is_set(t) || ((t->scalar_type() == at::kInt || t->scalar_type() == at::kLong) && t->dim() == 1 && (n < 0 || t->size(0) == n) &&
                          t->device() == device && t->is_contiguous());
}

int32_t index_code(const OptTensor& t) { return is_set(t) && t->scalar_type() == at::kLong ? HSTU_IDX_I64 : HSTU_IDX_I32; }

Pair rotary(const Tensor& q, const Tensor& k, const Tensor& frequencies, const OptTensor& seq_offset, const OptTensor& start, const OptTensor& positions,
            bool interleaved, double magnitude, bool inverse)
{
    const at::ScalarType dtype = q.scalar_type();
    const at::Device device = q.device();
    if (device.is_cuda() && q.dim() == 3 && k.dim() == 3 && q.numel() != 0 && k.numel() != 0 && is_float(dtype) && k.scalar_type() == dtype &&
        k.device() == device && k.size(0) == q.size(0) && k.size(2) == q.size(2) && q.stride(2) == 1 && k.stride(2) == 1 && frequencies.dim() == 1 &&
        frequencies.scalar_type() == at::kDouble && frequencies.device() == device && frequencies.is_contiguous() && frequencies.size(0) >= 1 &&
        2 * frequencies.size(0) <= q.size(2) && q.size(1) <= 65536 && k.size(1) <= 65536 && q.size(2) >= 2 && q.size(2) <= 65536 &&
        is_set(seq_offset) != is_set(positions) && !(is_set(start) && is_set(positions)) && is_index(seq_offset, -1, device) &&
        (!is_set(seq_offset) || (seq_offset->size(0) >= 2 && is_index(start, seq_offset->size(0) - 1, device))) && is_index(positions, q.size(0), device)) {
        const c10::DeviceGuard guard(device);
        Tensor q_out = empty(q.sizes(), dtype, device), k_out = empty(k.sizes(), dtype, device);
        rotary_params p;
        std::memset(&p, 0, sizeof p);
        p.struct_size = sizeof p;
        p.dtype = dtype_code(dtype);
        p.q = q.data_ptr();
        p.k = k.data_ptr();
        p.q_out = q_out.data_ptr();
        p.k_out = k_out.data_ptr();
        p.frequencies = static_cast<const double*>(frequencies.data_ptr());
        p.positions = ptr(positions);
        p.seq_offset = ptr(seq_offset);
        p.start = ptr(start);
        p.rows = q.size(0);
        p.heads_q = q.size(1);
        p.heads_k = k.size(1);
        p.dim = q.size(2);
        p.pairs = frequencies.size(0);
        p.n_offsets = is_set(seq_offset) ? seq_offset->size(0) : 0;
        p.q_stride_row = q.stride(0);
        p.q_stride_head = q.stride(1);
        p.k_stride_row = k.stride(0);
        p.k_stride_head = k.stride(1);
        p.magnitude = magnitude;
        p.positions_dtype = index_code(positions);
        p.seq_offset_dtype = index_code(seq_offset);
        p.start_dtype = index_code(start);
        p.interleaved = interleaved;
        p.inverse = inverse;
        const int rc = rotary_fwd(&p, stream_of(q));
        TORCH_CHECK(rc == HSTU_OK, "rotary failed (", rc, "): ", hstu_last_error());
        return {q_out, k_out};
    }
    return in_python<Pair>(fallbacks.rotary, q, k, frequencies, seq_offset, start, positions, interleaved, magnitude, inverse);
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& frequencies, const OptTensor& seq_offset,
                                 const OptTensor& start, const OptTensor& positions, bool interleaved, double magnitude, bool inverse)
    {
        static const auto op = operator_handle<decltype(rotary)>("ops_rec::rotary", "");
        const at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({frequencies, unwrap(seq_offset), unwrap(start), unwrap(positions)});
        ctx->saved_data["ints"] = std::vector<int64_t>{interleaved ? 1 : 0, inverse ? 1 : 0};
        ctx->saved_data["magnitude"] = magnitude;
        const auto [q_out, k_out] = op.call(q, k, frequencies, seq_offset, start, positions, interleaved, magnitude, inverse);
        return {q_out, k_out};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        // (through the dispatcher from the top: a rotation of the gradients, which can be differentiated again)
        static const auto op = operator_handle<decltype(rotary)>("ops_rec::rotary", "");
        const variable_list s = ctx->get_saved_variables();
        const auto ints = ctx->saved_data["ints"].toIntVector();
        const auto [dq, dk] = op.call(grads[0], grads[1], s[0], wrap(s[1]), wrap(s[2]), wrap(s[3]), ints[0] != 0, ctx->saved_data["magnitude"].toDouble(), ints[1] == 0);
        return {dq, dk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Pair rotary_autograd(const Tensor& q, const Tensor& k, const Tensor& frequencies, const OptTensor& seq_offset, const OptTensor& start,
                     const OptTensor& positions, bool interleaved, double magnitude, bool inverse)
{
    refuse_tangents("rotary", q, k, frequencies);
    if (!at::GradMode::is_enabled() || !(needs_grad(q) || needs_grad(k) || needs_grad(frequencies))) {
        static const auto op = operator_handle<decltype(rotary)>("ops_rec::rotary", "");
        const at::AutoDispatchBelowADInplaceOrView below;
        return op.call(q, k, frequencies, seq_offset, start, positions, interleaved, magnitude, inverse);
    }
    TORCH_CHECK_NOT_IMPLEMENTED(!needs_grad(frequencies), "rotary: frequencies is a non-differentiable input; do not pass one with requires_grad=True");
    const variable_list out = RotaryFunction::apply(q, k, frequencies, seq_offset, start, positions, interleaved, magnitude, inverse);
    return {out[0], out[1]};
}

// -------------------------------------------------------------------------------------------------- gated projections ----

// all of the description but hidden and mixed; false when the call is not in canonical form
bool describe_gated_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, c10::string_view activation, gated_linear_params& p)
{
    const auto readable = [&](const Tensor& t) {
        return t.scalar_type() == x.scalar_type() && t.device() == x.device() && t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    };
    const int act = activation == "silu" ? OPS_REC_ACT_SILU : activation == "gelu" ? OPS_REC_ACT_GELU : activation == "sigmoid" ? OPS_REC_ACT_SIGMOID : -1;
    if (act < 0 || !x.device().is_cuda() || x.dim() != 2 || weight.dim() != 2 || x.numel() == 0 || weight.numel() == 0 ||
        (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kHalf) || !readable(x) || !readable(weight) || weight.size(0) % 16 != 0 ||
        x.size(1) % 8 != 0 || weight.size(1) != x.size(1) || (is_set(bias) && (bias->dim() != 1 || bias->size(0) != weight.size(0) || !readable(*bias)))) {
        return false;
    }
    std::memset(&p, 0, sizeof p);
    p.struct_size = sizeof p;
    p.activation = act;
    p.x = x.data_ptr();
    p.weight = weight.data_ptr();
    p.bias = ptr(bias);
    p.rows = x.size(0);
    p.cols = x.size(1);
    p.inner = weight.size(0) / 2;
    p.dtype = dtype_code(x.scalar_type());
    return true;
}

Pair gated_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, c10::string_view activation, bool keep)
{
    gated_linear_params p;
    if (describe_gated_linear(x, weight, bias, activation, p)) {
        const c10::DeviceGuard guard(x.device());
        Tensor hidden = empty({p.rows, p.inner}, x.scalar_type(), x.device());
        Tensor mixed = keep && p.cols > kept_columns ? empty({p.rows, 3 * p.inner}, at::kShort, x.device()) : empty({0}, at::kShort, x.device());
        p.hidden = hidden.data_ptr();
        p.mixed = ptr(mixed);
        const int rc = gated_linear_fwd(&p, stream_of(x));
        if (rc != HSTU_ERR_INVALID) {  // (refused: the Python implementation says so in its words)
            TORCH_CHECK(rc == HSTU_OK, "gated_linear failed (", rc, "): ", hstu_last_error());
            return {hidden, mixed};
        }
    }
    return in_python<Pair>(fallbacks.gated_linear, x, weight, bias, std::string(activation), keep);
}

using Three = std::tuple<Tensor, Tensor, Tensor>;

Three gated_linear_backward(const Tensor& grad_in, const Tensor& x, const Tensor& weight, const OptTensor& bias, const Tensor& mixed_in,
                            c10::string_view activation, std::array<bool, 3> wanted)
{
    const Tensor grad = contiguous(grad_in);
    gated_linear_bwd_params p;
    const auto readable = [&](const Tensor& t, int64_t cols, at::ScalarType dtype) {
        return t.dim() == 2 && t.size(0) == x.size(0) && t.size(1) == cols && t.scalar_type() == dtype && t.device() == x.device() &&
               t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    };
    if ((wanted[0] || wanted[1] || (wanted[2] && is_set(bias))) && describe_gated_linear(x, weight, bias, activation, p.fwd) &&
        readable(grad, p.fwd.inner, x.scalar_type()) && (mixed_in.numel() == 0 || readable(mixed_in, 3 * p.fwd.inner, at::kShort))) {
        const c10::DeviceGuard guard(x.device());
        const auto make = [&](bool want, at::IntArrayRef size) { return want ? empty(size, x.scalar_type(), x.device()) : empty({0}, x.scalar_type(), x.device()); };
        Tensor x_grad = make(wanted[0], x.sizes()), weight_grad = make(wanted[1], weight.sizes()), bias_grad = make(wanted[2] && is_set(bias), {weight.size(0)});
        p.struct_size = sizeof p;
        p.reserved0 = 0;
        p.fwd.mixed = mixed_in.numel() != 0 ? mixed_in.data_ptr() : nullptr;
        p.grad = grad.data_ptr();
        p.x_grad = ptr(x_grad);
        p.weight_grad = ptr(weight_grad);
        p.bias_grad = ptr(bias_grad);
        if (run_with_workspace(gated_linear_bwd_workspace_size, gated_linear_bwd, p, x, "gated_linear_backward")) {
            return {x_grad, weight_grad, bias_grad};
        }
    }
    return in_python<Three>(fallbacks.gated_linear_backward, grad, x, weight, bias, mixed_in, std::string(activation), wanted);
}

struct GatedLinearFunction : torch::autograd::Function<GatedLinearFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias, const std::string& activation, bool keep)
    {
        static const auto op = operator_handle<decltype(gated_linear)>("ops_rec::gated_linear", "");
        const at::AutoDispatchBelowADInplaceOrView below;
        const auto [hidden, mixed] = op.call(x, weight, bias, activation, keep);
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({mixed});
        ctx->save_for_backward({x, weight, unwrap(bias), mixed});
        ctx->saved_data["activation"] = activation;
        return {hidden, mixed};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        variable_list out(5);
        if (grads[0].defined()) {
            static const auto op = operator_handle<decltype(gated_linear_backward)>("ops_rec::gated_linear_backward", "");
            const variable_list s = ctx->get_saved_variables();
            const std::string activation = ctx->saved_data["activation"].toStringRef();
            const bool bias = s[2].defined();
            // (inputs are numbered as the tensors among them: the optional bias is the third)
            const std::array<bool, 3> wanted{ctx->needs_input_grad(0), ctx->needs_input_grad(1), bias && ctx->needs_input_grad(2)};
            const auto [dx, dw, db] = op.call(grads[0], s[0], s[1], wrap(s[2]), s[3], activation, wanted);
            out[0] = wanted[0] ? dx : Tensor();
            out[1] = wanted[1] ? dw : Tensor();
            out[2] = wanted[2] ? db : Tensor();
        }
        return out;
    }
};

Pair gated_linear_autograd(const Tensor& x, const Tensor& weight, const OptTensor& bias, c10::string_view activation, bool keep)
{
    refuse_tangents("gated_linear", x, weight, bias);
    if (!at::GradMode::is_enabled() || !(needs_grad(x) || needs_grad(weight) || needs_grad(bias))) {
        static const auto op = operator_handle<decltype(gated_linear)>("ops_rec::gated_linear", "");
        const at::AutoDispatchBelowADInplaceOrView below;
        return op.call(x, weight, bias, activation, keep);
    }
    const variable_list out = GatedLinearFunction::apply(x, weight, bias, std::string(activation), keep);
    return {out[0], out[1]};
}

}  // namespace

void ops_rec_binding::define_layer(py::module_& m)
{
    m.def("set_layer_fallbacks", [](py::object residual_norm_fn, py::object residual_norm_backward_fn, py::object norm_gate_fn, py::object norm_gate_backward_fn,
                                    py::object rotary_fn, py::object gated_linear_fn, py::object gated_linear_backward_fn, int64_t kept) {
        fallbacks.residual_norm = residual_norm_fn.release().ptr();
        fallbacks.residual_norm_backward = residual_norm_backward_fn.release().ptr();
        fallbacks.norm_gate = norm_gate_fn.release().ptr();
        fallbacks.norm_gate_backward = norm_gate_backward_fn.release().ptr();
        fallbacks.rotary = rotary_fn.release().ptr();
        fallbacks.gated_linear = gated_linear_fn.release().ptr();
        fallbacks.gated_linear_backward = gated_linear_backward_fn.release().ptr();
        kept_columns = kept;
    });
    m.def("kept_columns", [] { return kept_columns; });
}

TORCH_LIBRARY_IMPL(ops_rec, CUDA, m)
{
    m.impl("residual_norm", residual_norm);
    m.impl("residual_norm_backward", residual_norm_backward);
    m.impl("norm_gate", norm_gate);
    m.impl("norm_gate_backward", norm_gate_backward);
    m.impl("rotary", rotary);
    m.impl("gated_linear", gated_linear);
    m.impl("gated_linear_backward", gated_linear_backward);
}

TORCH_LIBRARY_IMPL(ops_rec, AutogradCUDA, m)
{
    m.impl("residual_norm", residual_norm_autograd);
    m.impl("norm_gate", norm_gate_autograd);
    m.impl("rotary", rotary_autograd);
    m.impl("gated_linear", gated_linear_autograd);
}
