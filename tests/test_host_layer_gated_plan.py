"""What gated_linear's backward would launch, asked of the C ABI without a GPU (nothing is launched)."""

import ctypes

from ops_rec import _native


def params(rows=1000, cols=64, inner=128):
    p = _native.GatedLinearBwdParams()
    p.struct_size = ctypes.sizeof(p)
    p.fwd.struct_size = ctypes.sizeof(p.fwd)
    p.fwd.x = p.fwd.weight = p.fwd.mixed = p.grad = p.x_grad = p.weight_grad = p.bias_grad = 0x1000  # never dereferenced
    p.fwd.rows, p.fwd.cols, p.fwd.inner, p.fwd.dtype = rows, cols, inner, _native.DT_BF16
    return p


def test_kernels_of_the_backward():
    name, chunks = _native.load().gated_linear_bwd_kernel_name, ctypes.c_int64(-1)
    p = params()
    assert name(ctypes.byref(p), 0, ctypes.byref(chunks)) == b"gated_stage" and chunks.value == 1
    for part in (1, 2):
        assert name(ctypes.byref(p), part, ctypes.byref(chunks)).startswith(b"gated_gemm_") and chunks.value >= 1
        assert name(ctypes.byref(p), part, None).startswith(b"gated_gemm_")
    p.fwd.mixed = None
    assert name(ctypes.byref(p), 0, None).startswith(b"gated_gemm_")
    p.x_grad = None
    assert name(ctypes.byref(p), 1, None) is None and "no part 1" in _native.last_error()
    assert name(ctypes.byref(p), 3, None) is None and name(ctypes.byref(p), -1, None) is None
    p.fwd.cols = 60
    assert name(ctypes.byref(p), 2, None) is None
    assert name(None, 0, None) is None


def test_tall_products_are_cut_where_a_descriptor_ends():
    """A chunk of the weight gradient's depth is at most the rows whose d_mixed lies behind one descriptor of 2^31 bytes."""
    name, chunks = _native.load().gated_linear_bwd_kernel_name, ctypes.c_int64(-1)
    for rows, inner in ((500, 1 << 21), (100000, 1 << 18), ((1 << 31) - 1, 8)):
        p = params(rows, 8, inner)
        assert name(ctypes.byref(p), 2, ctypes.byref(chunks)) is not None
        depth = -(-(-(-rows // chunks.value)) // 32) * 32
        assert depth * 2 * inner * 2 <= 1 << 31
