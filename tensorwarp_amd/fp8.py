"""Linear layers in 8-bit floating point (e4m3 codes as u8, f32 scales per 128 features), the rows that feed them, and token
sampling: thin calls into libtwmarlin_hip.so like those of quantize.py.  The reference has no counterpart; the kinds of arrays
are described in include/twmarlin.h.
"""
import ctypes as C

from . import _lib
from .quantize import _check

FP8_BLOCK = 128   # features (and weight columns) that share a scale


_DTYPES = {"f32": _lib.F32, "f16": _lib.F16}


def _dtype(t):
    return _DTYPES.get(t.dtype, -1)


def _ptr(t):
    return None if t is None else t.ptr


def gemm_fp8(device, a, a_scales, w, w_scales, m, n, k, c):
    """C [m, n] (f32 or f16) = A [m, k] x W [n, k]^T, both e4m3; a_scales [m, ceil(k / 128)], w_scales [ceil(n / 128), ceil(k / 128)].

    f32 results come from exact products and f32 sums.  So do f16 results of up to 16 rows; from 17 on they may come from the 8-bit
    matrix instructions, which cut the products of eight neighbouring features off below 2^-13 of the largest one's power of two before
    they add them (1.5e-5 of a result's norm; small products beside large ones that cancel are lost).  plan_fp8() says which; f32 results
    rounded by twm_cast_f32_to_f16 keep the exact ones.
    """
    _check(device._l.twm_gemm_fp8(device.handle, a.ptr, a_scales.ptr, w.ptr, w_scales.ptr, m, n, k, c.ptr, _dtype(c)))


def plan_fp8(m, n, k, dtype="f32"):
    """What gemm_fp8() launches for these sizes, as a line of text."""
    buf = C.create_string_buffer(256)
    _check(_lib.load().twm_plan_describe_fp8(m, n, k, _DTYPES.get(dtype, -1), buf, 256))
    return buf.value.decode()


def quantize_rows_fp8(device, x, q, scales, rows, cols):
    """x f32 or f16 [rows, cols] -> q e4m3 [rows, cols], scales f32 [rows, ceil(cols / 128)]."""
    _check(device._l.twm_quantize_rows_fp8(device.handle, x.ptr, _dtype(x), rows, cols, q.ptr, scales.ptr))


def swiglu_rows_fp8(device, gate_up, q, scales, ffn_dim, batch, paired=False):
    """swiglu_rows() with f32 or f16 rows in and e4m3 rows out."""
    _check(device._l.twm_swiglu_rows_fp8(device.handle, gate_up.ptr, _dtype(gate_up), batch, ffn_dim, int(paired), q.ptr, scales.ptr))


def geglu_rows_fp8(device, gate_up, q, scales, dim, batch, paired=False):
    """The same with the tanh form of gelu as the gate."""
    _check(device._l.twm_geglu_rows_fp8(device.handle, gate_up.ptr, _dtype(gate_up), batch, dim, int(paired), q.ptr, scales.ptr))


def add_rms_norm_fp8(device, x, residual, weight, eps, rows, cols, q, scales, sum=None, normed=None):
    """s = x + residual (None: x), y = s / sqrt(mean(s^2) + eps) * weight as e4m3 rows; sum (f32, may be the residual) receives
    s, normed (f16) receives y."""
    _check(device._l.twm_add_rms_norm_fp8(device.handle, x.ptr, _dtype(x), _ptr(residual), weight.ptr, eps, rows, cols, _ptr(sum),
                                          q.ptr, scales.ptr, _ptr(normed)))


def sample(device, logits, uniform, output, rows, cols, temperature=None, top_k=None, top_p=None, min_p=None):
    """One token per row of logits f32 [rows, cols] from uniform f32 [rows]; the rules are f32 (top_k i32) [rows] or None."""
    _check(device._l.twm_sample_f32(device.handle, logits.ptr, rows, cols, uniform.ptr, _ptr(temperature), _ptr(top_k), _ptr(top_p),
                                    _ptr(min_p), output.ptr))
