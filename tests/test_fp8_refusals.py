"""What the 8-bit floating point entry points and the sampler refuse, on the CPU: the checks come before anything touches a
device, so a context that is nothing but zeros will do."""
import ctypes as C

import pytest

from tensorwarp_amd import _lib

A, B = 0x1000, 0x2000   # addresses that are never read: every call here is refused, or has nothing to do


@pytest.fixture()
def ctx():
    return C.cast(C.create_string_buffer(1 << 14), C.c_void_p)


def gemm(ctx, a=A, a_s=A, w=A, w_s=A, m=4, n=32, k=128, c=B, dtype=_lib.F32):
    return _lib.load().twm_gemm_fp8(ctx, a, a_s, w, w_s, m, n, k, c, dtype)


def quantize(ctx, x=A, dtype=_lib.F32, rows=2, cols=256, q=B, scales=B):
    return _lib.load().twm_quantize_rows_fp8(ctx, x, dtype, rows, cols, q, scales)


def gated(name, ctx, x=A, dtype=_lib.F32, rows=2, cols=256, paired=0, q=B, scales=B):
    return getattr(_lib.load(), name)(ctx, x, dtype, rows, cols, paired, q, scales)


def norm(ctx, x=A, dtype=_lib.F32, residual=A, weight=A, eps=1e-6, rows=2, cols=256, total=B, q=B, scales=B, normed=B):
    return _lib.load().twm_add_rms_norm_fp8(ctx, x, dtype, residual, weight, eps, rows, cols, total, q, scales, normed)


def sample(ctx, logits=A, rows=2, cols=100, uniform=A, temperature=A, top_k=A, top_p=A, min_p=A, out=B):
    return _lib.load().twm_sample_f32(ctx, logits, rows, cols, uniform, temperature, top_k, top_p, min_p, out)


def refused(rc, code, text):
    assert rc == code
    assert text in _lib.load().twm_last_error(), _lib.load().twm_last_error()
    assert _lib.load().twm_last_error_kind() == 0


def test_null_contexts():
    for rc in (gemm(None), quantize(None), gated("twm_swiglu_rows_fp8", None), gated("twm_geglu_rows_fp8", None), norm(None), sample(None)):
        refused(rc, _lib.INVALID_HANDLE, b"null context")


def test_gemm_refusals(ctx):
    refused(gemm(ctx, k=120), _lib.SHAPE_ERROR, b"divisible by 16")
    refused(gemm(ctx, dtype=_lib.I32), _lib.UNSUPPORTED_OP, b"f16 or f32")
    for name in ("a", "a_s", "w", "w_s", "c"):
        refused(gemm(ctx, **{name: None}), _lib.INVALID_HANDLE, b"null pointer")
    for name in ("a", "w"):
        refused(gemm(ctx, **{name: A + 8}), _lib.SHAPE_ERROR, b"16-byte aligned")
    for name in ("a_s", "w_s", "c"):
        refused(gemm(ctx, **{name: A + 2}), _lib.SHAPE_ERROR, b"aligned to its elements")
    refused(gemm(ctx, c=B + 1, dtype=_lib.F16), _lib.SHAPE_ERROR, b"aligned to its elements")
    for name in ("m", "n"):
        refused(gemm(ctx, **{name: (1 << 24) + 16}), _lib.SHAPE_ERROR, b"beyond 2^24")
    refused(gemm(ctx, k=(1 << 20) + 16), _lib.SHAPE_ERROR, b"beyond 2^20")
    refused(gemm(ctx, m=1 << 20, n=(1 << 16) + 1), _lib.SHAPE_ERROR, b"more than 2^36")
    assert gemm(ctx, m=0) == _lib.OK and gemm(ctx, n=0, c=None) == _lib.OK


def test_row_refusals(ctx):
    calls = [lambda **kw: quantize(ctx, **kw), lambda **kw: gated("twm_swiglu_rows_fp8", ctx, **kw), lambda **kw: gated("twm_geglu_rows_fp8", ctx, **kw),
             lambda **kw: norm(ctx, **kw)]
    for call in calls:
        refused(call(dtype=_lib.U8), _lib.UNSUPPORTED_OP, b"f16 or f32")
        for name in ("x", "q", "scales"):
            refused(call(**{name: None}), _lib.INVALID_HANDLE, b"null pointer")
        refused(call(x=A + 2), _lib.SHAPE_ERROR, b"aligned to its elements")
        refused(call(x=A + 1, dtype=_lib.F16), _lib.SHAPE_ERROR, b"aligned to its elements")
        refused(call(scales=A + 2), _lib.SHAPE_ERROR, b"aligned to its elements")
        refused(call(rows=(1 << 24) + 1), _lib.SHAPE_ERROR, b"beyond 2^24")
        refused(call(cols=(1 << 24) + 1), _lib.SHAPE_ERROR, b"beyond 2^24")
        assert call(rows=0) == _lib.OK and call(cols=0, x=None) == _lib.OK
    for name in ("twm_swiglu_rows_fp8", "twm_geglu_rows_fp8"):
        refused(gated(name, ctx, cols=48, paired=1), _lib.SHAPE_ERROR, b"multiple of 32")
    refused(norm(ctx, weight=None), _lib.INVALID_HANDLE, b"null pointer")
    for name in ("residual", "weight", "total"):
        refused(norm(ctx, **{name: A + 2}), _lib.SHAPE_ERROR, b"aligned to its elements")
    refused(norm(ctx, normed=B + 1), _lib.SHAPE_ERROR, b"aligned to its elements")
    for eps in (-1e-6, float("nan")):
        refused(norm(ctx, eps=eps), _lib.SHAPE_ERROR, b"eps")


def test_sample_refusals(ctx):
    for name in ("logits", "uniform", "out"):
        refused(sample(ctx, **{name: None}), _lib.INVALID_HANDLE, b"null pointer")
    for name in ("logits", "uniform", "temperature", "top_k", "top_p", "min_p", "out"):
        refused(sample(ctx, **{name: A + 2}), _lib.SHAPE_ERROR, b"aligned to its elements")
    refused(sample(ctx, rows=(1 << 24) + 1), _lib.SHAPE_ERROR, b"beyond 2^24")
    refused(sample(ctx, cols=(1 << 24) + 1), _lib.SHAPE_ERROR, b"beyond 2^24")
    assert sample(ctx, rows=0, logits=None) == _lib.OK
