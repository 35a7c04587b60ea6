"""tensorwarp_amd: MI355X (gfx950) implementation of TensorWarp's TW-Marlin W4A16
quantized-linear path.  The product is libtwmarlin_hip.so (C ABI in include/twmarlin.h);
this package is the thin Python mirror of the reference's Rust interface used by tests
and the benchmark."""
from . import _lib  # noqa: F401
from .quantize import *  # noqa: F401,F403
from .quantize import (DeviceError, ExpertBank, GpuTensor, GraphCapture, MarlinWeight, TWMarlinWeights,  # noqa: F401
                       WarpDevice)
from .fp8 import (add_rms_norm_fp8, gemm_fp8, geglu_rows_fp8, plan_fp8, quantize_rows_fp8, sample, swiglu_rows_fp8)  # noqa: F401
from .kv import KvCache, KvSequences, attention_decode, attention_prompt, kv_append, kv_copy_pages, kv_layers  # noqa: F401

__version__ = "0.1.0"
