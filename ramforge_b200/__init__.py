"""ramforge_b200 - a B200 (sm_100a) decode engine for RAMforge's legacy executor.

The compute path is librfcuda.so (hand-written CUDA kernels + a C ABI,
include/rfcuda.h); this package holds its Python host mirror (engine.py),
ctypes bindings (_lib.py), the synthetic model generator (synth.py) and the
build script (build.py).
"""
from .engine import (DecodeEngine, KvView, QMatrix, RfError, decode_attention, dequantize_i8,  # noqa: F401
                     i8_matmul, kv_cache_read, kv_cache_write, layer_read_plan, norm_i8, qk_norm_rope, quantize_i8,
                     selftest_wait, should_keep_resident, swiglu_i8, tp_unique_id, tree_attention, verify_drafts,
                     verify_error_word, verify_greedy)

__all__ = ["DecodeEngine", "KvView", "QMatrix", "RfError", "decode_attention", "dequantize_i8", "i8_matmul",
           "kv_cache_read", "kv_cache_write", "layer_read_plan", "norm_i8", "qk_norm_rope", "quantize_i8",
           "selftest_wait", "should_keep_resident", "swiglu_i8", "tp_unique_id", "tree_attention", "verify_drafts",
           "verify_error_word", "verify_greedy"]
