"""Python access to libsneppx_quant.so (the HIP-backed quantized linear path).

Two layers, both thin ctypes bindings over the C-ABI in include/:

* `Library` - the reference's host-pointer quantization API
  (include/sneppx_quantization.h) with numpy in / numpy out, mirroring the
  return tuples of the reference's C functions (rc first, then outputs).
* device entry points (include/sneppx_qlinear.h) taking torch tensors that
  live on the GPU; they launch on torch's current stream unless a stream is
  given.  torch is only the allocator/stream plumbing here.

There is no fallback: if the shared library is missing, `load()` raises.
"""
from __future__ import annotations

import ctypes as C
import os

import numpy as np

try:  # torch first: its libamdhip64 must be the one the library binds to
    import torch
except ImportError:  # pragma: no cover - torch is part of the image
    torch = None

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libsneppx_quant.so")

# SNEPPXDtype ordinals (multidimensional_tensor_engine.h:27-41)
SNEPPX_FLOAT32 = 0
SNEPPX_FLOAT16 = 2
SNEPPX_BFLOAT16 = 3
SNEPPX_INT8 = 8

_f32p = np.ctypeslib.ndpointer(np.float32, flags="C")
_i8p = np.ctypeslib.ndpointer(np.int8, flags="C")
_u8p = np.ctypeslib.ndpointer(np.uint8, flags="C")
_sz = C.c_size_t
_vp = C.c_void_p

EXPORTS = {
    # reference surface
    "SNEPPX_quantize_int8_sym": (C.c_int, [_f32p, _i8p, _sz, C.POINTER(C.c_float)]),
    "SNEPPX_dequantize_int8_sym": (C.c_int, [_i8p, _f32p, _sz, C.c_float]),
    "SNEPPX_quantize_int8_asym": (C.c_int, [_f32p, _i8p, _sz, C.POINTER(C.c_float), C.POINTER(C.c_int32)]),
    "SNEPPX_dequantize_int8_asym": (C.c_int, [_i8p, _f32p, _sz, C.c_float, C.c_int32]),
    "SNEPPX_quantize_int8_channel": (C.c_int, [_f32p, _i8p, _sz, _sz, _f32p]),
    "SNEPPX_quantize_int4_sym": (C.c_int, [_f32p, _u8p, _sz, C.POINTER(C.c_float)]),
    "SNEPPX_dequantize_int4_sym": (C.c_int, [_u8p, _f32p, _sz, C.c_float]),
    "SNEPPX_float_to_fp8_e4m3": (C.c_uint8, [C.c_float]),
    "SNEPPX_fp8_e4m3_to_float": (C.c_float, [C.c_uint8]),
    "SNEPPX_quantize_fp8_e4m3": (C.c_int, [_f32p, _u8p, _sz]),
    "SNEPPX_dequantize_fp8_e4m3": (C.c_int, [_u8p, _f32p, _sz]),
    "SNEPPX_float_to_fp8_e5m2": (C.c_uint8, [C.c_float]),
    "SNEPPX_fp8_e5m2_to_float": (C.c_float, [C.c_uint8]),
    "SNEPPX_quantize_fp8_e5m2": (C.c_int, [_f32p, _u8p, _sz]),
    "SNEPPX_dequantize_fp8_e5m2": (C.c_int, [_u8p, _f32p, _sz]),
    "SNEPPX_awq_scale_weights": (C.c_int, [_f32p, _sz, _sz, _f32p, _f32p]),
    "SNEPPX_awq_quantize": (C.c_int, [_f32p, _i8p, _vp, _f32p, _sz, _sz, C.c_int]),
    "SNEPPX_gptq_quantize": (C.c_int, [_f32p, _sz, _sz, C.c_int, C.c_int, _i8p, _f32p, _vp, C.c_int]),
    "SNEPPX_gptq_compute_hessian": (C.c_int, [_f32p, _f32p, _sz, _sz]),
    "SNEPPX_gptq_quantize_block": (C.c_int, [_f32p, _f32p, _f32p, C.POINTER(C.c_float),
                                             C.POINTER(C.c_int32), _sz, C.c_int, C.c_int]),
    "SNEPPX_quant_params_create": (C.c_int, [_vp, C.c_int]),
    "SNEPPX_quant_mode_name": (C.c_char_p, [C.c_int]),
    # device entry points
    "SNEPPX_qlinear_last_error": (C.c_char_p, []),
    "SNEPPX_dev_quantize_int8_channel": (C.c_int, [_vp, _vp, _vp, _sz, _sz, _vp]),
    "SNEPPX_dev_quantize_int8_channel_rounding": (C.c_int, [_vp, _vp, _vp, _sz, _sz, C.c_int, _vp]),
    "SNEPPX_dev_fake_quant": (C.c_int, [_vp, _vp, _sz, C.c_float, C.c_int, _vp]),
    "SNEPPX_dev_quantize_w4_awq": (C.c_int, [_vp, _vp, _vp, _vp, _sz, _sz, C.c_int, _vp]),
    "SNEPPX_dev_quantize_w4_gptq": (C.c_int, [_vp, _vp, _sz, _vp, _vp, _sz, _sz, _vp]),
    "SNEPPX_dev_quantize_fp8_e4m3_scaled": (C.c_int, [_vp, _vp, _vp, _sz, _vp]),
    "SNEPPX_qlinear_w8_gemv": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "SNEPPX_qlinear_w4a16": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _sz, _vp, _vp, C.c_int, _sz, _sz,
                                       _sz, C.c_int, _vp]),
    "SNEPPX_qlinear_w4a16_noalloc": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _sz, _vp, _vp, C.c_int, _sz, _sz,
                                               _sz, C.c_int, _vp]),
    "SNEPPX_qlinear_w4_actorder_prepare": (C.c_int, [_vp, _vp, _sz, _vp, _vp, _sz, _sz, _vp]),
    "SNEPPX_qlinear_w4a16_actorder": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, C.c_int, _sz, _sz,
                                                _sz, C.c_int, _vp]),
    "SNEPPX_qlinear_silu_mul": (C.c_int, [_vp, _vp, _sz, _sz, _vp]),
    "SNEPPX_qlinear_w4a16_swiglu": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz, C.c_int, _vp]),
    "SNEPPX_qlinear_w4a16_mlp": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, C.c_int, _sz, _sz,
                                           _sz, _sz, C.c_int, _vp]),
    "SNEPPX_qlinear_silu_mul_quant_int8": (C.c_int, [_vp, _vp, _vp, _sz, _sz, _vp]),
    "SNEPPX_dev_quantize_int8_channel_bf16": (C.c_int, [_vp, _vp, _vp, _sz, _sz, _vp]),
    "SNEPPX_qlinear_w8a8_i8": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "SNEPPX_qlinear_i8_gemm_i32": (C.c_int, [_vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "SNEPPX_qlinear_w8a8_fp8": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    # quantized weights on disk + model-zoo int8 (include/sneppx_qstore.h)
    "SNEPPX_qstore_open": (_vp, [C.c_char_p]),
    "SNEPPX_qstore_close": (None, [_vp]),
    "SNEPPX_qstore_count": (_sz, [_vp]),
    "SNEPPX_qstore_name": (C.c_char_p, [_vp, _sz]),
    "SNEPPX_qstore_info": (C.c_int, [_vp, C.c_char_p, C.POINTER(C.c_int), C.POINTER(_sz),
                                     C.POINTER(_sz), C.POINTER(_sz)]),
    "SNEPPX_qstore_data": (_vp, [_vp, C.c_char_p, C.POINTER(_sz)]),
    "SNEPPX_qstore_read_device": (C.c_int, [_vp, C.c_char_p, _vp, _sz, _vp]),
    "SNEPPX_qstore_metadata": (C.c_char_p, [_vp, C.c_char_p]),
    "SNEPPX_qstore_writer_open": (_vp, [C.c_char_p]),
    "SNEPPX_qstore_writer_add_host": (C.c_int, [_vp, C.c_char_p, C.c_int, C.POINTER(_sz), _sz, _vp]),
    "SNEPPX_qstore_writer_add_device": (C.c_int, [_vp, C.c_char_p, C.c_int, C.POINTER(_sz), _sz, _vp,
                                                  _vp]),
    "SNEPPX_qstore_writer_set_metadata": (C.c_int, [_vp, C.c_char_p, C.c_char_p]),
    "SNEPPX_qstore_writer_close": (C.c_int, [_vp]),
    "SNEPPX_qstore_save_w4": (C.c_int, [_vp, C.c_char_p, _vp, _vp, _vp, _vp, _sz, _sz, C.c_int, _sz,
                                        _vp]),
    "SNEPPX_qstore_query_w4": (C.c_int, [_vp, C.c_char_p, C.POINTER(_sz), C.POINTER(_sz),
                                         C.POINTER(_sz), C.POINTER(C.c_int), C.POINTER(C.c_int),
                                         C.POINTER(C.c_int)]),
    "SNEPPX_qstore_load_w4": (C.c_int, [_vp, C.c_char_p, _vp, _vp, _vp, _vp, _vp]),
    "SNEPPX_qstore_save_w8": (C.c_int, [_vp, C.c_char_p, _vp, _vp, _sz, _sz, _vp]),
    "SNEPPX_qstore_query_w8": (C.c_int, [_vp, C.c_char_p, C.POINTER(_sz), C.POINTER(_sz)]),
    "SNEPPX_qstore_load_w8": (C.c_int, [_vp, C.c_char_p, _vp, _vp, _vp]),
    "SNEPPX_quantize_int8_modelzoo": (C.c_int, [_f32p, _i8p, _sz, C.POINTER(C.c_float)]),
    "SNEPPX_dev_quantize_int8_modelzoo": (C.c_int, [_vp, _vp, _vp, _sz, _vp]),
    # quantized layers for the reference's linear call sites (include/sneppx_qlayer.h)
    "SNEPPX_qlayer_create_kn": (_vp, [_f32p, _sz, _sz, C.c_int, C.c_int, _vp]),
    "SNEPPX_qlayer_create_kn_device": (_vp, [_vp, _sz, _sz, C.c_int, C.c_int, _vp]),
    "SNEPPX_qlayer_load": (_vp, [_vp, C.c_char_p, _vp]),
    "SNEPPX_qlayer_save": (C.c_int, [_vp, _vp, C.c_char_p, _vp]),
    "SNEPPX_qlayer_destroy": (None, [_vp]),
    "SNEPPX_qlayer_set_bias": (C.c_int, [_vp, _f32p, _vp]),
    "SNEPPX_qlayer_set_bias_device": (C.c_int, [_vp, _vp, _vp]),
    "SNEPPX_qlayer_in_features": (_sz, [_vp]),
    "SNEPPX_qlayer_out_features": (_sz, [_vp]),
    "SNEPPX_qlayer_format": (C.c_int, [_vp]),
    "SNEPPX_qlayer_forward_f32": (C.c_int, [_vp, _vp, _vp, _sz, _vp]),
    "SNEPPX_qlayer_forward_bf16": (C.c_int, [_vp, _vp, _vp, _sz, _vp]),
    "SNEPPX_qlayer_matmul_host": (C.c_int, [_vp, _f32p, _f32p, _sz]),
    # MX formats (include/sneppx_mx.h)
    "SNEPPX_mx_bits": (C.c_int, [C.c_int]),
    "SNEPPX_mx_default_block": (C.c_int, [C.c_int]),
    "SNEPPX_mx_packed_bytes": (_sz, [C.c_int, _sz, _sz, C.c_int]),
    "SNEPPX_mx_scale_count": (_sz, [C.c_int, _sz, _sz, C.c_int]),
    "SNEPPX_dev_quantize_mx": (C.c_int, [_vp, _vp, _vp, _sz, _sz, C.c_int, C.c_int, _vp]),
    "SNEPPX_dev_dequantize_mx": (C.c_int, [_vp, _vp, _vp, _sz, _sz, C.c_int, C.c_int, _vp]),
    "SNEPPX_qlinear_mxfp4_gemm": (C.c_int, [_vp, _vp, _vp, _vp, _vp, C.c_int, _sz, _sz, _sz, _vp]),
    "SNEPPX_qlinear_mx_gemm": (C.c_int, [_vp, _vp, _vp, _vp, C.c_int, _vp, C.c_int, _sz, _sz, _sz, _vp]),
    "SNEPPX_qlinear_mx_gemm_mfma": (C.c_int, [_vp, _vp, _vp, _vp, C.c_int, _vp, C.c_int, _sz, _sz, _sz, _vp]),
    "SNEPPX_qlinear_mx_gemm_bs": (C.c_int, [_vp, _vp, _vp, _vp, C.c_int, C.c_int, _vp, C.c_int, _sz, _sz, _sz,
                                            _vp]),
    "SNEPPX_mx_to_mfma": (C.c_int, [_vp, _vp, _vp, _vp, _sz, _sz, C.c_int, _vp, _vp]),
    # paged key-value cache (include/sneppx_kv.h)
    "SNEPPX_kv_append": (C.c_int, [_vp, _vp, _sz, _vp, _sz, _sz, _vp, _vp, _vp, _vp, _sz, _vp, _vp, _sz, _vp]),
    "SNEPPX_kv_attention": (C.c_int, [_vp, _vp, _sz, _vp, _sz, C.c_int, _vp, _sz, _vp, _sz, _sz, _sz, C.c_float,
                                      C.c_int, _vp]),
    "SNEPPX_kv_evict": (C.c_int, [_vp, _vp, _sz, _vp, _vp, _vp, _sz, _sz, _sz, _sz, _vp]),
    "SNEPPX_kv_append_rotated": (C.c_int, [_vp, _vp, _vp, _sz, _vp, _sz, _sz, _vp, _sz, _vp, _sz, _sz, _vp, _vp, _vp,
                                           _vp, _vp]),
    "SNEPPX_kv_reserve": (C.c_int, [_vp, _sz, _sz, _vp, _sz, _vp, _vp, _vp, _sz, _vp, _vp, _vp, _vp, _sz, _vp]),
    "SNEPPX_kv_release": (C.c_int, [_vp, _sz, _sz, _vp, _sz, _vp, _sz, _vp]),
    "SNEPPX_kv_share": (C.c_int, [_vp, _sz, _sz, _vp, _sz, _vp, _vp, _vp, _vp, _sz, _vp]),
    "SNEPPX_kv_attention_shared": (C.c_int, [_vp, _vp, _sz, _vp, _sz, C.c_int, _vp, _sz, _vp, _sz, _sz, _sz, _vp, _vp,
                                             _sz, _sz, _sz, C.c_float, _vp]),
    "SNEPPX_kv_key_bounds": (C.c_int, [_vp, _vp, _vp, _sz, _vp, _vp, _sz, _sz, _vp]),
    "SNEPPX_kv_pick": (C.c_int, [_vp, _vp, _vp, _sz, _sz, _vp, _sz, _vp, _sz, _sz, _sz, _sz, _sz, _vp, _vp, _vp]),
    "SNEPPX_kv_attention_picked": (C.c_int, [_vp, _vp, _sz, _vp, _sz, C.c_int, _vp, _sz, _vp, _sz, _sz, C.c_float,
                                             C.c_int, _vp]),
    # rotary positions (include/sneppx_rotary.h)
    "SNEPPX_rotary_frequencies": (C.c_int, [_vp, C.POINTER(C.c_float), _sz, C.c_double, C.c_int, C.c_double, C.c_double,
                                            C.c_double, C.c_double]),
    "SNEPPX_rotary_apply": (C.c_int, [_vp, _vp, _sz, _vp, _sz, _sz, _vp, _sz, _vp, _sz, _sz, _sz, _vp, _sz, _vp]),
    # thin HIP ABI
    "snx_hip_device_count": (C.c_int, [C.POINTER(C.c_int)]),
    "snx_hip_event_create": (C.c_int, [C.POINTER(_vp)]),
    "snx_hip_event_destroy": (C.c_int, [_vp]),
    "snx_hip_event_record": (C.c_int, [_vp, _vp]),
    "snx_hip_event_sync": (C.c_int, [_vp]),
    "snx_hip_event_elapsed_ms": (C.c_int, [C.POINTER(C.c_float), _vp, _vp]),
    "snx_hip_stream_sync": (C.c_int, [_vp]),
    "snx_hip_device_info": (C.c_int, [C.c_char_p, _sz, C.POINTER(C.c_int), C.POINTER(C.c_int)]),
    "SNEPPX_qlinear_release_workspaces": (C.c_int, [_vp]),
    "SNEPPX_qlinear_noalloc_reset": (C.c_int, [_vp]),
    "SNEPPX_qlinear_w8a8_i8_dyn": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "SNEPPX_qlinear_w8a8_fp8_dyn": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "snx_hip_stream_begin_capture": (C.c_int, [_vp]),
    "snx_hip_stream_end_capture": (C.c_int, [_vp, C.POINTER(_vp)]),
    "snx_hip_graph_launch": (C.c_int, [_vp, _vp]),
    "snx_hip_graph_destroy": (C.c_int, [_vp]),
    "snx_workspace_count": (C.c_long, []),
}


class QuantParams(C.Structure):
    """SNEPPXQuantParams (quantization.h:42-48)."""
    _fields_ = [("scale", C.c_float), ("zero_point", C.c_int32), ("qmin", C.c_float),
                ("qmax", C.c_float), ("scale_max", C.c_float)]


class SneppxError(RuntimeError):
    pass


def _ptr(t):
    if t is None:
        return None
    return C.c_void_p(t.data_ptr())


def _bias_ptr(bias, n, like):
    """Pointer of an optional bias after checking what the kernels read: fp32,
    contiguous, on the output's device, exactly n elements (2F for the stacked
    gate/up of the SwiGLU form).  Anything else raises ValueError rather than
    letting a kernel read past the end or reinterpret bf16 bits."""
    if bias is None:
        return None
    if not isinstance(bias, torch.Tensor):
        raise ValueError("bias must be a torch tensor on the device (fp32 [N])")
    if bias.dtype != torch.float32:
        raise ValueError(f"bias must be float32, got {bias.dtype}")
    if not bias.is_contiguous():
        raise ValueError("bias must be contiguous")
    if bias.device != like.device:
        raise ValueError(f"bias is on {bias.device}, the output on {like.device}")
    if bias.numel() != n:
        raise ValueError(f"bias has {bias.numel()} elements, the linear needs {n}")
    return C.c_void_p(bias.data_ptr())


class Library:
    """ctypes view of libsneppx_quant.so."""

    def __init__(self, path: str = LIB_PATH):
        if not os.path.exists(path):
            raise SneppxError(f"{path} is not built; run `make -C sneppx-alg_amd` "
                              "(or __graft_entry__.build()) - there is no CPU fallback")
        self.path = path
        self.lib = C.CDLL(path)
        self.fn = {}
        for name, (res, args) in EXPORTS.items():
            f = getattr(self.lib, name)
            f.restype, f.argtypes = res, args
            self.fn[name] = f

    def last_error(self) -> str:
        return self.fn["SNEPPX_qlinear_last_error"]().decode()

    def check(self, rc: int, what: str) -> None:
        if rc != 0:
            raise SneppxError(f"{what} failed: {self.last_error()}")

    # ---------------- reference host API (numpy) -------------------------
    def quantize_int8_sym(self, x):
        x = np.ascontiguousarray(x, np.float32).ravel()
        q = np.zeros(x.size, np.int8)
        s = C.c_float(0)
        rc = self.fn["SNEPPX_quantize_int8_sym"](x, q, x.size, C.byref(s))
        return rc, q, np.float32(s.value)

    def dequantize_int8_sym(self, q, scale):
        q = np.ascontiguousarray(q, np.int8).ravel()
        y = np.zeros(q.size, np.float32)
        return self.fn["SNEPPX_dequantize_int8_sym"](q, y, q.size, scale), y

    def quantize_int8_asym(self, x):
        x = np.ascontiguousarray(x, np.float32).ravel()
        q = np.zeros(x.size, np.int8)
        s, z = C.c_float(0), C.c_int32(0)
        rc = self.fn["SNEPPX_quantize_int8_asym"](x, q, x.size, C.byref(s), C.byref(z))
        return rc, q, np.float32(s.value), int(z.value)

    def dequantize_int8_asym(self, q, scale, zp):
        q = np.ascontiguousarray(q, np.int8).ravel()
        y = np.zeros(q.size, np.float32)
        return self.fn["SNEPPX_dequantize_int8_asym"](q, y, q.size, scale, zp), y

    def quantize_int8_channel(self, x):
        x = np.ascontiguousarray(x, np.float32)
        rows, cols = x.shape
        q = np.zeros((rows, cols), np.int8)
        s = np.zeros(rows, np.float32)
        rc = self.fn["SNEPPX_quantize_int8_channel"](x, q, rows, cols, s)
        return rc, q, s

    def quantize_int4_sym(self, x):
        x = np.ascontiguousarray(x, np.float32).ravel()
        p = np.zeros((x.size + 1) // 2, np.uint8)
        s = C.c_float(0)
        rc = self.fn["SNEPPX_quantize_int4_sym"](x, p, x.size, C.byref(s))
        return rc, p, np.float32(s.value)

    def dequantize_int4_sym(self, packed, n, scale):
        packed = np.ascontiguousarray(packed, np.uint8)
        y = np.zeros(n, np.float32)
        return self.fn["SNEPPX_dequantize_int4_sym"](packed, y, n, scale), y

    def quantize_fp8(self, x, fmt="e4m3"):
        x = np.ascontiguousarray(x, np.float32).ravel()
        c = np.zeros(x.size, np.uint8)
        return self.fn[f"SNEPPX_quantize_fp8_{fmt}"](x, c, x.size), c

    def dequantize_fp8(self, c, fmt="e4m3"):
        c = np.ascontiguousarray(c, np.uint8).ravel()
        y = np.zeros(c.size, np.float32)
        return self.fn[f"SNEPPX_dequantize_fp8_{fmt}"](c, y, c.size), y

    def awq_scale_weights(self, w, act_scales):
        w = np.array(w, np.float32, order="C", copy=True)
        rows, cols = w.shape
        s = np.zeros((rows, cols), np.float32)
        a = np.ascontiguousarray(act_scales, np.float32)
        rc = self.fn["SNEPPX_awq_scale_weights"](w, rows, cols, a, s)
        return rc, w, s

    def awq_quantize(self, w, group_size, act_scales=None):
        w = np.ascontiguousarray(w, np.float32)
        rows, cols = w.shape
        g = group_size if group_size > 0 else 128
        q = np.zeros((rows, cols), np.int8)
        s = np.zeros((rows, (cols + g - 1) // g), np.float32)
        a = None if act_scales is None else np.ascontiguousarray(act_scales, np.float32)
        rc = self.fn["SNEPPX_awq_quantize"](w, q, None if a is None else a.ctypes.data_as(_vp),
                                            s, rows, cols, group_size)
        return rc, q, s

    def gptq_compute_hessian(self, act):
        act = np.ascontiguousarray(act, np.float32)
        n, dim = act.shape
        h = np.zeros((dim, dim), np.float32)
        return self.fn["SNEPPX_gptq_compute_hessian"](h, act, n, dim), h

    def gptq_quantize_block(self, w, h_inv, bits, sym):
        w = np.array(w, np.float32, order="C", copy=True)
        h = np.array(h_inv, np.float32, order="C", copy=True)
        qw = np.zeros(w.size, np.float32)
        s, z = C.c_float(0), C.c_int32(-7)
        rc = self.fn["SNEPPX_gptq_quantize_block"](w, h, qw, C.byref(s), C.byref(z), w.size, bits, sym)
        return rc, w, qw, np.float32(s.value), int(z.value)

    def gptq_quantize(self, w, group_size, bits, sym, with_zeros=True):
        w = np.array(w, np.float32, order="C", copy=True)
        rows, cols = w.shape
        g = group_size if group_size > 0 else 128
        ng = (cols + g - 1) // g
        q = np.full((rows, cols), 0x55, np.int8)
        s = np.zeros((rows, ng), np.float32)
        z = np.full((rows, ng), -7, np.int32) if with_zeros else None
        rc = self.fn["SNEPPX_gptq_quantize"](w, rows, cols, group_size, bits, q, s,
                                             None if z is None else z.ctypes.data_as(_vp), sym)
        return rc, w, q, s, z

    def quant_params_create(self, mode):
        p = QuantParams()
        rc = self.fn["SNEPPX_quant_params_create"](C.cast(C.pointer(p), _vp), mode)
        return rc, (p.scale, p.zero_point, p.qmin, p.qmax, p.scale_max)

    def quant_mode_name(self, mode):
        return self.fn["SNEPPX_quant_mode_name"](mode).decode()

    # ---------------- device entry points (torch tensors on the GPU) -------
    @staticmethod
    def _stream(stream):
        if stream is not None:
            return C.c_void_p(stream)
        return C.c_void_p(torch.cuda.current_stream().cuda_stream)

    def dev_quantize_int8_channel(self, w, q, scales, stream=None, half_even=False):
        rows, cols = w.shape
        if half_even:
            self.check(self.fn["SNEPPX_dev_quantize_int8_channel_rounding"](
                _ptr(w), _ptr(q), _ptr(scales), rows, cols, 1, self._stream(stream)),
                "dev_quantize_int8_channel_rounding")
        else:
            self.check(self.fn["SNEPPX_dev_quantize_int8_channel"](
                _ptr(w), _ptr(q), _ptr(scales), rows, cols, self._stream(stream)), "dev_quantize_int8_channel")

    def dev_fake_quant(self, x, out, scale, bits, stream=None):
        self.check(self.fn["SNEPPX_dev_fake_quant"](
            _ptr(x), _ptr(out), x.numel(), scale, bits, self._stream(stream)), "dev_fake_quant")

    def dev_quantize_w4_awq(self, w, qweight, scales, qzeros, group, stream=None):
        N, K = w.shape
        self.check(self.fn["SNEPPX_dev_quantize_w4_awq"](
            _ptr(w), _ptr(qweight), _ptr(scales), _ptr(qzeros), N, K, group, self._stream(stream)),
            "dev_quantize_w4_awq")

    def dev_quantize_w4_gptq(self, w, g_idx, G, qweight, scales, stream=None):
        N, K = w.shape
        self.check(self.fn["SNEPPX_dev_quantize_w4_gptq"](
            _ptr(w), _ptr(g_idx), G, _ptr(qweight), _ptr(scales), N, K, self._stream(stream)),
            "dev_quantize_w4_gptq")

    def dev_quantize_fp8_e4m3_scaled(self, x, out, scale, stream=None):
        self.check(self.fn["SNEPPX_dev_quantize_fp8_e4m3_scaled"](
            _ptr(x), _ptr(out), _ptr(scale), x.numel(), self._stream(stream)), "dev_quantize_fp8_e4m3_scaled")

    def qlinear_w8_gemv(self, x, qweight, scales, y, stream=None, bias=None):
        M, K = x.shape
        N = qweight.shape[0]
        self.check(self.fn["SNEPPX_qlinear_w8_gemv"](
            _ptr(x), _ptr(qweight), _ptr(scales), _bias_ptr(bias, N, y), _ptr(y), M, N, K, self._stream(stream)),
            "qlinear_w8_gemv")

    def qlinear_w4a16(self, x, qweight, scales, qzeros, g_idx, G, y, group, stream=None, bias=None):
        M, K = x.shape
        N = qweight.shape[0]
        ydt = SNEPPX_FLOAT32 if y.dtype == torch.float32 else SNEPPX_BFLOAT16
        self.check(self.fn["SNEPPX_qlinear_w4a16"](
            _ptr(x), _ptr(qweight), _ptr(scales), _ptr(qzeros), _ptr(g_idx), G, _bias_ptr(bias, N, y), _ptr(y),
            ydt, M, N, K, group, self._stream(stream)), "qlinear_w4a16")

    def qlinear_w4a16_noalloc(self, x, qweight, scales, qzeros, g_idx, G, y, group, stream=None,
                              bias=None):
        """SNEPPX_qlinear_w4a16_noalloc: as qlinear_w4a16, scratch from the
        library's static device array instead of a workspace."""
        M, K = x.shape
        N = qweight.shape[0]
        ydt = SNEPPX_FLOAT32 if y.dtype == torch.float32 else SNEPPX_BFLOAT16
        self.check(self.fn["SNEPPX_qlinear_w4a16_noalloc"](
            _ptr(x), _ptr(qweight), _ptr(scales), _ptr(qzeros), _ptr(g_idx), G, _bias_ptr(bias, N, y), _ptr(y),
            ydt, M, N, K, group, self._stream(stream)), "qlinear_w4a16_noalloc")

    def qlinear_noalloc_reset(self, stream=None):
        """SNEPPX_qlinear_noalloc_reset: for a program that has let calls of
        qlinear_w4a16_noalloc overlap."""
        self.check(self.fn["SNEPPX_qlinear_noalloc_reset"](self._stream(stream)), "qlinear_noalloc_reset")

    def qlinear_w4_actorder_prepare(self, qweight, g_idx, G, qweight_sorted, perm, stream=None):
        N, K8 = qweight.shape
        self.check(self.fn["SNEPPX_qlinear_w4_actorder_prepare"](
            _ptr(qweight), _ptr(g_idx), G, _ptr(qweight_sorted), _ptr(perm), N, K8 * 8,
            self._stream(stream)), "qlinear_w4_actorder_prepare")

    def qlinear_w4a16_actorder(self, x, qweight_sorted, scales, qzeros, perm, y, group, stream=None,
                               bias=None):
        M, K = x.shape
        N = qweight_sorted.shape[0]
        ydt = SNEPPX_FLOAT32 if y.dtype == torch.float32 else SNEPPX_BFLOAT16
        self.check(self.fn["SNEPPX_qlinear_w4a16_actorder"](
            _ptr(x), _ptr(qweight_sorted), _ptr(scales), _ptr(qzeros), _ptr(perm), _bias_ptr(bias, N, y), _ptr(y),
            ydt, M, N, K, group, self._stream(stream)), "qlinear_w4a16_actorder")

    def qlinear_w4a16_swiglu(self, x, qweight, scales, qzeros, out, group, stream=None, bias=None):
        """out [M][F] = bf16(silu(x . Wg^T) * (x . Wu^T)), qweight the stacked [2F][K/8]."""
        M, K = x.shape
        F = out.shape[1]
        self.check(self.fn["SNEPPX_qlinear_w4a16_swiglu"](
            _ptr(x), _ptr(qweight), _ptr(scales), _ptr(qzeros), _bias_ptr(bias, 2 * F, out), _ptr(out), M, F, K, group,
            self._stream(stream)), "qlinear_w4a16_swiglu")

    def qlinear_w4a16_mlp(self, x, gate_up, down, y, group, stream=None, gu_bias=None, dn_bias=None):
        """y [M][N] = down(silu(x . Wg^T) * (x . Wu^T)): gate_up = (qweight [2F][H/8],
        scales, qzeros) of the stacked gate/up projection, down = (qweight [N][F/8],
        scales, qzeros)."""
        M, H = x.shape
        gq, gs, gz = gate_up
        dq, ds, dz = down
        F = gq.shape[0] // 2
        N = dq.shape[0]
        ydt = SNEPPX_FLOAT32 if y.dtype == torch.float32 else SNEPPX_BFLOAT16
        self.check(self.fn["SNEPPX_qlinear_w4a16_mlp"](
            _ptr(x), _ptr(gq), _ptr(gs), _ptr(gz), _bias_ptr(gu_bias, 2 * F, y), _ptr(dq), _ptr(ds), _ptr(dz),
            _bias_ptr(dn_bias, N, y), _ptr(y), ydt, M, H, F, N, group, self._stream(stream)), "qlinear_w4a16_mlp")

    def qlinear_silu_mul(self, gate_up, out, stream=None):
        T, F2 = gate_up.shape
        self.check(self.fn["SNEPPX_qlinear_silu_mul"](
            _ptr(gate_up), _ptr(out), T, F2 // 2, self._stream(stream)), "qlinear_silu_mul")

    def qlinear_silu_mul_quant_int8(self, gate_up, q, scales, stream=None):
        T, F2 = gate_up.shape
        self.check(self.fn["SNEPPX_qlinear_silu_mul_quant_int8"](
            _ptr(gate_up), _ptr(q), _ptr(scales), T, F2 // 2, self._stream(stream)),
            "qlinear_silu_mul_quant_int8")

    def dev_quantize_int8_channel_bf16(self, x, q, scales, stream=None):
        rows, cols = x.shape
        self.check(self.fn["SNEPPX_dev_quantize_int8_channel_bf16"](
            _ptr(x), _ptr(q), _ptr(scales), rows, cols, self._stream(stream)),
            "dev_quantize_int8_channel_bf16")

    def qlinear_w8a8_i8(self, A, sA, W, sW, out, stream=None, bias=None):
        M, K = A.shape
        N = W.shape[0]
        self.check(self.fn["SNEPPX_qlinear_w8a8_i8"](
            _ptr(A), _ptr(sA), _ptr(W), _ptr(sW), _bias_ptr(bias, N, out), _ptr(out), M, N, K, self._stream(stream)),
            "qlinear_w8a8_i8")

    def qlinear_w8a8_dyn(self, A, W, sW, out, fp8=False, stream=None, bias=None):
        """C4 from bf16 activations: A quantized inside the call (int8 per
        token, or fp8 per tensor), then the W8A8 GEMM."""
        M, K = A.shape
        N = W.shape[0]
        name = "SNEPPX_qlinear_w8a8_fp8_dyn" if fp8 else "SNEPPX_qlinear_w8a8_i8_dyn"
        self.check(self.fn[name](_ptr(A), _ptr(W), _ptr(sW), _bias_ptr(bias, N, out), _ptr(out), M, N, K,
                                 self._stream(stream)), name[7:])

    def qlinear_i8_gemm_i32(self, A, W, Cm, stream=None):
        M, K = A.shape
        N = W.shape[0]
        self.check(self.fn["SNEPPX_qlinear_i8_gemm_i32"](
            _ptr(A), _ptr(W), _ptr(Cm), M, N, K, self._stream(stream)), "qlinear_i8_gemm_i32")

    def qlinear_w8a8_fp8(self, A, sA, W, sW, out, stream=None, bias=None):
        M, K = A.shape
        N = W.shape[0]
        self.check(self.fn["SNEPPX_qlinear_w8a8_fp8"](
            _ptr(A), _ptr(sA), _ptr(W), _ptr(sW), _bias_ptr(bias, N, out), _ptr(out), M, N, K, self._stream(stream)),
            "qlinear_w8a8_fp8")

    # ---------------- model-zoo int8 (weights.c:225-252) -------------------
    def quantize_int8_modelzoo(self, x):
        x = np.ascontiguousarray(x, np.float32).ravel()
        q = np.zeros(x.size, np.int8)
        m = C.c_float(0)
        rc = self.fn["SNEPPX_quantize_int8_modelzoo"](x, q, x.size, C.byref(m))
        return rc, q, np.float32(m.value)

    def dev_quantize_int8_modelzoo(self, x, q, mult, stream=None):
        self.check(self.fn["SNEPPX_dev_quantize_int8_modelzoo"](
            _ptr(x), _ptr(q), _ptr(mult), x.numel(), self._stream(stream)), "dev_quantize_int8_modelzoo")

    # ---------------- quantized weights on disk (safetensors) --------------
    def qstore_open(self, path):
        h = self.fn["SNEPPX_qstore_open"](os.fsencode(path))
        if not h:
            raise SneppxError(f"qstore_open failed: {self.last_error()}")
        return QStore(self, h)

    def qstore_writer(self, path):
        h = self.fn["SNEPPX_qstore_writer_open"](os.fsencode(path))
        if not h:
            raise SneppxError(f"qstore_writer_open failed: {self.last_error()}")
        return QStoreWriter(self, h)

    # ---------------- quantized layers (reference [K, N] weights) ------------
    def qlayer_create_kn(self, w_kn, fmt="w4", group=128, stream=None):
        """w_kn: numpy fp32 [K, N] (host) or a torch fp32 [K, N] device tensor."""
        code = {"w8": 0, "w4": 1}[fmt]
        if isinstance(w_kn, np.ndarray):
            w = np.ascontiguousarray(w_kn, np.float32)
            K, N = w.shape
            h = self.fn["SNEPPX_qlayer_create_kn"](w, K, N, code, group, self._stream(stream))
        else:
            K, N = w_kn.shape
            h = self.fn["SNEPPX_qlayer_create_kn_device"](_ptr(w_kn), K, N, code, group, self._stream(stream))
        if not h:
            raise SneppxError(f"qlayer_create_kn failed: {self.last_error()}")
        return QLayer(self, h)

    def qlayer_load(self, store, prefix, stream=None):
        h = self.fn["SNEPPX_qlayer_load"](store.h, prefix.encode(), self._stream(stream))
        if not h:
            raise SneppxError(f"qlayer_load failed: {self.last_error()}")
        return QLayer(self, h)

    # ---------------- MX formats (mx_formats.py semantics) ------------------
    def _mx_block(self, fmt, block_size):
        # the reference's `block_size or spec.block_size`, per tensor when <= 0
        if block_size is None:
            return 0
        return block_size if block_size > 0 else -1

    def dev_quantize_mx(self, x, fmt, block_size=None, stream=None):
        """x: float32 device tensor [rows, cols] (or [n]); returns (packed uint8,
        scales int8) device tensors laid out as quantize_mx returns them."""
        code = MX_FORMATS.index(fmt)
        x2 = x if x.dim() == 2 else x.reshape(1, -1)
        rows, cols = x2.shape
        bs = self._mx_block(fmt, block_size)
        nbytes = self.fn["SNEPPX_mx_packed_bytes"](code, rows, cols, bs)
        nsc = self.fn["SNEPPX_mx_scale_count"](code, rows, cols, bs)
        if nbytes == 0 or nsc == 0:
            raise SneppxError(f"dev_quantize_mx: bad block size {block_size}")
        packed = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        scales = torch.empty(nsc, dtype=torch.int8, device=x.device)
        self.check(self.fn["SNEPPX_dev_quantize_mx"](
            _ptr(x2), _ptr(packed), _ptr(scales), rows, cols, code, bs, self._stream(stream)),
            "dev_quantize_mx")
        if nsc > 1 or self.fn["SNEPPX_mx_default_block"](code) > 0 and bs >= 0:
            scales = scales.reshape(rows, -1)
        return packed, scales

    def dev_dequantize_mx(self, packed, scales, shape, fmt, block_size=None, stream=None):
        code = MX_FORMATS.index(fmt)
        rows, cols = (1, shape[0]) if len(shape) == 1 else shape
        y = torch.empty((rows, cols), dtype=torch.float32, device=packed.device)
        self.check(self.fn["SNEPPX_dev_dequantize_mx"](
            _ptr(packed), _ptr(scales), _ptr(y), rows, cols, code, self._mx_block(fmt, block_size),
            self._stream(stream)), "dev_dequantize_mx")
        return y.reshape(shape)

    def qlinear_mxfp4_gemm(self, A, sA, W, sW, out, M, N, K, stream=None):
        ydt = SNEPPX_FLOAT32 if out.dtype == torch.float32 else SNEPPX_BFLOAT16
        self.check(self.fn["SNEPPX_qlinear_mxfp4_gemm"](
            _ptr(A), _ptr(sA), _ptr(W), _ptr(sW), _ptr(out), ydt, M, N, K, self._stream(stream)),
            "qlinear_mxfp4_gemm")

    def qlinear_mx_gemm(self, A, sA, W, sW, fmt, out, M, N, K, stream=None, mfma_form=False):
        """out = A W^T for block-32 MX operands of format `fmt` (FP8 / FP6 / FP4);
        mfma_form: operands already converted by mx_to_mfma."""
        ydt = SNEPPX_FLOAT32 if out.dtype == torch.float32 else SNEPPX_BFLOAT16
        name = "SNEPPX_qlinear_mx_gemm_mfma" if mfma_form else "SNEPPX_qlinear_mx_gemm"
        self.check(self.fn[name](
            _ptr(A), _ptr(sA), _ptr(W), _ptr(sW), MX_FORMATS.index(fmt), _ptr(out), ydt, M, N, K,
            self._stream(stream)), name[7:])

    def qlinear_mx_gemm_bs(self, A, sA, W, sW, fmt, out, M, N, K, block_size=None, stream=None):
        """out = A W^T for MX operands quantized with `block_size` (the rule of
        dev_quantize_mx: None = the format's default, <= 0 per tensor)."""
        ydt = SNEPPX_FLOAT32 if out.dtype == torch.float32 else SNEPPX_BFLOAT16
        self.check(self.fn["SNEPPX_qlinear_mx_gemm_bs"](
            _ptr(A), _ptr(sA), _ptr(W), _ptr(sW), MX_FORMATS.index(fmt), self._mx_block(fmt, block_size),
            _ptr(out), ydt, M, N, K, self._stream(stream)), "qlinear_mx_gemm_bs")

    def mx_to_mfma(self, packed, scales, rows, cols, fmt, stream=None):
        """(packed, scales, rounded) in the matrix cores' encoding; rounded is an
        int32 device counter of the elements that rounded half to even."""
        out_p, out_s = torch.empty_like(packed), torch.empty_like(scales)
        rounded = torch.zeros(1, dtype=torch.int32, device=packed.device)
        self.check(self.fn["SNEPPX_mx_to_mfma"](
            _ptr(packed), _ptr(scales), _ptr(out_p), _ptr(out_s), rows, cols, MX_FORMATS.index(fmt),
            _ptr(rounded), self._stream(stream)), "mx_to_mfma")
        return out_p, out_s, rounded

    # ---------------- paged key-value cache ----------------------------------
    def kv_cache(self, pages, page_size, kv_heads, head_dim, dtype="bf16", weights=False, positions=False,
                 device="cuda"):
        """A KVCache of `pages` pages in new memory ("bf16" or "int8");
        weights / positions: with the planes that eviction goes by."""
        if dtype not in ("bf16", "int8"):
            raise ValueError(f"dtype must be 'bf16' or 'int8', got {dtype!r}")
        shape, planes = (pages, kv_heads, page_size, head_dim), (pages, kv_heads, page_size)
        k, v = (torch.empty(shape, dtype=torch.int8 if dtype == "int8" else torch.bfloat16, device=device)
                for _ in range(2))
        ks, vs = (torch.zeros(planes, device=device) if dtype == "int8" else None for _ in range(2))
        return KVCache(self, k, v, ks, vs, torch.zeros(planes, device=device) if weights else None,
                       torch.zeros(planes, dtype=torch.int32, device=device) if positions else None)

    def kv_cache_from(self, k, v, k_scales=None, v_scales=None, weights=None, positions=None):
        """A KVCache over tensors that the caller has (layouts of include/sneppx_kv.h)."""
        return KVCache(self, k, v, k_scales, v_scales, weights, positions)

    def kv_pages(self, pages, page_size, device="cuda"):
        """KVPages of a pool in which every page is free."""
        return KVPages(self, torch.zeros(pages, dtype=torch.int32, device=device), page_size)

    def kv_pages_from(self, refs, page_size):
        """KVPages over counts that the caller has: int32 [pages]."""
        return KVPages(self, refs, page_size)

    # ---------------- rotary positions ---------------------------------------
    def rotary_frequencies(self, dims, base=10000.0, scaling=None, factor=1.0, original=0.0, low=1.0, high=4.0):
        """SNEPPX_rotary_frequencies: (float64 numpy [dims / 2], magnitude); scaling None,
        "linear", "base", "bands" or "ramp"."""
        if scaling is not None and scaling not in ROTARY_SCALINGS:
            raise ValueError(f"scaling must be None or one of {ROTARY_SCALINGS}, got {scaling!r}")
        _no_count(dims=dims)
        freqs, magnitude = np.zeros(dims // 2, np.float64), C.c_float(0)
        self.check(self.fn["SNEPPX_rotary_frequencies"](
            freqs.ctypes.data_as(_vp), C.byref(magnitude), dims, base,
            0 if scaling is None else 1 + ROTARY_SCALINGS.index(scaling), factor, original, low, high),
            "rotary_frequencies")
        return freqs, magnitude.value

    def rotary(self, head_dim, dims=None, base=10000.0, interleaved=False, q_norm=None, k_norm=None, eps=1e-6,
               device="cuda", **scaling):
        """A Rotary of the frequencies that rotary_frequencies(dims, base, **scaling) gives
        (dims: head_dim unless given)."""
        freqs, magnitude = self.rotary_frequencies(head_dim if dims is None else dims, base, **scaling)
        return Rotary(self, torch.from_numpy(freqs).to(device), head_dim, interleaved, magnitude, q_norm, k_norm, eps)

    def rotary_from(self, freqs, head_dim, interleaved=False, magnitude=1.0, q_norm=None, k_norm=None, eps=1e-6):
        """A Rotary over tensors that the caller has."""
        return Rotary(self, freqs, head_dim, interleaved, magnitude, q_norm, k_norm, eps)

    # ---------------- HIP events on an explicit stream ----------------------
    def event(self):
        e = C.c_void_p()
        self.check(self.fn["snx_hip_event_create"](C.byref(e)), "event_create")
        return e

    def record(self, ev, stream=None):
        self.check(self.fn["snx_hip_event_record"](ev, self._stream(stream)), "event_record")

    def capture(self, fn, stream=None):
        """A HIP graph of everything fn() issues on `stream` (an executable
        graph handle; replay with graph_launch, free with graph_destroy)."""
        st = self._stream(stream)
        self.check(self.fn["snx_hip_stream_begin_capture"](st), "stream_begin_capture")
        try:
            fn()
        finally:
            g = C.c_void_p()
            rc = self.fn["snx_hip_stream_end_capture"](st, C.byref(g))
        self.check(rc, "stream_end_capture")
        return g

    def graph_launch(self, g, stream=None):
        self.check(self.fn["snx_hip_graph_launch"](g, self._stream(stream)), "graph_launch")

    def graph_destroy(self, g):
        self.check(self.fn["snx_hip_graph_destroy"](g), "graph_destroy")

    def elapsed_ms(self, a, b):
        self.check(self.fn["snx_hip_event_sync"](b), "event_sync")
        ms = C.c_float(0)
        self.check(self.fn["snx_hip_event_elapsed_ms"](C.byref(ms), a, b), "event_elapsed")
        return ms.value

    def device_info(self):
        buf = C.create_string_buffer(128)
        cu, clk = C.c_int(0), C.c_int(0)
        self.check(self.fn["snx_hip_device_info"](buf, 128, C.byref(cu), C.byref(clk)), "device_info")
        return buf.value.decode(), cu.value, clk.value


# SNEPPXMXFormat order (include/sneppx_mx.h = MX_FORMATS of mx_formats.py)
MX_FORMATS = ["mxfp8_e4m3", "mxfp8_e5m2", "mxfp6_e3m2", "mxfp6_e2m3", "mxfp4_e2m1", "nvfp4_e2m1"]

# SNEPPXRotaryScaling (include/sneppx_rotary.h), without SNEPPX_ROTARY_PLAIN
ROTARY_SCALINGS = ["linear", "base", "bands", "ramp"]

# dtype codes of include/sneppx_qstore.h (= the reference's SNEPPXSafetensorsDType)
QST_DTYPES = ["F32", "F16", "F64", "I64", "I32", "I16", "I8", "U8", "BOOL", "BF16", "F8_E5M2",
              "F8_E4M3FN"]
QST_NUMPY = {"F32": np.float32, "F16": np.float16, "F64": np.float64, "I64": np.int64,
             "I32": np.int32, "I16": np.int16, "I8": np.int8, "U8": np.uint8, "BOOL": np.bool_,
             "BF16": np.uint16, "F8_E5M2": np.uint8, "F8_E4M3FN": np.uint8}


def _shape_arg(shape):
    return (_sz * max(len(shape), 1))(*shape), len(shape)


class QStore:
    """A safetensors file opened by SNEPPX_qstore_open (read-only mapping)."""

    def __init__(self, lib, handle):
        self.L, self.h = lib, C.c_void_p(handle)

    def close(self):
        if self.h:
            self.L.fn["SNEPPX_qstore_close"](self.h)
            self.h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def names(self):
        n = self.L.fn["SNEPPX_qstore_count"](self.h)
        return [self.L.fn["SNEPPX_qstore_name"](self.h, i).decode() for i in range(n)]

    def info(self, name):
        dt, nd, nb = C.c_int(0), _sz(0), _sz(0)
        shape = (_sz * 8)()
        if self.L.fn["SNEPPX_qstore_info"](self.h, name.encode(), C.byref(dt), shape, C.byref(nd),
                                           C.byref(nb)):
            return None
        return dt.value, tuple(shape[i] for i in range(nd.value)), nb.value

    def host(self, name):
        """Copy of a tensor's bytes as a numpy array of its dtype and shape."""
        inf = self.info(name)
        if inf is None:
            raise KeyError(name)
        dt, shape, nb = inf
        n = _sz(0)
        p = self.L.fn["SNEPPX_qstore_data"](self.h, name.encode(), C.byref(n))
        raw = np.frombuffer(C.string_at(p, n.value), np.uint8) if n.value else np.zeros(0, np.uint8)
        npdt = QST_NUMPY[QST_DTYPES[dt]] if 0 <= dt < len(QST_DTYPES) else np.uint8
        return raw.view(npdt).reshape(shape) if dt >= 0 else raw

    def metadata(self, key):
        v = self.L.fn["SNEPPX_qstore_metadata"](self.h, key.encode())
        return None if v is None else v.decode()

    def read_device(self, name, t, stream=None):
        self.L.check(self.L.fn["SNEPPX_qstore_read_device"](
            self.h, name.encode(), _ptr(t), t.numel() * t.element_size(), self.L._stream(stream)),
            "qstore_read_device")

    def query_w4(self, prefix):
        N, K, G = _sz(0), _sz(0), _sz(0)
        group, hz, hg = C.c_int(0), C.c_int(0), C.c_int(0)
        self.L.check(self.L.fn["SNEPPX_qstore_query_w4"](
            self.h, prefix.encode(), C.byref(N), C.byref(K), C.byref(G), C.byref(group),
            C.byref(hz), C.byref(hg)), "qstore_query_w4")
        return N.value, K.value, G.value, group.value, bool(hz.value), bool(hg.value)

    def load_w4(self, prefix, qweight, scales, qzeros=None, g_idx=None, stream=None):
        self.L.check(self.L.fn["SNEPPX_qstore_load_w4"](
            self.h, prefix.encode(), _ptr(qweight), _ptr(scales), _ptr(qzeros), _ptr(g_idx),
            self.L._stream(stream)), "qstore_load_w4")

    def query_w8(self, prefix):
        N, K = _sz(0), _sz(0)
        self.L.check(self.L.fn["SNEPPX_qstore_query_w8"](self.h, prefix.encode(), C.byref(N), C.byref(K)),
                     "qstore_query_w8")
        return N.value, K.value

    def load_w8(self, prefix, q, scales, stream=None):
        self.L.check(self.L.fn["SNEPPX_qstore_load_w8"](
            self.h, prefix.encode(), _ptr(q), _ptr(scales), self.L._stream(stream)), "qstore_load_w8")


class QStoreWriter:
    """Accumulates tensors and metadata; close() writes the file."""

    def __init__(self, lib, handle):
        self.L, self.h = lib, C.c_void_p(handle)

    def add_host(self, name, dtype, arr):
        arr = np.array(arr, order="C", copy=True)   # keeps 0-d arrays 0-d
        shape, nd = _shape_arg(arr.shape)
        self.L.check(self.L.fn["SNEPPX_qstore_writer_add_host"](
            self.h, name.encode(), QST_DTYPES.index(dtype), shape, nd, arr.ctypes.data_as(_vp)),
            "qstore_writer_add_host")

    def add_device(self, name, dtype, t, stream=None):
        shape, nd = _shape_arg(tuple(t.shape))
        self.L.check(self.L.fn["SNEPPX_qstore_writer_add_device"](
            self.h, name.encode(), QST_DTYPES.index(dtype), shape, nd, _ptr(t), self.L._stream(stream)),
            "qstore_writer_add_device")

    def set_metadata(self, key, value):
        self.L.check(self.L.fn["SNEPPX_qstore_writer_set_metadata"](self.h, key.encode(), value.encode()),
                     "qstore_writer_set_metadata")

    def save_w4(self, prefix, qweight, scales, qzeros, g_idx, N, K, group, G, stream=None):
        self.L.check(self.L.fn["SNEPPX_qstore_save_w4"](
            self.h, prefix.encode(), _ptr(qweight), _ptr(scales), _ptr(qzeros), _ptr(g_idx), N, K,
            group, G, self.L._stream(stream)), "qstore_save_w4")

    def save_w8(self, prefix, q, scales, stream=None):
        N, K = q.shape
        self.L.check(self.L.fn["SNEPPX_qstore_save_w8"](
            self.h, prefix.encode(), _ptr(q), _ptr(scales), N, K, self.L._stream(stream)), "qstore_save_w8")

    def close(self):
        h, self.h = self.h, None
        if h:
            self.L.check(self.L.fn["SNEPPX_qstore_writer_close"](h), "qstore_writer_close")


class _KVCacheStruct(C.Structure):
    """SNEPPXKVCache (include/sneppx_kv.h)."""
    _fields_ = [("k", _vp), ("v", _vp), ("k_scales", _vp), ("v_scales", _vp), ("weights", _vp), ("positions", _vp),
                ("dtype", C.c_int), ("pages", _sz), ("page_size", _sz), ("kv_heads", _sz), ("head_dim", _sz)]


_COUNTS = 1 << 63       # (ctypes passes a size_t on modulo 2^64)


def _no_count(**counts):
    for name, n in counts.items():
        if not 0 <= n < _COUNTS:
            raise ValueError(f"{name} must be a count, got {n!r}")


_BF16, _BF16_OR_F32 = ((torch.bfloat16,), (torch.bfloat16, torch.float32)) if torch else ((), ())


class _OnDevice:
    """What calls on a handle's device share: self.L, self.device, self._index and self.head_dim."""

    _what = "handle"

    # (the library's workspaces and launches are the current device's.  Asked in line, as
    # is torch's current stream by its number: a function around every call takes 0.2 us,
    # current_stream(), which makes an object, 2.8)
    def _elsewhere(self, fn):
        """fn on the handle's device, which is not the current one."""
        if self._index is None:
            raise ValueError(f"the {self._what} is on {self.device}: its calls run on a GPU")

        def run(*args):
            with torch.cuda.device(self._index):
                return fn(*args)
        return run

    # (the checks are on the way of every call: few look-ups of a tensor's attributes,
    # which take 0.1 us each)
    def _check(self, t, name, dtype, shape):
        """The address of a contiguous tensor of this type and shape on the handle's device."""
        try:
            if t.dtype is dtype and t.shape == shape and t.device == self.device and t.is_contiguous():
                return t.data_ptr()
        except AttributeError:
            pass
        got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else repr(t)
        raise ValueError(f"{name} must be a contiguous {dtype} {tuple(shape)} tensor on {self.device}, got {got}")

    def _rows(self, t, name, heads, dtypes):
        """[n, heads, head_dim] whose rows are contiguous: its address, row stride, n and heads."""
        try:
            (n, h, d), (step, s1, s2) = t.shape, t.stride()
            if d == self.head_dim and s2 == 1 and (s1 == d or h == 1) and (h == heads or not heads) \
                    and t.dtype in dtypes and t.device == self.device:
                return t.data_ptr(), step, n, h
        except (AttributeError, TypeError, ValueError):
            pass
        got = f"{t.dtype} {tuple(t.shape)} (strides {t.stride()}) on {t.device}" \
            if isinstance(t, torch.Tensor) else repr(t)
        raise ValueError(f"{name} must be [n, {heads or 'q_heads'}, {self.head_dim}] with contiguous rows, "
                         f"{' or '.join(map(str, dtypes))}, on {self.device}; got {got}")

    def _tables(self, tables, lengths):
        if not isinstance(tables, torch.Tensor) or tables.dim() != 2:
            raise ValueError("tables must be an int32 tensor [rows, width]")
        shape = n, width = tables.shape
        return self._check(tables, "tables", torch.int32, shape), width, \
            self._check(lengths, "lengths", torch.int32, (n,)), n


class KVCache(_OnDevice):
    """A paged key-value pool (include/sneppx_kv.h): k, v [pages, kv_heads,
    page_size, head_dim] in bf16 or int8; k_scales, v_scales (int8), weights
    (fp32) and positions (int32) [pages, kv_heads, page_size].

    Calls take the rows' block tables (int32 [rows, width]) and lengths (int32
    [rows], the call's new tokens included) on the cache's device, and run there
    on torch's current stream of that device unless one is given."""

    _what = "cache"

    def __init__(self, lib, k, v, k_scales=None, v_scales=None, weights=None, positions=None):
        if not isinstance(k, torch.Tensor) or k.dim() != 4 or k.dtype not in (torch.bfloat16, torch.int8):
            raise ValueError("k must be a bf16 or int8 tensor [pages, kv_heads, page_size, head_dim]")
        self.L, self.device, self._index = lib, k.device, k.device.index if k.is_cuda else None
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        i8 = k.dtype == torch.int8
        planes = k.shape[:3]
        for t, name, dtype, shape, needed in (
                (k, "k", k.dtype, k.shape, True), (v, "v", k.dtype, k.shape, True),
                (k_scales, "k_scales", torch.float32, planes, i8), (v_scales, "v_scales", torch.float32, planes, i8),
                (weights, "weights", torch.float32, planes, False),
                (positions, "positions", torch.int32, planes, False)):
            if t is None and not needed:
                continue
            self._check(t, name, dtype, shape)
        if not i8 and (k_scales is not None or v_scales is not None):
            raise ValueError("a bf16 cache has no scales")
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self.weights, self.positions = weights, positions
        self._c = _KVCacheStruct(*(None if t is None else t.data_ptr()
                                   for t in (k, v, k_scales, v_scales, weights, positions)),
                                 SNEPPX_INT8 if i8 else SNEPPX_BFLOAT16, *(k.shape[i] for i in (0, 2, 1, 3)))
        self._p = C.cast(C.pointer(self._c), _vp)
        self._append, self._attention, self._evict = (
            lib.fn[f"SNEPPX_kv_{n}"] for n in ("append", "attention", "evict"))
        self._append_rotated, self._shared, self._bounds, self._pick, self._picked = (
            lib.fn[f"SNEPPX_kv_{n}"] for n in ("append_rotated", "attention_shared", "key_bounds", "pick",
                                               "attention_picked"))

    def append(self, k, v, tables, lengths, next_pos=None, starts=None, k_stored=None, v_stored=None, stream=None):
        """SNEPPX_kv_append: k, v bf16 [tokens, kv_heads, head_dim], slices of
        wider rows among them; starts int32 [rows + 1], without it one token
        per row; k_stored, v_stored bf16 [tokens, kv_heads, head_dim]."""
        kp, ks, tokens, heads = self._rows(k, "k", self.kv_heads, _BF16)
        vp, vs, v_tokens, _ = self._rows(v, "v", self.kv_heads, _BF16)
        tb, width, ln, n = self._tables(tables, lengths)
        if v_tokens != tokens:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ")
        np_ = None if next_pos is None else self._check(next_pos, "next_pos", torch.int32, (n,))
        st = None if starts is None else self._check(starts, "starts", torch.int32, (n + 1,))
        stored = tokens, heads, self.head_dim
        ko = None if k_stored is None else self._check(k_stored, "k_stored", torch.bfloat16, stored)
        vo = None if v_stored is None else self._check(v_stored, "v_stored", torch.bfloat16, stored)
        run = self._append if self._index is not None and torch._C._cuda_getDevice() == self._index \
            else self._elsewhere(self._append)
        rc = run(self._p, kp, ks, vp, vs, tokens, st, ko, vo, tb, width, ln, np_, n,
                 stream if stream is not None else torch._C._cuda_getCurrentRawStream(self._index))
        if rc:
            self.L.check(rc, "kv_append")

    def attention(self, q, out, tables, lengths, max_length, scale=None, accumulate=False, stream=None):
        """SNEPPX_kv_attention: q bf16 [rows, q_heads, head_dim], out the same
        in bf16 or fp32; scale 1 / sqrt(head_dim) unless given."""
        qp, qs, rows, heads = self._rows(q, "q", 0, _BF16)
        op, os_, out_rows, _ = self._rows(out, "out", heads, _BF16_OR_F32)
        tb, width, ln, n = self._tables(tables, lengths)
        if rows != n or out_rows != n:
            raise ValueError(f"q has {rows} rows and out {out_rows}, tables {n}")
        if not 0 <= max_length < _COUNTS:
            _no_count(max_length=max_length)
        run = self._attention if self._index is not None and torch._C._cuda_getDevice() == self._index \
            else self._elsewhere(self._attention)
        rc = run(self._p, qp, qs, op, os_, SNEPPX_BFLOAT16 if out.dtype is torch.bfloat16 else SNEPPX_FLOAT32, tb, width,
                 ln, n, heads, max_length, self.head_dim ** -0.5 if scale is None else scale, int(accumulate),
                 stream if stream is not None else torch._C._cuda_getCurrentRawStream(self._index))
        if rc:
            self.L.check(rc, "kv_attention")

    def evict(self, tables, lengths, next_pos, new_lengths, max_length, budget, recent, stream=None):
        """SNEPPX_kv_evict; new_lengths int32 [rows] or None."""
        tb, width, ln, n = self._tables(tables, lengths)
        np_ = self._check(next_pos, "next_pos", torch.int32, (n,))
        nl = None if new_lengths is None else self._check(new_lengths, "new_lengths", torch.int32, (n,))
        if not 0 <= max_length | budget | recent < _COUNTS:      # (the sign and high bits of any)
            _no_count(max_length=max_length, budget=budget, recent=recent)
        run = self._evict if self._index is not None and torch._C._cuda_getDevice() == self._index \
            else self._elsewhere(self._evict)
        rc = run(self._p, tb, width, ln, np_, nl, n, max_length, budget, recent,
                 stream if stream is not None else torch._C._cuda_getCurrentRawStream(self._index))
        if rc:
            self.L.check(rc, "kv_evict")

    def append_rotated(self, rotary, q, k, v, slots, positions, q_out=None, k_stored=None, v_stored=None, stream=None):
        """SNEPPX_kv_append_rotated: q bf16 [tokens, q_heads, head_dim] turned into q_out
        (without q_out in place), or None; k, v bf16 [tokens, kv_heads, head_dim], slots and
        positions int32 [tokens]."""
        kp, ks, tokens, heads = self._rows(k, "k", self.kv_heads, _BF16)
        vp, vs, v_tokens, _ = self._rows(v, "v", self.kv_heads, _BF16)
        qp = qs = op = os_ = None
        q_heads, q_tokens = 0, tokens
        if q is not None:
            qp, qs, q_tokens, q_heads = self._rows(q, "q", 0, _BF16)
            op, os_ = qp, qs
            if q_out is not None:
                op, os_, o_tokens, _ = self._rows(q_out, "q_out", q_heads, _BF16)
                if o_tokens != tokens:
                    raise ValueError(f"q_out has {o_tokens} tokens, k {tokens}")
        if v_tokens != tokens or q_tokens != tokens:
            raise ValueError(f"k has {tokens} tokens, v {v_tokens}, q {q_tokens}")
        if not isinstance(rotary, Rotary) or rotary.device != self.device or rotary.head_dim != self.head_dim:
            raise ValueError(f"rotary must be a Rotary of heads of {self.head_dim} on {self.device}, got {rotary!r}")
        shape = (tokens,)
        sl, ps = self._check(slots, "slots", torch.int32, shape), self._check(positions, "positions", torch.int32, shape)
        stored = tokens, heads, self.head_dim
        ko = None if k_stored is None else self._check(k_stored, "k_stored", torch.bfloat16, stored)
        vo = None if v_stored is None else self._check(v_stored, "v_stored", torch.bfloat16, stored)
        run = self._append_rotated if self._index is not None and torch._C._cuda_getDevice() == self._index \
            else self._elsewhere(self._append_rotated)
        rc = run(self._p, rotary._p, qp, qs or 0, op, os_ or 0, q_heads, kp, ks, vp, vs, tokens, sl, ps, ko, vo,
                 stream if stream is not None else torch._C._cuda_getCurrentRawStream(self._index))
        if rc:
            self.L.check(rc, "kv_append_rotated")

    def attention_shared(self, q, out, tables, lengths, max_length, groups, prefix, max_prefix, max_own, scale=None,
                         stream=None):
        """SNEPPX_kv_attention_shared: groups int32 [n + 1] (first rows), prefix int32 [n]
        (tokens that a group's rows have in common); the others as in attention."""
        qp, qs, rows, heads = self._rows(q, "q", 0, _BF16)
        op, os_, out_rows, _ = self._rows(out, "out", heads, _BF16_OR_F32)
        tb, width, ln, n = self._tables(tables, lengths)
        if rows != n or out_rows != n:
            raise ValueError(f"q has {rows} rows and out {out_rows}, tables {n}")
        if not isinstance(prefix, torch.Tensor) or prefix.dim() != 1:
            raise ValueError("prefix must be an int32 tensor [groups]")
        many = prefix.shape[0]
        pf, gr = self._check(prefix, "prefix", torch.int32, (many,)), self._check(groups, "groups", torch.int32, (many + 1,))
        if not 0 <= max_length | max_prefix | max_own < _COUNTS:
            _no_count(max_length=max_length, max_prefix=max_prefix, max_own=max_own)
        run = self._shared if self._index is not None and torch._C._cuda_getDevice() == self._index \
            else self._elsewhere(self._shared)
        rc = run(self._p, qp, qs, op, os_, SNEPPX_BFLOAT16 if out.dtype is torch.bfloat16 else SNEPPX_FLOAT32, tb, width,
                 ln, n, heads, max_length, gr, pf, many, max_prefix, max_own,
                 self.head_dim ** -0.5 if scale is None else scale,
                 stream if stream is not None else torch._C._cuda_getCurrentRawStream(self._index))
        if rc:
            self.L.check(rc, "kv_attention_shared")

    def key_bounds(self, bounds, tables, lengths, counts=None, max_count=1, stream=None):
        """SNEPPX_kv_key_bounds: bounds bf16 [pages, kv_heads, 2, head_dim]; the pages of
        the last counts tokens (int32 [rows], none larger than max_count), or of one."""
        tb, width, ln, n = self._tables(tables, lengths)
        bp = self._check(bounds, "bounds", torch.bfloat16, (self.pages, self.kv_heads, 2, self.head_dim))
        ct = None if counts is None else self._check(counts, "counts", torch.int32, (n,))
        if not 0 <= max_count < _COUNTS:
            _no_count(max_count=max_count)
        run = self._bounds if self._index is not None and torch._C._cuda_getDevice() == self._index \
            else self._elsewhere(self._bounds)
        rc = run(self._p, bp, tb, width, ln, ct, max_count, n,
                 stream if stream is not None else torch._C._cuda_getCurrentRawStream(self._index))
        if rc:
            self.L.check(rc, "kv_key_bounds")

    def _picks(self, picked, lengths, name):
        """The addresses of page lists [rows, kv_heads, budget] and of their lengths, rows and budget."""
        if not isinstance(picked, torch.Tensor) or picked.dim() != 3:
            raise ValueError("picked must be an int32 tensor [rows, kv_heads, budget]")
        n, _, budget = picked.shape
        return self._check(picked, "picked", torch.int32, (n, self.kv_heads, budget)), \
            self._check(lengths, name, torch.int32, (n,)), n, budget

    def pick(self, q, bounds, tables, lengths, max_length, picked, picked_lengths, first=1, recent=1, stream=None):
        """SNEPPX_kv_pick: picked int32 [rows, kv_heads, budget], picked_lengths int32
        [rows]; the first `first` and last `recent` pages are always among them."""
        qp, qs, rows, heads = self._rows(q, "q", 0, _BF16)
        tb, width, ln, n = self._tables(tables, lengths)
        bp = self._check(bounds, "bounds", torch.bfloat16, (self.pages, self.kv_heads, 2, self.head_dim))
        pk, pl, pn, budget = self._picks(picked, picked_lengths, "picked_lengths")
        if rows != n or pn != n:
            raise ValueError(f"q has {rows} rows and picked {pn}, tables {n}")
        if not 0 <= max_length | first | recent < _COUNTS:
            _no_count(max_length=max_length, first=first, recent=recent)
        run = self._pick if self._index is not None and torch._C._cuda_getDevice() == self._index \
            else self._elsewhere(self._pick)
        rc = run(self._p, bp, qp, qs, heads, tb, width, ln, n, max_length, budget, first, recent, pk, pl,
                 stream if stream is not None else torch._C._cuda_getCurrentRawStream(self._index))
        if rc:
            self.L.check(rc, "kv_pick")

    def attention_picked(self, q, out, picked, picked_lengths, scale=None, accumulate=False, stream=None):
        """SNEPPX_kv_attention_picked: attention over the pages that pick has left."""
        qp, qs, rows, heads = self._rows(q, "q", 0, _BF16)
        op, os_, out_rows, _ = self._rows(out, "out", heads, _BF16_OR_F32)
        pk, pl, n, budget = self._picks(picked, picked_lengths, "picked_lengths")
        if rows != n or out_rows != n:
            raise ValueError(f"q has {rows} rows and out {out_rows}, picked {n}")
        run = self._picked if self._index is not None and torch._C._cuda_getDevice() == self._index \
            else self._elsewhere(self._picked)
        rc = run(self._p, qp, qs, op, os_, SNEPPX_BFLOAT16 if out.dtype is torch.bfloat16 else SNEPPX_FLOAT32, pk, budget,
                 pl, n, heads, self.head_dim ** -0.5 if scale is None else scale, int(accumulate),
                 stream if stream is not None else torch._C._cuda_getCurrentRawStream(self._index))
        if rc:
            self.L.check(rc, "kv_attention_picked")


class KVPages(_OnDevice):
    """Which pages of a pool are in use (include/sneppx_kv.h): refs int32 [pages], the
    number of rows that hold each.  Calls change refs, the rows' tables (int32 [rows,
    width], -1 where there is no page) and lengths (int32 [rows]) on the device, on
    torch's current stream unless one is given."""

    _what = "page counts"

    def __init__(self, lib, refs, page_size):
        if not isinstance(refs, torch.Tensor) or refs.dim() != 1 or refs.dtype != torch.int32 or not refs.is_contiguous():
            raise ValueError("refs must be a contiguous int32 tensor [pages]")
        _no_count(page_size=page_size)
        self.L, self.device, self._index = lib, refs.device, refs.device.index if refs.is_cuda else None
        self.refs, self.pages, self.page_size = refs, refs.shape[0], page_size
        self._p = refs.data_ptr()
        self._reserve, self._release, self._share = (lib.fn[f"SNEPPX_kv_{n}"] for n in ("reserve", "release", "share"))

    # (memory of torch's current stream may still be in use there)
    def _new(self, n, stream):
        """int32 [n] of the memory of the stream that a call writes it on."""
        if stream is None or self._index is None or stream == torch._C._cuda_getCurrentRawStream(self._index):
            return torch.empty(n, dtype=torch.int32, device=self.device)
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=self.device)):
            return torch.empty(n, dtype=torch.int32, device=self.device)

    def reserve(self, tables, lengths, slots, counts=None, next_pos=None, positions=None, starts=None, granted=None,
                stream=None):
        """SNEPPX_kv_reserve: slots (and positions) int32 [tokens]; counts, next_pos,
        granted int32 [rows], starts int32 [rows + 1].  Returns (starts, granted), new ones of
        the stream's memory where none are given."""
        tb, width, ln, n = self._tables(tables, lengths)
        if not isinstance(slots, torch.Tensor) or slots.dim() != 1:
            raise ValueError("slots must be an int32 tensor [tokens]")
        tokens, rows, int32, check = slots.shape, (n,), torch.int32, self._check
        if starts is None:
            starts = self._new(n + 1, stream)
        if granted is None:
            granted = self._new(n, stream)
        st, gr = check(starts, "starts", int32, (n + 1,)), check(granted, "granted", int32, rows)
        sl, ps = check(slots, "slots", int32, tokens), None if positions is None else check(positions, "positions", int32, tokens)
        np_ = None if next_pos is None else check(next_pos, "next_pos", int32, rows)
        ct = None if counts is None else check(counts, "counts", int32, rows)
        run = self._reserve if self._index is not None and torch._C._cuda_getDevice() == self._index \
            else self._elsewhere(self._reserve)
        rc = run(self._p, self.pages, self.page_size, tb, width, ln, np_, ct, n, st, gr, sl, ps, tokens[0],
                 stream if stream is not None else torch._C._cuda_getCurrentRawStream(self._index))
        if rc:
            self.L.check(rc, "kv_reserve")
        return starts, granted

    def release(self, tables, lengths, stream=None):
        """SNEPPX_kv_release: the pages behind the rows' lengths go back."""
        tb, width, ln, n = self._tables(tables, lengths)
        run = self._release if self._index is not None and torch._C._cuda_getDevice() == self._index \
            else self._elsewhere(self._release)
        rc = run(self._p, self.pages, self.page_size, tb, width, ln, n,
                 stream if stream is not None else torch._C._cuda_getCurrentRawStream(self._index))
        if rc:
            self.L.check(rc, "kv_release")

    def share(self, tables, lengths, sources, counts, next_pos=None, stream=None):
        """SNEPPX_kv_share: sources int32 [rows] (a row, or -1), counts int32 [rows]
        (tokens, of which whole pages are taken)."""
        tb, width, ln, n = self._tables(tables, lengths)
        sr, ct = self._check(sources, "sources", torch.int32, (n,)), self._check(counts, "counts", torch.int32, (n,))
        np_ = None if next_pos is None else self._check(next_pos, "next_pos", torch.int32, (n,))
        run = self._share if self._index is not None and torch._C._cuda_getDevice() == self._index \
            else self._elsewhere(self._share)
        rc = run(self._p, self.pages, self.page_size, tb, width, ln, np_, sr, ct, n,
                 stream if stream is not None else torch._C._cuda_getCurrentRawStream(self._index))
        if rc:
            self.L.check(rc, "kv_share")


class _RotaryStruct(C.Structure):
    """SNEPPXRotary (include/sneppx_rotary.h)."""
    _fields_ = [("freqs", _vp), ("dims", _sz), ("interleaved", C.c_int), ("magnitude", C.c_float), ("q_norm", _vp),
                ("k_norm", _vp), ("eps", C.c_float)]


class Rotary(_OnDevice):
    """The rotation of heads of head_dim to their positions (include/sneppx_rotary.h):
    freqs float64 [pairs], the first 2 * pairs elements of a head turn; q_norm and
    k_norm float32 [head_dim] (or None) normalise heads first."""

    _what = "rotary"

    def __init__(self, lib, freqs, head_dim, interleaved=False, magnitude=1.0, q_norm=None, k_norm=None, eps=1e-6):
        if not isinstance(freqs, torch.Tensor) or freqs.dim() != 1 or freqs.dtype != torch.float64:
            raise ValueError("freqs must be a float64 tensor [pairs]")
        self.L, self.device, self._index = lib, freqs.device, freqs.device.index if freqs.is_cuda else None
        self.head_dim, self.freqs, self.q_norm, self.k_norm = head_dim, freqs, q_norm, k_norm
        qn, kn = (None if t is None else self._check(t, name, torch.float32, (head_dim,))
                  for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")))
        self._c = _RotaryStruct(self._check(freqs, "freqs", torch.float64, freqs.shape), 2 * freqs.shape[0],
                                int(interleaved), magnitude, qn, kn, eps)
        self._p = C.cast(C.pointer(self._c), _vp)
        self._apply = lib.fn["SNEPPX_rotary_apply"]

    def apply(self, q, k, positions, q_out=None, k_out=None, stream=None):
        """SNEPPX_rotary_apply: q, k bf16 [tokens, heads, head_dim], slices of wider rows
        among them, or None; in place where no output is given.  positions int32 [tokens]."""
        if not isinstance(positions, torch.Tensor) or positions.dim() != 1:
            raise ValueError("positions must be an int32 tensor [tokens]")
        shape = tokens, = positions.shape
        ps = self._check(positions, "positions", torch.int32, shape)
        qp = qs = qo = qos = kp = ks = ko = kos = None
        qh = kh = 0
        qn = qon = kn = kon = tokens
        if q is not None:
            qp, qs, qn, qh = self._rows(q, "q", 0, _BF16)
            qo, qos, qon, _ = (qp, qs, qn, qh) if q_out is None else self._rows(q_out, "q_out", qh, _BF16)
        if k is not None:
            kp, ks, kn, kh = self._rows(k, "k", 0, _BF16)
            ko, kos, kon, _ = (kp, ks, kn, kh) if k_out is None else self._rows(k_out, "k_out", kh, _BF16)
        if not qn == qon == kn == kon == tokens:
            raise ValueError(f"q has {qn} tokens and its output {qon}, k has {kn} tokens and its output {kon}, "
                             f"positions {tokens}")
        run = self._apply if self._index is not None and torch._C._cuda_getDevice() == self._index \
            else self._elsewhere(self._apply)
        rc = run(self._p, qp, qs or 0, qo, qos or 0, qh, kp, ks or 0, ko, kos or 0, kh, self.head_dim, ps, tokens,
                 stream if stream is not None else torch._C._cuda_getCurrentRawStream(self._index))
        if rc:
            self.L.check(rc, "rotary_apply")


class QLayer:
    """SNEPPXQLayer: y = x . W for a reference-layout weight W [K, N]."""

    def __init__(self, lib, handle):
        self.L, self.h = lib, C.c_void_p(handle)
        self.K = lib.fn["SNEPPX_qlayer_in_features"](self.h)
        self.N = lib.fn["SNEPPX_qlayer_out_features"](self.h)
        self.format = ["w8", "w4"][lib.fn["SNEPPX_qlayer_format"](self.h)]

    def destroy(self):
        if self.h:
            self.L.fn["SNEPPX_qlayer_destroy"](self.h)
            self.h = None

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass

    def forward_f32(self, x, y, stream=None):
        M = x.shape[0]
        self.L.check(self.L.fn["SNEPPX_qlayer_forward_f32"](self.h, _ptr(x), _ptr(y), M,
                                                            self.L._stream(stream)), "qlayer_forward_f32")

    def forward_bf16(self, x, y, stream=None):
        M = x.shape[0]
        self.L.check(self.L.fn["SNEPPX_qlayer_forward_bf16"](self.h, _ptr(x), _ptr(y), M,
                                                             self.L._stream(stream)), "qlayer_forward_bf16")

    def set_bias(self, bias, stream=None):
        """bias: numpy fp32 [N] (host), a torch fp32 [N] device tensor, or None."""
        if bias is None:
            rc = self.L.fn["SNEPPX_qlayer_set_bias_device"](self.h, None, self.L._stream(stream))
        elif isinstance(bias, np.ndarray):
            rc = self.L.fn["SNEPPX_qlayer_set_bias"](self.h, np.ascontiguousarray(bias, np.float32),
                                                      self.L._stream(stream))
        else:
            n = self.L.fn["SNEPPX_qlayer_out_features"](self.h)
            rc = self.L.fn["SNEPPX_qlayer_set_bias_device"](self.h, _bias_ptr(bias, n, bias),
                                                             self.L._stream(stream))
        self.L.check(rc, "qlayer_set_bias")

    def matmul_host(self, x):
        x = np.ascontiguousarray(x, np.float32)
        M = x.shape[0]
        y = np.zeros((M, self.N), np.float32)
        self.L.check(self.L.fn["SNEPPX_qlayer_matmul_host"](self.h, x, y, M), "qlayer_matmul_host")
        return y

    def save(self, writer, prefix, stream=None):
        self.L.check(self.L.fn["SNEPPX_qlayer_save"](self.h, writer.h, prefix.encode(),
                                                     self.L._stream(stream)), "qlayer_save")


_LIB = None


def load() -> Library:
    global _LIB
    if _LIB is None:
        _LIB = Library()
    return _LIB
