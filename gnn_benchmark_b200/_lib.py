"""ctypes binding of libgnnagg.so, the C-ABI CUDA library (declared in include/gnnagg.h).

The library is the only compute path of this package: if it is missing, or a call returns a
non-zero status, a RuntimeError is raised.  There is no CPU or PyTorch fallback.
"""
import ctypes
import os

import torch

_PKG_DIR = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG_DIR, "libgnnagg.so")

OPS_PATH = os.path.join(_PKG_DIR, "_torch_ops.so")

_lib = None
_ops = None

_vp = ctypes.c_void_p
_i64 = ctypes.c_int64
_i32 = ctypes.c_int32
_sz = ctypes.c_size_t

# name -> (restype, argtypes); mirrors include/gnnagg.h one to one
SIGNATURES = {
    "gnnagg_version": (ctypes.c_int, []),
    "gnnagg_error_string": (ctypes.c_char_p, [ctypes.c_int]),
    "gnnagg_spmm_plan_bytes": (_sz, [_i64, _i64]),
    "gnnagg_spmm_plan_build": (ctypes.c_int, [_vp, _i64, _i64, _vp, _sz, _vp]),
    "gnnagg_spmm_scratch_bytes": (_sz, [_i64, _i64, _i32]),
    "gnnagg_spmm_csr_f32": (ctypes.c_int, [_vp, _vp, _vp, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _i32, _i32, _vp,
                                           _vp, _sz, _vp]),
    "gnnagg_spmm_csr_q": (ctypes.c_int, [_vp, _vp, _vp, _i64, _i64, _i64, _vp, _vp, _vp, _i32, _i32, _vp, _i64, _i32, _i32,
                                         _vp, _vp, _sz, _vp]),
    "gnnagg_spmm_csr_f32_static_scratch": (ctypes.c_int, [_vp, _vp, _vp, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _i32,
                                                          _i32, _vp, _vp]),
    "gnnagg_csr_to_csc_workspace_bytes": (_sz, [_i64, _i64, _i64]),
    "gnnagg_csr_to_csc": (ctypes.c_int, [_vp, _vp, _vp, _i64, _i64, _i64, _vp, _vp, _vp, _vp, _sz, _vp]),
    "gnnagg_csr_validate": (ctypes.c_int, [_vp, _vp, _i64, _i64, _i64, _vp, _vp]),
    "gnnagg_gather_rows_f32": (ctypes.c_int, [_vp, _i64, _vp, _i64, _i32, _vp, _i64, _vp]),
    "gnnagg_push_block": (ctypes.c_int, [_vp, _vp, _sz, _vp]),
    "gnnagg_push_rows": (ctypes.c_int, [_vp, _i64, _vp, _i32, _vp, _i32, _i32, _i32, _vp, _i64, _i64, _vp]),
    "gnnagg_scale_rows_f32": (ctypes.c_int, [_vp, _i64, _vp, _i64, _i32, _i32, _vp, _vp, _i64, _vp]),
    "gnnagg_quant_pack_rows": (ctypes.c_int, [_vp, _i64, _vp, _i32, _vp, _i32, _i64, _i32, _i32, _vp, _vp, _vp, _vp]),
    "gnnagg_spmm_quant_pack_scratch_bytes": (_sz, [_i64, _i64, _i32]),
    "gnnagg_spmm_quant_pack": (ctypes.c_int, [_vp, _vp, _vp, _i64, _i64, _i64, _vp, _i64, _i32, _vp, _i32, _i32, _vp, _vp, _vp,
                                              _vp, _vp, _sz, _vp]),
    "gnnagg_unpack_dequant_rows": (ctypes.c_int, [_vp, _i32, _vp, _i32, _i64, _i32, _vp, _vp, _vp, _i64, _vp]),
    "gnnagg_quant_v1_rows": (ctypes.c_int, [_vp, _i64, _i64, _i32, _vp, _vp, _vp, _vp]),
    "gnnagg_dequant_v1_rows": (ctypes.c_int, [_vp, _i64, _i32, _vp, _vp, _vp, _i64, _vp]),
    "gnnagg_cast_f32_to_bf16": (ctypes.c_int, [_vp, _vp, _i64, _vp]),
    "gnnagg_cast_bf16_to_f32": (ctypes.c_int, [_vp, _vp, _i64, _vp]),
    "gnnagg_dense_workspace_bytes": (_sz, [_i32, _i32]),
    "gnnagg_dense_tf32x3_f32": (ctypes.c_int, [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i32, _i32, _vp, _i32, _vp, _sz,
                                               _vp]),
    "gnnagg_dense_status": (ctypes.c_int, [_vp, _vp]),
    "gnnagg_dense_status_clear": (ctypes.c_int, [_vp, _vp]),
    "gnnagg_dense_stall_test": (ctypes.c_int, [_i32, _i64]),
    "gnnagg_dense_wgrad_workspace_bytes": (_sz, [_i32, _i32]),
    "gnnagg_dense_wgrad_tf32x3_f32": (ctypes.c_int, [_vp, _i64, _vp, _i64, _i64, _i32, _i32, _vp, _i64, _vp, _sz, _vp]),
    "gnnagg_dropout_ln_relu_partial_bytes": (_sz, [_i32]),
    "gnnagg_dropout_ln_relu_fwd": (ctypes.c_int, [_vp, _i64, _i64, _i32, _vp, _vp, ctypes.c_float, ctypes.c_float,
                                                  ctypes.c_uint64, _vp, _i64, _vp, _vp, _vp]),
    "gnnagg_relu_dropout_fwd": (ctypes.c_int, [_vp, _i64, _i64, _i32, ctypes.c_float, ctypes.c_uint64, _vp, _i64, _vp, _vp]),
    "gnnagg_relu_dropout_bwd": (ctypes.c_int, [_vp, _i64, _vp, _i64, _i32, ctypes.c_float, _vp, _i64, _vp]),
    "gnnagg_dropout_ln_relu_bwd": (ctypes.c_int, [_vp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _i64, _i32, ctypes.c_float,
                                                  _vp, _i64, _vp, _sz, _vp, _vp, _vp]),
    "gnnagg_rms_norm_fwd": (ctypes.c_int, [_vp, _i64, _vp, _i64, _vp, _i32, _i64, _i32, _i32, ctypes.c_float, _vp, _i64,
                                           _vp, _i64, _vp, _vp]),
    "gnnagg_rms_norm_fp8": (ctypes.c_int, [_vp, _i64, _vp, _i64, _vp, _i32, _i64, _i32, _i32, ctypes.c_float, _vp, _i64,
                                           _vp, _i64, _vp, _i64, _vp]),
    "gnnagg_rms_norm_partial_bytes": (_sz, [_i64, _i32, _i32]),
    "gnnagg_rms_norm_bwd": (ctypes.c_int, [_vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i32, _i64, _i32, _i32, _vp, _i64,
                                           _vp, _vp, _sz, _vp]),
    "gnnagg_fp8_quantize": (ctypes.c_int, [_vp, _i64, _i64, _i64, _i32, _i32, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64,
                                           _vp, _vp]),
    "gnnagg_fp8_matmul_workspace_bytes": (_sz, [_i64, _i64, _i64]),
    "gnnagg_fp8_matmul": (ctypes.c_int, [_vp, _i64, _vp, _i64, _i64, _i32, _vp, _i64, _vp, _i64, _i64, _i32, _i64, _i64,
                                         _i64, _vp, _i32, _i32, _vp, _i64, _i32, _vp, _sz, _vp]),
    "gnnagg_fp8_linear_kept_bytes": (_sz, [_i64, _i64, _i64, _i32, _i32]),
    "gnnagg_fp8_linear_scratch_bytes": (_sz, [_i64, _i64, _i64, _i32]),
    "gnnagg_fp8_linear_fwd": (ctypes.c_int, [_vp, _i64, _i32, _vp, _i64, _i32, _vp, _i32, _i64, _i64, _i64, _vp, _i32, _i32,
                                             _i32, _vp, _sz, _vp, _sz, _vp]),
    "gnnagg_fp8_linear_bwd": (ctypes.c_int, [_vp, _i64, _i32, _i64, _i64, _i64, _i32, _i32, _vp, _sz, _vp, _i32, _vp, _i32,
                                             _vp, _i32, _vp, _sz, _vp]),
    "gnnagg_fp8_matmul_status": (ctypes.c_int, [_vp]),
    "gnnagg_fp8_matmul_status_clear": (ctypes.c_int, [_vp]),
    "gnnagg_adamw_scalars_bytes": (_sz, []),
    "gnnagg_adamw_tick": (ctypes.c_int, [_vp, _vp] + [ctypes.c_double] * 5 + [_vp, _vp]),
    "gnnagg_adamw_step": (ctypes.c_int, [_vp, _i64, _i32, _i32] + [ctypes.c_double] * 5 + [_i64, _vp, _vp]),
}


def lib():
    """The loaded library.  Raises if libgnnagg.so has not been built
    (`python -m gnn_benchmark_b200.build`)."""
    global _lib
    if _lib is None:
        if not os.path.isfile(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -m gnn_benchmark_b200.build` "
                "(nvcc, sm_100a).  This package has no CPU fallback."
            )
        handle = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def ops():
    """The torch front end of the low-precision operators (csrc/torch/ops.cpp): the same C ABI, with argument checks,
    allocation and autograd nodes in C++.  Raises if _torch_ops.so has not been built."""
    global _ops
    if _ops is None:
        import importlib.util

        lib()
        if not os.path.isfile(OPS_PATH):
            raise RuntimeError(f"{OPS_PATH} is missing: build it with `python -m gnn_benchmark_b200.build`")
        spec = importlib.util.spec_from_file_location("_torch_ops", OPS_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        _ops = module
    return _ops


def check(rc: int, what: str) -> None:
    if rc != 0:
        msg = lib().gnnagg_error_string(rc).decode()
        raise RuntimeError(f"libgnnagg {what} failed (status {rc}): {msg}")


def stream_ptr(device=None) -> int:
    """cudaStream_t of torch's current stream on `device` (without building torch's Stream object: 2 us a call)."""
    index = None if device is None else torch.device(device).index
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None else index)


def ptr(t) -> int:
    """Device address of a tensor, 0 for None."""
    return 0 if t is None else t.data_ptr()


class device_of:
    """Makes a tensor's device current for a launch (kernels go to the current device) and puts the caller's
    back; free where it is current already."""

    __slots__ = ("index", "before")

    def __init__(self, t):
        self.index = t.device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def require_cuda(*tensors) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("libgnnagg kernels take CUDA tensors only (this package has no CPU fallback)")
