"""ctypes binding of libgk.so, the C ABI declared in include/gk.h.

This replaces the reference's NVRTC/driver-API launcher
(python/kingdom_ai/gpu_runtime.py:179-221, ``CudaModule.launch``): every
kernel launch goes through one exported C function that takes raw device
pointers, sizes and the current PyTorch stream. There is no fallback: if the
library is missing or a call fails, an exception is raised.
"""

from __future__ import annotations

import contextlib
import ctypes
import threading
from pathlib import Path

import torch

LIBRARY_PATH = Path(__file__).resolve().parent / "libgk.so"

c_void_p = ctypes.c_void_p
c_int = ctypes.c_int
c_int64 = ctypes.c_int64
c_uint64 = ctypes.c_uint64
c_double = ctypes.c_double
c_float = ctypes.c_float
c_size_t = ctypes.c_size_t


TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # GK_FP32, GK_BF16, GK_FP16


class PuctOptions(ctypes.Structure):
    _fields_ = [("c_puct", c_double), ("dirichlet_epsilon", c_double), ("fpu_enabled", c_int),
                ("fpu_reduction", c_double)]


class PuctBuffers(ctypes.Structure):
    _fields_ = [("needs_eval", c_void_p), ("leaf_bits", c_void_p), ("leaf_value", c_void_p),
                ("policy", c_void_p), ("noise", c_void_p), ("active", c_void_p), ("active_count", c_void_p),
                ("errors", c_void_p), ("leaf", c_void_p), ("root_allow", c_void_p), ("node_visits", c_void_p)]


class PuctResults(ctypes.Structure):
    _fields_ = [("actions", c_void_p), ("visits", c_void_p), ("policy", c_void_p), ("values", c_void_p),
                ("simulations", c_void_p), ("network_evaluations", c_void_p), ("priors", c_void_p),
                ("best_values", c_void_p), ("nodes", c_void_p), ("root_values", c_void_p),
                ("status", c_void_p)]


class NetStruct(ctypes.Structure):
    _fields_ = [("channels", c_int), ("blocks", c_int), ("conv_w", c_void_p), ("conv_b", c_void_p),
                ("head_w", c_void_p), ("head_b", c_void_p), ("pol_w", c_void_p), ("pol_b", c_void_p),
                ("val_w1", c_void_p), ("val_b1", c_void_p), ("val_w2", c_void_p), ("val_b2", c_void_p),
                ("norm", c_int), ("norm_w", c_void_p), ("norm_b", c_void_p), ("head_norm", c_void_p)]


class PolicyLossStruct(ctypes.Structure):
    _fields_ = [("logits", c_void_p), ("mask", c_void_p), ("target", c_void_p), ("actions", c_void_p),
                ("old_log_probs", c_void_p), ("advantages", c_void_p), ("reference_log_probs", c_void_p),
                ("denominator_ptr", c_void_p), ("rows", c_int64), ("cols", c_int64), ("logits_stride", c_int64),
                ("mask_stride", c_int64), ("target_stride", c_int64), ("clip_low", c_float), ("clip_high", c_float),
                ("kl_weight", c_float), ("target_weight", c_float), ("denominator", c_float), ("logits_type", c_int),
                ("target_type", c_int), ("loss", c_void_p), ("log_probs", c_void_p), ("stats", c_void_p),
                ("partials", c_void_p), ("grad", c_void_p)]


class LinearStruct(ctypes.Structure):
    _fields_ = [("x", c_void_p), ("w", c_void_p), ("bias", c_void_p), ("residual", c_void_p), ("y", c_void_p),
                ("pre", c_void_p), ("m", c_int64), ("n", c_int64), ("k", c_int64), ("x_stride", c_int64),
                ("w_stride", c_int64), ("residual_stride", c_int64), ("dtype", c_int), ("activation", c_int)]


class LinearGradStruct(ctypes.Structure):
    _fields_ = [("dy", c_void_p), ("kept", c_void_p), ("x", c_void_p), ("x_codes", c_void_p), ("x_scales", c_void_p),
                ("w", c_void_p), ("dx", c_void_p), ("dw", c_void_p), ("db", c_void_p), ("dz", c_void_p),
                ("m", c_int64), ("n", c_int64), ("k", c_int64), ("dy_stride", c_int64), ("x_stride", c_int64),
                ("w_stride", c_int64), ("dtype", c_int), ("activation", c_int)]


_SIGNATURES = {
    "gk_linear_forward": [ctypes.POINTER(LinearStruct), c_void_p, c_void_p, c_void_p],
    "gk_linear_backward": [ctypes.POINTER(LinearGradStruct), c_void_p, c_void_p, c_void_p],
    "gk_pack": [c_void_p, c_int64, c_int, c_int64, c_int64, c_void_p, c_void_p, c_void_p],
    "gk_unpack": [c_void_p, c_void_p, c_int64, c_int64, c_void_p, c_int64, c_int, c_void_p],
    "gk_policy_loss_parts": [c_int64, c_int64],
    "gk_policy_loss_forward": [ctypes.POINTER(PolicyLossStruct), c_void_p],
    "gk_policy_loss_backward": [ctypes.POINTER(PolicyLossStruct), c_void_p, c_int, c_void_p],
    "gk_initial_records": [c_void_p, c_int64, c_int, c_void_p],
    "gk_initial_bits": [c_void_p, c_int64, c_int, c_void_p],
    "gk_play_records": [c_void_p, c_void_p, c_int, c_void_p, c_int64, c_void_p],
    "gk_encode_records": [c_void_p, c_void_p, c_void_p, c_int64, c_void_p],
    "gk_records_to_bits": [c_void_p, c_void_p, c_void_p, c_int64, c_void_p],
    "gk_bits_to_records": [c_void_p, c_void_p, c_int64, c_void_p],
    "gk_play_bits": [c_void_p, c_void_p, c_int, c_void_p, c_int64, c_void_p],
    "gk_encode_bits": [c_void_p, c_void_p, c_void_p, c_int64, c_void_p],
    "gk_random_playouts": [c_uint64, c_uint64, c_int64, c_int, c_void_p, c_void_p, c_void_p],
    "gk_gen_positions": [c_uint64, c_uint64, c_int64, c_void_p, c_void_p],
    "gk_puct_buffers": [c_void_p, c_int64, c_int, ctypes.POINTER(PuctBuffers)],
    "gk_puct_begin": [c_void_p, c_int64, c_int, c_void_p, c_void_p],
    "gk_puct_root_tactics": [c_void_p, c_int64, c_int, c_void_p],
    "gk_replay_validate": [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_void_p, c_void_p],
    "gk_puct_noise": [c_void_p, c_int64, c_int, c_uint64, c_uint64, c_double, c_void_p],
    "gk_puct_select": [c_void_p, c_int64, c_int, ctypes.POINTER(PuctOptions), c_void_p],
    "gk_puct_hash_eval": [c_void_p, c_int64, c_int, c_void_p],
    "gk_puct_compact": [c_void_p, c_int64, c_int, c_void_p],
    "gk_puct_expand_backup": [c_void_p, c_int64, c_int, ctypes.POINTER(PuctOptions), c_int, c_void_p],
    "gk_puct_finish": [c_void_p, c_int64, c_int, ctypes.POINTER(PuctResults), c_void_p],
    "gk_puct_search_hash": [c_void_p, c_int64, c_int, c_void_p, ctypes.POINTER(PuctOptions),
                            ctypes.POINTER(PuctResults), c_void_p],
    "gk_mma_selftest": [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p],
    "gk_net_forward": [ctypes.POINTER(NetStruct), c_void_p, c_void_p, c_int64, c_void_p, c_void_p, c_void_p,
                       c_void_p, c_void_p],
    "gk_net_evaluate_puct": [ctypes.POINTER(NetStruct), c_void_p, c_int64, c_int, c_void_p, c_void_p, c_void_p],
}
_SIZE_FUNCTIONS = {
    "gk_puct_workspace_bytes": [c_int64, c_int],
    "gk_net_weight_bytes": [c_int, c_int],
    "gk_net_headfeat_bytes": [c_int64],
    "gk_linear_workspace_bytes": [ctypes.POINTER(LinearStruct)],
    "gk_linear_grad_workspace_bytes": [ctypes.POINTER(LinearGradStruct)],
}

_lock = threading.Lock()
_lib = None


def library():
    """Load libgk.so once; raise if it has not been built."""
    global _lib
    with _lock:
        if _lib is None:
            if not LIBRARY_PATH.exists():
                raise RuntimeError(f"{LIBRARY_PATH} is missing: build it with build_native.py "
                                   "(the CUDA path has no fallback)")
            lib = ctypes.CDLL(str(LIBRARY_PATH))
            for name, args in _SIGNATURES.items():
                fn = getattr(lib, name)
                fn.argtypes = args
                fn.restype = c_int
            for name, args in _SIZE_FUNCTIONS.items():
                fn = getattr(lib, name)
                fn.argtypes = args
                fn.restype = c_size_t
            _lib = lib
        return _lib


def register(name: str, argtypes, restype=c_int):
    """Bind an additional exported function (used by other modules)."""
    fn = getattr(library(), name)
    fn.argtypes = argtypes
    fn.restype = restype
    return fn


def call(name: str, *args) -> None:
    status = getattr(library(), name)(*args)
    if status != 0:
        if status == -22:
            raise ValueError(f"{name}: invalid argument")
        raise RuntimeError(f"{name} failed with CUDA error {status}")


def ptr(tensor: torch.Tensor | None):
    return None if tensor is None else c_void_p(tensor.data_ptr())


def stream_of(device: torch.device):
    return c_void_p(torch.cuda.current_stream(device).cuda_stream)


def launch_stream(device: torch.device, tensors):
    """The current stream of `device`; the tensors are marked as used on it, so
    that memory allocated on another stream is not reused under the launch."""
    stream = torch.cuda.current_stream(device)
    for tensor in tensors:
        tensor.record_stream(stream)
    return c_void_p(stream.cuda_stream)


def on_device(device: torch.device):
    """A context in which `device` is current (nothing to do if it already is)."""
    if torch.cuda.current_device() == device.index:
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def require_cuda(device) -> torch.device:
    resolved = torch.device(device)
    if resolved.type != "cuda":
        raise ValueError("the batched self-play engine requires a CUDA device")
    if not torch.cuda.is_available():
        raise RuntimeError("CUDA is unavailable")
    index = torch.cuda.current_device() if resolved.index is None else resolved.index
    if not 0 <= index < torch.cuda.device_count():
        raise ValueError("CUDA device index is unavailable")
    return torch.device("cuda", index)
