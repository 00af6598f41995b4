"""ctypes binding of ``libisingdiff.so`` (declared in ``include/isingdiff.h``).

The library is built in-tree by ``csrc/Makefile`` (``__graft_entry__.build()``).  There is
no CPU fallback: if the shared library is missing or a call fails, an exception is raised.
"""
from __future__ import annotations

import ctypes as C
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("ISINGDIFF_LIB") or os.path.join(_HERE, "libisingdiff.so")

IDM_FP32 = 0
IDM_BF16 = 1
IDM_UPDATE_SCORE = 0
IDM_UPDATE_DDPM = 1
NCONV = 11
NDENSE = 3
ABI_VERSION = 4
NOALLOC_SCRATCH_BYTES = 64 << 20


class IdmError(RuntimeError):
    pass


class ModelDesc(C.Structure):
    _fields_ = [
        ("channels", C.c_int32), ("base_filters", C.c_int32), ("batchnorm", C.c_int32), ("reserved", C.c_int32),
        ("conv_w", C.c_void_p * NCONV), ("conv_b", C.c_void_p * NCONV),
        ("bn_scale", C.c_void_p * NCONV), ("bn_shift", C.c_void_p * NCONV),
        ("dense_w", C.c_void_p * NDENSE), ("dense_b", C.c_void_p * NDENSE),
    ]


class SampleCfg(C.Structure):
    _fields_ = [
        ("T", C.c_int32), ("precision", C.c_int32), ("betas_host", C.c_void_p), ("seed", C.c_uint64),
        ("first_global_index", C.c_int64), ("init_state", C.c_int32), ("add_noise", C.c_int32),
        ("chunk", C.c_int64), ("update_rule", C.c_int32), ("reserved", C.c_int32), ("alpha_cumprod_host", C.c_void_p),
    ]


class ProfileEntry(C.Structure):
    _fields_ = [("name", C.c_char * 32), ("launches", C.c_int64), ("ms", C.c_double), ("flop", C.c_double),
                ("bytes", C.c_double)]


BITFLIP_NTENSOR = 68


class BitflipDesc(C.Structure):
    _fields_ = [("n_tensors", C.c_int32), ("reserved", C.c_int32), ("tensors", C.c_void_p * BITFLIP_NTENSOR)]


class BitflipCfg(C.Structure):
    _fields_ = [("T", C.c_int32), ("reserved", C.c_int32), ("emb_table_host", C.c_void_p), ("seed", C.c_uint64),
                ("first_global_index", C.c_int64), ("chunk", C.c_int64)]


MLP_MAXLAYERS = 8


class MlpDesc(C.Structure):
    _fields_ = [("n_layers", C.c_int32), ("reserved", C.c_int32), ("in_dim", C.c_int32 * MLP_MAXLAYERS),
                ("out_dim", C.c_int32 * MLP_MAXLAYERS), ("act", C.c_int32 * MLP_MAXLAYERS),
                ("w", C.c_void_p * MLP_MAXLAYERS), ("b", C.c_void_p * MLP_MAXLAYERS)]


IDM_DT_F32, IDM_DT_BF16, IDM_DT_F16 = 0, 1, 2
IDM_ACT_NONE, IDM_ACT_SWISH = 0, 1
ADAMW_BLOCK = 256


class GroupNormDesc(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("activation", C.c_int32), ("batch", C.c_int64), ("pixels", C.c_int64),
                ("channels", C.c_int32), ("groups", C.c_int32), ("x_sample", C.c_int64), ("x_pixel", C.c_int64),
                ("dy_sample", C.c_int64), ("dy_pixel", C.c_int64), ("shift_sample", C.c_int64), ("eps", C.c_float),
                ("aligned", C.c_int32)]


class AdamWCfg(C.Structure):
    _fields_ = [("param_dtype", C.c_int32), ("grad_dtype", C.c_int32), ("moment_bits", C.c_int32), ("reserved", C.c_int32),
                ("lr", C.c_double), ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double)]


# name -> (restype, argtypes); every symbol include/isingdiff.h declares
SIGNATURES = {
    "idm_abi_version": (C.c_int, []),
    "idm_last_error": (C.c_char_p, []),
    "idm_model_create": (C.c_int, [C.POINTER(C.c_void_p), C.c_int, C.POINTER(ModelDesc)]),
    "idm_model_destroy": (C.c_int, [C.c_void_p]),
    "idm_time_table": (C.c_int, [C.c_void_p, C.c_int, C.c_void_p]),
    "idm_forward": (C.c_int, [C.c_void_p, C.c_void_p, C.c_float, C.c_void_p, C.c_int64, C.c_int, C.c_int, C.c_int, C.c_void_p]),
    "idm_forward_noalloc": (C.c_int, [C.c_void_p, C.c_void_p, C.c_float, C.c_void_p, C.c_int64, C.c_int, C.c_int, C.c_int, C.c_void_p]),
    "idm_plan_chunk": (C.c_int, [C.c_void_p, C.c_int64, C.c_int, C.c_int, C.c_int, C.POINTER(C.c_int64), C.POINTER(C.c_int64)]),
    "idm_forward_taps": (C.c_int, [C.c_void_p, C.c_void_p, C.c_float, C.c_void_p, C.c_int64, C.c_int, C.c_int, C.c_int,
                                   C.POINTER(C.c_void_p), C.c_void_p]),
    "idm_sample": (C.c_int, [C.c_void_p, C.POINTER(SampleCfg), C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                             C.c_int64, C.c_int, C.c_int, C.c_void_p]),
    "idm_update": (C.c_int, [C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_float, C.c_int64, C.c_void_p]),
    "idm_philox_normal": (C.c_int, [C.c_int, C.c_void_p, C.c_int64, C.c_int64, C.c_uint64, C.c_int64, C.c_int32, C.c_void_p]),
    "idm_sign_project": (C.c_int, [C.c_int, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]),
    "idm_observe": (C.c_int, [C.c_int, C.c_void_p, C.c_int64, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                              C.c_void_p, C.c_void_p]),
    "idm_irfft2_sign": (C.c_int, [C.c_int, C.c_void_p, C.c_int64, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]),
    "idm_metropolis": (C.c_int, [C.c_int, C.c_void_p, C.c_int64, C.c_int, C.c_void_p, C.c_int, C.c_uint64, C.c_int64, C.c_int,
                                 C.c_void_p]),
    "idm_xy_metropolis": (C.c_int, [C.c_int, C.c_void_p, C.c_int64, C.c_int, C.c_float, C.c_float, C.c_int, C.c_uint64, C.c_int64, C.c_int,
                                    C.c_void_p]),
    "idm_xy_observe": (C.c_int, [C.c_int, C.c_void_p, C.c_int64, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]),
    "idm_comm_create": (C.c_int, [C.POINTER(C.c_void_p), C.POINTER(C.c_int), C.c_int]),
    "idm_allreduce_i64": (C.c_int, [C.c_void_p, C.POINTER(C.c_void_p), C.c_size_t, C.POINTER(C.c_void_p)]),
    "idm_comm_destroy": (C.c_int, [C.c_void_p]),
    "idm_set_option": (C.c_int, [C.c_void_p, C.c_char_p, C.c_int]),
    "idm_profile_begin": (C.c_int, [C.c_void_p]),
    "idm_profile_end": (C.c_int, [C.c_void_p, C.POINTER(ProfileEntry), C.c_int, C.POINTER(C.c_int)]),
    "idm_mlp_create": (C.c_int, [C.POINTER(C.c_void_p), C.c_int, C.POINTER(MlpDesc)]),
    "idm_mlp_destroy": (C.c_int, [C.c_void_p]),
    "idm_mlp_forward": (C.c_int, [C.c_void_p, C.c_void_p, C.c_float, C.c_void_p, C.c_int64, C.c_void_p]),
    "idm_mlp_forward_precision": (C.c_int, [C.c_void_p, C.c_void_p, C.c_float, C.c_void_p, C.c_int64, C.c_int, C.c_void_p]),
    "idm_mlp_sample": (C.c_int, [C.c_void_p, C.POINTER(SampleCfg), C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64,
                                 C.c_void_p]),
    "idm_bitflip_create": (C.c_int, [C.POINTER(C.c_void_p), C.c_int, C.POINTER(BitflipDesc)]),
    "idm_bitflip_destroy": (C.c_int, [C.c_void_p]),
    "idm_bitflip_set_precision": (C.c_int, [C.c_void_p, C.c_int]),
    "idm_bitflip_time": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p]),
    "idm_bitflip_forward": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_int, C.c_int,
                                      C.POINTER(C.c_void_p), C.c_void_p]),
    "idm_bitflip_sample": (C.c_int, [C.c_void_p, C.POINTER(BitflipCfg), C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64,
                                     C.c_int, C.c_int, C.c_void_p]),
    "idm_group_norm_workspace": (C.c_int, [C.POINTER(GroupNormDesc), C.c_int, C.POINTER(C.c_size_t)]),
    "idm_group_norm_forward": (C.c_int, [C.c_int, C.POINTER(GroupNormDesc)] + [C.c_void_p] * 8 + [C.c_size_t, C.c_void_p]),
    "idm_group_norm_backward": (C.c_int, [C.c_int, C.POINTER(GroupNormDesc)] + [C.c_void_p] * 12 + [C.c_size_t, C.c_void_p]),
    "idm_adamw_step": (C.c_int, [C.c_int, C.POINTER(AdamWCfg), C.c_int64] + [C.c_void_p] * 8 + [C.c_int64] + [C.c_void_p] * 3),
    "idm_adamw_moments": (C.c_int, [C.c_int] + [C.c_void_p] * 6 + [C.c_int64, C.c_void_p]),
}

_lib = _bound = None


def load():
    """Load the shared library (once) and bind every exported symbol."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise IdmError(f"{LIB_PATH} not found: build it with `make -C diffusion-model_amd/csrc` "
                           "(there is no CPU fallback)")
        # PyTorch bundles its own HIP runtime (same SONAME as /opt/rocm's).  Import it first so that
        # this library binds to the runtime that owns torch's device pointers and streams.
        import torch  # noqa: F401
        lib = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        if lib.idm_abi_version() != ABI_VERSION:
            raise IdmError("libisingdiff.so ABI version mismatch")
        _lib = lib
    return _lib


def host():
    """The compiled host side of the training operators (``idm_host.cpp``), bound to the library (once)."""
    global _bound
    if _bound is None:
        lib = load()
        import torch
        try:
            from . import _host
        except ImportError as e:
            raise IdmError(f"isingdiff/_host.so cannot be loaded ({e}): build it with `make -C diffusion-model_amd/csrc`") from None
        # the hipStream_t of a device's current stream; by torch's own short cut where it has one (0.1 us instead of 2)
        stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
        names = ("group_norm_workspace", "group_norm_forward", "group_norm_backward", "adamw_step", "adamw_moments")
        _host.bind(tuple(C.cast(getattr(lib, "idm_" + n), C.c_void_p).value for n in names), check, stream)
        _bound = _host
    return _bound


def check(rc: int):
    if rc != 0:
        msg = load().idm_last_error()
        raise IdmError(f"libisingdiff error {rc}: {msg.decode() if msg else '?'}")
