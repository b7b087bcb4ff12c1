"""ctypes binding of ``libmfcc_hip.so`` (the C ABI declared in ``include/mfcc_hip.h``).

There is no CPU fallback: if the shared library is missing or cannot be loaded the import of
this module's :func:`lib` raises, and every feature function built on it fails loudly.
"""
from __future__ import annotations

import ctypes as C
import os
from pathlib import Path

ABI_VERSION = 1

MFCC_OK = 0
MFCC_E_INVALID = -1
MFCC_E_UNSUPPORTED = -2
MFCC_E_HIP = -3
MFCC_E_WORKSPACE = -4
MFCC_E_NOMEM = -5

NOALLOC_SCRATCH_BYTES = 64 * 1024 * 1024   # MFCC_NOALLOC_SCRATCH_BYTES

PAD_CONSTANT = 0
PAD_REFLECT = 1


class MfccConfigC(C.Structure):
    """``struct mfcc_config`` -- field order and types must match include/mfcc_hip.h."""

    _fields_ = [
        ("struct_size", C.c_int32),
        ("n_fft", C.c_int32),
        ("hop_length", C.c_int32),
        ("win_length", C.c_int32),
        ("center", C.c_int32),
        ("pad_mode", C.c_int32),
        ("power", C.c_float),
        ("sr", C.c_double),
        ("n_mels", C.c_int32),
        ("fmin", C.c_double),
        ("fmax", C.c_double),
        ("htk", C.c_int32),
        ("mel_norm", C.c_int32),
        ("ref", C.c_float),
        ("amin", C.c_float),
        ("top_db", C.c_float),
        ("n_mfcc", C.c_int32),
        ("dct_type", C.c_int32),
        ("dct_norm", C.c_int32),
        ("lifter", C.c_float),
        ("window", C.POINTER(C.c_double)),
        ("mel_basis", C.POINTER(C.c_float)),
    ]


def _fields(text: str):
    """ctypes fields from "type name, name; ..." lines in the order of the C struct."""
    kinds = {"i32": C.c_int32, "i64": C.c_int64, "f32": C.c_float, "ptr": C.c_void_p, "size": C.c_size_t}
    out = []
    for group in text.split(";"):
        kind, _, names = group.strip().partition(" ")
        out += [(n.strip(), kinds[kind]) for n in names.split(",")]
    return out


class ConvArgsC(C.Structure):
    """``struct mfcc_conv_args`` -- field order and types must match include/mfcc_hip.h."""

    _fields_ = _fields("""i32 struct_size, dtype, channels, width, activation, n_seqs, zero_rest; i64 rows;
        ptr d_offsets, d_x; i64 x_stride; ptr d_weight, d_bias, d_initial, d_y; i64 y_stride; ptr d_state, d_dy;
        i64 dy_stride; ptr d_dstate, d_dx; i64 dx_stride; ptr d_dweight, d_dbias, d_dinitial, d_workspace;
        size workspace_bytes""")


class ScanArgsC(C.Structure):
    """``struct mfcc_scan_args`` -- field order and types must match include/mfcc_hip.h."""

    _fields_ = _fields("""i32 struct_size, dtype, channels, state, groups, softplus, n_seqs, zero_rest; i64 rows;
        ptr d_offsets, d_u; i64 u_stride; ptr d_delta; i64 delta_stride; ptr d_A, d_B; i64 B_stride; ptr d_C;
        i64 C_stride; ptr d_D, d_delta_bias, d_initial, d_y; i64 y_stride; ptr d_final, d_dy; i64 dy_stride;
        ptr d_dfinal, d_du, d_ddelta, d_dA, d_dB, d_dC, d_dD, d_ddelta_bias, d_dinitial, d_workspace;
        size workspace_bytes""")


class NormArgsC(C.Structure):
    """``struct mfcc_norm_args`` -- field order and types must match include/mfcc_hip.h."""

    _fields_ = _fields("""i32 struct_size, dtype, res_dtype, channels, groups, norm, gate_first; f32 eps, scale_value;
        i64 rows; ptr d_weight, d_bias, d_scale, d_x; i64 x_stride; ptr d_z; i64 z_stride; ptr d_residual;
        i64 residual_stride; ptr d_y; i64 y_stride; ptr d_r; i64 r_stride; ptr d_dy; i64 dy_stride; ptr d_dr;
        i64 dr_stride; ptr d_dx, d_dz, d_dresidual, d_dweight, d_dbias, d_dscale, d_workspace; size workspace_bytes""")


class LibraryError(RuntimeError):
    """A call into libmfcc_hip failed; ``code`` is the MFCC_E_* value."""

    def __init__(self, code: int, message: str):
        super().__init__(f"libmfcc_hip error {code}: {message}")
        self.code = code
        self.message = message


def library_path() -> Path:
    env = os.environ.get("MFCC_HIP_LIBRARY")
    if env:
        return Path(env)
    return Path(__file__).resolve().parent / "lib" / "libmfcc_hip.so"


# name -> (restype, argtypes); every symbol include/mfcc_hip.h declares.
SYMBOLS = {
    "mfcc_config_default": (None, [C.POINTER(MfccConfigC)]),
    "mfcc_abi_version": (C.c_int, []),
    "mfcc_last_error": (C.c_char_p, []),
    "mfcc_host_window": (C.c_int, [C.POINTER(MfccConfigC), C.POINTER(C.c_double)]),
    "mfcc_host_mel_basis": (C.c_int, [C.POINTER(MfccConfigC), C.POINTER(C.c_float)]),
    "mfcc_host_dct_basis": (C.c_int, [C.POINTER(MfccConfigC), C.POINTER(C.c_float)]),
    "mfcc_num_frames": (C.c_int64, [C.POINTER(MfccConfigC), C.c_int64]),
    "mfcc_batch_layout": (C.c_int, [C.POINTER(MfccConfigC), C.POINTER(C.c_int64), C.c_int32,
                                    C.POINTER(C.c_int64)]),
    "mfcc_plan_create": (C.c_int, [C.POINTER(MfccConfigC), C.POINTER(C.c_void_p)]),
    "mfcc_plan_destroy": (None, [C.c_void_p]),
    "mfcc_workspace_bytes": (C.c_size_t, [C.c_void_p, C.c_int64, C.c_int32]),
    "mfcc_execute": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                               C.c_int32, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p,
                               C.c_size_t, C.c_void_p]),
    "mfcc_execute_pcm16": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                     C.c_int32, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p,
                                     C.c_size_t, C.c_void_p]),
    "mfcc_execute_noalloc": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                       C.c_int32, C.c_int64, C.c_void_p, C.c_void_p]),
    "mfcc_workspace_status": (C.c_int, [C.c_void_p, C.c_void_p]),
    "mfcc_execute_spectrogram": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                           C.c_int32, C.c_int64, C.c_void_p, C.c_void_p,
                                           C.c_size_t, C.c_void_p]),
    "mfcc_plan_set_profiling": (C.c_int, [C.c_void_p, C.c_int]),
    "mfcc_plan_last_timings": (C.c_int, [C.c_void_p, C.POINTER(C.c_float), C.POINTER(C.c_float)]),
    "mfcc_plan_timing_history": (C.c_int, [C.c_void_p, C.c_int32, C.POINTER(C.c_float), C.POINTER(C.c_float)]),
    "mfcc_plan_front_kernel": (C.c_char_p, [C.c_void_p]),
    "mfcc_to_db": (C.c_int, [C.c_void_p, C.c_int64, C.c_int32, C.c_float, C.c_int32, C.c_float, C.c_float,
                             C.c_void_p, C.c_void_p, C.c_void_p]),
    "mfcc_dct": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p]),
    "mfcc_delta": (C.c_int, [C.c_void_p, C.c_void_p, C.POINTER(C.c_int64), C.c_int32, C.c_int32, C.c_int32, C.c_int32,
                             C.c_void_p, C.c_void_p]),
    "mfcc_host_pcm16_from_float": (C.c_int, [C.c_void_p, C.c_int64, C.c_void_p]),
    "mfcc_host_write_feature_file": (C.c_int, [C.c_char_p, C.c_char_p, C.c_void_p, C.c_int64, C.c_int64, C.c_int32,
                                               C.POINTER(C.c_char_p), C.POINTER(C.c_int32), C.POINTER(C.c_int64),
                                               C.POINTER(C.c_char_p)]),
    "mfcc_host_write_feature_files": (C.c_int, [C.c_int32, C.POINTER(C.c_char_p), C.c_char_p, C.POINTER(C.c_void_p),
                                                C.POINTER(C.c_int64), C.c_int64, C.c_int32, C.POINTER(C.c_char_p),
                                                C.POINTER(C.c_int32), C.POINTER(C.c_int64), C.POINTER(C.c_char_p)]),
    "mfcc_host_write_feature_files_mt": (C.c_int, [C.c_int32, C.POINTER(C.c_char_p), C.c_char_p, C.c_void_p,
                                                   C.c_void_p, C.c_int64, C.c_int32, C.POINTER(C.c_char_p),
                                                   C.POINTER(C.c_int32), C.c_void_p, C.POINTER(C.c_char_p), C.c_int32]),
    "mfcc_host_pack_range": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p, C.c_int64, C.c_int64, C.c_int64,
                                       C.c_int32]),
    "mfcc_host_file_error": (C.c_char_p, []),
    "mfcc_cmvn_accumulate": (C.c_int, [C.c_void_p, C.c_int64, C.c_int32, C.c_void_p, C.c_void_p]),
    "mfcc_cmvn_apply": (C.c_int, [C.c_void_p, C.c_int64, C.c_int32, C.c_void_p, C.c_double,
                                  C.c_void_p]),
    "mfcc_causal_conv": (C.c_int, [C.POINTER(ConvArgsC), C.c_void_p]),
    "mfcc_causal_conv_backward_workspace": (C.c_size_t, [C.POINTER(ConvArgsC)]),
    "mfcc_causal_conv_backward": (C.c_int, [C.POINTER(ConvArgsC), C.c_void_p]),
    "mfcc_causal_conv_step": (C.c_int, [C.c_int32] * 6 + [C.c_void_p, C.c_int64] + [C.c_void_p] * 6 + [C.c_int64, C.c_void_p]),
    "mfcc_selective_scan_workspace": (C.c_size_t, [C.POINTER(ScanArgsC)]),
    "mfcc_selective_scan": (C.c_int, [C.POINTER(ScanArgsC), C.c_void_p]),
    "mfcc_selective_scan_backward_workspace": (C.c_size_t, [C.POINTER(ScanArgsC)]),
    "mfcc_selective_scan_backward": (C.c_int, [C.POINTER(ScanArgsC), C.c_void_p]),
    "mfcc_selective_scan_step": (C.c_int, [C.POINTER(ScanArgsC), C.c_int32, C.c_void_p, C.c_void_p]),
    "mfcc_add_norm": (C.c_int, [C.POINTER(NormArgsC), C.c_void_p]),
    "mfcc_gate_norm": (C.c_int, [C.POINTER(NormArgsC), C.c_void_p]),
    "mfcc_norm_backward_workspace": (C.c_size_t, [C.POINTER(NormArgsC)]),
    "mfcc_add_norm_backward": (C.c_int, [C.POINTER(NormArgsC), C.c_void_p]),
    "mfcc_gate_norm_backward": (C.c_int, [C.POINTER(NormArgsC), C.c_void_p]),
}

_LIB = None


def lib() -> C.CDLL:
    """Load (once) and return the shared library with argument types set."""
    global _LIB
    if _LIB is not None:
        return _LIB
    path = library_path()
    if not path.exists():
        raise ImportError(
            f"{path} is missing: build it with `make -C speech_to_text_amd/csrc` "
            "(or __graft_entry__.build()); there is no CPU fallback for this package")
    handle = C.CDLL(str(path))
    for name, (restype, argtypes) in SYMBOLS.items():
        fn = getattr(handle, name)
        fn.restype = restype
        fn.argtypes = argtypes
    if handle.mfcc_abi_version() != ABI_VERSION:
        raise ImportError(f"{path}: ABI version {handle.mfcc_abi_version()} != {ABI_VERSION}")
    _LIB = handle
    return handle


def last_error() -> str:
    return lib().mfcc_last_error().decode("utf-8", "replace")


def check(code: int) -> None:
    if code != MFCC_OK:
        raise LibraryError(code, last_error())
