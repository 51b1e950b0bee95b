"""ctypes binding of libssd_b200.so, the C-ABI CUDA library.

The library is the only compute path: if the shared object is missing or
fails to load, importing this module raises.  There is no CPU fallback.
Signatures follow ``include/ssd_b200.h``.
"""
from __future__ import annotations

import ctypes
import os
from pathlib import Path

LIB_NAME = "libssd_b200.so"

SSD_OK = 0
SSD_FLAG_DT_SOFTPLUS = 1
SSD_FLAG_EXTENTS = 2


def head_parts_flag(parts: int) -> int:
    """SSD_FLAG_HEAD_PARTS of the header."""
    return (parts - 1) << 8


class SsdShape(ctypes.Structure):
    """Mirror of ``struct SsdShape``."""

    _fields_ = [
        ("batch", ctypes.c_int32),
        ("seqlen", ctypes.c_int32),
        ("nheads", ctypes.c_int32),
        ("headdim", ctypes.c_int32),
        ("dstate", ctypes.c_int32),
        ("tile", ctypes.c_int32),
        ("ngroups", ctypes.c_int32),
        ("flags", ctypes.c_uint32),
        ("dt_min", ctypes.c_float),
        ("dt_max", ctypes.c_float),
        ("valid_len", ctypes.c_int32),
    ]


def _args(name: str, pointers: str):
    """Mirror of one of the header's argument records: pointers, then the mode of D."""
    fields = [(f, ctypes.c_void_p) for f in pointers.split()] + [("d_mode", ctypes.c_int32)]
    return type(name, (ctypes.Structure,), {"_fields_": fields})


SsdForwardArgs = _args("SsdForwardArgs", "x dt dt_bias A bm cm D z initial_state y out final_state work status")
SsdBackwardArgs = _args("SsdBackwardArgs", "x dt dt_bias A bm cm D z y dout dfinal forward_work dx ddt dA dB dC dD dz "
                                           "d_dt_bias d_initial work status")

SSD_F32, SSD_BF16, SSD_F16 = 0, 1, 2


def _record(name: str, *groups):
    """Mirror of an argument record that is laid out as groups of (type, names)."""
    fields = [(f, kind) for kind, names in groups for f in names.split()]
    return type(name, (ctypes.Structure,), {"_fields_": fields})


_P, _I64, _I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
SsdNormArgs = _record("SsdNormArgs", (_P, "x residual weight static_scale out stream q scales rstd"),
                      (_I64, "rows x_stride residual_stride"), (_I32, "width dtype residual_f32 weight_f32 group"),
                      (ctypes.c_float, "eps"))
SsdNormGradArgs = _record("SsdNormGradArgs", (_P, "dout dstream stream addend weight rstd dx dresidual dweight work"),
                          (_I64, "rows dout_stride dstream_stride stream_stride addend_stride"),
                          (_I32, "width dtype residual_f32 weight_f32"))
SsdConvArgs = _record("SsdConvArgs", (_P, "x weight bias initial_state cu_seqlens out final_state"),
                      (_I64, "tokens batch_stride token_stride"), (_I32, "rows channels width dtype weight_f32 silu"))
SsdConvGradArgs = _record("SsdConvGradArgs", (SsdConvArgs, "forward"), (_P, "dout dfinal dx dinitial dweight dbias work"))
SsdConvStepArgs = _record("SsdConvStepArgs", (_P, "x weight bias state slots state_out out"),
                          (_I64, "x_stride state_stride state_out_stride"),
                          (_I32, "rows slot_count channels width dtype weight_f32 silu"))
SsdScanArgs = _record("SsdScanArgs", (_P, "x dt z bm cm A D dt_bias initial_state cu_seqlens out final_state checkpoints work"),
                      (_I64, "tokens"), (_I64 * 2, "x_strides dt_strides z_strides"), (_I64 * 3, "b_strides c_strides"),
                      (_I32, "rows channels dstate groups dtype softplus"))
SsdScanGradArgs = _record("SsdScanGradArgs", (SsdScanArgs, "forward"),
                          (_P, "dout dfinal dx ddt dz dbm dcm dA dD d_dt_bias dinitial work"))
SsdScanStepArgs = _record("SsdScanStepArgs", (_P, "x dt z bm cm A D dt_bias state slots state_out out"),
                          (_I64, "x_stride dt_stride z_stride"), (_I64 * 2, "b_strides c_strides"),
                          (_I64, "state_stride state_out_stride"),
                          (_I32, "rows slot_count channels dstate groups dtype softplus"))


def library_path() -> Path:
    override = os.environ.get("SSD_B200_LIBRARY")
    if override:
        return Path(override)
    return Path(__file__).resolve().parent / LIB_NAME


def _load() -> ctypes.CDLL:
    path = library_path()
    if not path.exists():
        raise ImportError(
            f"{path} not found: build it with `python mamba-ascendc_b200/build.py` "
            "(ascend_kernel has no fallback path)"
        )
    return ctypes.CDLL(str(path))


lib = _load()

_p = ctypes.c_void_p
_shape_p = ctypes.POINTER(SsdShape)

# name -> (restype, argtypes); every symbol declared in include/ssd_b200.h
SIGNATURES = {
    "ssd_error_string": (ctypes.c_char_p, [ctypes.c_int]),
    "ssd_check_shape": (ctypes.c_int, [_shape_p]),
    "ssd_buffer_bytes": (ctypes.c_size_t, [_shape_p, ctypes.c_int]),
    "ssd_selftest_wait_expiry": (ctypes.c_int, [_p, ctypes.c_int, _p]),
    "ssd_selftest_tile_walk": (ctypes.c_int, [_shape_p, ctypes.c_int, ctypes.c_int, ctypes.c_int, _p]),
    "ssd_selftest_split_walk": (ctypes.c_int, [_shape_p] + [ctypes.c_int] * 5 + [_p]),
    "ssd_selftest_head_split": (ctypes.c_int, [ctypes.c_longlong] + [ctypes.c_int] * 4),
    "ssd_selftest_umma": (ctypes.c_int, [_p, _p, _p, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, _p, _p]),
    "ssd_dt_cumsum": (ctypes.c_int, [_shape_p, _p, _p, _p, _p, _p, _p]),
    "ssd_recurrent_fwd": (ctypes.c_int, [_shape_p] + [_p] * 7 + [ctypes.c_int] + [_p] * 5),
    "ssd_chunk_state": (ctypes.c_int, [_shape_p, _p, _p, _p, _p, _p, ctypes.c_int, _p, _p]),
    "ssd_state_passing_fwd": (ctypes.c_int, [_shape_p, _p, _p, _p, _p, _p]),
    "ssd_chunk_scan_fwd": (ctypes.c_int, [_shape_p] + [_p] * 9),
    "ssd_chunk_scan_copy_fwd": (ctypes.c_int, [_shape_p] + [_p] * 10),
    "ssd_state_passing_bwd": (ctypes.c_int, [_shape_p] + [_p] * 7),
    "ssd_chunk_state_scan_supported": (ctypes.c_int, [_shape_p]),
    "ssd_chunk_state_scan": (ctypes.c_int, [_shape_p] + [_p] * 7 + [ctypes.c_int, _p, _p]),
    "ssd_state_fold": (ctypes.c_int, [_shape_p, _p, _p, _p, _p, ctypes.c_int, _p]),
    "ssd_chunk_dx_bwd": (ctypes.c_int, [_shape_p] + [_p] * 15 + [_p, ctypes.c_int, _p, _p]),
    "ssd_chunk_dbc_bwd": (ctypes.c_int, [_shape_p] + [_p] * 13),
    "ssd_dbc_split": (ctypes.c_int, [_shape_p]),
    "ssd_chunk_dbc_split_bwd": (ctypes.c_int, [_shape_p] + [_p] * 11 + [ctypes.c_int, _p, _p, _p]),
    "ssd_dt_finalize_bwd": (ctypes.c_int, [_shape_p] + [_p] * 5),
    "ssd_dt_finalize_bias_bwd": (ctypes.c_int, [_shape_p] + [_p] * 6),
    "ssd_gate_partial_floats": (ctypes.c_size_t, [_shape_p]),
    "ssd_gate_skip_fwd": (ctypes.c_int, [_shape_p, _p, _p, _p, ctypes.c_int, _p, _p, _p]),
    "ssd_gate_skip_bwd": (ctypes.c_int, [_shape_p, _p, _p, _p, _p, ctypes.c_int, _p, _p, _p, _p, _p, _p]),
    "ssd_block_rmsnorm_fwd": (ctypes.c_int, [_p, ctypes.c_longlong, _p, ctypes.c_longlong, _p, _p, ctypes.c_longlong,
                                            ctypes.c_int, ctypes.c_float, _p]),
    "ssd_block_conv_silu_fwd": (ctypes.c_int, [_p, ctypes.c_longlong, _p, _p, _p, _p, _p, ctypes.c_int, ctypes.c_int,
                                              ctypes.c_int, ctypes.c_int, _p]),
    "ssd_block_skip_rmsnorm_fwd": (ctypes.c_int, [_p, ctypes.c_longlong, _p, _p, ctypes.c_int, _p, ctypes.c_longlong, _p, _p,
                                                 ctypes.c_longlong, ctypes.c_int, ctypes.c_float, _p]),
    "ssd_block_conv_split_fwd": (ctypes.c_int, [_p, ctypes.c_longlong] + [_p] * 8 + [ctypes.c_int] * 5 + [_p]),
    "ssd_linear_work_bytes": (ctypes.c_size_t, [ctypes.c_int, ctypes.c_int]),
    "ssd_linear_pays": (ctypes.c_int, [ctypes.c_longlong, ctypes.c_int, ctypes.c_int]),
    "ssd_linear_fwd": (ctypes.c_int, [_p, _p, _p, _p, ctypes.c_longlong, ctypes.c_int, ctypes.c_int, _p, _p, _p]),
    "ssd_rms_norm_fwd": (ctypes.c_int, [ctypes.POINTER(SsdNormArgs), _p]),
    "ssd_rms_norm_work_bytes": (ctypes.c_size_t, [ctypes.c_int64, ctypes.c_int, ctypes.c_int]),
    "ssd_rms_norm_bwd": (ctypes.c_int, [ctypes.POINTER(SsdNormGradArgs), _p]),
    "ssd_short_conv_fwd": (ctypes.c_int, [ctypes.POINTER(SsdConvArgs), _p]),
    "ssd_short_conv_work_bytes": (ctypes.c_size_t, [ctypes.POINTER(SsdConvArgs)]),
    "ssd_short_conv_bwd": (ctypes.c_int, [ctypes.POINTER(SsdConvGradArgs), _p]),
    "ssd_short_conv_step": (ctypes.c_int, [ctypes.POINTER(SsdConvStepArgs), _p]),
    "ssd_selective_scan_work_bytes": (ctypes.c_size_t, [ctypes.POINTER(SsdScanArgs)]),
    "ssd_selective_scan_checkpoint_bytes": (ctypes.c_size_t, [ctypes.POINTER(SsdScanArgs)]),
    "ssd_selective_scan_fwd": (ctypes.c_int, [ctypes.POINTER(SsdScanArgs), _p]),
    "ssd_selective_scan_grad_work_bytes": (ctypes.c_size_t, [ctypes.POINTER(SsdScanArgs)]),
    "ssd_selective_scan_bwd": (ctypes.c_int, [ctypes.POINTER(SsdScanGradArgs), _p]),
    "ssd_selective_scan_step": (ctypes.c_int, [ctypes.POINTER(SsdScanStepArgs), _p]),
    "ssd_use_state_scan": (ctypes.c_int, [_shape_p, ctypes.c_int]),
    "ssd_forward_work_bytes": (ctypes.c_size_t, [_shape_p]),
    "ssd_backward_work_bytes": (ctypes.c_size_t, [_shape_p, ctypes.c_int, ctypes.c_int]),
    "ssd_forward": (ctypes.c_int, [_shape_p, ctypes.POINTER(SsdForwardArgs), ctypes.c_int, _p]),
    "ssd_backward": (ctypes.c_int, [_shape_p, ctypes.POINTER(SsdBackwardArgs), ctypes.c_int, _p]),
    "ssd_static_scratch_bytes": (ctypes.c_size_t, []),
    "ssd_forward_static": (ctypes.c_int, [_shape_p] + [_p] * 9),
}

# test-only entry points; a library built with ``build.py --product-only`` does not have them
TEST_HOOKS = {"ssd_selftest_umma", "ssd_selftest_wait_expiry", "ssd_selftest_tile_walk", "ssd_selftest_split_walk",
              "ssd_selftest_head_split"}

for _name, (_res, _args) in SIGNATURES.items():
    if _name in TEST_HOOKS and not hasattr(lib, _name):
        continue
    _fn = getattr(lib, _name)  # AttributeError here means the header and the build disagree
    _fn.restype = _res
    _fn.argtypes = _args


def error_string(code: int) -> str:
    return lib.ssd_error_string(int(code)).decode()


def check(code: int, op: str) -> None:
    """Raise the reference's style of error (``RuntimeError("<op>: <message>")``) for a failed call."""
    if code != SSD_OK:
        raise RuntimeError(f"{op}: {error_string(code)} (code {code})")


def _load_calls():
    """The extension module of csrc/torch_calls.cpp, bound to the library above."""
    import importlib

    import torch  # noqa: F401  (the module links against its libraries)

    try:
        module = importlib.import_module(__package__ + "._calls")
    except ImportError as error:
        raise ImportError(f"{Path(__file__).resolve().parent / '_calls.so'} is missing or belongs to another torch: build it with "
                          f"`python mamba-ascendc_b200/build.py` ({error})") from error
    module.bind({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in SIGNATURES if hasattr(lib, name)})
    return module


class _Calls:
    """The operators' calls; the module is loaded by the first of them, as the SSD does without it."""

    def __getattr__(self, name: str):
        if name.startswith("_"):
            raise AttributeError(name)
        module = _load_calls()
        self.__dict__.update((n, f) for n, f in vars(module).items() if not n.startswith("_"))
        return getattr(module, name)


calls = _Calls()
