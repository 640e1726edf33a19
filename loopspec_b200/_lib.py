"""ctypes binding of libloopspec_engine.so (declared in include/loopspec_engine.h).

The library is built in-tree (loopspec_b200/libloopspec_engine.so) by
`loopspec_b200.build.build()`. There is no fallback: if the library is missing
or fails to load, `lib()` raises, and every engine entry point fails loudly.
"""

from __future__ import annotations

import ctypes
import os
import struct
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libloopspec_engine.so")

LS_OK, LS_EINVAL, LS_ECAPACITY, LS_ECUDA, LS_EDEVICE, LS_EPIPELINE = 0, -1, -2, -3, -4, -5

FAMILY = {"ouro": 0, "raven": 1}
LAYOUT = {"ouro": 0, "raven_pre": 1, "olmo_post": 2}

_i32, _i64, _f32, _f64, _u64 = (ctypes.c_int32, ctypes.c_int64, ctypes.c_float,
                                ctypes.c_double, ctypes.c_uint64)


class ModelCfg(ctypes.Structure):
    _fields_ = [
        ("family", _i32), ("layout", _i32),
        ("hidden", _i32), ("n_heads", _i32), ("n_kv_heads", _i32), ("head_dim", _i32),
        ("intermediate", _i32), ("vocab", _i32),
        ("n_pre_layers", _i32), ("n_core_layers", _i32), ("n_post_layers", _i32),
        ("stages", _i32),
        ("rope_theta", _f32), ("rms_eps", _f32), ("embed_scale", _f32), ("init_std", _f32),
        ("init_seed", _u64),
        ("qk_norm", _i32), ("adapter_bias", _i32), ("tie_embeddings", _i32),
    ]


class SchedCfg(ctypes.Structure):
    _fields_ = [
        ("step_size", _i32), ("second_step", _i32),
        ("max_context", _i32), ("max_prompt", _i32),
        ("kv_slots", _i32), ("request_rows", _i32),
        ("use_graphs", _i32), ("use_pdl", _i32), ("max_requests", _i32), ("device_loop", _i32),
    ]


class Stats(ctypes.Structure):
    _fields_ = [
        ("pipeline_cycles", _i64), ("pre_rows", _i64), ("recurrent_rows", _i64),
        ("post_rows", _i64), ("verified_proposals", _i64), ("first_rejections", _i64),
        ("second_verifications", _i64), ("second_acceptances", _i64),
        ("second_rejections", _i64), ("decode_tokens", _i64),
        ("decode_device_ms", _f64), ("decode_host_s", _f64), ("prefill_device_ms", _f64),
        ("h2d_bytes", _i64), ("d2h_bytes", _i64), ("decode_kernel_launches", _i64),
        ("pre_calls", _i64), ("core_calls", _i64), ("core_kv_positions", _i64), ("post_calls", _i64), ("host_syncs", _i64),
    ]

    def as_dict(self):
        return {name: getattr(self, name) for name, _ in self._fields_}


_VP = ctypes.c_void_p


class SlotsArgs(ctypes.Structure):
    _fields_ = [
        ("lens", _VP), ("delta", _VP), ("block_table", _VP), ("table_stride", _i64), ("free_blocks", _VP),
        ("free_count", _VP), ("slots", _VP), ("positions", _VP), ("requests", _VP), ("token_start", _VP),
        ("lens_out", _VP), ("free_count_out", _VP), ("status", _VP),
        ("n_requests", _i32), ("table_width", _i32), ("free_capacity", _i32), ("n_blocks", _i32),
        ("page_size", _i32), ("base", _i32), ("max_tokens", _i32),
    ]


class QkNormArgs(ctypes.Structure):
    _fields_ = [
        ("qkv", _VP), ("qkv_stride", _i64), ("q_weight", _VP), ("k_weight", _VP), ("rope", _VP),
        ("positions", _VP), ("slots", _VP), ("k_pool", _VP), ("v_pool", _VP), ("slot_stride", _i64),
        ("q_out", _VP), ("q_out_stride", _i64), ("status", _VP),
        ("qkv_type", _i32), ("weight_type", _i32), ("cache_type", _i32), ("n_tokens", _i32),
        ("n_heads", _i32), ("n_kv_heads", _i32), ("head_dim", _i32), ("max_positions", _i32), ("rot", _i32),
        ("interleaved", _i32), ("n_slots", _i32), ("eps", _f32),
    ]


class PrefixAttentionArgs(ctypes.Structure):
    _fields_ = [
        ("q", _VP), ("q_stride", _i64), ("k_pool", _VP), ("v_pool", _VP), ("slot_stride", _i64),
        ("prefix_table", _VP), ("block_table", _VP), ("table_stride", _i64), ("lens", _VP),
        ("token_start", _VP), ("out", _VP), ("out_stride", _i64), ("workspace", _VP),
        ("workspace_bytes", _u64), ("status", _VP),
        ("q_type", _i32), ("cache_type", _i32), ("n_tokens", _i32), ("n_requests", _i32),
        ("n_heads", _i32), ("n_kv_heads", _i32), ("head_dim", _i32), ("prefix_len", _i32),
        ("max_new", _i32), ("max_len", _i32), ("page_size", _i32), ("n_slots", _i32), ("scale", _f32),
    ]


_CODES = {_VP: "P", _i64: "q", _u64: "Q", _i32: "i", _f32: "f"}


def packer(args):
    """pack(*fields) -> the bytes of the argument struct `args`, in field order.
    A call of one of these operators takes a few microseconds; packing costs a
    third of one, filling a ctypes Structure several."""
    form = struct.Struct("@" + "".join(_CODES[kind] for _, kind in args._fields_) + "0P")
    assert form.size == ctypes.sizeof(args)
    return form.pack


DECIDE_FN = ctypes.CFUNCTYPE(ctypes.c_int64, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_int32)
CYCLE_FN = ctypes.CFUNCTYPE(None, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int64), ctypes.c_int32)
COMMIT_FN = ctypes.CFUNCTYPE(ctypes.c_int32, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int64), ctypes.c_int32)
RETAIN_FN = ctypes.CFUNCTYPE(None, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int64), ctypes.c_int32,
                             ctypes.c_int32)

_P = ctypes.c_void_p
TP_HANDLE_BYTES = 128   # LS_TP_HANDLE_BYTES
_PI64 = ctypes.POINTER(_i64)
_PF32 = ctypes.POINTER(_f32)

# (name, restype, argtypes) for every symbol of include/loopspec_engine.h
SIGNATURES = [
    ("ls_create", _i32, [ctypes.POINTER(ModelCfg), ctypes.POINTER(SchedCfg), _i32, ctypes.POINTER(_P)]),
    ("ls_load_weight", _i32, [_P, ctypes.c_char_p, _P, _i32, _PI64, _i32]),
    ("ls_finalize", _i32, [_P]),
    ("ls_tp_init", _i32, [_P, _i32, _i32, _P]),
    ("ls_tp_attach", _i32, [_P, _P]),
    ("ls_debug_tp_silent_peer", _i32, [_P, _i32]),
    ("ls_prefill", _i32, [_P, _PI64, _i32, _PF32, _PI64]),
    ("ls_set_sampling", _i32, [_P, _f32, _i32, _f32, _u64]),
    ("ls_cycle", _i32, [_P, _PI64, _i32, _PI64, _PF32]),
    ("ls_retain", _i32, [_P, _PI64, _PI64, _i32]),
    ("ls_generate", _i32, [_P, _PI64, _i32, _i32, _i32, _i64, _PI64, ctypes.POINTER(_i32),
                           ctypes.POINTER(Stats)]),
    ("ls_generate_stream", _i32, [_P, _PI64, _i32, _i32, _i32, _i64, COMMIT_FN, _P, _PI64,
                                  ctypes.POINTER(_i32), ctypes.POINTER(Stats)]),
    ("ls_generate_batch", _i32, [_P, _PI64, ctypes.POINTER(_i32), _i32, _i32, _i32, _i64,
                                 ctypes.POINTER(_u64), _PI64, ctypes.POINTER(_i32),
                                 ctypes.POINTER(Stats), ctypes.POINTER(Stats)]),
    ("ls_generate_batch_sampling", _i32, [_P, _PI64, ctypes.POINTER(_i32), _i32, _i32, _i32, _i64,
                                          ctypes.POINTER(_u64), ctypes.POINTER(ctypes.c_float),
                                          ctypes.POINTER(_i32), ctypes.POINTER(ctypes.c_float), _PI64,
                                          ctypes.POINTER(_i32), ctypes.POINTER(Stats),
                                          ctypes.POINTER(Stats)]),
    ("ls_device_loop_simulate", _i32, [_i32, _i32, _i32, _i64, _i32, _i64, DECIDE_FN, CYCLE_FN,
                                       RETAIN_FN, _P, _PI64, ctypes.POINTER(_i32),
                                       ctypes.POINTER(Stats)]),
    ("ls_pipeline_simulate", _i32, [_i32, _i32, _i32, _i64, _i32, _i64, DECIDE_FN, CYCLE_FN,
                                    RETAIN_FN, _P, _PI64, ctypes.POINTER(_i32),
                                    ctypes.POINTER(Stats)]),
    ("ls_time_role", _i32, [_P, _i32, _i32, _i32, _i32, ctypes.POINTER(_f64)]),
    ("ls_time_gemm", _i32, [_P, _i32, _i32, _i32, ctypes.POINTER(_f64)]),
    ("ls_time_core_gemms", _i32, [_P, _i32, _i32, ctypes.POINTER(_f64), ctypes.POINTER(_f64)]),
    ("ls_role_kernel_count", _i32, [_P, _i32, _i32, ctypes.POINTER(_i32)]),
    ("ls_debug_gemm", _i32, [_P, _i32, _i32, _PF32, _PF32]),
    ("ls_gemm_splits", _i32, [_P, _i32, ctypes.POINTER(_i32), ctypes.POINTER(_i32), ctypes.POINTER(_i32)]),
    ("ls_debug_kv", _i32, [_P, ctypes.POINTER(_P), ctypes.POINTER(_P), ctypes.POINTER(_i32),
                           ctypes.POINTER(_i32)]),
    ("ls_decode_attention_workspace_bytes", ctypes.c_size_t, [_i32, _i32, _i32, _i32, _i32]),
    ("ls_decode_attention", _i32, [_P, _P, _P, _P, _P, _P, _i32, _i32, _i32, _i32, _i32, _i32,
                                   _i32, _P, ctypes.c_size_t, _P, _P]),
    ("ls_decode_attention_noalloc", _i32, [_P, _P, _P, _P, _P, _P, _i32, _i32, _i32, _i32, _i32,
                                           _i32, _i32, _P, _P]),
    ("ls_decode_attention_noalloc_limit", ctypes.c_size_t, []),
    ("ls_check_status", _i32, [_P, _P]),
    ("ls_build_slots", _i32, [ctypes.c_char_p, _P]),
    ("ls_qk_norm_rope", _i32, [ctypes.c_char_p, _P]),
    ("ls_prefix_attention_workspace_bytes", ctypes.c_size_t, [_i32] * 8),
    ("ls_prefix_attention", _i32, [ctypes.c_char_p, _P]),
    ("ls_destroy", _i32, [_P]),
    ("ls_last_error", ctypes.c_char_p, [_P]),
    ("ls_version", ctypes.c_char_p, []),
]

_LIB = None


def lib():
    """Load the engine library once; raise if it is missing (no CPU fallback)."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(
                f"{LIB_PATH} is missing: build it with `python -c 'import loopspec_b200.build as b; b.build()'`")
        handle = ctypes.CDLL(LIB_PATH)
        for name, res, args in SIGNATURES:
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _LIB = handle
    return _LIB


_FACTS = None


def tensor_facts():
    """facts and pointers of csrc/tensor_facts.cpp: tensor arguments looked over
    in one call each, for the operators whose whole call takes microseconds."""
    global _FACTS
    if _FACTS is None:
        import torch
        how = "build it with `python -m loopspec_b200.build`"
        try:
            from . import _tensor_facts
        except ImportError as e:
            raise ImportError(f"{e}: {how}") from e
        here = (torch.__version__.split("+")[0], *sys.version_info[:2])
        if _tensor_facts.made_for != here:      # its reading of tensors goes by the layout of that version's objects
            raise ImportError(f"the tensor module was made for torch and Python {_tensor_facts.made_for}, not {here}: {how}")
        _FACTS = _tensor_facts.facts, _tensor_facts.pointers
    return _FACTS


BF16, F16, F32, I32, BYTE = range(5)   # type codes: LS_BF16, LS_F16, LS_F32, and those of index and scratch tensors


class EngineError(RuntimeError):
    def __init__(self, code, message):
        super().__init__(f"[{code}] {message}")
        self.code = code


def check(code, handle=None):
    if code != LS_OK:
        raise EngineError(code, lib().ls_last_error(handle).decode())
