"""ctypes binding of libfermix_b200.so (the C ABI declared in include/fermix_b200.h).

The library is built in-tree (``python -m fermix_b200.build``) and loaded from
``fermix_b200/_lib/``. There is no fallback: if the library is missing or cannot be
loaded, every call raises.
"""

import ctypes
import os
import threading

LIB_DIR = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_lib")
LIB_PATH = os.path.join(LIB_DIR, "libfermix_b200.so")

FX_F32, FX_F64, FX_C64, FX_C128, FX_BF16 = 0, 1, 2, 3, 4
FX_PREC_DEFAULT, FX_PREC_TF32X3, FX_PREC_IEEE = 0, 1, 2
FX_OP_SLOGDET, FX_OP_SLOGPF = 0, 1
FX_ERR_TIMEOUT = 8
FX_WAIT_POLLS_DEFAULT = 1 << 26
FX_NORM_MAX_WIDTH, FX_ATTN_MAX_DIM, FX_BUCKET_MAX, FX_BUCKET_MAX_EDGE = 8192, 128, 256, 2048

# every symbol include/fermix_b200.h declares, with its ctypes signature
_vp, _i, _i64, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
SIGNATURES = {
    "fermix_slogdet": (_i, [_vp, _i, _i, _i64, _i64, _vp, _vp, _vp, _vp, _vp, _sz]),
    "fermix_slogdet_grad": (_i, [_vp, _i, _i, _i64, _i64, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp, _sz]),
    "fermix_slogpf": (_i, [_vp, _i, _i, _i64, _i64, _i, _vp, _vp, _vp, _vp, _vp, _sz]),
    "fermix_slogpf_grad": (_i, [_vp, _i, _i, _i64, _i64, _i, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp, _sz]),
    "fermix_slogdet_grad_static": (_i, [_vp, _i, _i, _i64, _i64, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp]),
    "fermix_slogdet_gather": (
        _i, [_vp, _i, _i, _i64, _i64, _vp, _i64, _i64, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp, _sz]),
    "fermix_slogdet_gather_workspace_bytes": (_sz, [_i, _i, _i64, _i64, _i]),
    "fermix_slogdet_ratio": (_i, [_vp, _i, _i64, _i64, _i64, _vp, _vp, _vp, _vp, _vp]),
    "fermix_slogdet_update": (_i, [_vp, _i, _i64, _i64, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz]),
    "fermix_slogdet_update_workspace_bytes": (_sz, [_i, _i64, _i64, _i64]),
    "fermix_slogpf_ratio": (_i, [_vp, _i, _i64, _i64, _vp, _vp, _vp, _vp, _vp]),
    "fermix_slogpf_update": (_i, [_vp, _i, _i64, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz]),
    "fermix_slogpf_update_workspace_bytes": (_sz, [_i, _i64, _i64]),
    "fermix_slogpf_ratio_k": (_i, [_vp, _i, _i64, _i64, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _sz]),
    "fermix_slogpf_update_k": (_i, [_vp, _i, _i64, _i64, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz]),
    "fermix_slogpf_move_k_workspace_bytes": (_sz, [_i, _i64, _i64, _i64]),
    "fermix_workspace_bytes": (_sz, [_i, _i, _i64, _i64, _i]),
    "fermix_check_prec": (_i, [_i, _i]),
    "fermix_strerror": (ctypes.c_char_p, [_i]),
    "fermix_version": (_i, []),
    "fermix_selftest_umma": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _vp, _vp]),
    "fermix_selftest_fma_rate": (_i, [_vp, _i, _i, _i, _vp]),
    "fermix_device_status": (_i, [_i]),
    "fermix_set_wait_polls": (ctypes.c_uint, [ctypes.c_uint]),
    "fermix_slogdet_planar": (_i, [_vp, _i, _i, _i64, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _sz]),
    "fermix_slogdet_grad_planar": (
        _i, [_vp, _i, _i, _i64, _i64, _vp, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _sz]),
    "fermix_slogpf_planar": (_i, [_vp, _i, _i, _i64, _i64, _i, _vp, _vp, _vp, _vp, _vp, _vp, _sz]),
    "fermix_slogpf_grad_planar": (
        _i, [_vp, _i, _i, _i64, _i64, _i, _vp, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _sz]),
    "fermix_workspace_bytes_planar": (_sz, [_i, _i, _i64, _i64, _i]),
    # include/fermix_b200_block.h
    "fermix_residual_norm": (_i, [_vp, _vp]),
    "fermix_residual_norm_grad": (_i, [_vp, _vp, _vp, _sz]),
    "fermix_residual_norm_grad_workspace_bytes": (_sz, [_vp]),
    "fermix_position_bias": (_i, [_vp, _vp]),
    "fermix_position_bias_grad": (_i, [_vp, _vp, _vp, _sz]),
    "fermix_position_bias_grad_workspace_bytes": (_sz, [_vp]),
    "fermix_biased_attention": (_i, [_vp, _vp, _vp, _sz]),
    "fermix_biased_attention_workspace_bytes": (_sz, [_vp]),
    "fermix_biased_attention_grad": (_i, [_vp, _vp, _vp, _sz]),
    "fermix_biased_attention_grad_workspace_bytes": (_sz, [_vp]),
    # include/fermix_b200_xla.h
    "fermix_xla_custom_call": (None, [_vp, _vp, ctypes.c_char_p, _sz]),
    "fermix_xla_last_error": (_i, [_i]),
}



def _fields(kind, names):
    return [(n, kind) for n in names.split()]


_i32, _f32, _i64x3 = ctypes.c_int32, ctypes.c_float, ctypes.c_int64 * 3


class NormArgs(ctypes.Structure):
    """fx_norm_args (include/fermix_b200_block.h)."""

    _fields_ = (_fields(_i32, "dtype kind gate_mode dgate_f32") + _fields(_f32, "eps") + _fields(_i32, "reserved") + _fields(_i64, "groups rows width") +
                _fields(_vp, "x f gate scale post_weight post_bias pre_weight pre_bias r z grad_r grad_z dx df dgate "
                        "dscale dpost_weight dpost_bias dpre_weight dpre_bias"))


class Buckets(ctypes.Structure):
    """fx_buckets."""

    _fields_ = (_fields(_i32, "num_buckets two_sided num_edges reserved") + _fields(_vp, "edges q_pos k_pos") +
                _fields(_i64, "q_pos_stride k_pos_stride"))


class BiasArgs(ctypes.Structure):
    """fx_bias_args."""

    _fields_ = (_fields(_i32, "dtype reserved") + _fields(_i64, "batch heads q_len k_len") + [("buckets", Buckets)] +
                _fields(_vp, "table out grad dtable"))


class AttnArgs(ctypes.Structure):
    """fx_attn_args."""

    _fields_ = (_fields(_i32, "dtype causal") + _fields(_i64, "batch heads kv_heads q_len k_len dim") +
                _fields(_f32, "scale") + _fields(_i32, "reserved") + [("buckets", Buckets)] +
                _fields(_vp, "q k v table") + _fields(_i64x3, "q_stride k_stride v_stride") +
                _fields(_vp, "key_mask") + _fields(_i64, "mask_stride") + _fields(_vp, "out") +
                _fields(_i64x3, "out_stride") + _fields(_vp, "lse dout") + _fields(_i64x3, "dout_stride") +
                _fields(_vp, "dq dk dv dtable") + _fields(_i64x3, "dq_stride dk_stride dv_stride") + _fields(_vp, "lse_low"))


_lib = None
_lock = threading.Lock()


class FermixError(RuntimeError):
    """A non-zero status from the CUDA library."""


def lib():
    """The loaded library (raises if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise FermixError(
                    f"{LIB_PATH} is missing: build it with `python -m fermix_b200.build` "
                    "(fermix_b200 has no CPU fallback)"
                )
            h = ctypes.CDLL(LIB_PATH)
            for name, (res, args) in SIGNATURES.items():
                fn = getattr(h, name)
                fn.restype = res
                fn.argtypes = args
            _lib = h
    return _lib


def device_status(clear=False):
    """The kernels' status on the current CUDA device (synchronises it): 0, or
    FX_ERR_TIMEOUT when a kernel gave up a bounded wait since the last clear (its members'
    outputs are NaN). Entry points are stream-ordered, so they cannot return it."""
    return lib().fermix_device_status(int(clear))


def check(status):
    if status != 0:
        msg = lib().fermix_strerror(status).decode()
        raise FermixError(f"fermix_b200 error {status}: {msg}")
