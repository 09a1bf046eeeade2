"""ctypes binding of libdkz.so, the C ABI declared in include/dkz_ops.h, and of
its companions libdkz_dense.so (include/dkz_dense.h) and libdkz_lm.so (include/dkz_lm.h).

This is the Python-side equivalent of the extern declarations a Zig host would
write against the same header. Every exported symbol is listed in SIGNATURES;
tests check the table against the header and the built library.

There is deliberately no fallback: if a library has not been built (or cannot
be loaded), load(), load_dense() and load_lm() raise and nothing runs.
"""

from __future__ import annotations

import ctypes as C
import os
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libdkz.so"
DENSE_LIB_NAME = "libdkz_dense.so"
LM_LIB_NAME = "libdkz_lm.so"

_p = C.c_void_p
_i = C.c_int
_f = C.c_float
_sz = C.c_size_t
_u = C.c_uint
_u64 = C.c_ulonglong

# name -> (restype, argtypes), in the order of include/dkz_ops.h.
SIGNATURES: dict[str, tuple] = {
    "dkz_init": (_i, [_i]),
    "dkz_device_count": (_i, [C.POINTER(_i)]),
    "dkz_device_name": (_i, [_i, C.c_char_p, _i]),
    "dkz_mem_info": (_i, [C.POINTER(_sz), C.POINTER(_sz)]),
    "dkz_malloc": (_i, [C.POINTER(_p), _sz]),
    "dkz_free": (_i, [_p]),
    "dkz_memset_zero": (_i, [_p, _sz]),
    "dkz_copy_to_device": (_i, [_p, _p, _sz]),
    "dkz_copy_to_host": (_i, [_p, _p, _sz]),
    "dkz_synchronize": (_i, []),
    "dkz_error_string": (C.c_char_p, [_i]),
    "dkz_set_sync_after_launch": (None, [_i]),
    "dkz_get_sync_after_launch": (_i, []),
    "dkz_last_error_context": (C.c_char_p, []),
    "dkz_set_stream": (_i, [_p]),
    "dkz_get_stream": (_p, []),
    "dkz_fill": (_i, [_p, _i, _f]),
    "dkz_copy": (_i, [_i, _p, _p]),
    "dkz_axpy": (_i, [_i, _f, _p, _p]),
    "dkz_scal": (_i, [_i, _f, _p]),
    "dkz_mul": (_i, [_i, _p, _p]),
    "dkz_add_scalar": (_i, [_i, _f, _p]),
    "dkz_constrain": (_i, [_i, _f, _p]),
    "dkz_rand_uniform": (_i, [_i, _p, C.c_uint]),
    "dkz_activate_array": (_i, [_p, _i, _i]),
    "dkz_gradient_array": (_i, [_p, _i, _i, _p]),
    "dkz_add_bias": (_i, [_p, _p, _i, _i, _i]),
    "dkz_scale_bias": (_i, [_p, _p, _i, _i, _i]),
    "dkz_backward_bias": (_i, [_p, _p, _i, _i, _i]),
    "dkz_backward_scale": (_i, [_p, _p, _i, _i, _i, _p]),
    "dkz_mean": (_i, [_p, _i, _i, _i, _p]),
    "dkz_variance": (_i, [_p, _p, _i, _i, _i, _p]),
    "dkz_normalize": (_i, [_p, _p, _p, _i, _i, _i]),
    "dkz_mean_delta": (_i, [_p, _p, _i, _i, _i, _p]),
    "dkz_variance_delta": (_i, [_p, _p, _p, _p, _i, _i, _i, _p]),
    "dkz_normalize_delta": (_i, [_p, _p, _p, _p, _p, _i, _i, _i, _p]),
    "dkz_softmax": (_i, [_p, _i, _i, _i, _i, _i, _i, _f, _p]),
    "dkz_softmax_layer_forward": (_i, [_i, _i, _i, _f, _p, _p, _p, _p, _p]),
    "dkz_softmax_cross_entropy": (_i, [_i, _p, _p, _p, _p]),
    "dkz_l2": (_i, [_i, _p, _p, _p, _p]),
    "dkz_l1": (_i, [_i, _p, _p, _p, _p]),
    "dkz_smooth_l1": (_i, [_i, _p, _p, _p, _p]),
    "dkz_forward_maxpool": (_i, [_i, _i, _i, _i, _i, _i, _i, _p, _p, _p]),
    "dkz_backward_maxpool": (_i, [_i, _i, _i, _i, _i, _i, _i, _p, _p, _p]),
    "dkz_forward_avgpool": (_i, [_i, _i, _i, _i, _p, _p]),
    "dkz_backward_avgpool": (_i, [_i, _i, _i, _i, _p, _p]),
    "dkz_shortcut": (_i, [_i, _i, _i, _i, _p, _i, _i, _i, _f, _f, _p]),
    "dkz_im2col": (_i, [_p, _i, _i, _i, _i, _i, _i, _p]),
    "dkz_col2im": (_i, [_p, _i, _i, _i, _i, _i, _i, _p]),
    "dkz_gemm": (_i, [_i, _i, _i, _i, _i, _f, _p, _i, _p, _i, _f, _p, _i]),
    "dkz_convolution_forward": (_i, [_i] * 9 + [_p] * 3),
    "dkz_convolution_weight_gradient": (_i, [_i] * 9 + [_p] * 3),
    "dkz_convolution_data_gradient": (_i, [_i] * 9 + [_p] * 3),
    "dkz_dropout": (_i, [_p, _i, _p, _f, _f]),
    "dkz_adam_update": (_i, [_p, _p, _p, _p, _f, _f, _f, _f, _f, _i, _i, _i]),
    "dkz_batchnorm_forward": (_i, [_i, _i, _i, _i, _i] + [_p] * 10),
    "dkz_batchnorm_backward": (_i, [_i, _i, _i, _i] + [_p] * 11),
    "dkz_batchnorm_backward_noalloc": (_i, [_i, _i, _i, _i] + [_p] * 11),
}

# The same for include/dkz_dense.h.
_drop = [_f, _f, _u, _u64]  # prob, scale, seed, first
DENSE_SIGNATURES: dict[str, tuple] = {
    "dkz_dense_last_error_context": (C.c_char_p, []),
    "dkz_seeded_dropout": (_i, [_i, _i, _p, _p, *_drop, _i, _p]),
    "dkz_linear_forward_workspace": (_i, [_i] * 4 + [C.POINTER(_sz)]),
    "dkz_linear_forward": (_i, [_i] * 5 + _drop + [_p] * 7 + [_sz]),
    "dkz_linear_backward_workspace": (_i, [_i] * 4 + [C.POINTER(_sz)]),
    "dkz_linear_backward": (_i, [_i] * 5 + _drop + [_p] * 5 + [_f] + [_p] * 4 + [_sz]),
    "dkz_linear_cross_entropy_forward_workspace": (_i, [_i] * 4 + [C.POINTER(_sz)] * 2),
    "dkz_linear_cross_entropy_forward": (_i, [_i] * 4 + [_p] * 7 + [_sz]),
    "dkz_linear_cross_entropy_backward_workspace": (_i, [_i] * 4 + [C.POINTER(_sz)] * 2),
    "dkz_linear_cross_entropy_backward": (_i, [_i] * 4 + [_p] * 6 + [_f, _f] + [_p] * 4 + [_sz]),
}

# The same for include/dkz_lm.h.
LM_SIGNATURES: dict[str, tuple] = {
    "dkz_lm_last_error_context": (C.c_char_p, []),
    "dkz_gated_forward_workspace": (_i, [_i] * 4 + [C.POINTER(_sz)]),
    "dkz_gated_forward": (_i, [_i] * 5 + [_p] * 6 + [_sz]),
    "dkz_gated_backward_workspace": (_i, [_i] * 4 + [C.POINTER(_sz)]),
    "dkz_gated_backward": (_i, [_i] * 5 + [_p] * 5 + [_f] + [_p] * 4 + [_sz]),
    "dkz_token_log_probs_workspace": (_i, [_i] * 4 + [C.POINTER(_sz)]),
    "dkz_token_log_probs": (_i, [_i] * 4 + [_p, _f, _i, _p, _i] + [_p] * 6 + [_sz]),
    "dkz_token_log_probs_backward": (_i, [_i] * 4 + [_p, _f, _i] + [_p] * 5 + [_f, _p]),
    "dkz_distillation_workspace": (_i, [_i] * 3 + [C.POINTER(_sz)]),
    "dkz_distillation": (_i, [_i] * 4 + [_p, _f, _i] + [_p] * 3 + [_f] + [_p] * 3 + [_sz]),
}

_LIB: C.CDLL | None = None
_DENSE: C.CDLL | None = None
_LM: C.CDLL | None = None


def _open(p: Path, signatures: dict[str, tuple]) -> C.CDLL:
    if not p.exists():
        raise ImportError(
            f"{p} is not built; the HIP tensor-op libraries are required "
            "(build them with `python -m darknet_zig_amd.build`)"
        )
    lib = C.CDLL(str(p))
    for name, (res, args) in signatures.items():
        fn = getattr(lib, name)  # AttributeError names a missing export
        fn.restype = res
        fn.argtypes = args
    return lib


def _path() -> Path:
    env = os.environ.get("DKZ_LIBRARY")
    return Path(env) if env else LIB_PATH


def load(path: Path | str | None = None) -> C.CDLL:
    """Loads libdkz.so (once) and declares every signature. Raises if absent.

    $DKZ_LIBRARY names another build of the library, as $DARKNET_KERNELS names
    another code object in the reference (gpu.zig:240-244).
    """
    global _LIB
    if _LIB is not None and path is None:
        return _LIB
    lib = _open(Path(path) if path is not None else _path(), SIGNATURES)
    if path is None:
        _LIB = lib
    return lib


def load_dense() -> C.CDLL:
    """Loads libdkz_dense.so (once), which lies beside libdkz.so and shares its
    stream and sync-after-launch switch. Raises if absent."""
    global _DENSE
    if _DENSE is None:
        load()
        _DENSE = _open(_path().resolve().parent / DENSE_LIB_NAME, DENSE_SIGNATURES)
    return _DENSE


def load_lm() -> C.CDLL:
    """Loads libdkz_lm.so (once), as load_dense()."""
    global _LM
    if _LM is None:
        load()
        _LM = _open(_path().resolve().parent / LM_LIB_NAME, LM_SIGNATURES)
    return _LM
