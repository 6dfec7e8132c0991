"""ctypes binding of libta_nn.so (include/ta_nn.h): attention with a learned relative position bias, a teacher's top logits and
distillation from them, on gfx950.  ``relative.py`` and ``distill.py`` are the public side; like ``_hip`` this module has no
fallback: a missing library, symbol or device raises.  Calls run on the tensors' device and its current torch stream, allocate
nothing and never synchronise (legal inside ``torch.cuda.graph`` capture)."""
import ctypes
import os

import torch
from torch.autograd import forward_ad

from ._hip import HipExtensionError

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("TA_NN_LIB", os.path.join(_HERE, "lib", "libta_nn.so"))
ABI_VERSION = 1

_i64, _int, _f32, _f64, _vp = ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_double, ctypes.c_void_p

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MASK_NONE, MASK_BOOL, MASK_FLOAT = 0, 1, 2             # MASK_FLOAT + element type


class AttentionArgs(ctypes.Structure):
    """ta_nn_attention_args, field by field"""
    _fields_ = ([(n, _int) for n in ("dtype", "batch", "heads", "kv_heads", "m", "n", "dim")]
                + [(n, _vp) for n in ("q", "k", "v")]
                + [(n, _i64) for n in ("q_sb", "q_sh", "q_sm", "k_sb", "k_sh", "k_sn", "v_sb", "v_sh", "v_sn")]
                + [("scale", _f32), ("table_dtype", _int), ("buckets", _int), ("table", _vp), ("distances", _int), ("first", _int),
                   ("index", _vp), ("index_t", _vp), ("index_stride", _i64), ("index_t_stride", _i64), ("mask_kind", _int),
                   ("mask_period", _int), ("mask", _vp)]
                + [(n, _i64) for n in ("mask_sb", "mask_sh", "mask_sm", "mask_sn")]
                + [("key_lengths", _vp), ("query_start", _vp), ("start", _int), ("causal", _int), ("out", _vp)]
                + [(n, _i64) for n in ("o_sb", "o_sh", "o_sm")]
                + [("stats", _vp), ("workspace", _vp), ("grad", _vp)]
                + [(n, _i64) for n in ("g_sb", "g_sh", "g_sm")]
                + [(n, _vp) for n in ("dq", "dk", "dv")]
                + [(n, _i64) for n in ("dq_sb", "dq_sh", "dq_sm", "dk_sb", "dk_sh", "dk_sn", "dv_sb", "dv_sh", "dv_sn")]
                + [(n, _vp) for n in ("dtable", "pair_order", "pair_starts")])


_args_p = ctypes.POINTER(AttentionArgs)

# name -> (restype, argtypes): mirrors include/ta_nn.h one to one
SIGNATURES = {
    "ta_nn_abi_version": (_int, []),
    "ta_nn_last_error": (ctypes.c_char_p, []),
    "ta_nn_attention_workspace": (_i64, [_args_p, _int]),
    "ta_nn_attention": (_int, [_args_p, _vp]),
    "ta_nn_attention_backward": (_int, [_args_p, _vp]),
    "ta_nn_top_logits": (_int, [_vp, _int, _i64, _i64, _int, _int, _f32, _vp, _vp, _vp, _vp]),
    "ta_nn_distil": (_int, [_vp, _int, _i64, _i64, _int, _vp, _vp, _int, _int, _vp, _vp, _f64, _f32, _vp, _vp, _vp, _vp, _i64, _vp]),
    "ta_nn_distil_backward": (_int, [_vp, _int, _i64, _i64, _int, _vp, _vp, _int, _int, _vp, _vp, _f64, _f32, _vp, _vp, _int, _vp, _vp,
                                     _i64, _vp]),
    "ta_nn_distil_total": (_int, [_vp, _vp, _i64, _int, _vp, _vp, _vp]),
}

_lib = None


def bind(lib):
    for name, (restype, argtypes) in SIGNATURES.items():
        try:
            fn = getattr(lib, name)
        except AttributeError:
            raise HipExtensionError("%s does not export %s (stale build?)" % (LIB_PATH, name))
        fn.restype, fn.argtypes = restype, argtypes
    if lib.ta_nn_abi_version() != ABI_VERSION:
        raise HipExtensionError("libta_nn.so ABI %d, binding %d" % (lib.ta_nn_abi_version(), ABI_VERSION))
    return lib


def load():
    global _lib
    if _lib is None:
        if not os.path.isfile(LIB_PATH):
            raise HipExtensionError("%s is missing: build it with `make -C transferattack_amd/csrc` "
                                    "(python -c 'import __graft_entry__ as g; g.build()')" % LIB_PATH)
        try:
            _lib = bind(ctypes.CDLL(LIB_PATH))
        except OSError as exc:
            raise HipExtensionError("cannot load %s: %s" % (LIB_PATH, exc))
    return _lib


def _check(rc, what):
    if rc != 0:
        raise HipExtensionError("%s failed (rc=%d): %s" % (what, rc, load().ta_nn_last_error().decode("utf-8", "replace")))


def _on_device(t, name):
    if not t.is_cuda:
        raise HipExtensionError("%s is on %s: the HIP path needs tensors on a HIP device (no CPU fallback)" % (name, t.device))


def _launch(name, like, *args):
    fn = getattr(_lib or load(), name)
    dev = like.get_device()
    # (what torch.cuda.current_stream(dev).cuda_stream is, without the objects; torch builds without a GPU do not have it)
    raw_stream = torch._C._cuda_getCurrentRawStream
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):                   # the launch needs the tensor's device current in this thread
            rc = fn(*args, raw_stream(dev))
    else:
        rc = fn(*args, raw_stream(dev))
    if rc != 0:
        _check(rc, name)


def check_tensor(t, name, like=None, dtypes=None):
    """a tensor on a HIP device -- ``like``'s -- of one of ``dtypes``"""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch.Tensor" % name)
    _on_device(t, name)
    if like is not None and t.get_device() != like.get_device():
        raise ValueError("%s is on %s, not on %s" % (name, t.device, like.device))
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError("%s must be %s, got %s" % (name, " or ".join(str(d).replace("torch.", "") for d in dtypes), t.dtype))
    return t


def no_tangents(*tensors):
    """forward-mode derivatives do not pass through the kernels: a dual tensor is refused rather than its tangent dropped"""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("forward-mode derivatives are not implemented for this operator")


def kept(*tensors):
    """what ``ctx.save_for_backward`` takes: it refuses tensors made under ``torch.inference_mode`` (a teacher's answers), whose changes
    nobody counts, so those are copied"""
    return tuple(t.clone() if t is not None and t.is_inference() else t for t in tensors)


def ptr(t):
    return None if t is None else t.data_ptr()
