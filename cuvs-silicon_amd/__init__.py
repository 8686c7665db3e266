"""ctypes binding of libcvs_hip (the C ABI declared in include/cvs_hip.h).

Python host code for tests and benchmarks.  It loads the in-tree shared
library built by ``make -C cuvs-silicon_amd`` and raises if it is missing:
there is no CPU fallback.

Errors map like the C++ front-end does (reference src/cagra.cpp:26-32,
:100-111): CVS_ERR_INVALID_ARGUMENT / CVS_ERR_UNSUPPORTED -> ValueError,
everything else -> RuntimeError.
"""
from __future__ import annotations

import array
import ctypes
import os
import sys
import weakref
from ctypes import POINTER, byref, c_char_p, c_double, c_float, c_int, c_int64, c_size_t, c_uint32, c_uint64, c_void_p

import numpy as np

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
LIB_DIR = os.path.join(PKG_DIR, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libcvs_hip.so")
CXX_LIB_PATH = os.path.join(LIB_DIR, "libcuvs_silicon.so")
SYNTH_LIB_PATH = os.path.join(LIB_DIR, "libcvs_synth.so")

CVS_OK = 0
CVS_ERR_INVALID_ARGUMENT = 1
CVS_ERR_RUNTIME = 2
CVS_ERR_NO_DEVICE = 3
CVS_ERR_OUT_OF_MEMORY = 4
CVS_ERR_UNSUPPORTED = 5

BF_MAX_DIM = 16384
BF_MAX_K = 1024
CAGRA_MAX_DIM = 8192
CAGRA_MAX_ITOPK = 512
CAGRA_MAX_WIDTH = 16

# Every extern "C" symbol declared in include/cvs_hip.h: name -> (restype, argtypes).
_SIGNATURES = {
    "cvs_last_error": (c_char_p, []),
    "cvs_dispatch_count": (c_uint64, []),
    "cvs_reset_dispatch_count": (None, []),
    "cvs_device_count": (c_int, [POINTER(c_int)]),
    "cvs_context_create": (c_int, [c_int, POINTER(c_void_p)]),
    "cvs_calibrate_stream_read": (c_int, [c_void_p, c_size_t, c_int, c_int, POINTER(c_double)]),
    "cvs_context_destroy": (c_int, [c_void_p]),
    "cvs_context_synchronize": (c_int, [c_void_p]),
    "cvs_context_device_info": (c_int, [c_void_p, c_char_p, c_size_t, POINTER(c_int), POINTER(c_int64)]),
    "cvs_context_set_timing": (c_int, [c_void_p, c_int]),
    "cvs_context_kernel_time": (c_int, [c_void_p, c_char_p, POINTER(c_double), POINTER(c_uint64)]),
    "cvs_device_alloc": (c_int, [c_void_p, c_size_t, POINTER(c_void_p)]),
    "cvs_device_free": (c_int, [c_void_p, c_void_p]),
    "cvs_copy_to_device": (c_int, [c_void_p, c_void_p, c_void_p, c_size_t]),
    "cvs_copy_to_host": (c_int, [c_void_p, c_void_p, c_void_p, c_size_t]),
    "cvs_dataset_create": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int, POINTER(c_void_p)]),
    "cvs_dataset_destroy": (c_int, [c_void_p]),
    "cvs_dataset_shape": (c_int, [c_void_p, POINTER(c_int64), POINTER(c_int64)]),
    "cvs_dataset_rows": (c_int, [c_void_p, POINTER(c_void_p)]),
    "cvs_bf_search": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_void_p, c_void_p]),
    "cvs_bf_search_async": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_void_p, c_void_p]),
    "cvs_cagra_index_create": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int, c_void_p, c_uint32, c_int,
                                       c_void_p, c_uint32, POINTER(c_void_p)]),
    "cvs_cagra_index_destroy": (c_int, [c_void_p]),
    "cvs_cagra_index_set_traversal": (c_int, [c_void_p, c_int]),
    "cvs_cagra_build_reference": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int, c_uint32, c_void_p, c_int,
                                          c_void_p]),
    "cvs_cagra_build_reference_ex": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int, c_uint32, c_int64, c_int64,
                                             c_void_p, c_int, c_void_p]),
    "cvs_cagra_index_edge_distances": (c_int, [c_void_p, c_void_p, c_void_p, c_int]),
    "cvs_cagra_search_teams": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_uint32, c_uint32, c_uint32,
                                       c_uint32, c_void_p, c_void_p]),
    "cvs_cagra_search_teams_async": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_uint32, c_uint32,
                                             c_uint32, c_uint32, c_void_p, c_void_p]),
    "cvs_cagra_search": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_uint32, c_uint32, c_uint32,
                                 c_void_p, c_void_p]),
    "cvs_cagra_search_async": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_uint32, c_uint32, c_uint32,
                                       c_void_p, c_void_p, c_void_p]),
}

class RefBuildStats(ctypes.Structure):
    _fields_ = [("graph_degree", c_uint32), ("clusters", c_uint32), ("kmeans_iterations", c_uint32),
                ("descent_iterations", c_uint32), ("descent_changed_nodes", c_uint32),
                ("seconds_kmeans", c_double), ("seconds_seed", c_double), ("seconds_descent", c_double),
                ("seconds_total", c_double), ("pq_iterations", c_uint32), ("seconds_pq", c_double)]

    def as_dict(self):
        return {name: getattr(self, name) for name, _ in self._fields_}


class BuildStats(ctypes.Structure):
    """cvs_build_stats (include/cvs_hip.h)."""
    _fields_ = [("iterations", c_uint32), ("intermediate_degree", c_uint32), ("graph_degree", c_uint32),
                ("final_update_rate", c_double), ("seconds_seed", c_double), ("seconds_descent", c_double),
                ("seconds_prune", c_double), ("seconds_total", c_double), ("join_ms", c_double),
                ("join_bytes", c_double), ("join_members", c_uint64), ("updates_emitted", c_uint64),
                ("updates_kept", c_uint64), ("insertions", c_uint64), ("seconds_rescore", c_double)]

    def as_dict(self):
        return {name: getattr(self, name) for name, _ in self._fields_}


_SIGNATURES["cvs_cagra_build"] = (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int, c_uint32, c_uint32, c_uint32,
                                          c_float, c_uint64, c_void_p, c_int, POINTER(BuildStats)])


class BuildOptions(ctypes.Structure):
    """cvs_build_options (include/cvs_hip.h)."""
    _fields_ = [("rescore_fp32", c_int), ("intermediate_out", c_void_p), ("graph_mode", c_int),
                ("reverse_edges", c_uint32)]


GRAPH_DETOUR, GRAPH_KNN = 0, 1


_SIGNATURES["cvs_cagra_build_ex"] = (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int, c_uint32, c_uint32,
                                             c_uint32, c_float, c_uint64, POINTER(BuildOptions), c_void_p, c_int,
                                             POINTER(BuildStats)])

_SIGNATURES["cvs_cagra_optimize"] = (c_int, [c_void_p, c_void_p, c_int64, c_uint32, c_int, c_uint32, c_uint32,
                                             c_void_p, c_int])
_SIGNATURES["cvs_bf_search_noalloc"] = (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_void_p, c_void_p])
_SIGNATURES["cvs_cagra_nav_nodes"] = (c_int, [c_int64, c_void_p, POINTER(c_int64)])
_SIGNATURES["cvs_cagra_entry_points"] = (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_void_p])
_SIGNATURES["cvs_cagra_entry_points_async"] = (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_void_p])
_SIGNATURES["cvs_cagra_search_reference"] = (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_uint32,
                                                     c_uint32, c_void_p, c_void_p, c_void_p])
_SIGNATURES["cvs_cagra_search_reference_async"] = (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_uint32,
                                                           c_uint32, c_void_p, c_void_p, c_void_p])
_SIGNATURES["cvs_calibrate_gather_read"] = (c_int, [c_void_p, c_size_t, c_int64, c_int, c_int, c_int, POINTER(c_double)])
_SIGNATURES["cvs_calibrate_mfma"] = (c_int, [c_void_p, c_void_p, c_size_t, c_int, c_int64, c_int, c_int,
                                             POINTER(c_double)])
_SIGNATURES["cvs_cagra_search_record_async"] = (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_uint32,
                                                        c_uint32, c_uint32, c_void_p, c_void_p, c_void_p, c_void_p,
                                                        c_uint32])
_SIGNATURES["cvs_cagra_replay_gathers"] = (c_int, [c_void_p, c_void_p, c_void_p, c_uint32, c_void_p, c_int64, c_int,
                                                   c_int, POINTER(c_double)])
_SIGNATURES["cvs_context_bf_escalations"] = (c_int, [c_void_p, POINTER(c_uint64), POINTER(c_uint64), c_int])



class Heads(ctypes.Structure):
    """cvs_heads (include/cvs_hip.h)."""
    _fields_ = [("data", c_void_p), ("tokens", c_int64), ("token_stride", c_int64), ("head_stride", c_int64),
                ("heads", c_int), ("head_dim", c_int), ("type", c_int)]


FP16, BF16 = 0, 1
ATTN_MAX_DIM = 128

_HEADS = POINTER(Heads)
_SIGNATURES["cvs_context_create_on_stream"] = (c_int, [c_int, c_void_p, POINTER(c_void_p)])
_SIGNATURES["cvs_context_stream"] = (c_int, [c_void_p, POINTER(c_void_p)])
_SIGNATURES["cvs_prompt_plan_create"] = (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int, c_int, c_int,
                                                 POINTER(c_void_p)])
_SIGNATURES["cvs_prompt_plan_destroy"] = (c_int, [c_void_p])
_SIGNATURES["cvs_prompt_attention_async"] = (c_int, [c_void_p, c_void_p, _HEADS, _HEADS, _HEADS, _HEADS, c_void_p,
                                                     c_float])
_SIGNATURES["cvs_kv_cache_create"] = (c_int, [c_void_p, c_int, c_int64, c_int, c_int, c_int, c_int,
                                              POINTER(c_void_p)])
_SIGNATURES["cvs_kv_cache_destroy"] = (c_int, [c_void_p])
_SIGNATURES["cvs_kv_cache_pages"] = (c_int, [c_void_p, POINTER(c_int64), POINTER(c_int64)])
_SIGNATURES["cvs_kv_sequence_create"] = (c_int, [c_void_p, c_int64, c_void_p])
_SIGNATURES["cvs_kv_sequence_fork"] = (c_int, [c_void_p, c_int64, c_int64, c_int64, c_void_p])
_SIGNATURES["cvs_kv_sequence_extend"] = (c_int, [c_void_p, c_void_p, c_void_p, c_int64])
_SIGNATURES["cvs_kv_sequence_truncate"] = (c_int, [c_void_p, c_int64, c_int64])
_SIGNATURES["cvs_kv_sequence_free"] = (c_int, [c_void_p, c_void_p, c_int64])
_SIGNATURES["cvs_kv_sequence_pages"] = (c_int, [c_void_p, c_void_p, c_int64, c_void_p, c_void_p, c_int64,
                                                POINTER(c_int64)])
_SIGNATURES["cvs_kv_cache_compact"] = (c_int, [c_void_p, POINTER(c_int64)])
_SIGNATURES["cvs_kv_plan_create"] = (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int, POINTER(c_void_p)])
_SIGNATURES["cvs_kv_plan_destroy"] = (c_int, [c_void_p])
_SIGNATURES["cvs_kv_write_async"] = (c_int, [c_void_p, c_void_p, c_int, c_int, _HEADS, c_int64, _HEADS, c_int64])
_SIGNATURES["cvs_kv_read_async"] = (c_int, [c_void_p, c_void_p, c_int, c_int, _HEADS, c_int64, _HEADS, c_int64])
_SIGNATURES["cvs_kv_attention_async"] = (c_int, [c_void_p, c_void_p, c_int, _HEADS, _HEADS, c_void_p, c_float])



class RotaryScaling(ctypes.Structure):
    """cvs_rotary_scaling (include/cvs_hip.h)."""
    _fields_ = [("kind", c_int), ("factor", c_double), ("original_length", c_double), ("low", c_double),
                ("high", c_double)]


class HeadNorm(ctypes.Structure):
    """cvs_head_norm (include/cvs_hip.h)."""
    _fields_ = [("weight", c_void_p), ("type", c_int), ("eps", c_float)]


FP32 = 2
ROTARY_HALVES, ROTARY_NEIGHBOURS = 0, 1
SCALINGS = {None: 0, "linear": 1, "base": 2, "turns": 3}

_NORM = POINTER(HeadNorm)
_SIGNATURES["cvs_rotary_frequencies"] = (c_int, [c_int, c_double, POINTER(RotaryScaling), c_void_p])
_SIGNATURES["cvs_rotary_create"] = (c_int, [c_void_p, c_int, c_int, c_void_p, c_float, POINTER(c_void_p)])
_SIGNATURES["cvs_rotary_destroy"] = (c_int, [c_void_p])
_SIGNATURES["cvs_rotate_async"] = (c_int, [c_void_p, c_void_p, c_void_p, _HEADS, _HEADS])
_SIGNATURES["cvs_norm_rotate_async"] = (c_int, [c_void_p, c_void_p, c_void_p, _HEADS, _HEADS, _NORM, _HEADS, _HEADS,
                                                _NORM])
_SIGNATURES["cvs_kv_append_async"] = (c_int, [c_void_p, c_void_p, c_int, c_void_p, c_void_p, _HEADS, _NORM, _HEADS,
                                              _HEADS, _HEADS, _NORM])


class ScoreOptions(ctypes.Structure):
    """cvs_scores (include/cvs_hip.h)."""
    _fields_ = [("cap", c_float), ("slopes", c_void_p)]


_SCORES = POINTER(ScoreOptions)
_SIGNATURES["cvs_prompt_plan_create_prefix"] = (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int, c_int,
                                                        POINTER(c_void_p)])
_SIGNATURES["cvs_prompt_attention_scored_async"] = (c_int, [c_void_p, c_void_p, _HEADS, _HEADS, _HEADS, _HEADS,
                                                            c_void_p, c_float, _SCORES])
_SIGNATURES["cvs_kv_attention_scored_async"] = (c_int, [c_void_p, c_void_p, c_int, _HEADS, _HEADS, c_void_p, c_float,
                                                        _SCORES])

# The bucketing permutation seed of the reference (src/metal_context.mm:803).
DEFAULT_BUILD_SEED = 0xFEDCBA9876543210

_lib = None


def library_path() -> str:
    return LIB_PATH


def load() -> ctypes.CDLL:
    """Loads libcvs_hip.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with `make -C {PKG_DIR}`")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def exported_symbols():
    return list(_SIGNATURES)


class CvsError(RuntimeError):
    pass


def _check(status: int) -> None:
    if status == CVS_OK:
        return
    msg = load().cvs_last_error().decode()
    if status in (CVS_ERR_INVALID_ARGUMENT, CVS_ERR_UNSUPPORTED):
        raise ValueError(msg)
    raise RuntimeError(f"cvs error {status}: {msg}")


def cagra_nav_nodes(n: int) -> np.ndarray:
    """Navigation (seed) node ids of an n-row graph index, as the
    reference's cagra::build picks them (src/cagra.cpp:63-72)."""
    cnt = c_int64(0)
    _check(load().cvs_cagra_nav_nodes(int(n), None, byref(cnt)))
    out = np.empty(cnt.value, np.uint32)
    _check(load().cvs_cagra_nav_nodes(int(n), out.ctypes.data_as(c_void_p), byref(cnt)))
    return out


def device_count() -> int:
    n = c_int(0)
    _check(load().cvs_device_count(byref(n)))
    return n.value


def dispatch_count() -> int:
    return int(load().cvs_dispatch_count())


def reset_dispatch_count() -> None:
    load().cvs_reset_dispatch_count()


def _f32(a) -> np.ndarray:
    return np.ascontiguousarray(a, dtype=np.float32)


class DeviceArray:
    """A device allocation with numpy shape/dtype bookkeeping."""

    def __init__(self, ctx: "Context", shape, dtype):
        self.ctx = ctx
        self.shape = tuple(int(s) for s in shape)
        self.dtype = np.dtype(dtype)
        self.nbytes = int(np.prod(self.shape)) * self.dtype.itemsize
        p = c_void_p()
        _check(load().cvs_device_alloc(ctx.handle, max(self.nbytes, 1), byref(p)))
        self.ptr = p

    @classmethod
    def from_host(cls, ctx: "Context", host: np.ndarray) -> "DeviceArray":
        host = np.ascontiguousarray(host)
        arr = cls(ctx, host.shape, host.dtype)
        if arr.nbytes:
            _check(load().cvs_copy_to_device(ctx.handle, arr.ptr, host.ctypes.data_as(c_void_p), arr.nbytes))
        return arr

    def to_host(self) -> np.ndarray:
        out = np.empty(self.shape, dtype=self.dtype)
        if self.nbytes:
            _check(load().cvs_copy_to_host(self.ctx.handle, out.ctypes.data_as(c_void_p), self.ptr, self.nbytes))
        return out

    def rows(self, lo: int, hi: int) -> "DeviceArray":
        """A view of rows [lo, hi) of this array: same memory, not owned
        (its free() does nothing); it must not outlive this array."""
        if not 0 <= lo <= hi <= self.shape[0]:
            raise ValueError(f"rows [{lo}, {hi}) outside [0, {self.shape[0]})")
        view = DeviceArray.__new__(DeviceArray)
        view.ctx = self.ctx
        view.shape = (hi - lo,) + self.shape[1:]
        view.dtype = self.dtype
        view.nbytes = int(np.prod(view.shape)) * self.dtype.itemsize
        row_bytes = int(np.prod(self.shape[1:])) * self.dtype.itemsize
        view.ptr = c_void_p(self.ptr.value + lo * row_bytes)
        view._view_of = self
        return view

    def free(self) -> None:
        if getattr(self, "_view_of", None) is not None:
            return
        if self.ptr is not None and self.ctx.handle is not None:
            _check(load().cvs_device_free(self.ctx.handle, self.ptr))
        self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


# Element types of attention operands by the name of their dtype (numpy's and
# torch's); numpy has no bfloat16, so a DeviceArray of uint16 holds those.
_HEAD_TYPES = {"float16": FP16, "torch.float16": FP16, "fp16": FP16, "half": FP16, "uint16": BF16, "bf16": BF16,
               "bfloat16": BF16, "torch.bfloat16": BF16}


def _head_type(dtype) -> int:
    t = _HEAD_TYPES.get(dtype)
    if t is None:
        t = _HEAD_TYPES.get(str(dtype))
        if t is None:
            raise ValueError(f"type {dtype}: attention takes float16 or bfloat16")
        _HEAD_TYPES[dtype] = t  # a torch dtype's name takes longer to make than all else here
    return t


def _no_gradient(what: str) -> None:
    """The calls compute no gradients: a torch tensor that requires grad would
    lose it without a word, and is refused while gradients are recorded."""
    if sys.modules["torch"].is_grad_enabled():
        raise ValueError(f"{what} requires grad, and attention has no backward pass: detach it, or call under no_grad")


def _heads(ctx: "Context", x, what: str, layered: bool = False):
    """The cvs_heads view of a (tokens, heads, head_dim) device array, a
    DeviceArray or a torch tensor on the context's device, whose last axis is
    contiguous; with layered, of (layers, tokens, heads, head_dim) as well.
    Returns (view, layers, layer stride)."""
    shape = x.shape
    if len(shape) == 3:
        layers, layer = 1, 0
        tokens, heads, dim = shape
    elif layered and len(shape) == 4:
        layers, tokens, heads, dim = shape
        layer = None
    else:
        raise ValueError(f"{what} must be (tokens, heads, head_dim)" + (" or (layers, ...)" if layered else ""))
    if isinstance(x, DeviceArray):
        if x.ctx.device != ctx.device:
            raise ValueError(f"{what} must be on the context's device")
        ptr, by_token, by_head = x.ptr.value, heads * dim, dim
        if layer is None:
            layer = tokens * by_token
    elif hasattr(x, "data_ptr"):
        if x.get_device() != ctx.device:  # -1 for a tensor that is on no GPU
            raise ValueError(f"{what} must be on the context's device")
        if x.requires_grad:
            _no_gradient(what)
        if layer is None:
            layer, by_token, by_head, step = x.stride()
        else:
            by_token, by_head, step = x.stride()
        if step != 1 and dim > 1:
            raise ValueError(f"{what}: the last axis must be contiguous")
        ptr = x.data_ptr()
    else:
        raise ValueError(f"{what} must be a DeviceArray or a torch tensor")
    dtype = x.dtype
    kind = _HEAD_TYPES[dtype] if dtype in _HEAD_TYPES else _head_type(dtype)
    return Heads(ptr, tokens, by_token, by_head, heads, dim, kind), layers, layer


def _lse(ctx: "Context", lse, heads: int, tokens: int):
    """Device address of a (heads, tokens) float32 array, or None."""
    if lse is None:
        return None
    if tuple(lse.shape) != (heads, tokens) or str(lse.dtype) not in ("float32", "torch.float32"):
        raise ValueError(f"lse must be a float32 device array of shape {(heads, tokens)}")
    if isinstance(lse, DeviceArray):
        if lse.ctx.device != ctx.device:
            raise ValueError("lse must be on the context's device")
        return lse.ptr
    if not lse.is_cuda or lse.device.index != ctx.device or not lse.is_contiguous():
        raise ValueError("lse must be contiguous and on the context's device")
    if lse.requires_grad:
        _no_gradient("lse")
    return lse.data_ptr()


_KINDS = {}  # dtypes' names: making a torch dtype's takes longer than all else in a call


def _vector(ctx: "Context", x, what: str, length: int, dtypes):
    """Device address of an array of `length` elements of one of `dtypes`,
    contiguous, and which of them."""
    kind = _KINDS.get(x.dtype)
    if kind is None:
        kind = _KINDS[x.dtype] = str(x.dtype).replace("torch.", "")
    shape = x.shape
    if len(shape) != 1 or shape[0] != length or kind not in dtypes:
        raise ValueError(f"{what} must be {length} elements of {' or '.join(dtypes)}, in one dimension")
    if isinstance(x, DeviceArray):
        if x.ctx.device != ctx.device:
            raise ValueError(f"{what} must be on the context's device")
        return x.ptr.value, kind
    if not hasattr(x, "data_ptr"):
        raise ValueError(f"{what} must be a DeviceArray or a torch tensor")
    if x.get_device() != ctx.device:
        raise ValueError(f"{what} must be on the context's device")
    if length > 1 and x.stride(0) != 1:
        raise ValueError(f"{what} must be contiguous")
    if x.requires_grad:
        _no_gradient(what)
    return x.data_ptr(), kind


# A norm's weight: fp32 or the type of the heads.
_WEIGHT_TYPES = {FP16: ("float32", "float16"), BF16: ("float32", "bfloat16", "uint16")}


def _norm(ctx: "Context", weight, heads, eps: float, what: str):
    """The cvs_head_norm of heads, None without a weight."""
    if weight is None:
        return None
    ptr, kind = _vector(ctx, weight, what, heads.head_dim, _WEIGHT_TYPES[heads.type])
    return HeadNorm(ptr, FP32 if kind == "float32" else heads.type, eps)


def _open(rotary):
    """The handle of a rotary, None without one: a closed one's is none as well, but it is no call without rotation."""
    if rotary is None:
        return None
    if rotary.handle is None:
        raise ValueError("the rotary is closed")
    return rotary.handle


def _scores(ctx: "Context", cap: float, slopes, heads: int):
    """The cvs_scores of a call."""
    if slopes is None:
        return ScoreOptions(cap, None)
    return ScoreOptions(cap, _vector(ctx, slopes, "slopes", heads, ("float32",))[0])


def _ready(ctx: "Context", x, out, weight, eps: float, what: str):
    """Heads, their output and norm as C takes them; None, all three, without heads."""
    if x is None:
        if out is not None or weight is not None:
            raise ValueError(f"an output or a weight of {what} without {what}")
        return None, None, None
    if out is None:
        raise ValueError(f"{what} needs {what}_out")
    h = _heads(ctx, x, what)[0]
    return h, _heads(ctx, out, what + "_out")[0], _norm(ctx, weight, h, eps, what + "_weight")


def _raw_stream(torch, device: int) -> int:
    """The address of torch's current stream."""
    try:
        return torch._C._cuda_getCurrentRawStream(device)  # a twentieth of the time of making the stream's object
    except AttributeError:
        return torch.cuda.current_stream(device).cuda_stream


def _i64(a, n=None) -> array.array:
    """A list of whole numbers as 64-bit ones."""
    if n is not None and len(a) != n:
        raise ValueError(f"{n} values are needed, {len(a)} given")
    return array.array("q", a)


def _at(a: array.array):
    """The address of its numbers."""
    return a.buffer_info()[0]


class Context:
    """One device + one HIP stream (C: cvs_context).  stream: None for a
    stream of its own, or the address of a HIP stream of the caller's (a torch
    stream's cuda_stream) that the context works on, in order with the
    caller's own work there.

    Calls on torch tensors are in order with torch's current stream of the
    device: where that is not the context's, the context's waits for what is
    on it before the call, and it waits for the call.  DeviceArrays are in
    order on the context's stream alone."""

    def __init__(self, device: int = 0, stream: int = None):
        h = c_void_p()
        if stream is None:
            _check(load().cvs_context_create(int(device), byref(h)))
        else:
            _check(load().cvs_context_create_on_stream(int(device), c_void_p(int(stream)), byref(h)))
        self.handle = h
        self.device = int(device)
        p = c_void_p()
        _check(load().cvs_context_stream(h, byref(p)))
        self.stream = p.value or 0
        # What was made on this context (datasets, graph indexes, caches,
        # prompt plans): the C library refuses to destroy a context that still
        # owns any, so close() closes the live ones first.
        self._children = weakref.WeakSet()

    def _behind_torch(self, *arrays):
        """Before a call on these arrays: if some are torch tensors and torch's
        current stream is not the context's, the context's stream waits for it.
        Returns what the call has to be followed by: None or a function that
        makes torch's stream wait for the call."""
        for x in arrays:
            if x is not None and not isinstance(x, DeviceArray):
                break
        else:
            return None
        if self.handle is None:
            return None  # closed: the call refuses
        torch = sys.modules["torch"]
        if _raw_stream(torch, self.device) == self.stream:
            return None
        theirs = torch.cuda.current_stream(self.device)
        ours = (torch.cuda.ExternalStream(self.stream, device=self.device) if self.stream
                else torch.cuda.default_stream(self.device))
        ours.wait_stream(theirs)
        return lambda: theirs.wait_stream(ours)

    def _adopt(self, child) -> None:
        self._children.add(child)

    def close(self) -> None:
        if self.handle is not None:
            for child in list(self._children):
                child.close()
            _check(load().cvs_context_destroy(self.handle))
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def synchronize(self) -> None:
        _check(load().cvs_context_synchronize(self.handle))

    def device_info(self):
        name = ctypes.create_string_buffer(256)
        cu = c_int(0)
        mem = c_int64(0)
        _check(load().cvs_context_device_info(self.handle, name, 256, byref(cu), byref(mem)))
        return {"name": name.value.decode(), "compute_units": cu.value, "total_mem_bytes": mem.value}

    def calibrate_stream_read(self, nbytes: int, workgroups: int, reps: int = 20) -> float:
        """Achievable streaming-read rate in GB/s (C: cvs_calibrate_stream_read)."""
        gbs = c_double(0)
        _check(load().cvs_calibrate_stream_read(self.handle, int(nbytes), int(workgroups), int(reps), byref(gbs)))
        return gbs.value

    def calibrate_gather_read(self, row_bytes: int, n_rows: int, workgroups: int, rows_per_team: int,
                              reps: int = 10) -> float:
        """Achievable rate of random whole-row gathers in GB/s (C:
        cvs_calibrate_gather_read)."""
        gbs = c_double(0)
        _check(load().cvs_calibrate_gather_read(self.handle, int(row_bytes), int(n_rows), int(workgroups),
                                                int(rows_per_team), int(reps), byref(gbs)))
        return gbs.value

    def calibrate_mfma(self, data_ptr, nbytes: int, workgroups: int, ksteps: int, from_lds: bool = False,
                       reps: int = 5) -> float:
        """fp16 MFMA rate in TFLOP/s of the large-batch scan's register
        block on the fp16 data at device address data_ptr (an int or a
        c_void_p; C:
        cvs_calibrate_mfma)."""
        tf = c_double(0)
        ptr = data_ptr if isinstance(data_ptr, c_void_p) else c_void_p(int(data_ptr))
        _check(load().cvs_calibrate_mfma(self.handle, ptr, int(nbytes), int(workgroups),
                                         int(ksteps), 1 if from_lds else 0, int(reps), byref(tf)))
        return tf.value

    def set_timing(self, enable: bool) -> None:
        _check(load().cvs_context_set_timing(self.handle, 1 if enable else 0))

    def kernel_time(self, kernel: str):
        """(total_ms, launches) of `kernel` since the last query."""
        ms = c_double(0)
        n = c_uint64(0)
        _check(load().cvs_context_kernel_time(self.handle, kernel.encode(), byref(ms), byref(n)))
        return ms.value, int(n.value)

    def bf_escalations(self, reset: bool = False):
        """(escalated, rescanned): brute-force queries whose fp16 selection
        was not certified and were re-ranked exactly over more rows, and how
        many of those over every row (C: cvs_context_bf_escalations)."""
        esc = c_uint64(0)
        full = c_uint64(0)
        _check(load().cvs_context_bf_escalations(self.handle, byref(esc), byref(full), 1 if reset else 0))
        return int(esc.value), int(full.value)

    def dataset(self, rows) -> "Dataset":
        return Dataset(self, rows)

    def prompt_plan(self, q_lengths, heads: int, kv_heads: int, k_lengths=None, causal: bool = True,
                    prefixes=None) -> "PromptPlan":
        return PromptPlan(self, q_lengths, heads, kv_heads, k_lengths, causal, prefixes)

    def prompt_attention_async(self, plan: "PromptPlan", q, k, v, out, lse=None, scale: float = 0.0, cap: float = 0.0,
                               slopes=None) -> None:
        """Attention over packed sequences (C: cvs_prompt_attention_async):
        q, out (query tokens, heads, head_dim), k, v (key tokens, kv_heads,
        head_dim); lse, when given, (heads, query tokens) float32; scale 0:
        1 / sqrt(head_dim).  Scores are capped to cap * tanh(score / cap) where
        it is not 0, and lose slopes[head] (float32) times their distance."""
        hq, hk, hv, ho = (_heads(self, x, w)[0] for x, w in ((q, "q"), (k, "k"), (v, "v"), (out, "out")))
        hl = _lse(self, lse, hq.heads, hq.tokens)
        sc = _scores(self, cap, slopes, hq.heads) if cap or slopes is not None else None
        after = self._behind_torch(q, k, v, out, lse, slopes)
        _check(load().cvs_prompt_attention_scored_async(self.handle, plan.handle, hq, hk, hv, ho, hl, scale, sc))
        if after:
            after()

    def rotary(self, dims: int, base: float = 10000.0, interleaved: bool = False, scaling: str = None,
               factor: float = 1.0, original_length: float = 0.0, low: float = 1.0, high: float = 32.0,
               magnitude: float = 1.0, frequencies=None) -> "Rotary":
        """Rotary positions of the first `dims` channels of heads: frequencies
        of a base, scaled if need be (rotary_frequencies), or the given ones."""
        if frequencies is None:
            frequencies = rotary_frequencies(dims, base, scaling, factor, original_length, low, high)
        return Rotary(self, dims, frequencies, interleaved, magnitude)

    def rotate_async(self, rotary: "Rotary", positions, x, out) -> None:
        """x (tokens, heads, head_dim) rotated to out, which may be x itself;
        positions (tokens,) int64 (C: cvs_rotate_async)."""
        hx, ho = _heads(self, x, "x")[0], _heads(self, out, "out")[0]
        at = _vector(self, positions, "positions", hx.tokens, ("int64",))[0]
        after = self._behind_torch(positions, x, out)
        _check(load().cvs_rotate_async(self.handle, rotary.handle, at, hx, ho))
        if after:
            after()

    def norm_rotate_async(self, rotary, positions, q, q_out, k=None, k_out=None, q_weight=None, k_weight=None,
                          eps: float = 1e-6) -> None:
        """Queries and keys (tokens, heads, head_dim), normed where they have
        a weight (head_dim,) and rotated where there is a rotary, to their
        outputs in one pass (C: cvs_norm_rotate_async)."""
        hq, hqo, nq = _ready(self, q, q_out, q_weight, eps, "q")
        hk, hko, nk = _ready(self, k, k_out, k_weight, eps, "k")
        if hq is None and hk is None:
            raise ValueError("neither q nor k")
        at = None
        if positions is not None:
            at = _vector(self, positions, "positions", (hq or hk).tokens, ("int64",))[0]
        after = self._behind_torch(q, q_out, k, k_out, q_weight, k_weight, positions)
        _check(load().cvs_norm_rotate_async(self.handle, _open(rotary), at, hq, hqo, nq, hk, hko, nk))
        if after:
            after()

    def kv_cache(self, layers: int, pages: int, page_tokens: int, kv_heads: int, head_dim: int,
                 dtype="bf16") -> "KvCache":
        return KvCache(self, layers, pages, page_tokens, kv_heads, head_dim, dtype)

    def cagra_index(self, rows, graph, seeds=None, traversal_bits: int = 32) -> "CagraIndex":
        return CagraIndex(self, rows, graph, seeds, traversal_bits)

    def cagra_build_reference(self, rows, graph_degree: int = 64, exact_limit: int = None, pq_limit: int = None):
        """The reference's own build algorithm on the GPU (exact seeding for
        n <= 50,000; IVF k-means + per-cluster seeding, random bucketing and
        2-hop nn-descent up to 200,000; product-quantised seeding above).
        exact_limit / pq_limit replace those two sizes (tests).  Returns
        (graph, stats)."""
        st = RefBuildStats()
        rows = _f32(rows)
        n, d = rows.shape
        g = max(min(int(graph_degree), n - 1), 1)
        host = np.empty((n, g), np.uint32)
        if exact_limit is None and pq_limit is None:
            _check(load().cvs_cagra_build_reference(self.handle, rows.ctypes.data_as(c_void_p), n, d, 0,
                                                    int(graph_degree), host.ctypes.data_as(c_void_p), 0, byref(st)))
        else:
            _check(load().cvs_cagra_build_reference_ex(
                self.handle, rows.ctypes.data_as(c_void_p), n, d, 0, int(graph_degree),
                50000 if exact_limit is None else int(exact_limit), 200000 if pq_limit is None else int(pq_limit),
                host.ctypes.data_as(c_void_p), 0, byref(st)))
        return host, st.as_dict()

    def cagra_build(self, rows, intermediate_degree: int = 128, graph_degree: int = 64, max_iterations: int = 20,
                    termination_threshold: float = 0.001, seed: int = DEFAULT_BUILD_SEED, out: "DeviceArray" = None,
                    rescore_fp32: bool = False, intermediate_out: "DeviceArray" = None,
                    graph_mode: int = GRAPH_DETOUR, reverse_edges: int = 0):
        """GPU graph build.  Returns (graph, stats): graph is a host uint32
        array (n, g), or `out` (a device array of that shape) when given.
        rescore_fp32 re-ranks the final intermediate lists by exact fp32
        distances before pruning, intermediate_out (a uint32 device array
        (n, list width)) receives the lists the graph is made from, and
        graph_mode picks how (GRAPH_DETOUR: detour pruning, with the last
        `reverse_edges` kept edges of each row giving way to reverse edges;
        GRAPH_KNN: the nearest graph_degree entries) (cvs_cagra_build_ex)."""
        st = BuildStats()
        if isinstance(rows, DeviceArray):
            n, d = rows.shape
            rptr, rdev = rows.ptr, 1
        else:
            rows = _f32(rows)
            n, d = rows.shape
            rptr, rdev = rows.ctypes.data_as(c_void_p), 0
        g = min(int(graph_degree), max(int(intermediate_degree), int(graph_degree)), n - 1)
        if out is not None:
            if out.shape != (n, g) or out.dtype != np.uint32:
                raise ValueError(f"out must be a uint32 device array of shape {(n, g)}")
            gptr, gdev, host = out.ptr, 1, None
        else:
            host = np.empty((n, max(g, 1)), np.uint32)
            gptr, gdev = host.ctypes.data_as(c_void_p), 0
        if intermediate_out is not None:
            kd = min(max(int(intermediate_degree), int(graph_degree)), n - 1)
            if intermediate_out.shape != (n, kd) or intermediate_out.dtype != np.uint32:
                raise ValueError(f"intermediate_out must be a uint32 device array of shape {(n, kd)}")
        if rescore_fp32 or intermediate_out is not None or graph_mode != GRAPH_DETOUR or reverse_edges:
            opts = BuildOptions(rescore_fp32=int(bool(rescore_fp32)),
                                intermediate_out=intermediate_out.ptr if intermediate_out is not None else None,
                                graph_mode=int(graph_mode), reverse_edges=int(reverse_edges))
            _check(load().cvs_cagra_build_ex(self.handle, rptr, n, d, rdev, int(intermediate_degree),
                                             int(graph_degree), int(max_iterations), float(termination_threshold),
                                             int(seed), byref(opts), gptr, gdev, byref(st)))
        else:
            _check(load().cvs_cagra_build(self.handle, rptr, n, d, rdev, int(intermediate_degree),
                                          int(graph_degree), int(max_iterations), float(termination_threshold),
                                          int(seed), gptr, gdev, byref(st)))
        return (out if out is not None else host), st.as_dict()

    def cagra_optimize(self, knn, graph_degree: int, reverse_edges: int = 0, out: "DeviceArray" = None):
        """Detour pruning of caller k-NN lists (n, width) uint32, nearest
        first, with the last `reverse_edges` kept edges of each row giving way
        to reverse edges (cvs_cagra_optimize).  Returns a host (n,
        graph_degree) uint32 graph, or `out` when given."""
        if isinstance(knn, DeviceArray):
            n, kd = knn.shape
            kptr, kdev = knn.ptr, 1
        else:
            knn = np.ascontiguousarray(knn, np.uint32)
            if knn.ndim != 2:
                raise ValueError("knn must be a 2-D array")
            n, kd = knn.shape
            kptr, kdev = knn.ctypes.data_as(c_void_p), 0
        g = int(graph_degree)
        if out is not None:
            if out.shape != (n, g) or out.dtype != np.uint32:
                raise ValueError(f"out must be a uint32 device array of shape {(n, g)}")
            gptr, gdev, host = out.ptr, 1, None
        else:
            host = np.empty((n, max(g, 1)), np.uint32)
            gptr, gdev = host.ctypes.data_as(c_void_p), 0
        _check(load().cvs_cagra_optimize(self.handle, kptr, int(n), int(kd), kdev, g, int(reverse_edges), gptr,
                                         gdev))
        return out if out is not None else host


class Dataset:
    """Device-resident dataset (C: cvs_dataset)."""

    def __init__(self, ctx: Context, rows):
        self.ctx = ctx
        h = c_void_p()
        if isinstance(rows, DeviceArray):
            n, d = rows.shape
            _check(load().cvs_dataset_create(ctx.handle, rows.ptr, n, d, 1, byref(h)))
        else:
            rows = _f32(rows)
            if rows.ndim != 2:
                raise ValueError("dataset must be a 2-D array")
            n, d = rows.shape
            _check(load().cvs_dataset_create(ctx.handle, rows.ctypes.data_as(c_void_p), n, d, 0, byref(h)))
        self.handle = h
        self.n, self.d = int(n), int(d)
        ctx._adopt(self)

    def close(self) -> None:
        # A dataset dies with its context (Context.close closes it first).
        if self.handle is not None and self.ctx.handle is not None:
            _check(load().cvs_dataset_destroy(self.handle))
        self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def bf_search(self, queries, k: int):
        """Exact k-NN of host queries; returns (neighbors u32 [q,k], distances f32 [q,k])."""
        queries = _f32(queries)
        if queries.ndim != 2 or queries.shape[1] != self.d:
            raise ValueError("queries must be (q, d)")
        q = queries.shape[0]
        nbr = np.empty((q, k), dtype=np.uint32)
        dist = np.empty((q, k), dtype=np.float32)
        _check(load().cvs_bf_search(self.ctx.handle, self.handle, queries.ctypes.data_as(c_void_p), q, int(k),
                                    nbr.ctypes.data_as(c_void_p), dist.ctypes.data_as(c_void_p)))
        return nbr, dist

    def bf_search_noalloc(self, queries: DeviceArray, k: int, nbr: DeviceArray, dist: DeviceArray) -> None:
        """bf_search_async with the library's per-device scratch array
        (cvs_bf_search_noalloc): no device allocation."""
        _check(load().cvs_bf_search_noalloc(self.ctx.handle, self.handle, queries.ptr, queries.shape[0], int(k),
                                            nbr.ptr, dist.ptr))

    def bf_search_async(self, queries: DeviceArray, k: int, nbr: DeviceArray, dist: DeviceArray) -> None:
        _check(load().cvs_bf_search_async(self.ctx.handle, self.handle, queries.ptr, queries.shape[0], int(k),
                                          nbr.ptr, dist.ptr))


class CagraIndex:
    """Device-resident graph index (C: cvs_cagra_index): rows, neighbour lists
    and seed (navigation) node ids."""

    def __init__(self, ctx: Context, rows, graph, seeds=None, traversal_bits: int = 32):
        self.ctx = ctx
        h = c_void_p()
        graph_dev = isinstance(graph, DeviceArray)
        if graph_dev:
            n_g, degree = graph.shape
            gptr = graph.ptr
        else:
            graph = np.ascontiguousarray(graph, np.uint32)
            if graph.ndim != 2:
                raise ValueError("graph must be a 2-D array")
            n_g, degree = graph.shape
            gptr = graph.ctypes.data_as(c_void_p)
        seeds = np.ascontiguousarray(seeds if seeds is not None else np.zeros(0, np.uint32), np.uint32)
        if isinstance(rows, DeviceArray):
            n, d = rows.shape
            rptr, rdev = rows.ptr, 1
        else:
            rows = _f32(rows)
            if rows.ndim != 2:
                raise ValueError("dataset must be a 2-D array")
            n, d = rows.shape
            rptr, rdev = rows.ctypes.data_as(c_void_p), 0
        if n_g != n:
            raise ValueError("graph must have one row per dataset row")
        _check(load().cvs_cagra_index_create(ctx.handle, rptr, n, d, rdev, gptr, degree, 1 if graph_dev else 0,
                                             seeds.ctypes.data_as(c_void_p) if len(seeds) else None, len(seeds),
                                             byref(h)))
        self.handle = h
        self.n, self.d, self.degree = int(n), int(d), int(degree)
        ctx._adopt(self)
        self.set_traversal(traversal_bits)

    def edge_distances(self, out: "DeviceArray" = None):
        """Exact squared L2 length of every graph edge, (n, degree) float32
        (+inf where the entry is not a row id); into `out` (a device array)
        when given, else returned as a host array."""
        if out is not None:
            if out.shape != (self.n, self.degree) or out.dtype != np.float32:
                raise ValueError(f"out must be a float32 device array of shape {(self.n, self.degree)}")
            _check(load().cvs_cagra_index_edge_distances(self.ctx.handle, self.handle, out.ptr, 1))
            return out
        host = np.empty((self.n, self.degree), np.float32)
        _check(load().cvs_cagra_index_edge_distances(self.ctx.handle, self.handle,
                                                     host.ctypes.data_as(c_void_p), 0))
        return host

    def search_record_async(self, queries: DeviceArray, k: int, nbr: DeviceArray, dist: DeviceArray,
                            stats: DeviceArray, record: DeviceArray, itopk_size: int = 64, search_width: int = 1,
                            max_iterations: int = 0) -> None:
        """search_async that also records each query's evaluated row ids
        (C: cvs_cagra_search_record_async); record is (q, cap) uint32."""
        _check(load().cvs_cagra_search_record_async(self.ctx.handle, self.handle, queries.ptr, queries.shape[0],
                                                    int(k), int(itopk_size), int(search_width), int(max_iterations),
                                                    nbr.ptr, dist.ptr, stats.ptr, record.ptr, record.shape[1]))

    def replay_gathers(self, record: DeviceArray, stats: DeviceArray, bits: int, reps: int = 5) -> float:
        """Mean ms of gathering the recorded rows alone (C:
        cvs_cagra_replay_gathers)."""
        ms = c_double(0)
        _check(load().cvs_cagra_replay_gathers(self.ctx.handle, self.handle, record.ptr, record.shape[1], stats.ptr,
                                               record.shape[0], int(bits), int(reps), byref(ms)))
        return ms.value

    def entry_points(self, queries) -> np.ndarray:
        """Per-query entry node: the nearest seed (navigation) node, as the
        reference picks it (C: cvs_cagra_entry_points)."""
        queries = _f32(queries)
        out = np.empty(queries.shape[0], np.uint32)
        _check(load().cvs_cagra_entry_points(self.ctx.handle, self.handle, queries.ctypes.data_as(c_void_p),
                                             queries.shape[0], out.ctypes.data_as(c_void_p)))
        return out

    def search_reference(self, queries, k: int, beam_size: int, max_iter: int, entry_nodes=None):
        """The reference's own beam search (C: cvs_cagra_search_reference):
        one entry node per query (None: the hashed fallback), beam and
        iteration cap as given."""
        queries = _f32(queries)
        q = queries.shape[0]
        ent = None
        if entry_nodes is not None:
            ent = np.ascontiguousarray(entry_nodes, np.uint32)
            if ent.shape != (q,):
                raise ValueError("entry_nodes must hold one id per query")
        nbr = np.empty((q, k), np.uint32)
        dist = np.empty((q, k), np.float32)
        _check(load().cvs_cagra_search_reference(self.ctx.handle, self.handle, queries.ctypes.data_as(c_void_p), q,
                                                 int(k), int(beam_size), int(max_iter),
                                                 None if ent is None else ent.ctypes.data_as(c_void_p),
                                                 nbr.ctypes.data_as(c_void_p), dist.ctypes.data_as(c_void_p)))
        return nbr, dist

    def search_reference_async(self, queries: DeviceArray, k: int, nbr: DeviceArray, dist: DeviceArray,
                               beam_size: int, max_iter: int, entry_nodes: DeviceArray = None) -> None:
        _check(load().cvs_cagra_search_reference_async(self.ctx.handle, self.handle, queries.ptr, queries.shape[0],
                                                       int(k), int(beam_size), int(max_iter),
                                                       None if entry_nodes is None else entry_nodes.ptr, nbr.ptr,
                                                       dist.ptr))

    def entry_points_async(self, queries: DeviceArray, out: DeviceArray) -> None:
        _check(load().cvs_cagra_entry_points_async(self.ctx.handle, self.handle, queries.ptr, queries.shape[0],
                                                   out.ptr))

    def set_traversal(self, bits: int) -> None:
        """16: candidates evaluated on the fp16 copy, final list re-ranked in
        fp32; 32: every evaluation on the fp32 rows."""
        _check(load().cvs_cagra_index_set_traversal(self.handle, int(bits)))
        self.traversal_bits = int(bits)

    def close(self) -> None:
        # An index dies with its context (Context.close closes it first).
        if self.handle is not None and self.ctx.handle is not None:
            _check(load().cvs_cagra_index_destroy(self.handle))
        self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def search(self, queries, k: int, itopk_size: int = 64, search_width: int = 1, max_iterations: int = 0):
        """Graph search of host queries; returns (neighbors u32 [q,k], distances f32 [q,k])."""
        queries = _f32(queries)
        if queries.ndim != 2 or queries.shape[1] != self.d:
            raise ValueError("queries must be (q, d)")
        q = queries.shape[0]
        nbr = np.empty((q, k), dtype=np.uint32)
        dist = np.empty((q, k), dtype=np.float32)
        _check(load().cvs_cagra_search(self.ctx.handle, self.handle, queries.ctypes.data_as(c_void_p), q, int(k),
                                       int(itopk_size), int(search_width), int(max_iterations),
                                       nbr.ctypes.data_as(c_void_p), dist.ctypes.data_as(c_void_p)))
        return nbr, dist

    def search_teams(self, queries, k: int, teams: int, itopk_size: int = 32, search_width: int = 1,
                     max_iterations: int = 0):
        """Multi-team graph search of host queries (C: cvs_cagra_search_teams):
        `teams` searches per query with `itopk_size`-entry lists, merged."""
        queries = _f32(queries)
        if queries.ndim != 2 or queries.shape[1] != self.d:
            raise ValueError("queries must be (q, d)")
        q = queries.shape[0]
        nbr = np.empty((q, k), dtype=np.uint32)
        dist = np.empty((q, k), dtype=np.float32)
        _check(load().cvs_cagra_search_teams(self.ctx.handle, self.handle, queries.ctypes.data_as(c_void_p), q, int(k),
                                             int(itopk_size), int(search_width), int(max_iterations), int(teams),
                                             nbr.ctypes.data_as(c_void_p), dist.ctypes.data_as(c_void_p)))
        return nbr, dist

    def search_teams_async(self, queries: DeviceArray, k: int, nbr: DeviceArray, dist: DeviceArray, teams: int,
                           itopk_size: int = 32, search_width: int = 1, max_iterations: int = 0) -> None:
        _check(load().cvs_cagra_search_teams_async(self.ctx.handle, self.handle, queries.ptr, queries.shape[0], int(k),
                                                   int(itopk_size), int(search_width), int(max_iterations),
                                                   int(teams), nbr.ptr, dist.ptr))

    def search_async(self, queries: DeviceArray, k: int, nbr: DeviceArray, dist: DeviceArray, itopk_size: int = 64,
                     search_width: int = 1, max_iterations: int = 0, stats: DeviceArray | None = None) -> None:
        _check(load().cvs_cagra_search_async(self.ctx.handle, self.handle, queries.ptr, queries.shape[0], int(k),
                                             int(itopk_size), int(search_width), int(max_iterations), nbr.ptr,
                                             dist.ptr, stats.ptr if stats is not None else None))


class PromptPlan:
    """How a batch of packed sequences is worked on, for every layer of a
    model (C: cvs_prompt_plan)."""

    def __init__(self, ctx: Context, q_lengths, heads: int, kv_heads: int, k_lengths=None, causal: bool = True,
                 prefixes=None):
        self.ctx = ctx
        self.handle = None
        n = len(q_lengths)
        h = c_void_p()
        ql, kl = _i64(q_lengths), None if k_lengths is None else _i64(k_lengths, n)
        kl_at = None if kl is None else _at(kl)
        if prefixes is None:
            _check(load().cvs_prompt_plan_create(ctx.handle, _at(ql), kl_at, n, int(heads), int(kv_heads),
                                                 1 if causal else 0, byref(h)))
        else:
            if not causal:
                raise ValueError("prefixes belong to a causal plan")
            seen = _i64(prefixes, n)
            _check(load().cvs_prompt_plan_create_prefix(ctx.handle, _at(ql), kl_at, _at(seen), n, int(heads),
                                                        int(kv_heads), byref(h)))
        self.handle = h
        ctx._adopt(self)

    def close(self) -> None:
        # A plan dies with its context (Context.close closes it first).
        if self.handle is not None and self.ctx.handle is not None:
            _check(load().cvs_prompt_plan_destroy(self.handle))
        self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def rotary_frequencies(dims: int, base: float = 10000.0, scaling: str = None, factor: float = 1.0,
                       original_length: float = 0.0, low: float = 1.0, high: float = 32.0) -> np.ndarray:
    """Radians a position of each pair of channels (C: cvs_rotary_frequencies):
    base^(-2i/dims), for contexts longer than the trained one scaled "linear",
    by "base", or by the "turns" of a pair over original_length positions."""
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {list(SCALINGS)}")
    out = np.empty(max(int(dims), 0) // 2, np.float64)
    _check(load().cvs_rotary_frequencies(int(dims), base, RotaryScaling(SCALINGS[scaling], factor, original_length, low,
                                                                        high), out.ctypes.data))
    return out


class Rotary:
    """Rotary positions of a model's heads (C: cvs_rotary)."""

    def __init__(self, ctx: Context, dims: int, frequencies, interleaved: bool = False, magnitude: float = 1.0):
        self.ctx = ctx
        self.handle = None
        f = np.ascontiguousarray(frequencies, np.float64)
        if f.shape != (max(int(dims), 0) // 2,):
            raise ValueError(f"{dims} channels have {int(dims) // 2} frequencies, {f.shape} given")
        h = c_void_p()
        _check(load().cvs_rotary_create(ctx.handle, int(dims), ROTARY_NEIGHBOURS if interleaved else ROTARY_HALVES,
                                        f.ctypes.data, magnitude, byref(h)))
        self.handle = h
        ctx._adopt(self)

    def close(self) -> None:
        # A rotary dies with its context (Context.close closes it first).
        if self.handle is not None and self.ctx.handle is not None:
            _check(load().cvs_rotary_destroy(self.handle))
        self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class KvCache:
    """Paged cache of attention keys and values whose sequences share pages
    (C: cvs_kv_cache).  Sequences are ids; plans name the newest tokens of
    some of them."""

    def __init__(self, ctx: Context, layers: int, pages: int, page_tokens: int, kv_heads: int, head_dim: int,
                 dtype="bf16"):
        self.ctx = ctx
        self.handle = None
        h = c_void_p()
        _check(load().cvs_kv_cache_create(ctx.handle, int(layers), int(pages), int(page_tokens), int(kv_heads),
                                          int(head_dim), _head_type(dtype), byref(h)))
        self.handle = h
        self.layers, self.kv_heads, self.head_dim = int(layers), int(kv_heads), int(head_dim)
        self.page_tokens = int(page_tokens)
        self._plans = weakref.WeakSet()
        ctx._adopt(self)

    def close(self) -> None:
        # A cache dies with its context (Context.close closes it first), its plans with it.
        if self.handle is not None and self.ctx.handle is not None:
            for plan in list(self._plans):
                plan.close()
            _check(load().cvs_kv_cache_destroy(self.handle))
        self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def free_pages(self) -> int:
        free = c_int64(0)
        _check(load().cvs_kv_cache_pages(self.handle, None, byref(free)))
        return free.value

    def sequences(self, n: int) -> list:
        """n new sequences without tokens."""
        ids = array.array("q", bytes(8 * n))
        _check(load().cvs_kv_sequence_create(self.handle, n, _at(ids)))
        return ids.tolist()

    def sequence(self) -> int:
        return self.sequences(1)[0]

    def fork(self, parent: int, n: int, length: int = -1) -> list:
        """n new sequences of the parent's first `length` tokens (-1: all), on
        its pages."""
        ids = array.array("q", bytes(8 * n))
        _check(load().cvs_kv_sequence_fork(self.handle, int(parent), int(length), n, _at(ids)))
        return ids.tolist()

    def extend(self, seqs, tokens) -> None:
        """Room for tokens[i] more tokens in seqs[i]; RuntimeError and no change
        when the free pages do not suffice."""
        n = len(seqs)
        ids, more = _i64(seqs), _i64(tokens, n)
        _check(load().cvs_kv_sequence_extend(self.handle, _at(ids), _at(more), n))

    def truncate(self, seq: int, length: int) -> None:
        _check(load().cvs_kv_sequence_truncate(self.handle, int(seq), int(length)))

    def free(self, seqs) -> None:
        ids = _i64(seqs)
        _check(load().cvs_kv_sequence_free(self.handle, _at(ids), len(ids)))

    def lengths(self, seqs) -> list:
        ids, out = _i64(seqs), array.array("q", bytes(8 * len(seqs)))
        _check(load().cvs_kv_sequence_pages(self.handle, _at(ids), len(ids), _at(out), None, 0, None))
        return out.tolist()

    def pages(self, seqs) -> np.ndarray:
        """The sequences' page ids, one list behind another."""
        ids, count = _i64(seqs), c_int64(0)
        _check(load().cvs_kv_sequence_pages(self.handle, _at(ids), len(ids), None, None, 0, byref(count)))
        out = np.empty(count.value, np.uint32)
        _check(load().cvs_kv_sequence_pages(self.handle, _at(ids), len(ids), None, out.ctypes.data, count.value, None))
        return out

    def compact(self) -> int:
        """Moves the live pages to the front; returns their number."""
        live = c_int64(0)
        _check(load().cvs_kv_cache_compact(self.handle, byref(live)))
        return live.value

    def plan(self, seqs, tokens, heads: int = 0) -> "KvPlan":
        """The newest tokens[i] tokens of seqs[i] as rows to write, read and,
        with a number of query heads, query."""
        return KvPlan(self, seqs, tokens, heads)

    def _move(self, call, plan, k, v, layer: int) -> None:
        (hk, nk, lk), (hv, nv, lv) = _heads(self.ctx, k, "k", True), _heads(self.ctx, v, "v", True)
        if nk != nv:
            raise ValueError("k and v must have the same layers")
        if nk:
            after = self.ctx._behind_torch(k, v)
            _check(call(self.handle, plan.handle, layer, nk, hk, lk, hv, lv))
            if after:
                after()

    def write_async(self, plan: "KvPlan", k, v, layer: int = 0) -> None:
        """Writes the plan's tokens: k, v (tokens, kv_heads, head_dim) of one
        layer, or (layers, tokens, kv_heads, head_dim) of `layer` and on."""
        self._move(load().cvs_kv_write_async, plan, k, v, layer)

    def read_async(self, plan: "KvPlan", k, v, layer: int = 0) -> None:
        """Reads the plan's tokens into k, v (shapes as write_async)."""
        self._move(load().cvs_kv_read_async, plan, k, v, layer)

    def append_async(self, plan: "KvPlan", k, v, layer: int = 0, rotary: "Rotary" = None, positions=None,
                     k_weight=None, q=None, q_out=None, q_weight=None, eps: float = 1e-6) -> None:
        """Writes the plan's tokens (tokens, kv_heads, head_dim) into a layer,
        keys normed where they have a weight and rotated where there is a
        rotary, at positions (tokens,) int64 or their places in their
        sequences; queries q (tokens, heads, head_dim), made ready in the same
        way, go to q_out (C: cvs_kv_append_async)."""
        hk, hv = _heads(self.ctx, k, "k")[0], _heads(self.ctx, v, "v")[0]
        nk = _norm(self.ctx, k_weight, hk, eps, "k_weight")
        hq, hqo, nq = _ready(self.ctx, q, q_out, q_weight, eps, "q")
        at = None if positions is None else _vector(self.ctx, positions, "positions", hk.tokens, ("int64",))[0]
        after = self.ctx._behind_torch(k, v, q, q_out, k_weight, q_weight, positions)
        _check(load().cvs_kv_append_async(self.handle, plan.handle, layer, _open(rotary), at, hk, nk, hv, hq, hqo, nq))
        if after:
            after()

    def attention_async(self, plan: "KvPlan", q, out, layer: int = 0, lse=None, scale: float = 0.0, cap: float = 0.0,
                        slopes=None) -> None:
        """Attention of the plan's tokens over a layer (C:
        cvs_kv_attention_async): q, out (tokens, heads, head_dim); lse, when
        given, (heads, tokens) float32; scale 0: 1 / sqrt(head_dim); cap and
        slopes as in prompt_attention_async."""
        hq, ho = _heads(self.ctx, q, "q")[0], _heads(self.ctx, out, "out")[0]
        hl = _lse(self.ctx, lse, hq.heads, hq.tokens)
        sc = _scores(self.ctx, cap, slopes, hq.heads) if cap or slopes is not None else None
        after = self.ctx._behind_torch(q, out, lse, slopes)
        _check(load().cvs_kv_attention_scored_async(self.handle, plan.handle, layer, hq, ho, hl, scale, sc))
        if after:
            after()


class KvPlan:
    """The newest tokens of some sequences of a cache (C: cvs_kv_plan)."""

    def __init__(self, cache: KvCache, seqs, tokens, heads: int = 0):
        self.cache = cache
        self.handle = None
        n = len(seqs)
        h = c_void_p()
        ids, newest = _i64(seqs), _i64(tokens, n)
        _check(load().cvs_kv_plan_create(cache.handle, _at(ids), _at(newest), n, int(heads), byref(h)))
        self.handle = h
        cache._plans.add(self)

    def close(self) -> None:
        # A plan dies with its cache (KvCache.close closes it first).
        if self.handle is not None and self.cache.handle is not None and self.cache.ctx.handle is not None:
            _check(load().cvs_kv_plan_destroy(self.handle))
        self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- synthetic data (lib/libcvs_synth.so) ---------------------------------
STREAM_BASE = 1
STREAM_QUERIES = 2
_synth = None


def _synth_lib():
    global _synth
    if _synth is None:
        if not os.path.exists(SYNTH_LIB_PATH):
            raise RuntimeError(f"{SYNTH_LIB_PATH} is missing: build it with `make -C {PKG_DIR}`")
        lib = ctypes.CDLL(SYNTH_LIB_PATH)
        lib.cvs_synth_clustered.restype = None
        lib.cvs_synth_clustered.argtypes = [c_uint64, c_uint32, c_int64, c_int64, c_int64, c_int, c_double, c_void_p]
        lib.cvs_synth_normal.restype = c_double
        lib.cvs_synth_normal.argtypes = [c_uint64, c_uint32, c_uint64, c_uint64]
        _synth = lib
    return _synth


def synth_clustered(seed: int, stream: int, n: int, d: int, n_centers: int = 64, sigma: float = 0.3,
                    row0: int = 0) -> np.ndarray:
    """Rows [row0, row0+n) of the clustered L2-normalised distribution."""
    out = np.empty((int(n), int(d)), dtype=np.float32)
    _synth_lib().cvs_synth_clustered(int(seed), int(stream), int(row0), int(n), int(d), int(n_centers),
                                     float(sigma), out.ctypes.data_as(c_void_p))
    return out


def synth_normal(seed: int, stream: int, row: int, col: int) -> float:
    return float(_synth_lib().cvs_synth_normal(int(seed), int(stream), int(row), int(col)))
