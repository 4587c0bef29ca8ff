"""ctypes binding of the C-ABI library ``libspn.so`` (see ``include/spn.h``).

The product path has NO fallback: if the library is missing or a call fails, a
``RuntimeError`` is raised.  PyTorch tensors only provide device memory and the
current HIP stream; every signature is plain pointers, sizes and strides.
"""
from __future__ import annotations

import ctypes
import os
from typing import Optional

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("SPN_LIB") or os.path.join(_HERE, "libspn.so")   # SPN_LIB: A/B a variant build (tools/)
_lib: Optional[ctypes.CDLL] = None

c_void_p, c_int, c_long, c_float = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float


class SpnError(RuntimeError):
    pass


class SpnMissing(SpnError, AttributeError):
    """The loaded library was built before this entry point was added."""


class _Library(ctypes.CDLL):
    def __getattr__(self, name):
        try:
            return super().__getattr__(name)
        except AttributeError:
            raise SpnMissing(f"{LIB_PATH} has no {name}: rebuild it") from None


def load() -> ctypes.CDLL:
    """Load libspn.so (built by ``scoreperformer_amd.build``); raises if it is absent."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise SpnError(f"{LIB_PATH} not found: run `python -m scoreperformer_amd.build` "
                           f"(the HIP extension is mandatory; there is no fallback path)")
        handle = _Library(LIB_PATH)
        if handle.spn_abi_version() != ABI_VERSION:
            raise SpnError(f"{LIB_PATH} has ABI version {handle.spn_abi_version()}, this package needs {ABI_VERSION}: rebuild it")
        # (a library of the same version built before an entry point was added serves everything else)
        for name, result in _RESULTS.items():
            if hasattr(handle, name):
                getattr(handle, name).restype = result
        for name, types in _SIGNATURES.items():
            if hasattr(handle, name):
                getattr(handle, name).argtypes = types
        _lib = handle
        _apply_env_tuning(_lib)
    return _lib


# Argument types of entry points whose callers pass plain Python numbers and addresses (one conversion in C instead of a ctypes object per
# argument: the calls of a decode step are bound by the host)
_P, _I, _L, _F, _Z = c_void_p, c_int, c_long, c_float, ctypes.c_size_t
_SIGNATURES = {
    "spn_paged_plan": [_P] * 3 + [_L] + [_P] * 5 + [_I] * 5 + [_P, _Z, _P],
    "spn_paged_plan_workspace_bytes": [_I] * 2,
    "spn_paged_release": [_P] * 3 + [_L] + [_P] * 2 + [_I] * 4 + [_P, _P],
    "spn_paged_append": [_P] * 2 + [_I] + [_L] * 4 + [_P] * 2 + [_I, _P, _L] + [_I] * 3 + [_P],
    "spn_paged_attn": [_P, _L, _L, _P, _P, _I, _P, _L, _P, _P, _P, _L, _L] + [_I] * 6 + [_F, _P, _Z, _P],
    "spn_paged_attn_workspace_bytes": [_I] * 6,
    "spn_embed_bwd_det_workspace_floats": [_I] * 2,
}

# what the entry points return that do not return a status
_RESULTS = {
    "spn_last_error": ctypes.c_char_p, "spn_tuning_name": ctypes.c_char_p, "spn_attn_dropbits_elems": c_long, "spn_attn_band_elems": c_long,
    "spn_gemm_workspace_bytes": _Z, "spn_paged_attn_workspace_bytes": _Z, "spn_paged_plan_workspace_bytes": _Z,
    "spn_embed_bwd_det_workspace_floats": c_long,
}

ABI_VERSION = 10
TUNING_EPOCH = 0

# The library itself never reads the environment (include/spn.h): tuning knobs are set explicitly.  For A/B runs from the
# shell this binding maps SPN_<KNOB> variables onto spn_set_tuning once, at load (e.g. SPN_ATTN_BAND=0, SPN_GEMM_VARIANT=9).
_ENV_ALIASES = {"gemm_split_blocks": ("SPN_GEMM_SPLIT_BLOCKS", "SPN_GEMM_PP_SPLIT_BLOCKS")}


def _apply_env_tuning(lib) -> None:
    for i in range(lib.spn_tuning_count()):
        name = lib.spn_tuning_name(c_int(i)).decode()
        for env in _ENV_ALIASES.get(name, ("SPN_" + name.upper(),)):
            val = os.environ.get(env)
            if val is not None:
                lib.spn_set_tuning(name.encode(), ctypes.c_double(float(val)))


def set_tuning(name: str, value: float) -> None:
    """Set a process-wide tuning knob of libspn.so (names: csrc/tuning.h)."""
    lib = load()
    if lib.spn_set_tuning(name.encode(), ctypes.c_double(float(value))) != 0:
        raise SpnError(f"unknown tuning knob {name!r}")
    global TUNING_EPOCH
    TUNING_EPOCH += 1   # shape-keyed host caches that depend on a knob (ops._gemm_ws_bytes) key on it


def get_tuning(name: str) -> float:
    lib = load()
    out = ctypes.c_double(0.0)
    if lib.spn_get_tuning(name.encode(), ctypes.byref(out)) != 0:
        raise SpnError(f"unknown tuning knob {name!r}")
    return out.value


def ptr(t: Optional[torch.Tensor]):
    return c_void_p(0) if t is None else c_void_p(t.data_ptr())


def stream_ptr() -> c_void_p:
    return c_void_p(torch.cuda.current_stream().cuda_stream)


def raw_stream(index: int) -> int:
    """The current stream of GPU `index` as a number (what stream_ptr() wraps, without building a torch.cuda.Stream: 0.1 us instead of 2.9)."""
    return torch._C._cuda_getCurrentRawStream(index)


def call(name: str, *args) -> None:
    lib = load()
    fn = getattr(lib, name)
    rc = fn(*args)
    if rc != 0:
        raise SpnError(f"{name} failed (rc={rc}): {lib.spn_last_error().decode()}")


def require_gpu(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise SpnError("scoreperformer_amd ops run only on an AMD GPU (HIP device tensors); "
                           "there is no CPU fallback in the product path")
