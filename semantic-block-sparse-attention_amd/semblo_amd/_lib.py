"""ctypes binding of libsbsa.so, the C ABI declared in include/sbsa.h.

The library is loaded from ``semblo_amd/_lib/libsbsa.so`` (built in-tree by
``build.py``).  There is no fallback: if the library is missing or a tensor
is not on a ROCm device, the call raises.
"""
from __future__ import annotations

import ctypes
import os
from pathlib import Path

import torch

LIB_PATH = Path(__file__).resolve().parent / "_lib" / "libsbsa.so"

P = ctypes.c_void_p
I64 = ctypes.c_int64
I32 = ctypes.c_int
F32 = ctypes.c_float
SZ = ctypes.c_size_t

# name -> (restype, argtypes), in the order of include/sbsa.h
SIGNATURES = {
    "sbsa_abi_version": (I32, []),
    "sbsa_route_vectors": (I32, [P, I64, I64, I32, I32, P, I64, P]),
    "sbsa_key_space": (I32, [P, I64, I64, I32, I32, P, P, P]),
    "sbsa_kmeans_assign": (I32, [P, I64, P, I64, P, I32, I32, P, P]),
    "sbsa_kmeans_update": (I32, [P, I64, P, I64, P, I32, I32, P, P, P, SZ, P]),
    "sbsa_kmeans_member_bits_bytes": (SZ, [I64, I32]),
    "sbsa_kmeans_iterate": (I32, [P, P, I64, P, I64, I32, I32, P, P, P, P, P, I32, P, P, P, P, SZ,
                                     I32, I32, P]),
    "sbsa_kmeans_centroids": (I32, [I32, P, P, P, P, I64, P, I32, I32, P, P, P]),
    "sbsa_bucket_layout_workspace_bytes": (SZ, [I64, I32]),
    "sbsa_bucket_layout": (I32, [P, I64, I32, I32, P, P, P, I64, P, P, P, SZ, P]),
    "sbsa_kmeans_draw_ints": (I64, [I64, I32, I32, I32]),
    "sbsa_kmeans_draw_scratch_ints": (I64, [I64, I64, I32, I32]),
    "sbsa_kmeans_draws": (I32, [ctypes.c_uint32, I64, I64, I32, I32, I32, P, P]),
    "sbsa_kmeans_draws_after": (I32, [ctypes.c_uint32, I32, I32, I64, I64, I32, I32, I32, P, P]),
    "sbsa_kmeans_fit_workspace_bytes": (SZ, [I64, I64, I32, I32, I32, I32, I32]),
    "sbsa_kmeans_fit": (I32, [P, I64, I64, I64, I32, I32, I32, P, I64, I32, I32, I32, I32, P, P, P, I64, P, P,
                              P, P, SZ, P]),
    "sbsa_kmeans_fit_counted": (I32, [P, I64, I64, I64, I32, I32, I32, P, I64, I32, I32, I32, I32, P, P, P, I64, P,
                                      P, P, P, P, SZ, P]),
    "sbsa_pack_kv": (I32, [P, P, I64, I64, I32, I32, P, I64, I64, P, P]),
    "sbsa_score_select": (I32, [P, I64, I64, P, P, P, I64, I64, I32, I32, I32, I32, I32, I32,
                                F32, F32, F32, I32, I32, P, P, P, P, P, P, P]),
    "sbsa_causal_sizes": (I32, [P, I64, P, P, I32, I32, I64, P, P]),
    "sbsa_reverse_index_ints": (I64, [I32, I32, I32]),
    "sbsa_reverse_index": (I32, [P, I32, I32, I32, P, P, P, P, P, I64, P, P]),
    "sbsa_prefill_items_bound": (I64, [I64, I32, I32, I32, I32]),
    "sbsa_prefill_items_max_queries": (I64, [I32, I32, I32]),
    "sbsa_prefill_items": (I32, [P, I32, I32, I32, I32, I32, P, P, P, P, I64, I64, P, P]),
    "sbsa_plan_chunks": (I32, [P, I64, I64, P, P, I64, P, P, I64, I32, I32, I32, I32, I32, I32, F32, F32, F32, I32,
                               I32, P, P, P, P, P, P, P, P, P, P, I64, I64, I64, P, P]),
    "sbsa_prefill_item_rows": (I32, []),
    "sbsa_prefill_attend": (I32, [P, I64, I64, I32, I32, I32, I32, P, I64, P, P, I64, I64, P, P,
                                  I32, P, P, P, P, P, P, P, I64, I64, P, I64, I64, F32, I32, P]),
    "sbsa_prefill_combine": (I32, [P, P, P, P, P, P, P, I64, I64, P, P, I64, I64, P, I32, I32,
                                   I32, I32, I32, P, P]),
    "sbsa_decode_workspace_bytes": (SZ, [I32, I32, I32, I32, I32, I32]),
    "sbsa_decode_step": (I32, [P, I64, P, I64, I32, P, P, I64, P, P, P, P, P, I64, P, I64, I32, P, I64,
                               I32, P, P, P, I32, I32, I32, I32, F32, F32, F32, I32, I32, F32, I32,
                               I32, P, SZ, P, I64, P, P, P]),
    "sbsa_decode_scratch_bytes": (SZ, []),
    "sbsa_decode_step_noalloc": (I32, [P, I64, P, I64, I32, P, P, I64, P, P, P, P, P, I64, P, I64,
                                       I32, P, I64, I32, P, P, P, I32, I32, I32, I32, F32, F32,
                                       F32, I32, I32, F32, I32, I32, P, I64, P, P, P]),
    "sbsa_nearest_cluster": (I32, [P, I64, I64, I64, I32, I32, I32, P, I32, P, P]),
    "sbsa_append_rows": (I32, [P, I64, I32, I32, P, P, P, P, P, P, P]),
    "sbsa_append_kv": (I32, [P, P, I64, I64, I64, I32, I32, P, I64, P, I64, P, I64, P, I64, P, P,
                             I32, P, P]),
    "sbsa_relayout_runs": (I32, [P, P, I64, I64, I64, I32, I32, P, I64, P, P, I32, P, I64, P, I64,
                                 P, I64, P]),
    "sbsa_gather_rows": (I32, [P, I64, I32, I32, P, I64, I64, I64, P, P, I64, I64, P]),
    "sbsa_repack_runs": (I32, [P, P, I64, I32, I32, I64, P, I64, P, P, I32, P, I64, P, I64, P]),
    "sbsa_rotary": (I32, [P, I64, I64, P, I64, I64, I32, P, I64, I64, P, I64, I64, I32, P, I32, I64, I64, I64, I32,
                          I32, I32, P, P, F32, I32, P]),
    "sbsa_cache8_append": (I32, [P, P, I64, I64, P, I64, I64, I64, P, P, I64, P]),
    "sbsa_cache8_attend_workspace_bytes": (SZ, [P, I32, I64, I64, I32, I32]),
    "sbsa_cache8_attend": (I32, [P, P, I64, I64, I32, I64, P, I64, F32, P, I64, I64, P, I32, P, SZ, P]),
    "sbsa_cache8_evict": (I32, [P, P, P, P, P, P, P, P, I32, I32, I32, I32, I32, I32, P]),
}

ERRORS = {1: "bad argument", 2: "unsupported shape", 3: "kernel launch failed",
          4: "buffer below its capacity bound"}

_LIB = None


def load() -> ctypes.CDLL:
    """Load libsbsa.so once; raise if it was not built."""
    global _LIB
    if _LIB is not None:
        return _LIB
    path = Path(os.environ.get("SBSA_LIB", LIB_PATH))
    if not path.exists():
        raise RuntimeError(
            f"libsbsa.so is not built ({path}); run "
            "`python semantic-block-sparse-attention_amd/build.py` (needs hipcc)")
    lib = ctypes.CDLL(str(path))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _LIB = lib
    return lib


def call(name: str, *args) -> int:
    """Call an entry point; raise RuntimeError on a nonzero status."""
    rc = getattr(load(), name)(*args)
    if rc != 0:
        raise RuntimeError(f"{name} failed: {ERRORS.get(rc, rc)}")
    return rc


def query(name: str, *args):
    """Call a size/bound query (no status code)."""
    return getattr(load(), name)(*args)


def ptr(t: torch.Tensor | None) -> int | None:
    """Device address of a tensor (None for a missing optional tensor)."""
    if t is None:
        return None
    if not t.is_cuda:
        raise RuntimeError("libsbsa works on ROCm device tensors only; got a CPU tensor")
    return t.data_ptr()


# The current device without torch.cuda's check that the GPU is initialised (a tensor of it is there)
_CURRENT_DEVICE = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
# The handle itself, without the Stream object around it (a tenth of the time), where torch has the call
_RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream(device: torch.device | None = None) -> int:
    """The current torch stream's hipStream_t."""
    if _RAW_STREAM is not None and device is not None and device.index is not None:
        return _RAW_STREAM(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def require_device(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("the semblo_amd kernels run on the GPU only (no CPU fallback)")


def require_one_device(first: torch.Tensor, *others: torch.Tensor | None) -> None:
    """Every tensor of a call lies on one ROCm device."""
    require_device(first)
    device = first.get_device()
    for t in others:
        if t is not None and t.get_device() != device:
            raise RuntimeError(f"one call's tensors lie on {first.device} and {t.device}")


def rows_like(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of x's shape [tokens, heads, dim], type and device (``empty`` takes 2.2 us of the host,
    ``empty_like`` 1.2 and ``empty_strided`` 1.3)."""
    if x.is_contiguous():
        return torch.empty_like(x)
    t, h, d = x.shape
    return torch.empty_strided((t, h, d), (h * d, d, 1), dtype=x.dtype, device=x.device)


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two tensors meet."""
    def span(t):
        if t.numel() == 0:
            return 0, 0
        first = t.data_ptr()
        return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def rows_overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether [tokens, heads, dim] tensors share memory: as ``overlap``, but columns of one buffer's rows are told apart."""
    if not overlap(a, b):
        return False
    (st, sh, _), size = a.stride(), a.element_size()
    ends = [((t.shape[1] - 1) * t.stride(1) + t.shape[2]) * size for t in (a, b)]
    at = (b.data_ptr() - a.data_ptr()) % (st * size) if st else 0
    return b.stride(0) != st or at < ends[0] or at + ends[1] > st * size


def call_on(device: torch.device, name: str, *args) -> int:
    """``call`` with the device's current torch stream as the last argument, the device made current
    for the launch where it is not."""
    if device.type != "cuda" or device.index == _CURRENT_DEVICE():
        rc = getattr(_LIB or load(), name)(*args, stream(device))
        if rc != 0:
            raise RuntimeError(f"{name} failed: {ERRORS.get(rc, rc)}")
        return rc
    with torch.cuda.device(device):
        return call(name, *args, stream(device))
