"""ctypes binding of the C-ABI library ``libsoupb200.so`` (declared in include/soupb200.h).

The library is built in-tree by ``auspex_soup_demo_b200.build``. Loading fails
loudly (:class:`SoupLibraryError`) when it is missing: there is no fallback
implementation. Every call goes to the CUDA stream torch considers current
for the tensor's device.
"""

from __future__ import annotations

import array
import ctypes
import os
import threading

import torch
from torch.autograd import forward_ad

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libsoupb200.so")

SOUP_OK = 0
SOUP_ERR_INVALID = 1
SOUP_ERR_UNSUPPORTED = 2
SOUP_ERR_CUDA = 3
SOUP_ERR_WORKSPACE = 4
SOUP_ERR_DEVICE = 5

F32, F16, BF16 = 0, 1, 2
_DTYPE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


class SoupLibraryError(RuntimeError):
    """The compiled library is missing or does not load."""


class SoupError(RuntimeError):
    """An entry point returned a non-zero status."""

    def __init__(self, fn: str, status: int, detail: str):
        super().__init__(f"{fn} failed with status {status}: {detail}")
        self.status = status


c_i64 = ctypes.c_int64
c_int = ctypes.c_int
c_f = ctypes.c_float
c_d = ctypes.c_double
c_vp = ctypes.c_void_p
c_sz = ctypes.c_size_t
P_I64 = ctypes.POINTER(ctypes.c_int64)

# name -> (restype, argtypes)
_SIGNATURES = {
    "soup_version": (c_int, []),
    "soup_last_error": (ctypes.c_char_p, []),
    "soup_device_error": (c_int, [c_vp, ctypes.POINTER(c_int)]),
    "soup_set_wait_limit_ns": (c_int, [ctypes.c_uint64]),
    "soup_gemm_wait_expiry_check": (c_int, [c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, ctypes.c_uint64,
                                            c_vp]),
    "soup_rmsnorm_fwd": (c_int, [c_vp, c_i64, c_vp, c_vp, c_i64, c_vp, c_i64, c_i64, c_f, c_int,
                                 c_int, c_vp]),
    "soup_rmsnorm_bwd_workspace_bytes": (c_sz, [c_i64, c_i64]),
    "soup_rmsnorm_bwd": (c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_vp, c_vp, c_i64, c_vp, c_vp,
                                 c_sz, c_i64, c_i64, c_int, c_int, c_vp]),
    "soup_rmsnorm_bwd_noalloc": (c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_vp, c_vp, c_i64, c_vp,
                                         c_i64, c_i64, c_int, c_int, c_vp]),
    "soup_swiglu_fwd": (c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_int, c_vp]),
    "soup_swiglu_bwd": (c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_vp, c_i64,
                                c_i64, c_i64, c_int, c_vp]),
    "soup_rope": (c_int, [c_vp, P_I64, c_vp, P_I64, c_i64, c_vp, P_I64, c_vp, P_I64, c_i64, c_vp,
                          c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_int, c_int, c_int, c_vp]),
    "soup_qk_norm_rope": (c_int, [c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp]),
    "soup_qk_norm_rope_bwd_workspace_bytes": (c_sz, [c_i64, c_i64, c_i64, c_i64, c_i64]),
    "soup_qk_norm_rope_bwd": (c_int, [c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp,
                                      c_vp, c_vp, c_sz, c_vp]),
    "soup_tensor_addresses": (c_int, [c_vp, c_vp, c_vp, c_int, c_int, c_int, c_int, c_vp]),
    "soup_grad_square_workspace_bytes": (c_sz, [c_i64]),
    "soup_grad_square": (c_int, [c_vp, c_vp, c_int, c_int, c_vp, c_sz, ctypes.POINTER(c_int), c_vp]),
    "soup_adamw_multi": (c_int, [c_vp, c_vp, c_vp, c_vp, c_int, c_int, c_int, c_vp, c_vp, c_vp, c_vp, c_d, c_d,
                                 c_d, c_d, c_d, c_d, c_vp, c_int, c_vp, c_vp, c_int, c_vp, c_vp]),
    "soup_multi_lora_state_bytes": (c_sz, [c_i64, c_i64, c_i64]),
    "soup_multi_lora_fwd": (c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_vp, c_vp, c_vp, c_vp, c_int, c_i64, c_i64,
                                    c_i64, c_i64, c_i64, c_i64, c_vp, c_i64, c_vp, c_sz, c_vp]),
    "soup_multi_lora_bwd_workspace_bytes": (c_sz, [c_i64, c_i64, c_i64]),
    "soup_multi_lora_bwd": (c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_vp, c_vp, c_vp, c_vp, c_int, c_i64,
                                    c_i64, c_i64, c_i64, c_i64, c_i64, c_vp, c_sz, c_vp, c_i64, c_vp, c_int, c_vp,
                                    c_int, c_vp, c_sz, c_vp]),
    "soup_ce_rows": (c_int, [c_vp, c_i64, c_vp, c_vp, c_vp, c_vp, c_i64, c_i64, c_f, c_i64, c_int,
                             c_int, c_vp]),
    "soup_ce_linear_workspace_bytes": (c_sz, [c_i64, c_i64, c_i64]),
    "soup_ce_linear": (c_int, [c_vp, c_i64, c_vp, c_i64, c_int, c_vp, c_i64, c_vp, c_i64, c_i64,
                               c_i64, c_f, c_i64, c_vp, c_vp, c_vp, c_vp, c_vp, c_int, c_vp, c_int,
                               c_int, c_vp, c_sz, c_vp]),
    "soup_ce_linear_dweight": (c_int, [c_vp, c_sz, c_vp, c_i64, c_int, c_i64, c_i64, c_i64, c_vp,
                                       c_vp, c_int, c_int, c_vp]),
    "soup_ce_vp_workspace_bytes": (c_sz, [c_i64, c_i64, c_i64]),
    "soup_ce_vp_forward": (c_int, [c_vp, c_i64, c_vp, c_i64, c_int, c_vp, c_i64, c_i64, c_i64, c_i64,
                                   c_vp, c_vp, c_sz, c_vp]),
    "soup_ce_vp_combine": (c_int, [c_vp, c_int, c_vp, c_i64, c_i64, c_i64, c_vp, c_vp, c_vp, c_vp,
                                   c_vp, c_vp]),
    "soup_ce_vp_backward": (c_int, [c_vp, c_sz, c_vp, c_i64, c_vp, c_i64, c_int, c_vp, c_i64, c_vp,
                                    c_i64, c_i64, c_i64, c_i64, c_vp, c_f, c_i64, c_vp, c_int, c_vp,
                                    c_int, c_int, c_vp]),
    "soup_set_stage_events": (c_int, [ctypes.POINTER(c_vp), c_int]),
    "soup_attention_fwd": (c_int, [c_vp, P_I64, c_vp, P_I64, c_vp, P_I64, c_i64, c_i64, c_i64, c_i64,
                                   c_i64, c_f, c_int, c_vp, c_vp, c_vp]),
    "soup_attention_bwd_workspace_bytes": (c_sz, [c_i64, c_i64, c_i64]),
    "soup_attention_bwd": (c_int, [c_vp, P_I64, c_vp, P_I64, c_vp, P_I64, c_vp, c_vp, c_vp, c_i64,
                                   c_i64, c_i64, c_i64, c_i64, c_f, c_int, c_vp, c_vp, c_vp, c_vp,
                                   c_sz, c_vp]),
    "soup_attention_window_fwd": (c_int, [c_vp, P_I64, c_vp, P_I64, c_vp, P_I64, c_i64, c_i64, c_i64,
                                          c_i64, c_i64, c_f, c_i64, c_i64, c_vp, c_vp, c_vp]),
    "soup_attention_window_bwd_workspace_bytes": (c_sz, [c_i64, c_i64, c_i64, c_i64, c_i64, c_i64]),
    "soup_attention_window_bwd": (c_int, [c_vp, P_I64, c_vp, P_I64, c_vp, P_I64, c_vp, c_vp, c_vp, c_i64,
                                          c_i64, c_i64, c_i64, c_i64, c_f, c_i64, c_i64, c_vp, c_vp, c_vp,
                                          c_vp, c_sz, c_vp]),
    "soup_head_logps_state_bytes": (c_sz, [c_i64, c_i64, c_i64]),
    "soup_head_logps_workspace_bytes": (c_sz, [c_i64, c_i64, c_i64, c_int]),
    "soup_head_logps_fwd": (c_int, [c_vp, c_i64, c_vp, c_i64, c_int, c_vp, c_i64, c_i64, c_i64, c_i64,
                                    c_vp, c_vp, c_vp, c_sz, c_vp, c_sz, c_vp]),
    "soup_head_logps_bwd": (c_int, [c_vp, c_sz, c_vp, c_i64, c_int, c_vp, c_i64, c_vp, c_i64, c_i64,
                                    c_i64, c_vp, c_int, c_vp, c_int, c_int, c_vp, c_sz, c_vp]),
    "soup_preference_loss_workspace_bytes": (c_sz, [c_i64, c_i64]),
    "soup_preference_loss_fwd": (c_int, [c_vp, c_i64, c_vp, c_i64, c_int, c_vp, c_i64, c_i64, c_i64, c_i64,
                                         c_d, c_d, c_int, c_vp, c_vp, c_vp, c_vp, c_sz, c_vp]),
    "soup_preference_loss_bwd": (c_int, [c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_i64, c_vp, c_vp]),
    "soup_policy_loss_workspace_bytes": (c_sz, [c_i64, c_i64]),
    "soup_policy_loss_fwd": (c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_i64,
                                     c_i64, c_i64, c_d, c_d, c_f, c_int, c_vp, c_vp, c_vp, c_vp, c_vp,
                                     c_vp, c_sz, c_vp]),
    "soup_policy_loss_bwd": (c_int, [c_vp, c_vp, c_vp, c_i64, c_i64, c_vp, c_vp]),
    "soup_swiglu_q8_fwd": (c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_vp, c_vp, c_i64, c_vp, c_vp,
                                   c_i64, c_i64, c_i64, c_int, c_vp]),
    "soup_swiglu_q8_bwd": (c_int, [c_vp, c_i64, c_vp, c_vp, c_i64, c_vp, c_vp, c_i64, c_vp, c_i64, c_vp,
                                   c_i64, c_vp, c_i64, c_i64, c_i64, c_int, c_vp]),
    "soup_q8_quantize": (c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_int, c_vp]),
    "soup_nf4_quantize": (c_int, [c_vp, c_i64, c_int, c_int, ctypes.POINTER(c_f), c_vp, c_vp, c_vp]),
    "soup_nf4_dequant": (c_int, [c_vp, c_vp, c_i64, c_int, ctypes.POINTER(c_f), c_vp, c_int, c_vp]),
    "soup_gemm_stream_k_workspace_bytes": (c_sz, []),
    "soup_gemm_set_stream_k_workspace": (c_int, [c_vp, c_sz]),
    "soup_gemm_set_stream_k_min_saved": (c_int, [c_int]),
    "soup_gemm_bf16": (c_int, [c_vp, c_i64, c_int, c_vp, c_i64, c_int, c_vp, c_i64, c_int, c_i64,
                               c_i64, c_i64, c_f, c_int, c_vp]),
    "soup_gemm_bf16_lora_swiglu": (c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_i64,
                                           c_vp, c_int, c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_i64,
                                           c_vp]),
    "soup_gemm_bf16_lora_dswiglu": (c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_vp, c_i64,
                                            c_i64, c_vp, c_i64, c_i64, c_i64, c_i64, c_vp]),
    "soup_adamw_flat": (c_int, [c_vp, c_vp, c_vp, c_vp, c_i64, c_vp, c_f, c_f, c_f, c_f, c_f, c_vp,
                                c_int, c_i64, c_f, c_vp]),
    "soup_gemm_bf16_lora": (c_int, [c_vp, c_i64, c_int, c_vp, c_i64, c_int, c_vp, c_i64, c_vp, c_i64,
                                    c_i64, c_vp, c_vp, c_i64, c_int, c_i64, c_i64, c_i64, c_f, c_int,
                                    c_vp]),
    "soup_lora_rank_gemm": (c_int, [c_vp, c_i64, c_int, c_vp, c_i64, c_i64, c_i64, c_i64, c_vp, c_i64,
                                    c_vp, c_i64, c_vp, c_i64, c_int, c_f, c_vp]),
    "soup_lora_rank_dual_workspace_bytes": (c_sz, [c_i64, c_i64, c_i64]),
    "soup_lora_rank_dual": (c_int, [c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_i64, c_vp, c_i64,
                                    c_vp, c_i64, c_vp, c_sz, c_vp]),
    "soup_lora_rank_grad_group": (c_int, [c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_i64, c_int, c_int,
                                          c_vp, c_vp, c_vp, c_vp, c_f, c_vp]),
}

_lib = None
_lock = threading.Lock()


def lib() -> ctypes.CDLL:
    """Load (once) and return the library; raise SoupLibraryError if absent."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(LIB_PATH):
            raise SoupLibraryError(
                f"{LIB_PATH} is not built; run `python -m auspex_soup_demo_b200.build` "
                "(nvcc with sm_100a support is required)")
        try:
            handle = ctypes.CDLL(LIB_PATH)
        except OSError as exc:  # pragma: no cover - depends on the host
            raise SoupLibraryError(f"cannot load {LIB_PATH}: {exc}") from exc
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def exported_symbols():
    """Names the binding expects the library to export."""
    return list(_SIGNATURES)


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE[dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {dtype}; expected float32, float16 or bfloat16") from None


def check(fn: str, status: int) -> None:
    if status != SOUP_OK:
        detail = lib().soup_last_error()
        raise SoupError(fn, status, detail.decode() if detail else "")


def stream_of(t: torch.Tensor) -> int:
    """The raw handle of the stream torch considers current for t's device (without
    the Stream object of torch.cuda.current_stream, which costs 3 us a call). A tensor
    that is not on a CUDA device is refused here: its raw handle would be the current
    device's, and the kernel would read host memory."""
    if not t.is_cuda:
        raise ValueError(f"expected a CUDA tensor, got one on {t.device}")
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def once_differentiable(backward):
    """``torch.autograd.function.once_differentiable`` whose checks (3 us a call) run only
    when a graph of the backward itself is asked for (create_graph)."""
    checked = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return (checked if torch.is_grad_enabled() else backward)(ctx, *grads)

    return run


def differentiated(*tensors) -> bool:
    """Whether a call on these tensors (or None) has to go through its autograd Function: a
    gradient is wanted, or forward-mode derivatives may be (tangents do not show in
    requires_grad), which the Function refuses."""
    if forward_ad._current_level >= 0:
        return True
    for t in tensors:
        if t is not None and t.requires_grad:
            return torch.is_grad_enabled()
    return False


def call(fn: str, device: torch.device, *args) -> None:
    """Invoke entry point `fn` with `device` current; raise on failure."""
    f = getattr(lib(), fn)
    if device.index is not None and device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            if fn in _GEMM_ENTRY_POINTS:
                _ensure_stream_k()
            check(fn, f(*args))
    else:
        if fn in _GEMM_ENTRY_POINTS:
            _ensure_stream_k()
        check(fn, f(*args))


# --------------------------------------------------------------------------
# Stream-K scratch of the tcgen05 GEMMs: one zero-filled buffer per device,
# registered with the library before the first GEMM on that device (the
# kernels leave it zero-filled). SOUP_STREAM_K=0 in the environment, or
# set_stream_k(False), runs every GEMM's last wave as a partial wave instead.
# Launches on one device share the buffer, so GEMMs of this library must not
# run concurrently on unordered streams of one device.
# --------------------------------------------------------------------------
STREAM_K = os.environ.get("SOUP_STREAM_K", "1") != "0"
_GEMM_ENTRY_POINTS = {
    "soup_gemm_bf16", "soup_gemm_bf16_lora", "soup_gemm_bf16_lora_swiglu",
    "soup_gemm_bf16_lora_dswiglu", "soup_ce_linear", "soup_ce_linear_dweight",
    "soup_ce_vp_forward", "soup_ce_vp_backward",
}
_sk_buffers = {}  # device index -> registered buffer


def _ensure_stream_k() -> None:
    """Register the current device's stream-K buffer, once. Skipped while a
    CUDA graph is being captured (the zero-fill would become part of the
    graph): launches then run without the stream-K tail."""
    idx = torch.cuda.current_device()
    if idx in _sk_buffers or not STREAM_K:
        return
    if torch.cuda.is_current_stream_capturing():
        return
    with _lock:
        if idx in _sk_buffers:
            return
        nbytes = int(lib().soup_gemm_stream_k_workspace_bytes())
        buf = torch.zeros(nbytes, dtype=torch.uint8, device=torch.device("cuda", idx))
        torch.cuda.synchronize(idx)  # zero before any stream's first GEMM reads it
        check("soup_gemm_set_stream_k_workspace",
              lib().soup_gemm_set_stream_k_workspace(buf.data_ptr(), nbytes))
        _sk_buffers[idx] = buf


def set_stream_k(enabled: bool) -> None:
    """Turn the GEMMs' stream-K tail on or off for later launches (devices with
    a registered buffer; the others get one on their next GEMM when enabled).
    Synchronises those devices first."""
    global STREAM_K
    STREAM_K = bool(enabled)
    for idx, buf in list(_sk_buffers.items()):
        with torch.cuda.device(idx):
            torch.cuda.synchronize(idx)
            if enabled:
                check("soup_gemm_set_stream_k_workspace",
                      lib().soup_gemm_set_stream_k_workspace(buf.data_ptr(), buf.numel()))
            else:
                check("soup_gemm_set_stream_k_workspace", lib().soup_gemm_set_stream_k_workspace(None, 0))


def ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


_table_reader = None


def _reader():
    """(soup_tensor_addresses bound with the interpreter's lock held, its reader: the function
    that fills a DLPack table from a torch tensor, PyList_GetItem, None)"""
    global _table_reader
    if _table_reader is None:
        lib()  # built and loadable
        fn = ctypes.PyDLL(LIB_PATH).soup_tensor_addresses
        fn.restype, fn.argtypes = _SIGNATURES["soup_tensor_addresses"]
        capsule = ctypes.pythonapi.PyCapsule_GetPointer
        capsule.restype, capsule.argtypes = c_vp, [ctypes.py_object, ctypes.c_char_p]
        api = capsule(torch.Tensor.__dlpack_c_exchange_api__, b"dlpack_exchange_api")
        # DLPackExchangeAPI: version (two 32-bit numbers), an older interface, then five
        # functions, of which the fourth fills a DLTensor that does not own anything
        major = ctypes.cast(api, ctypes.POINTER(ctypes.c_uint32))[0]
        read = ctypes.cast(api + 16, ctypes.POINTER(c_vp))[3]
        if major != 1 or not read:
            raise SoupLibraryError(f"torch's DLPack exchange interface has version {major} or cannot fill a DLTensor")
        item = ctypes.cast(ctypes.pythonapi.PyList_GetItem, c_vp).value
        _table_reader = fn, (c_vp * 3)(read, item, id(None))
    return _table_reader


def tensor_addresses(tensors: list, sizes: array.array, code: int, device: torch.device):
    """The addresses (array of 64-bit numbers) of a list of tensors of these sizes (array of
    int64): dense, of one type (its code) and on one device; or the index of the first
    that is not so, or is None. One call for all of them: asking each of hundreds of
    tensors for its size, type, device and layout from Python costs a step more than its
    kernels."""
    fn, reader = _table_reader or _reader()
    n, out = len(sizes), array.array("q", sizes)
    if len(tensors) != n:
        raise ValueError(f"{len(tensors)} tensors and {n} sizes")
    status = fn(reader, id(tensors), sizes.buffer_info()[0], n, code, 2 if device.type == "cuda" else 1, device.index or 0,
                out.buffer_info()[0])
    if status > 0:
        check("soup_tensor_addresses", status)
    return out if status == 0 else -1 - status


def dense(t: torch.Tensor) -> torch.Tensor:
    """t contiguous and 16-byte aligned, copied only if it is not. For tensors that a
    forward saved in that form: a saved-tensor hook (activation offloading) may hand
    back the same values in another layout."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    return t.detach().clone(memory_format=torch.contiguous_format)


def i64_array(values):
    return (ctypes.c_int64 * len(values))(*values)


def device_error(device: torch.device) -> int:
    """Read and clear the device error word (synchronises the current stream).
    After a GEMM wait error (codes 0x101-0x104) the device's stream-K buffer is
    zeroed again, since an aborted launch may have left ready flags set."""
    out = c_int(0)
    with torch.cuda.device(device):
        check("soup_device_error",
              lib().soup_device_error(torch.cuda.current_stream(device).cuda_stream,
                                      ctypes.byref(out)))
        idx = torch.cuda.current_device()
        if 0x101 <= out.value <= 0x104 and _sk_buffers.get(idx) is not None:
            torch.cuda.synchronize(idx)
            _sk_buffers[idx].zero_()
            torch.cuda.synchronize(idx)
    return out.value


# --------------------------------------------------------------------------
# Scratch buffers, one per (device, stream), grown on demand.
# --------------------------------------------------------------------------
_scratch = {}


def scratch(device: torch.device, nbytes: int) -> torch.Tensor:
    """A uint8 device buffer of at least `nbytes` for the current stream."""
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    buf = _scratch.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
        _scratch[key] = buf
    return buf


def release_scratch() -> None:
    _scratch.clear()
