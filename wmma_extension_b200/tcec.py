"""ctypes binding of the C ABI in ``include/tcec.h`` for torch CUDA tensors.

PyTorch is used for device memory and streams only; all arithmetic happens in
the sm_100a kernels of ``libtcec_b200.so``.  There is no CPU or eager fallback:
if the shared library is missing, or no sm_100 device is present, calls raise.

Policy names follow the reference's fragment type and error-correction tags
(``half`` / ``tf32`` x ``with_ec`` / ``without_ec``,
include/wmma_extension/tcec/detail/policy.hpp:12-20).
"""
from __future__ import annotations

import contextlib
import ctypes
import os
import sys
from typing import Optional, Sequence

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libtcec_b200.so")

ROW_MAJOR, COL_MAJOR = 0, 1
POLICIES = {"fp16_ec": 0, "tf32_ec": 1, "fp16_no_ec": 2, "tf32_no_ec": 3}
OK, ERR_INVALID_ARGUMENT, ERR_UNSUPPORTED, ERR_CUDA, ERR_TIMEOUT, ERR_ALLOC, ERR_TOO_LARGE, ERR_COMM = range(8)
COMM_ID_BYTES = 128
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # of the dense operands of products on operands held in few bits

EXPORTED_SYMBOLS = (
    "tcec_sgemm",
    "tcec_sgemm_batched",
    "tcec_sgemm_strided_batched",
    "tcec_packed_bytes",
    "tcec_packed_row_offset",
    "tcec_pack_a",
    "tcec_pack_b",
    "tcec_sgemm_packed",
    "tcec_q4_bytes",
    "tcec_pack_q4",
    "tcec_pack_q4_codes",
    "tcec_unpack_q4",
    "tcec_gemm_q4_workspace_bytes",
    "tcec_gemm_q4",
    "tcec_q8_bytes",
    "tcec_pack_q8",
    "tcec_unpack_q8",
    "tcec_wgrad_q8_workspace_bytes",
    "tcec_wgrad_q8",
    "tcec_split",
    "tcec_cgemm",
    "tcec_sgemm_cublas",
    "tcec_sgemm_batched_cublas",
    "tcec_sgemm_host",
    "tcec_sgemm_multi",
    "tcec_sgemm_batched_multi",
    "tcec_comm_set_library",
    "tcec_comm_unique_id",
    "tcec_comm_init_rank",
    "tcec_comm_destroy",
    "tcec_sgemm_column_shard",
    "tcec_sgemm_column_shard_host",
    "tcec_sgemm_static",
    "tcec_static_scratch_bytes",
    "tcec_static_status",
    "tcec_set_option",
    "tcec_get_option",
    "tcec_device_status",
    "tcec_workspace_bytes",
    "tcec_destroy",
    "tcec_status_string",
    "tcec_version",
)

_lib = None

# The common calls in native code (csrc/tcec_binding.cpp): one 32 x 32 x 32 product, calls in a row, 10.6 -> 6.6 us, 64 rows packed
# and multiplied by packed 4096 x 4096 24.6 -> 22.7.  It answers None to whatever is not plain float32 CUDA tensors of the current
# device, and the code here takes the call.
try:
    from . import _binding

    if _binding.built_for != f"torch {torch.__version__}, Python {sys.version_info[0]}.{sys.version_info[1]}":
        _binding = None  # tensors may be laid out in another way there
except (ImportError, AttributeError):  # not built, or it does not load here: this file does it all
    _binding = None


class TcecError(RuntimeError):
    def __init__(self, status: int, what: str):
        self.status = status
        super().__init__(f"{what}: status {status} ({status_string(status)})")


def load() -> ctypes.CDLL:
    """Load the in-tree shared library; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
            "(there is no fallback path)"
        )
    lib = ctypes.CDLL(LIB_PATH)
    i, ll, f, p, sz = ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_void_p, ctypes.c_size_t
    lib.tcec_sgemm.argtypes = [i, i, i, i, i, i, f, p, ll, p, ll, f, p, ll, i, p]
    lib.tcec_sgemm.restype = i
    lib.tcec_sgemm_batched.argtypes = [i, i, i, i, i, i, f, p, ll, p, ll, f, p, ll, i, i, p]
    lib.tcec_sgemm_batched.restype = i
    lib.tcec_sgemm_strided_batched.argtypes = [i, i, i, i, i, i, f, p, ll, ll, p, ll, ll, f, p, ll, ll, i, i, p]
    lib.tcec_sgemm_strided_batched.restype = i
    lib.tcec_packed_bytes.argtypes = [i, i, i]
    lib.tcec_packed_bytes.restype = sz
    lib.tcec_packed_row_offset.argtypes = [i, i, i]
    lib.tcec_packed_row_offset.restype = sz
    lib.tcec_pack_a.argtypes = [i, i, i, p, ll, p, i, p]
    lib.tcec_pack_a.restype = i
    lib.tcec_pack_b.argtypes = [i, i, i, p, ll, p, i, p]
    lib.tcec_pack_b.restype = i
    lib.tcec_sgemm_packed.argtypes = [i, i, i, i, f, p, p, f, p, ll, i, p]
    lib.tcec_sgemm_packed.restype = i
    fp = ctypes.POINTER(ctypes.c_float)
    lib.tcec_sgemm_cublas.argtypes = [i, i, i, i, i, fp, p, i, p, i, fp, p, i, i, p]
    lib.tcec_sgemm_cublas.restype = i
    lib.tcec_sgemm_batched_cublas.argtypes = [i, i, i, i, i, fp, p, i, p, i, fp, p, i, i, i, p]
    lib.tcec_sgemm_batched_cublas.restype = i
    lib.tcec_sgemm_static.argtypes = [i, i, i, i, i, i, f, p, ll, p, ll, f, p, ll, i, p]
    lib.tcec_sgemm_static.restype = i
    lib.tcec_static_scratch_bytes.argtypes = []
    lib.tcec_static_scratch_bytes.restype = sz
    lib.tcec_static_status.argtypes = [ctypes.POINTER(i)]
    lib.tcec_static_status.restype = i
    lib.tcec_sgemm_host.argtypes = [i, i, i, i, i, i, f, p, ll, p, ll, f, p, ll, i, i, p]
    lib.tcec_sgemm_host.restype = i
    ip, pp, llp = ctypes.POINTER(i), ctypes.POINTER(p), ctypes.POINTER(ll)
    lib.tcec_sgemm_multi.argtypes = [i, ip, i, i, i, i, ip, i, f, p, ll, pp, llp, f, pp, llp, i, pp]
    lib.tcec_sgemm_multi.restype = i
    lib.tcec_sgemm_batched_multi.argtypes = [i, ip, i, i, i, i, i, i, f, pp, ll, ll, pp, ll, ll, f, pp, ll, ll, ip, i, pp]
    lib.tcec_sgemm_batched_multi.restype = i
    lib.tcec_comm_set_library.argtypes = [ctypes.c_char_p]
    lib.tcec_comm_set_library.restype = i
    lib.tcec_comm_unique_id.argtypes = [p]
    lib.tcec_comm_unique_id.restype = i
    lib.tcec_comm_init_rank.argtypes = [i, i, p]
    lib.tcec_comm_init_rank.restype = i
    lib.tcec_comm_destroy.argtypes = []
    lib.tcec_comm_destroy.restype = i
    lib.tcec_sgemm_column_shard.argtypes = [i, i, i, i, i, i, i, f, p, ll, p, ll, f, p, ll, i, p]
    lib.tcec_sgemm_column_shard.restype = i
    lib.tcec_sgemm_column_shard_host.argtypes = [i, i, i, i, i, i, i, f, p, ll, p, ll, f, p, ll, i, i, p]
    lib.tcec_sgemm_column_shard_host.restype = i
    lib.tcec_cgemm.argtypes = [i, i, i, i, i, i, fp, p, ll, p, ll, fp, p, ll, i, p]
    lib.tcec_cgemm.restype = i
    lib.tcec_q4_bytes.argtypes = [i, i, i]
    lib.tcec_q4_bytes.restype = sz
    lib.tcec_pack_q4.argtypes = [i, i, i, p, ll, i, i, i, p, p]
    lib.tcec_pack_q4.restype = i
    lib.tcec_pack_q4_codes.argtypes = [i, i, p, ll, p, i, p, i, p, p]
    lib.tcec_pack_q4_codes.restype = i
    lib.tcec_unpack_q4.argtypes = [i, i, i, p, i, p, ll, i, p]
    lib.tcec_unpack_q4.restype = i
    lib.tcec_gemm_q4_workspace_bytes.argtypes = [i, i, i, i]
    lib.tcec_gemm_q4_workspace_bytes.restype = sz
    lib.tcec_gemm_q4.argtypes = [i, i, i, i, i, f, p, ll, i, p, i, f, p, ll, i, p, sz, p]
    lib.tcec_gemm_q4.restype = i
    lib.tcec_q8_bytes.argtypes = [i, i]
    lib.tcec_q8_bytes.restype = sz
    lib.tcec_pack_q8.argtypes = [i, i, i, p, ll, i, p, p]
    lib.tcec_pack_q8.restype = i
    lib.tcec_unpack_q8.argtypes = [i, i, i, p, p, ll, i, p]
    lib.tcec_unpack_q8.restype = i
    lib.tcec_wgrad_q8_workspace_bytes.argtypes = [i, i, i, i]
    lib.tcec_wgrad_q8_workspace_bytes.restype = sz
    lib.tcec_wgrad_q8.argtypes = [i, i, i, i, i, f, p, ll, i, p, f, p, ll, i, p, sz, p]
    lib.tcec_wgrad_q8.restype = i
    lib.tcec_split.argtypes = [p, p, p, sz, i, p]
    lib.tcec_split.restype = i
    lib.tcec_set_option.argtypes = [ctypes.c_char_p, i]
    lib.tcec_set_option.restype = i
    lib.tcec_get_option.argtypes = [ctypes.c_char_p, ctypes.POINTER(i)]
    lib.tcec_get_option.restype = i
    lib.tcec_device_status.argtypes = [ctypes.POINTER(i)]
    lib.tcec_device_status.restype = i
    lib.tcec_workspace_bytes.argtypes = [i, i, i, i, i]
    lib.tcec_workspace_bytes.restype = sz
    lib.tcec_destroy.argtypes = []
    lib.tcec_destroy.restype = i
    lib.tcec_status_string.argtypes = [i]
    lib.tcec_status_string.restype = ctypes.c_char_p
    lib.tcec_version.argtypes = []
    lib.tcec_version.restype = ctypes.c_char_p
    if _binding is not None:
        _binding.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
            lib.tcec_sgemm, lib.tcec_sgemm_strided_batched, lib.tcec_pack_a, lib.tcec_pack_b, lib.tcec_sgemm_packed,
            lib.tcec_packed_bytes)))
        if hasattr(_binding, "bind_codes"):
            _binding.bind_codes(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
                lib.tcec_q4_bytes, lib.tcec_pack_q4, lib.tcec_unpack_q4, lib.tcec_gemm_q4_workspace_bytes, lib.tcec_gemm_q4, lib.tcec_q8_bytes,
                lib.tcec_pack_q8, lib.tcec_unpack_q8, lib.tcec_wgrad_q8_workspace_bytes, lib.tcec_wgrad_q8)))
    _lib = lib  # last: other threads go into the binding as soon as they see it
    return lib


def status_string(status: int) -> str:
    return load().tcec_status_string(status).decode()


def _check(status: int, what: str) -> None:
    if status != OK:
        raise TcecError(status, what)


def _answer(done, what: str) -> torch.Tensor:
    """What _binding returned: the result, or a status."""
    if done.__class__ is int:
        raise TcecError(done, what)
    return done


def _policy(policy) -> int:
    if isinstance(policy, str):
        return POLICIES[policy]
    return int(policy)


def _layout_ld(t: torch.Tensor):
    """(layout, leading dimension) of a 2-D view, from its strides."""
    r, c = t.shape[-2:]
    s0, s1 = t.stride()[-2:]
    if s1 == 1 and (s0 >= c or r == 1):
        return ROW_MAJOR, max(s0, c)
    if s0 == 1 and (s1 >= r or c == 1):
        return COL_MAJOR, max(s1, r)
    raise ValueError("matrix must have unit stride along rows or columns")


def _require_cuda_f32(*ts: torch.Tensor) -> None:
    for t in ts:
        if not t.is_cuda or t.dtype != torch.float32:
            raise ValueError("operands must be float32 CUDA tensors")


def _require_room(c: torch.Tensor, shape, *operands: torch.Tensor) -> None:
    """`c` holds a result of this shape (a larger one takes it in its first rows and columns), on the operands' device."""
    if c.dim() < len(shape) or any(have < want for have, want in zip(c.shape[-len(shape):], shape)) or 0 in c.shape[:-len(shape)]:
        raise ValueError(f"the result needs {tuple(shape)}, c is {tuple(c.shape)}")
    _require_one_device(c, *operands)


def _require_one_device(first: torch.Tensor, *others: torch.Tensor) -> None:
    if any(t.device != first.device for t in others):
        raise ValueError("operands must be on one device")


def _require_packed(t: torch.Tensor, rows: int, k: int, policy) -> None:
    """`t` is a packed operand of this size, or room for one."""
    if not t.is_cuda or not t.is_contiguous() or t.numel() * t.element_size() < packed_bytes(rows, k, policy):
        raise ValueError(f"a packed operand of {rows} rows and k = {k} takes {packed_bytes(rows, k, policy)} consecutive bytes on a GPU")


# torch's own short ways to the current device and to a device's current stream as a number: a Stream object costs 3 us and a
# device switch 1.5 us of a 12 us call.  They are not public; without them the public ones serve.
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_ptr() -> int:
    """The current stream of the current device."""
    return torch.cuda.current_stream().cuda_stream if _raw_stream is None else _raw_stream(_current_device())


_HERE_ALREADY = contextlib.nullcontext()


def _on(device):
    """Makes `device` current for a call; nothing to do when it is already."""
    return _HERE_ALREADY if getattr(device, "index", None) == _current_device() else torch.cuda.device(device)


def set_option(name: str, value: int) -> None:
    _check(load().tcec_set_option(name.encode(), int(value)), f"tcec_set_option({name})")


def get_option(name: str) -> int:
    v = ctypes.c_int(0)
    _check(load().tcec_get_option(name.encode(), ctypes.byref(v)), f"tcec_get_option({name})")
    return v.value


def device_status() -> int:
    """Synchronise and raise if a kernel gave up a bounded wait."""
    detail = ctypes.c_int(0)
    st = load().tcec_device_status(ctypes.byref(detail))
    if st != OK:
        raise TcecError(st, f"device status word {detail.value}")
    return detail.value


def sgemm(a: torch.Tensor, b: torch.Tensor, c: Optional[torch.Tensor] = None, *, alpha: float = 1.0,
          beta: float = 0.0, policy="fp16_ec") -> torch.Tensor:
    """C = alpha * A @ B + beta * C for 2-D float32 CUDA tensors (row- or column-major views)."""
    if _binding is not None and _lib is not None:
        done = _binding.sgemm(a, b, c, alpha, beta, policy)
        if done is not None:
            return _answer(done, "tcec_sgemm")
    _require_cuda_f32(a, b)
    m, k = a.shape
    k2, n = b.shape
    if k != k2:
        raise ValueError("inner dimensions differ")
    if c is None:
        c = a.new_empty((m, n))
    _require_cuda_f32(c)
    _require_room(c, (m, n), a, b)
    la, lda = _layout_ld(a)
    lb, ldb = _layout_ld(b)
    lc, ldc = _layout_ld(c)
    with _on(a.device):
        st = load().tcec_sgemm(la, lb, lc, m, n, k, alpha, a.data_ptr(), lda, b.data_ptr(), ldb, beta,
                               c.data_ptr(), ldc, _policy(policy), _stream_ptr())
    _check(st, "tcec_sgemm")
    return c


def cgemm(a: torch.Tensor, b: torch.Tensor, c: Optional[torch.Tensor] = None, *, alpha: complex = 1.0,
          beta: complex = 0.0, policy="fp16_ec") -> torch.Tensor:
    """C = alpha * A @ B + beta * C for 2-D complex64 CUDA tensors (row- or column-major views)."""
    for t in (a, b) + ((c,) if c is not None else ()):
        if not t.is_cuda or t.dtype != torch.complex64:
            raise ValueError("operands must be complex64 CUDA tensors")
    m, k = a.shape
    k2, n = b.shape
    if k != k2:
        raise ValueError("inner dimensions differ")
    if c is None:
        c = a.new_empty((m, n))
    _require_room(c, (m, n), a, b)
    la, lda = _layout_ld(a)
    lb, ldb = _layout_ld(b)
    lc, ldc = _layout_ld(c)
    al = (ctypes.c_float * 2)(complex(alpha).real, complex(alpha).imag)
    be = (ctypes.c_float * 2)(complex(beta).real, complex(beta).imag)
    with _on(a.device):
        st = load().tcec_cgemm(la, lb, lc, m, n, k, al, a.data_ptr(), lda, b.data_ptr(), ldb, be,
                               c.data_ptr(), ldc, _policy(policy), _stream_ptr())
    _check(st, "tcec_cgemm")
    return c


def sgemm_static(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, *, alpha: float = 1.0, beta: float = 0.0,
                 policy="fp16_ec") -> torch.Tensor:
    """``sgemm`` through the entry point that allocates nothing (``tcec_sgemm_static``).

    For callers that cannot allocate device memory when they need the product; the split
    operands go to a fixed array inside the library, so the problem must fit it
    (``TcecError`` with ``ERR_TOO_LARGE`` otherwise) and ``c`` must be supplied.  Calls that
    overlap on the GPU share that array and race: keep them on one stream.
    """
    _require_cuda_f32(a, b, c)
    m, k = a.shape
    k2, n = b.shape
    if k != k2 or tuple(c.shape) != (m, n):
        raise ValueError("shape mismatch")
    la, lda = _layout_ld(a)
    lb, ldb = _layout_ld(b)
    lc, ldc = _layout_ld(c)
    with _on(a.device):
        st = load().tcec_sgemm_static(la, lb, lc, m, n, k, alpha, a.data_ptr(), lda, b.data_ptr(), ldb, beta,
                                      c.data_ptr(), ldc, _policy(policy), _stream_ptr())
    _check(st, "tcec_sgemm_static")
    return c


def static_status() -> int:
    """Synchronise and raise if a kernel launched by ``sgemm_static`` gave up a bounded wait."""
    detail = ctypes.c_int(0)
    st = load().tcec_static_status(ctypes.byref(detail))
    if st != OK:
        raise TcecError(st, f"static status word {detail.value}")
    return detail.value


def sgemm_strided_batched(a: torch.Tensor, b: torch.Tensor, c: Optional[torch.Tensor] = None, *,
                          alpha: float = 1.0, beta: float = 0.0, policy="fp16_ec") -> torch.Tensor:
    """Batched product of 3-D tensors [batch, m, k] x [batch, k, n] with a uniform batch stride."""
    if _binding is not None and _lib is not None:
        done = _binding.strided(a, b, c, alpha, beta, policy)
        if done is not None:
            return _answer(done, "tcec_sgemm_strided_batched")
    _require_cuda_f32(a, b)
    batch, m, k = a.shape
    _, k2, n = b.shape
    if k != k2 or b.shape[0] != batch:
        raise ValueError("shape mismatch")
    if c is None:
        c = a.new_empty((batch, m, n))
    _require_cuda_f32(c)
    _require_room(c, (batch, m, n), a, b)
    la, lda = _layout_ld(a)
    lb, ldb = _layout_ld(b)
    lc, ldc = _layout_ld(c)
    with _on(a.device):
        st = load().tcec_sgemm_strided_batched(
            la, lb, lc, m, n, k, alpha, a.data_ptr(), lda, a.stride(0), b.data_ptr(), ldb, b.stride(0), beta,
            c.data_ptr(), ldc, c.stride(0), batch, _policy(policy), _stream_ptr())
    _check(st, "tcec_sgemm_strided_batched")
    return c


def sgemm_batched(a_list: Sequence[torch.Tensor], b_list: Sequence[torch.Tensor],
                  c_list: Sequence[torch.Tensor], *, alpha: float = 1.0, beta: float = 0.0,
                  policy="fp16_ec") -> Sequence[torch.Tensor]:
    """Pointer-array batch: one independent matrix per list entry, equal shapes and strides."""
    batch = len(a_list)
    if batch == 0:
        return c_list
    _require_cuda_f32(*a_list, *b_list, *c_list)
    m, k = a_list[0].shape
    _, n = b_list[0].shape
    la, lda = _layout_ld(a_list[0])
    lb, ldb = _layout_ld(b_list[0])
    lc, ldc = _layout_ld(c_list[0])
    dev = a_list[0].device

    def ptrs(ts):
        return torch.tensor([t.data_ptr() for t in ts], dtype=torch.int64).to(dev)

    pa, pb, pc = ptrs(a_list), ptrs(b_list), ptrs(c_list)
    with _on(dev):
        st = load().tcec_sgemm_batched(la, lb, lc, m, n, k, alpha, pa.data_ptr(), lda, pb.data_ptr(), ldb, beta,
                                       pc.data_ptr(), ldc, batch, _policy(policy), _stream_ptr())
        _check(st, "tcec_sgemm_batched")
        # the pointer tables must outlive the kernels that read them
        torch.cuda.current_stream().synchronize()
    return c_list


def packed_bytes(rows: int, k: int, policy="fp16_ec") -> int:
    return int(load().tcec_packed_bytes(rows, k, _policy(policy)))


def packed_row_offset(row: int, k: int, policy="fp16_ec") -> int:
    return int(load().tcec_packed_row_offset(row, k, _policy(policy)))


def pack_a(a: torch.Tensor, policy="fp16_ec", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Split A (m x k) once into operand panels; returns the uint8 panel buffer."""
    if _binding is not None and _lib is not None:
        done = _binding.pack_a(a, policy, out)
        if done is not None:
            return _answer(done, "tcec_pack_a")
    _require_cuda_f32(a)
    m, k = a.shape
    la, lda = _layout_ld(a)
    if out is None:
        out = a.new_empty(packed_bytes(m, k, policy), dtype=torch.uint8)
    _require_packed(out, m, k, policy)
    _require_one_device(a, out)
    with _on(a.device):
        st = load().tcec_pack_a(la, m, k, a.data_ptr(), lda, out.data_ptr(), _policy(policy), _stream_ptr())
    _check(st, "tcec_pack_a")
    return out


def pack_b(b: torch.Tensor, policy="fp16_ec", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Split B (k x n) once into operand panels; returns the uint8 panel buffer."""
    if _binding is not None and _lib is not None:
        done = _binding.pack_b(b, policy, out)
        if done is not None:
            return _answer(done, "tcec_pack_b")
    _require_cuda_f32(b)
    k, n = b.shape
    lb, ldb = _layout_ld(b)
    if out is None:
        out = b.new_empty(packed_bytes(n, k, policy), dtype=torch.uint8)
    _require_packed(out, n, k, policy)
    _require_one_device(b, out)
    with _on(b.device):
        st = load().tcec_pack_b(lb, k, n, b.data_ptr(), ldb, out.data_ptr(), _policy(policy), _stream_ptr())
    _check(st, "tcec_pack_b")
    return out


def sgemm_packed(a_packed: torch.Tensor, b_packed: torch.Tensor, m: int, n: int, k: int,
                 c: Optional[torch.Tensor] = None, *, alpha: float = 1.0, beta: float = 0.0,
                 policy="fp16_ec") -> torch.Tensor:
    """C = alpha * A @ B + beta * C on operands packed by pack_a / pack_b."""
    if _binding is not None and _lib is not None:
        done = _binding.sgemm_packed(a_packed, b_packed, m, n, k, c, alpha, beta, policy)
        if done is not None:
            return _answer(done, "tcec_sgemm_packed")
    if c is None:
        c = torch.empty((m, n), dtype=torch.float32, device=a_packed.device)
    _require_cuda_f32(c)
    _require_packed(a_packed, m, k, policy)
    _require_packed(b_packed, n, k, policy)
    _require_room(c, (m, n), a_packed, b_packed)
    lc, ldc = _layout_ld(c)
    with _on(c.device):
        st = load().tcec_sgemm_packed(lc, m, n, k, alpha, a_packed.data_ptr(), b_packed.data_ptr(), beta,
                                      c.data_ptr(), ldc, _policy(policy), _stream_ptr())
    _check(st, "tcec_sgemm_packed")
    return c


# ---------------------------------------------------------------- operands held in few bits
def _dense_type(t: torch.Tensor, what: str) -> int:
    """The type of a dense operand: a matrix in float32, float16 or bfloat16 on a GPU."""
    if not t.is_cuda or t.dtype not in TYPES or t.dim() != 2:
        raise ValueError(f"{what} must be a float32, float16 or bfloat16 CUDA matrix")
    return TYPES[t.dtype]


def _result_type(dtype: torch.dtype, operand: torch.Tensor) -> int:
    if dtype != operand.dtype and dtype != torch.float32:
        raise ValueError(f"the result is float32 or of the operand's type {operand.dtype}, not {dtype}")
    return TYPES[dtype]


def _exact_result(c: Optional[torch.Tensor], shape, dtype: Optional[torch.dtype], operand: torch.Tensor, beta: float) -> torch.Tensor:
    """`c` as given, or a new one of `dtype` (the operand's type by default)."""
    if c is None:
        if beta != 0.0:
            raise ValueError("beta needs a c")
        return operand.new_empty(shape, dtype=dtype or operand.dtype)
    if dtype is not None and c.dtype != dtype:
        raise ValueError(f"c is {c.dtype}, not {dtype}")
    if not c.is_cuda or tuple(c.shape) != tuple(shape):
        raise ValueError(f"c must be a CUDA matrix of {tuple(shape)}")
    _require_one_device(c, operand)
    return c


def _require_extents(*sizes: int) -> None:
    """The library counts rows and columns in 32 bits; ctypes would cut off the rest."""
    if any(not 0 <= s <= 0x7FFFFFFF for s in sizes):
        raise ValueError(f"sizes must be 0 to 2147483647, not {sizes}")


def _require_bytes(t: torch.Tensor, need: int, what: str) -> None:
    if not t.is_cuda or not t.is_contiguous() or t.numel() * t.element_size() < need:
        raise ValueError(f"{what} takes {need} consecutive bytes on a GPU")


def _scratch(need: int, device) -> Optional[torch.Tensor]:
    """From torch's allocator, so that a captured graph has its own."""
    return torch.empty(need, dtype=torch.uint8, device=device) if need else None


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def q4_bytes(n: int, k: int, group: int = 128) -> int:
    """Bytes of weights (n x k) packed by pack_q4 or pack_q4_codes."""
    if group not in (32, 64, 128):
        raise ValueError("group must be 32, 64 or 128")
    _require_extents(n, k)
    return int(load().tcec_q4_bytes(n, k, group))


def pack_q4(w: torch.Tensor, group: int = 128, scale: torch.dtype = torch.float16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Weights w (n x k, outputs first) in 4 bits, with a scale (float16 or bfloat16) and a zero point for every `group` of k.

    Returns the uint8 buffer that gemm_q4 takes.  Every value is brought to the nearest of its group's 16 steps
    (``tcec_pack_q4``); unpack_q4 gives the values that the codes stand for.
    """
    if _binding is not None and _lib is not None:
        done = _binding.pack_q4(w, group, scale, out)
        if done is not None:
            return _answer(done, "tcec_pack_q4")
    kind = _dense_type(w, "w")
    if scale not in (torch.float16, torch.bfloat16):
        raise ValueError("scale must be float16 or bfloat16")
    n, k = w.shape
    need = q4_bytes(n, k, group)
    lw, ldw = _layout_ld(w)
    if out is None:
        out = torch.empty(need, dtype=torch.uint8, device=w.device)
    _require_bytes(out, need, "packed weights of this size")
    _require_one_device(w, out)
    with _on(w.device):
        st = load().tcec_pack_q4(lw, n, k, w.data_ptr(), ldw, kind, group, TYPES[scale], out.data_ptr(), _stream_ptr())
    _check(st, "tcec_pack_q4")
    return out


def pack_q4_codes(codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, *, k: int, group: int = 128,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Lays out 4-bit codes that exist already: w[j, i] = scales[j, i // group] * (code - zeros[j, i // group]).

    ``codes``: uint8 [n, ceil(k / 2)], the code of an even i in the low half of its byte; ``scales``: float16 or bfloat16
    [n, ceil(k / group)]; ``zeros``: uint8 of the same shape, or None for 8.
    """
    if not codes.is_cuda or codes.dtype != torch.uint8 or codes.dim() != 2 or k < 0 or codes.shape[1] != (k + 1) // 2:
        raise ValueError("codes must be a uint8 CUDA matrix of ceil(k / 2) columns")
    n = codes.shape[0]
    need = q4_bytes(n, k, group)
    shape = (n, -(-k // group))
    if not scales.is_cuda or scales.dtype not in (torch.float16, torch.bfloat16) or tuple(scales.shape) != shape:
        raise ValueError(f"scales must be a float16 or bfloat16 CUDA matrix of {shape}")
    if zeros is not None and (not zeros.is_cuda or zeros.dtype != torch.uint8 or tuple(zeros.shape) != shape):
        raise ValueError(f"zeros must be a uint8 CUDA matrix of {shape}")
    if codes.stride(1) != 1 or (n > 1 and codes.stride(0) < codes.shape[1]):
        codes = codes.contiguous()
    scales = scales.contiguous()
    zeros = None if zeros is None else zeros.contiguous()
    if out is None:
        out = torch.empty(need, dtype=torch.uint8, device=codes.device)
    _require_bytes(out, need, "packed weights of this size")
    _require_one_device(codes, scales, out, *(() if zeros is None else (zeros,)))
    with _on(codes.device):
        st = load().tcec_pack_q4_codes(n, k, codes.data_ptr(), max(codes.stride(0), codes.shape[1]), scales.data_ptr(),
                                       TYPES[scales.dtype], _ptr(zeros), group, out.data_ptr(), _stream_ptr())
    _check(st, "tcec_pack_q4_codes")
    return out


def unpack_q4(packed: torch.Tensor, n: int, k: int, group: int = 128, dtype: torch.dtype = torch.float32,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The weights (n x k) that a packed buffer stands for, rounded to the result's type."""
    if _binding is not None and _lib is not None:
        done = _binding.unpack_q4(packed, n, k, group, dtype, out)
        if done is not None:
            return _answer(done, "tcec_unpack_q4")
    need = q4_bytes(n, k, group)
    _require_bytes(packed, need, "packed weights of this size")
    if out is None:
        out = torch.empty((n, k), dtype=dtype, device=packed.device)
    kind = _dense_type(out, "the result")
    if tuple(out.shape) != (n, k):
        raise ValueError(f"the result must be {(n, k)}")
    _require_one_device(packed, out)
    lw, ldw = _layout_ld(out)
    with _on(packed.device):
        st = load().tcec_unpack_q4(lw, n, k, packed.data_ptr(), group, out.data_ptr(), ldw, kind, _stream_ptr())
    _check(st, "tcec_unpack_q4")
    return out


def gemm_q4(x: torch.Tensor, packed: torch.Tensor, n: int, c: Optional[torch.Tensor] = None, *, group: int = 128, alpha: float = 1.0,
            beta: float = 0.0, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """C = alpha * X @ W^T + beta * C for X (m x k, float32, float16 or bfloat16) and weights W (n x k) packed by pack_q4.

    From one token to a whole prompt.  The result is of X's type, or of ``dtype`` (X's or float32).
    """
    if _binding is not None and _lib is not None:
        done = _binding.gemm_q4(x, packed, n, c, group, alpha, beta, dtype)
        if done is not None:
            return _answer(done, "tcec_gemm_q4")
    kind = _dense_type(x, "x")
    m, k = x.shape
    _require_extents(m)
    need = q4_bytes(n, k, group)
    _require_bytes(packed, need, "packed weights of this size")
    c = _exact_result(c, (m, n), dtype, x, beta)
    kind_c = _result_type(c.dtype, x)
    _require_one_device(x, packed)
    lx, ldx = _layout_ld(x)
    lc, ldc = _layout_ld(c)
    lib = load()
    with _on(x.device):
        need = int(lib.tcec_gemm_q4_workspace_bytes(m, n, k, kind))
        scratch = _scratch(need, x.device)
        st = lib.tcec_gemm_q4(lx, lc, m, n, k, alpha, x.data_ptr(), ldx, kind, packed.data_ptr(), group, beta, c.data_ptr(), ldc, kind_c,
                              _ptr(scratch), need, _stream_ptr())
    _check(st, "tcec_gemm_q4")
    return c


def q8_bytes(m: int, k: int) -> int:
    """Bytes of activations (m x k) packed by pack_q8."""
    _require_extents(m, k)
    return int(load().tcec_q8_bytes(m, k))


def pack_q8(x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Activations x (m tokens x k features) in 8 bits, with a scale for every 128 tokens of a feature, to be kept for wgrad_q8."""
    if _binding is not None and _lib is not None:
        done = _binding.pack_q8(x, out)
        if done is not None:
            return _answer(done, "tcec_pack_q8")
    kind = _dense_type(x, "x")
    m, k = x.shape
    need = q8_bytes(m, k)
    lx, ldx = _layout_ld(x)
    if out is None:
        out = torch.empty(need, dtype=torch.uint8, device=x.device)
    _require_bytes(out, need, "packed activations of this size")
    _require_one_device(x, out)
    with _on(x.device):
        st = load().tcec_pack_q8(lx, m, k, x.data_ptr(), ldx, kind, out.data_ptr(), _stream_ptr())
    _check(st, "tcec_pack_q8")
    return out


def unpack_q8(packed: torch.Tensor, m: int, k: int, dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The activations (m x k) that a packed buffer stands for, rounded to the result's type."""
    if _binding is not None and _lib is not None:
        done = _binding.unpack_q8(packed, m, k, dtype, out)
        if done is not None:
            return _answer(done, "tcec_unpack_q8")
    _require_bytes(packed, q8_bytes(m, k), "packed activations of this size")
    if out is None:
        out = torch.empty((m, k), dtype=dtype, device=packed.device)
    kind = _dense_type(out, "the result")
    if tuple(out.shape) != (m, k):
        raise ValueError(f"the result must be {(m, k)}")
    _require_one_device(packed, out)
    lx, ldx = _layout_ld(out)
    with _on(packed.device):
        st = load().tcec_unpack_q8(lx, m, k, packed.data_ptr(), out.data_ptr(), ldx, kind, _stream_ptr())
    _check(st, "tcec_unpack_q8")
    return out


def wgrad_q8(dy: torch.Tensor, packed: torch.Tensor, k: int, c: Optional[torch.Tensor] = None, *, alpha: float = 1.0, beta: float = 0.0,
             dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """C = alpha * dY^T @ X + beta * C: the gradient (n x k) of a layer's weights from the gradient dY (m x n, float32, float16 or
    bfloat16) of its outputs and its input X (m x k), kept by pack_q8.  beta = 1 adds up over batches.

    The result is of dY's type, or of ``dtype`` (dY's or float32).
    """
    if _binding is not None and _lib is not None:
        done = _binding.wgrad_q8(dy, packed, k, c, alpha, beta, dtype)
        if done is not None:
            return _answer(done, "tcec_wgrad_q8")
    kind = _dense_type(dy, "dy")
    m, n = dy.shape
    _require_extents(n)
    _require_bytes(packed, q8_bytes(m, k), "packed activations of this size")
    c = _exact_result(c, (n, k), dtype, dy, beta)
    kind_c = _result_type(c.dtype, dy)
    _require_one_device(dy, packed)
    ly, ldy = _layout_ld(dy)
    lc, ldc = _layout_ld(c)
    lib = load()
    with _on(dy.device):
        need = int(lib.tcec_wgrad_q8_workspace_bytes(m, n, k, kind))
        scratch = _scratch(need, dy.device)
        st = lib.tcec_wgrad_q8(ly, lc, m, n, k, alpha, dy.data_ptr(), ldy, kind, packed.data_ptr(), beta, c.data_ptr(), ldc, kind_c,
                               _ptr(scratch), need, _stream_ptr())
    _check(st, "tcec_wgrad_q8")
    return c


def _require_host_f32(*ts: torch.Tensor) -> None:
    for t in ts:
        if t.is_cuda or t.dtype != torch.float32:
            raise ValueError("host operands must be float32 CPU tensors")


def sgemm_host(a_host: torch.Tensor, b_host: torch.Tensor, c_host: torch.Tensor, *, alpha: float = 1.0,
               beta: float = 0.0, policy="fp16_ec", panel_rows: int = 0,
               device: Optional[torch.device] = None) -> torch.Tensor:
    """C = alpha * A @ B + beta * C for operands in (pinned) HOST memory, through ``tcec_sgemm_host``.

    B is copied and split once; A travels in row panels, so that the copy-in of panel p+1, the
    GEMM on panel p and the copy-out of panel p-1 overlap on three streams.  The call returns
    when everything is queued: ``c_host`` is complete once the current CUDA stream has reached
    the end of the call's work (synchronise it before reading).
    """
    _require_host_f32(a_host, b_host, c_host)
    m, k = a_host.shape
    k2, n = b_host.shape
    if k != k2 or tuple(c_host.shape) != (m, n):
        raise ValueError("shape mismatch")
    la, lda = _layout_ld(a_host)
    lb, ldb = _layout_ld(b_host)
    lc, ldc = _layout_ld(c_host)
    torch.cuda.init()
    dev = device or torch.device("cuda", torch.cuda.current_device())
    with _on(dev):
        st = load().tcec_sgemm_host(la, lb, lc, m, n, k, alpha, a_host.data_ptr(), lda, b_host.data_ptr(), ldb, beta,
                                    c_host.data_ptr(), ldc, _policy(policy), int(panel_rows), _stream_ptr())
    _check(st, "tcec_sgemm_host")
    return c_host


# ---------------------------------------------------------------- several GPUs
def comm_unique_id() -> bytes:
    """Rank 0's communicator id (``tcec_comm_unique_id``), to be handed to every rank."""
    buf = ctypes.create_string_buffer(COMM_ID_BYTES)
    _check(load().tcec_comm_unique_id(buf), "tcec_comm_unique_id")
    return buf.raw


def comm_init_rank(nranks: int, rank: int, uid: bytes) -> None:
    """Creates this process's communicator on the current device (``tcec_comm_init_rank``)."""
    if len(uid) != COMM_ID_BYTES:
        raise ValueError("communicator id has the wrong size")
    buf = ctypes.create_string_buffer(uid, COMM_ID_BYTES)
    _check(load().tcec_comm_init_rank(int(nranks), int(rank), buf), "tcec_comm_init_rank")


def comm_destroy() -> None:
    _check(load().tcec_comm_destroy(), "tcec_comm_destroy")


def _opt_mat(t: Optional[torch.Tensor]):
    if t is None:
        return ROW_MAJOR, 0, None
    la, lda = _layout_ld(t)
    return la, lda, t.data_ptr()


def sgemm_column_shard(a: Optional[torch.Tensor], b_local: torch.Tensor, c_local: torch.Tensor, m: int, k: int, *,
                       root: int = 0, alpha: float = 1.0, beta: float = 0.0, policy="fp16_ec") -> torch.Tensor:
    """This rank's part of the column-sharded GEMM (``tcec_sgemm_column_shard``): ``a`` (m x k) is
    needed on ``root`` only; ``b_local`` is k x n_local, ``c_local`` m x n_local, on the current device."""
    _require_cuda_f32(b_local, c_local)
    la, lda, ap = _opt_mat(a)
    lb, ldb = _layout_ld(b_local)
    lc, ldc = _layout_ld(c_local)
    with _on(c_local.device):
        st = load().tcec_sgemm_column_shard(root, la, lb, lc, m, b_local.shape[1], k, alpha, ap, lda, b_local.data_ptr(),
                                            ldb, beta, c_local.data_ptr(), ldc, _policy(policy), _stream_ptr())
    _check(st, "tcec_sgemm_column_shard")
    return c_local


def sgemm_column_shard_host(a_host: Optional[torch.Tensor], b_host: torch.Tensor, c_host: torch.Tensor, m: int, k: int,
                            *, root: int = 0, alpha: float = 1.0, beta: float = 0.0, policy="fp16_ec",
                            panel_rows: int = 2048) -> torch.Tensor:
    """The same with host operands (``tcec_sgemm_column_shard_host``): copy-in, broadcast, GEMM and
    copy-out pipelined in row panels; complete when the current stream has reached the end of it."""
    _require_host_f32(b_host, c_host)
    la, lda, ap = _opt_mat(a_host)
    lb, ldb = _layout_ld(b_host)
    lc, ldc = _layout_ld(c_host)
    torch.cuda.init()
    st = load().tcec_sgemm_column_shard_host(root, la, lb, lc, m, b_host.shape[1], k, alpha, ap, lda, b_host.data_ptr(),
                                             ldb, beta, c_host.data_ptr(), ldc, _policy(policy), int(panel_rows),
                                             _stream_ptr())
    _check(st, "tcec_sgemm_column_shard_host")
    return c_host


def _parr(ctype, values):
    return (ctype * len(values))(*values)


def sgemm_multi(a: torch.Tensor, b_blocks: Sequence[torch.Tensor], c_blocks: Sequence[torch.Tensor], *,
                alpha: float = 1.0, beta: float = 0.0, policy="fp16_ec") -> Sequence[torch.Tensor]:
    """One process driving several GPUs (``tcec_sgemm_multi``): block i of B and C lives on its own
    device, A on the device of block 0.  Returns when everything is queued on every device's current stream."""
    devices = [t.device.index for t in c_blocks]
    m, k = a.shape
    la, lda = _layout_ld(a)
    lays = [(_layout_ld(bb), _layout_ld(cc)) for bb, cc in zip(b_blocks, c_blocks)]
    if len({(x[0][0], x[1][0]) for x in lays}) != 1:
        raise ValueError("blocks must share their layouts")
    lb, lc = lays[0][0][0], lays[0][1][0]
    streams = [torch.cuda.current_stream(t.device).cuda_stream for t in c_blocks]
    st = load().tcec_sgemm_multi(
        len(devices), _parr(ctypes.c_int, devices), la, lb, lc, m, _parr(ctypes.c_int, [t.shape[1] for t in b_blocks]), k,
        alpha, a.data_ptr(), lda, _parr(ctypes.c_void_p, [t.data_ptr() for t in b_blocks]),
        _parr(ctypes.c_longlong, [x[0][1] for x in lays]), beta, _parr(ctypes.c_void_p, [t.data_ptr() for t in c_blocks]),
        _parr(ctypes.c_longlong, [x[1][1] for x in lays]), _policy(policy), _parr(ctypes.c_void_p, streams))
    _check(st, "tcec_sgemm_multi")
    return c_blocks


def sgemm_batched_multi(a_parts: Sequence[torch.Tensor], b_parts: Sequence[torch.Tensor],
                        c_parts: Sequence[torch.Tensor], *, alpha: float = 1.0, beta: float = 0.0,
                        policy="fp16_ec") -> Sequence[torch.Tensor]:
    """A batch divided among several GPUs driven by one process (``tcec_sgemm_batched_multi``):
    part i ([count_i, m, k] x [count_i, k, n]) lives on its own device; no collective."""
    devices = [t.device.index for t in c_parts]
    _, m, k = a_parts[0].shape
    n = b_parts[0].shape[2]
    la, lda = _layout_ld(a_parts[0])
    lb, ldb = _layout_ld(b_parts[0])
    lc, ldc = _layout_ld(c_parts[0])
    streams = [torch.cuda.current_stream(t.device).cuda_stream for t in c_parts]
    st = load().tcec_sgemm_batched_multi(
        len(devices), _parr(ctypes.c_int, devices), la, lb, lc, m, n, k, alpha,
        _parr(ctypes.c_void_p, [t.data_ptr() for t in a_parts]), lda, a_parts[0].stride(0),
        _parr(ctypes.c_void_p, [t.data_ptr() for t in b_parts]), ldb, b_parts[0].stride(0), beta,
        _parr(ctypes.c_void_p, [t.data_ptr() for t in c_parts]), ldc, c_parts[0].stride(0),
        _parr(ctypes.c_int, [t.shape[0] for t in a_parts]), _policy(policy), _parr(ctypes.c_void_p, streams))
    _check(st, "tcec_sgemm_batched_multi")
    return c_parts


def split(x: torch.Tensor, policy="fp16_ec"):
    """Element-wise hi / scaled-lo split, widened to float32 (for bit-exact checks)."""
    _require_cuda_f32(x)
    x = x.contiguous()
    hi = torch.empty_like(x)
    lo = torch.empty_like(x)
    with _on(x.device):
        st = load().tcec_split(x.data_ptr(), hi.data_ptr(), lo.data_ptr(), x.numel(), _policy(policy), _stream_ptr())
    _check(st, "tcec_split")
    return hi, lo


def workspace_bytes(m: int, n: int, k: int, batch: int = 1, policy="fp16_ec") -> int:
    return int(load().tcec_workspace_bytes(m, n, k, batch, _policy(policy)))


def destroy() -> None:
    _check(load().tcec_destroy(), "tcec_destroy")
