"""Operands held in few bits, without a GPU: sizes, and what is refused before anything is launched."""
import ctypes

import pytest
import torch

from wmma_extension_b200 import tcec

BAD = tcec.ERR_INVALID_ARGUMENT
F32, F16, BF16 = 0, 1, 2


def test_bytes_of_packed_operands():
    lib = tcec.load()
    # blocks of 128 x 128 codes, and four bytes for every group of a row
    assert tcec.q4_bytes(128, 128, 128) == 8192 + 512
    assert tcec.q4_bytes(129, 129, 32) == 4 * (8192 + 4 * 512)
    assert tcec.q4_bytes(0, 128) == 0 and tcec.q4_bytes(128, 0) == 0
    assert lib.tcec_q4_bytes(128, 128, 48) == 0 and lib.tcec_q4_bytes(-1, 128, 128) == 0
    with pytest.raises(ValueError, match="group"):
        tcec.q4_bytes(128, 128, 256)
    assert tcec.q8_bytes(1, 1) == 16384 + 512 and tcec.q8_bytes(128, 129) == 2 * (16384 + 512)
    assert lib.tcec_q8_bytes(-1, 4) == 0 and tcec.q8_bytes(0, 4) == 0
    # sizes whose product passes 32 bits
    assert tcec.q4_bytes(1 << 20, 1 << 20, 128) == (1 << 26) * (8192 + 512)
    assert tcec.q8_bytes(1 << 20, 1 << 20) == (1 << 26) * (16384 + 512)


def test_workspaces():
    lib = tcec.load()
    assert lib.tcec_gemm_q4_workspace_bytes(1, 4096, 4096, F32) == 0  # one token needs none
    # many: panels of the dense operand, 32 KB a block of 128 x 128, three times in FP32
    assert lib.tcec_gemm_q4_workspace_bytes(1000, 4096, 4096, BF16) == 8 * 32 * 32768
    assert lib.tcec_gemm_q4_workspace_bytes(1000, 4096, 4096, F32) == 3 * 8 * 32 * 32768
    assert lib.tcec_gemm_q4_workspace_bytes(1000, 4096, 4096, 3) == 0
    assert lib.tcec_wgrad_q8_workspace_bytes(300, 40, 4096, F16) == 3 * 32768
    # few: 2 KB for every eight columns of a block, their units and the sums of up to four groups
    assert lib.tcec_wgrad_q8_workspace_bytes(300, 16, 4096, F16) == 3 * 2 * (2048 + 5 * 32)
    assert lib.tcec_gemm_q4_workspace_bytes(3, 4096, 4096, F32) == 32 * 2 * (2048 + 5 * 32)
    assert lib.tcec_wgrad_q8_workspace_bytes(300, 129, 4096, F32) == 3 * 2 * 3 * 32768


def _host(bytes_=1 << 16):
    """Memory that no refused call may touch, aligned to 16 bytes."""
    keep = ctypes.create_string_buffer(bytes_ + 16)
    at = ctypes.addressof(keep)
    return keep, at + (-at) % 16


def _gemm(lib, p, **change):
    a = dict(lx=0, lc=0, m=40, n=8, k=16, alpha=1.0, x=p, ldx=16, tx=F32, w=p + 8192, group=32, beta=0.0, c=p + 4096, ldc=8, tc=F32,
             ws=p + 1024 * 1024, wsb=1 << 20)
    a.update(change)
    return lib.tcec_gemm_q4(a["lx"], a["lc"], a["m"], a["n"], a["k"], a["alpha"], a["x"], a["ldx"], a["tx"], a["w"], a["group"], a["beta"],
                            a["c"], a["ldc"], a["tc"], a["ws"], a["wsb"], None)


def _wgrad(lib, p, **change):
    a = dict(ly=0, lc=0, m=16, n=8, k=4, alpha=1.0, y=p, ldy=8, ty=F32, x=p + 8192, beta=0.0, c=p + 4096, ldc=4, tc=F32, ws=p + 1024 * 1024,
             wsb=1 << 20)
    a.update(change)
    return lib.tcec_wgrad_q8(a["ly"], a["lc"], a["m"], a["n"], a["k"], a["alpha"], a["y"], a["ldy"], a["ty"], a["x"], a["beta"], a["c"],
                             a["ldc"], a["tc"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("change", [
    dict(lx=2), dict(lc=-1), dict(m=-1), dict(n=-1), dict(k=-1), dict(tx=3), dict(tc=5), dict(tx=F32, tc=F16), dict(tx=F16, tc=BF16),
    dict(group=16), dict(group=0), dict(ldx=15), dict(lx=1, ldx=39), dict(ldc=7), dict(lc=1, ldc=39), dict(x=None), dict(c=None),
    dict(w=None), dict(ws=None), dict(wsb=3 * 32768 - 1), "x unaligned", "c unaligned", "w unaligned", "ws unaligned", "c over x", "c over w",
    "c over ws", "ws over x", "ws over w",
])
def test_gemm_q4_refuses(change):
    lib = tcec.load()
    keep, p = _host()
    named = {"x unaligned": dict(x=p + 2), "c unaligned": dict(c=p + 4098), "w unaligned": dict(w=p + 8200), "ws unaligned": dict(ws=p + 8),
             "c over x": dict(c=p + 40 * 16 * 4 - 4), "c over w": dict(c=p + 8192 + 8), "c over ws": dict(ws=p + 4096),
             "ws over x": dict(ws=p), "ws over w": dict(ws=p + 8192)}
    assert _gemm(lib, p, **(named[change] if isinstance(change, str) else change)) == BAD
    assert bytes(keep) == bytes(len(keep))


@pytest.mark.parametrize("change", [
    dict(ly=2), dict(lc=9), dict(m=-1), dict(n=-1), dict(k=-1), dict(ty=-1), dict(tc=3), dict(ty=BF16, tc=F16), dict(ldy=7),
    dict(ly=1, ldy=15), dict(ldc=3), dict(y=None), dict(c=None), dict(x=None), dict(ws=None), dict(wsb=4 * (2048 + 5 * 32) - 1), "y unaligned",
    "x unaligned", "c over y", "c over x", "ws over y",
])
def test_wgrad_q8_refuses(change):
    lib = tcec.load()
    keep, p = _host()
    named = {"y unaligned": dict(y=p + 1), "x unaligned": dict(x=p + 8200), "c over y": dict(c=p + 16), "c over x": dict(c=p + 8192 + 16896 - 4),
             "ws over y": dict(ws=p)}
    assert _wgrad(lib, p, **(named[change] if isinstance(change, str) else change)) == BAD
    assert bytes(keep) == bytes(len(keep))


def test_packing_refuses():
    lib = tcec.load()
    keep, p = _host()
    out = p + 16384
    assert lib.tcec_pack_q4(2, 4, 4, p, 4, F32, 32, F16, out, None) == BAD
    assert lib.tcec_pack_q4(0, 4, 4, p, 3, F32, 32, F16, out, None) == BAD
    assert lib.tcec_pack_q4(0, 4, 4, p, 4, 7, 32, F16, out, None) == BAD
    assert lib.tcec_pack_q4(0, 4, 4, p, 4, F32, 31, F16, out, None) == BAD
    assert lib.tcec_pack_q4(0, 4, 4, p, 4, F32, 32, F32, out, None) == BAD  # scales have 16 bits
    assert lib.tcec_pack_q4(0, 4, 4, None, 4, F32, 32, F16, out, None) == BAD
    assert lib.tcec_pack_q4(0, 4, 4, p, 4, F32, 32, F16, out + 8, None) == BAD
    assert lib.tcec_pack_q4(0, 4, 4, out + 64, 4, F32, 32, F16, out, None) == BAD
    assert lib.tcec_pack_q4_codes(4, 5, p, 2, p + 64, F16, None, 32, out, None) == BAD  # five codes take three bytes
    assert lib.tcec_pack_q4_codes(4, 4, p, 2, p + 65, F16, None, 32, out, None) == BAD
    assert lib.tcec_pack_q4_codes(4, 4, p, 2, p + 64, F32, None, 32, out, None) == BAD
    assert lib.tcec_pack_q4_codes(4, 4, p, 2, p + 64, F16, out + 16, 32, out, None) == BAD
    assert lib.tcec_unpack_q4(0, 4, 4, out, 32, p, 3, F32, None) == BAD
    assert lib.tcec_unpack_q4(0, 4, 4, out + 4, 32, p, 4, F32, None) == BAD
    assert lib.tcec_unpack_q4(0, 4, 4, None, 32, p, 4, F32, None) == BAD
    assert lib.tcec_pack_q8(0, 4, 4, p, 3, F32, out, None) == BAD
    assert lib.tcec_pack_q8(0, 4, 4, p, 4, F32, None, None) == BAD
    assert lib.tcec_pack_q8(1, 4, 8, p, 3, F16, out, None) == BAD
    assert lib.tcec_unpack_q8(0, 4, 4, out, p + 1, 4, BF16, None) == BAD
    assert lib.tcec_unpack_q8(0, 4, 4, out, out + 16, 4, BF16, None) == BAD
    # nothing to do: nothing is looked at
    assert lib.tcec_pack_q4(0, 0, 4, None, 4, F32, 32, F16, None, None) == tcec.OK
    assert lib.tcec_pack_q8(0, 4, 0, None, 4, F32, None, None) == tcec.OK
    assert lib.tcec_unpack_q8(0, 0, 4, None, None, 4, F32, None) == tcec.OK
    assert _gemm(lib, p, m=0) == tcec.OK and _gemm(lib, p, n=0, w=None) == tcec.OK and _wgrad(lib, p, k=0) == tcec.OK
    assert bytes(keep) == bytes(len(keep))


def test_python_refuses_what_is_not_a_matrix_on_a_gpu():
    x = torch.zeros(4, 4)
    for call in (lambda: tcec.pack_q4(x), lambda: tcec.pack_q8(x), lambda: tcec.gemm_q4(x, x, 4), lambda: tcec.wgrad_q8(x, x, 4)):
        with pytest.raises(ValueError, match="CUDA matrix"):
            call()
    with pytest.raises(ValueError, match="uint8 CUDA"):
        tcec.pack_q4_codes(torch.zeros(4, 2, dtype=torch.uint8), x.half(), k=4)
    with pytest.raises(ValueError, match="consecutive bytes on a GPU"):
        tcec.unpack_q4(torch.zeros(1 << 16, dtype=torch.uint8), 4, 4)
    with pytest.raises(ValueError, match="consecutive bytes on a GPU"):
        tcec.unpack_q8(torch.zeros(1 << 16, dtype=torch.uint8), 4, 4)
