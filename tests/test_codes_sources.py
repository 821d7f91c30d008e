"""What the kernels for operands held in few bits must say in their source, as no run can show that it is missing."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wmma_extension_b200", "csrc")


def kernel(file, name):
    """The body of a kernel, without comments."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, file)).read())
    start = re.search(r"__global__[^;{]*\b" + name + r"\(const", text).start()
    return text[start:text.index("\n}\n", start)]


# Kernels that may start while the one before them on the stream still writes their operands load them by asm statements that the compiler may move, and
# tie these to the wait by the pointer (after_wait in sm100_ptx.cuh).
@pytest.mark.parametrize("file,name,read", [
    ("tcec_codes.cuh", "pack_q4_kernel", ["w"]),
    ("tcec_codes.cuh", "pack_q4_codes_kernel", ["codes", "scales", "zeros"]),
    ("tcec_codes.cuh", "unpack_q4_kernel", ["packed"]),
    ("tcec_codes.cuh", "pack_q8_kernel", ["x"]),
    ("tcec_codes.cuh", "unpack_q8_kernel", ["packed"]),
    ("tcec_stage.cuh", "stage_panels_kernel", ["src"]),
    ("tcec_stage.cuh", "stage_columns_kernel", ["src"]),
    ("tcec_gemv_q4.cuh", "gemv_q4_kernel", ["x", "staged", "c"]),
    ("tcec_gemv_q8.cuh", "gemv_q8_kernel", ["staged", "c"]),
])
def test_operands_are_read_through_pointers_that_are_known_after_the_wait(file, name, read):
    body = kernel(file, name)
    wait = body.rindex("wait_for_launch_before()")
    for field in read:
        uses = [m.start() for m in re.finditer(r"\bp\." + field + r"\b", body)]
        assert uses, field
        for at in uses:
            assert body[:at].endswith("after_wait("), (field, body[at - 40:at + 40])
            assert at > wait, field


def test_one_tokens_operands_are_handed_over_behind_a_warp_barrier():
    """Lanes write their part of x to shared memory and read what others wrote; votes and the barrier of the codes' copies order neither."""
    body = kernel("tcec_gemv_q4.cuh", "gemv_q4_kernel")
    written = body.rindex("*reinterpret_cast<uint2*>(to")
    read = body.index("*reinterpret_cast<const uint4*>(x_shared", written)
    assert "__syncwarp();" in body[written:read]


def test_indexes_at_the_largest_extents_stay_in_32_bits():
    """With up to 2^31 - 1 rows or columns no sum of an extent or an index and something else may pass that: it would be negative, and taken for inside."""
    bad = re.compile(r"\b[kf]0 \+ 4 <=|\+ kCodeRows - 1\) /|\(a \+ b - 1\) /|\+ Cfg::ROWS - 1\) /|- row0 \+ 15\)")
    for file in ("tcec_codes.cuh", "tcec_gemv_q4.cu", "tcec_gemv_q4.cuh", "tcec_gemv_q8.cu", "tcec_gemv_q8.cuh"):
        found = bad.findall(open(os.path.join(CSRC, file)).read())
        assert not found, (file, found)
