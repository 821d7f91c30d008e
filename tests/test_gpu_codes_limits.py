"""Operands held in few bits, on a B200, at the ends of what the header promises."""
import pytest
import torch

from test_gpu_codes import BF16, DEV, F16, F32, bound, check, randn, with_codes
from wmma_extension_b200 import tcec

pytestmark = pytest.mark.gpu


# Up to 32 columns of tokens code and zero point are multiplied apart, so what is rounded off is relative to sum |s| (q + z) |x|: the codes' part as
# bound() counts it, and the zero points' alike, whose sums of x are of eight values a thread and four exchanges, 11 roundings of 2^-24 where bound()
# has 8 * 2^-22.
@pytest.mark.parametrize("m,dtype", [(1, F32), (1, BF16), (2, F32), (2, BF16), (5, F32), (5, BF16), (9, F32), (9, BF16), (24, BF16)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("alike", [True, False])
def test_tokens_up_to_2_27_and_beyond(m, dtype, group, alike):
    """Values whose sums over a group pass 2^28, where a sum of values times 2^100 would be infinite: all alike, of one sign, or random."""
    n, k = 48, 400
    byte, s, z, w = with_codes(n, k, group, 71)
    z[::3] = 0  # a zero point of 0 makes NaN of an infinite sum
    each = torch.arange(k, device=DEV) // group
    q = torch.stack([byte & 15, byte >> 4], 2).reshape(n, -1)[:, :k].double()
    w = (q - z.double()[:, each]) * s.double()[:, each]
    sizes = (q + z.double()[:, each]) * s.double()[:, each]
    packed = tcec.pack_q4_codes(byte, s, z, k=k, group=group)
    base = torch.full((m, k), 1.5, device=DEV) if alike else randn(m, k, seed=m).clamp(-3.9, 3.9)
    for exponent in (*range(18, 28), 60, 90, 110):
        x = (base.double() * 2.0**exponent).to(dtype)
        exact = x.double() @ w.T
        check(tcec.gemm_q4(x, packed, n, group=group, dtype=F32), exact, bound(x.double().abs() @ sizes.T, exact, F32, k, 3 if dtype == F32 else 1))


@pytest.mark.parametrize("m,dtype", [(1, F32), (1, F16), (1, BF16), (4, F32), (12, F16), (24, BF16)])
def test_few_tokens_with_an_infinity_are_nan(m, dtype):
    """As include/tcec.h says: code and zero point are multiplied apart, q * inf - z * inf; the other tokens keep their results."""
    n, k = 40, 300
    byte, s, z, w = with_codes(n, k, 64, 73)
    z[5] = 0
    packed = tcec.pack_q4_codes(byte, s, z, k=k, group=64)
    x = randn(m, k, seed=m, dtype=dtype)
    clean = tcec.gemm_q4(x, packed, n, group=64)
    for value in (float("inf"), -float("inf")) if dtype == F16 else (float("inf"), -float("inf"), 2.0**122):
        bad = x.clone()
        bad[0, 70] = value
        got = tcec.gemm_q4(bad, packed, n, group=64)
        assert got[0].isnan().all() and torch.equal(got[1:], clean[1:])
    if dtype != F16:  # the largest value below them counts
        x[0, 70] = 2.0**122 * (1 - torch.finfo(dtype).eps)
        assert tcec.gemm_q4(x, packed, n, group=64, dtype=F32)[0].isfinite().all()


@pytest.mark.parametrize("m", [40, 300])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("group", [32, 128])
def test_many_tokens_with_an_infinity_are_infinite(m, dtype, group):
    n, k = 200, 300
    byte, s, z, w = with_codes(n, k, group, 73)
    packed = tcec.pack_q4_codes(byte, s, z, k=k, group=group)
    x = randn(m, k, seed=m, dtype=dtype)
    for value in (float("inf"), -float("inf")):
        x[3, 70] = value
        want = value * w[:, 70]  # NaN where the weight is 0
        got = tcec.gemm_q4(x, packed, n, group=group)[3].double()
        torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("n", [3, 9, 50])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gradients_of_an_infinity_are_infinite(n, dtype):
    m, k = 300, 200
    x = randn(m, k, seed=n)
    x[150, ::7] = 0.0
    packed = tcec.pack_q8(x)
    kept = tcec.unpack_q8(packed, m, k).double()
    dy = randn(m, n, seed=n + 1, dtype=dtype)
    for value in (float("inf"), -float("inf")):
        dy[150, 2] = value
        got = tcec.wgrad_q8(dy, packed, k)[2].double()
        torch.testing.assert_close(got, value * kept[150], rtol=0, atol=0, equal_nan=True)


def test_sizes_that_are_no_extents_are_refused():
    """Matrices without elements have such sizes too; 2^32 + 4 rows would be taken for four."""
    many, none = 2**32 + 4, torch.empty(0, dtype=torch.uint8, device=DEV)
    for call in (
        lambda: tcec.gemm_q4(torch.empty(many, 0, dtype=BF16, device=DEV), none, 1),
        lambda: tcec.gemm_q4(torch.empty(0, 4, dtype=BF16, device=DEV), none, many),
        lambda: tcec.gemm_q4(torch.empty(0, 4, dtype=BF16, device=DEV), none, -1),
        lambda: tcec.wgrad_q8(torch.empty(0, many, dtype=BF16, device=DEV), none, 1),
        lambda: tcec.wgrad_q8(torch.empty(0, 4, dtype=BF16, device=DEV), none, many),
        lambda: tcec.pack_q4(torch.empty(many, 0, device=DEV)),
        lambda: tcec.pack_q8(torch.empty(0, many, device=DEV)),
        lambda: tcec.pack_q4_codes(torch.empty(0, many // 2, dtype=torch.uint8, device=DEV), torch.empty(0, many // 128 + 1, dtype=F16, device=DEV), k=many),
        lambda: tcec.unpack_q4(none, many, 0),
        lambda: tcec.unpack_q8(none, 0, many),
        lambda: tcec.unpack_q8(none, 4, -1),
    ):
        with pytest.raises(ValueError, match="2147483647"):
            call()


@pytest.mark.parametrize("alpha", [float("inf"), float("nan"), -3.0])
@pytest.mark.parametrize("m", [1, 2, 12, 40])
def test_a_sum_over_nothing_is_nothing_times_anything(alpha, m):
    n = 150
    c, none = randn(m, n, seed=m), torch.empty(0, dtype=torch.uint8, device=DEV)
    want = 0.5 * c
    assert torch.equal(tcec.gemm_q4(c[:, :0], none, n, c.clone(), alpha=alpha, beta=0.5), want)
    assert torch.equal(tcec.gemm_q4(c[:, :0], none, n, alpha=alpha), torch.zeros(m, n, device=DEV))
    assert torch.equal(tcec.wgrad_q8(c[:0, :m], none, n, c.clone(), alpha=alpha, beta=0.5), want)
    assert torch.equal(tcec.wgrad_q8(c[:0, :m], none, n, alpha=alpha), torch.zeros(m, n, device=DEV))


def test_the_first_call_is_not_captured():
    """It is refused, and the next one outside works.  In a process of its own, as others have called before."""
    import subprocess
    import sys

    code = """
import torch
from wmma_extension_b200 import tcec
w = torch.full((128, 128), 15.0, device="cuda")  # a scale of 1
torch.cuda.synchronize()
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        tcec.pack_q4(w)
except (tcec.TcecError, RuntimeError) as e:
    print("refused", type(e).__name__)
for i in range(2):
    try:
        assert torch.equal(tcec.unpack_q4(tcec.pack_q4(w), 128, 128), w)
        print("worked", i)
    except Exception as e:
        print("failed", i, repr(e))
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert "refused" in run.stdout and "worked 0" in run.stdout and "worked 1" in run.stdout, (run.stdout, run.stderr)


# The last of the three bf16 parts of an FP32 value holds up to 2^-16 of it.  Where all values have it in full, and all terms have one sign, a product without it is off
# by nearly 2^-16 of their sum, and bound() allows 2^-17.2 at 256 terms.
def last_part_in_full(*shape, seed):
    return ((randn(*shape, seed=seed).abs() + 0.5).view(torch.int32) | 0x7F).view(F32)


def without_last_part(t):
    return (t.view(torch.int32) & ~0x7F).view(F32).double()


@pytest.mark.parametrize("m", [1, 5, 10, 40, 300])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_products_have_all_parts_of_fp32_tokens(m, group):
    n, k = 136, 256
    byte, s, z, w = with_codes(n, k, group, 75)
    z.zero_()
    w = torch.stack([byte & 15, byte >> 4], 2).reshape(n, -1).double() * s.double()[:, torch.arange(k, device=DEV) // group]
    packed = tcec.pack_q4_codes(byte, s, z, k=k, group=group)
    x = last_part_in_full(m, k, seed=m)
    exact = x.double() @ w.T
    tol = bound(exact, exact, F32, k, 3)
    assert ((without_last_part(x) @ w.T - exact).abs() > 1.5 * tol).all()  # this would be noticed
    check(tcec.gemm_q4(x, packed, n, group=group), exact, tol)


@pytest.mark.parametrize("n", [2, 10, 40, 300])
def test_gradients_have_all_parts_of_fp32(n):
    m, k = 256, 200
    packed = tcec.pack_q8(randn(m, k, seed=n).abs())
    kept = tcec.unpack_q8(packed, m, k).double()
    dy = last_part_in_full(m, n, seed=n + 1)
    exact = dy.double().T @ kept
    tol = bound(exact, exact, F32, m, 3)
    assert ((without_last_part(dy).T @ kept - exact).abs() > 1.5 * tol).all()
    check(tcec.wgrad_q8(dy, packed, k), exact, tol)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("step", [1, 3])
def test_one_token_and_one_output_as_columns_of_a_matrix(dtype, step):
    """A row whose elements lie `step` apart or more: x of one token, dY of one output, and results between other columns."""
    n, k = 150, 333
    byte, s, z, w = with_codes(n, k, 64, 77)
    packed = tcec.pack_q4_codes(byte, s, z, k=k, group=64)
    x = torch.full((k, step), float("nan"), device=DEV, dtype=dtype)
    x[:, step - 1] = randn(k, seed=78, dtype=dtype)
    row = x[:, step - 1:].T
    exact = row.double() @ w.T
    c = torch.full((n, 5), 7.0, device=DEV)
    tcec.gemm_q4(row, packed, n, c[:, 2:3].T, group=64)
    q = torch.stack([byte & 15, byte >> 4], 2).reshape(n, -1)[:, :k].double()
    each = torch.arange(k, device=DEV) // 64
    sizes = (q + z.double()[:, each]) * s.double()[:, each]
    check(c[:, 2:3].T, exact, bound(row.double().abs() @ sizes.T, exact, F32, k, 3 if dtype == F32 else 1))
    assert (c[:, [0, 1, 3, 4]] == 7.0).all()
    kept = tcec.pack_q8(randn(k, n, seed=79))
    values = tcec.unpack_q8(kept, k, n).double()
    g = torch.full((n, 5), 7.0, device=DEV)
    tcec.wgrad_q8(x[:, step - 1:], kept, n, g[:, 3:4].T)
    exact = row.double() @ values
    check(g[:, 3:4].T, exact, bound(row.double().abs() @ values.abs(), exact, F32, k, 3 if dtype == F32 else 1))
    assert (g[:, [0, 1, 2, 4]] == 7.0).all()


@pytest.mark.parametrize("n,k", [(1, 1), (130, 333), (257, 128)])
def test_codes_between_other_bytes_are_laid_out(n, k):
    byte, s, z, w = with_codes(n, k, 32, 81, BF16)
    wide = torch.full((n, byte.shape[1] + 3), 0xFF, dtype=torch.uint8, device=DEV)
    wide[:, 1:-2] = byte
    packed = tcec.pack_q4_codes(wide[:, 1:-2], s, z, k=k, group=32)
    assert torch.equal(packed, tcec.pack_q4_codes(byte, s, z, k=k, group=32))
    turned = byte.T.contiguous().T  # columns first: copied
    assert torch.equal(packed, tcec.pack_q4_codes(turned, s, z, k=k, group=32))
    assert torch.equal(tcec.unpack_q4(packed, n, k, group=32).double(), w)
