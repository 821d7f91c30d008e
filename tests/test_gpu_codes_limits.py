"""Operands held in few bits, on a B200, at the ends of what the header promises."""
import pytest
import torch

from test_gpu_codes import BF16, DEV, F32, bound, check, randn, with_codes
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
