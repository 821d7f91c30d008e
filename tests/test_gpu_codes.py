"""Operands held in few bits, on a B200, against plain arithmetic in 64 bits.

Tolerances.  A product's terms code * dense are exact, a group's sum is one of the tensor core's FP32 accumulator, which cuts off
what is below its last place: at most `terms` * 2^-22 of the largest partial sum for the `terms` additions of a group (a step of 16 products is
one addition, of which the operands are aligned before they are added; 8 steps a group, 24 with three parts).  Folding adds 2^-23 of the running sum for each group (a
fused multiply-add, and the final additions).  All of it is relative to sum |s| |code| |dense|, which is what `bound` computes; a result in
16 bits adds half a step of its own value.
"""
import ctypes

import pytest
import torch

from wmma_extension_b200 import tcec

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(*shape, seed, dtype=F32):
    return torch.randn(*shape, device=DEV, generator=gen(seed)).to(dtype)


def bound(magnitude, exact, dtype, summed, parts):
    """How far a product may be from 64 bits: `magnitude` = sum of the terms' magnitudes, `summed` terms of it."""
    groups = -(-summed // 32) + 8
    tol = magnitude * (8 * parts * 2.0**-22 + groups * 2.0**-24) + 1e-30
    # below the normal numbers steps no longer shrink: f16 values under 2^-14 lie 2^-24 apart, and half of that is 2^-14 * eps / 2
    kind = torch.finfo(dtype)
    return tol + exact.abs().clamp(min=kind.smallest_normal) * kind.eps / 2 * 1.01


def check(got, exact, tol):
    assert got.shape == exact.shape
    assert torch.isfinite(got).all()
    off = (got.double() - exact).abs() - tol
    assert off.max().item() <= 0, (off.max().item(), (got.double() - exact).abs().max().item())


# ---------------------------------------------------------------- 4-bit weights
def quantise(w, group, scale):
    """The definition in include/tcec.h: codes, scales and zero points of n x groups x group (the last group filled with zeros)."""
    n, k = w.shape
    count = -(-k // group)
    g = torch.zeros(n, count * group, dtype=torch.float64, device=w.device)
    g[:, :k] = w.double()
    g = g.reshape(n, count, group)
    lo, hi = g.amin(2).clamp(max=0), g.amax(2).clamp(min=0)
    s = ((hi - lo).float().double() / 15).float().to(scale).double()
    step = torch.where(s > 0, s, torch.ones_like(s))
    z = torch.round(-lo / step).clamp(0, 15)
    q = (torch.round(g / step[..., None]) + z[..., None]).clamp(0, 15)
    q, z = torch.where((s > 0)[..., None], q, torch.zeros_like(q)), torch.where(s > 0, z, torch.zeros_like(z))
    return q, s, z


def values(w, group, scale):
    q, s, z = quantise(w, group, scale)
    return ((q - z[..., None]) * s[..., None]).reshape(w.shape[0], -1)[:, :w.shape[1]]


SIZES = [(1, 1), (1, 128), (7, 33), (16, 96), (128, 128), (129, 257), (300, 1000)]


@pytest.mark.parametrize("n,k", SIZES + [(2500, 4001)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype,scale", [(F32, F16), (F16, BF16), (BF16, F16)])
def test_weights_go_to_the_nearest_of_16_steps(n, k, group, dtype, scale):
    w = randn(n, k, seed=n + k, dtype=dtype)
    packed = tcec.pack_q4(w, group=group, scale=scale)
    assert torch.equal(tcec.unpack_q4(packed, n, k, group=group).double(), values(w, group, scale))  # a code times a scale has 15 bits


@pytest.mark.parametrize("order", ["wide", "odd", "columns"])
def test_weights_of_any_stride(order):
    n, k = 130, 200
    w = randn(n, k, seed=3)
    there = {"wide": lambda: torch.empty(n, k + 8, device=DEV)[:, 4:4 + k], "odd": lambda: torch.empty(n, k + 1, device=DEV)[:, 1:],
             "columns": lambda: torch.empty(k, n + 3, device=DEV)[:, :n].T}[order]()
    there.copy_(w)
    packed = tcec.pack_q4(there)
    assert torch.equal(packed, tcec.pack_q4(w))
    out = torch.empty_strided(there.shape, there.stride(), device=DEV)
    assert torch.equal(tcec.unpack_q4(packed, n, k, out=out), tcec.unpack_q4(packed, n, k))


def test_weights_at_the_borders_between_steps():
    """Multiples of half a step: ties go to the even code, whatever the quotient's own rounding does."""
    w = torch.zeros(64, 128, device=DEV)
    for r in range(64):
        s = float(torch.tensor(0.1 * 1.37**(r - 32), dtype=F32).half())
        w[r] = (torch.arange(128, device=DEV) % 16 - 5).float() * s * 0.5
        w[r, 0], w[r, 1] = -6.0 * s, 9.0 * s  # fixes the scale at s, or next to it
        w[r, 64:] = torch.nextafter(w[r, 64:], torch.full((), 1e30, device=DEV))
    for scale in (F16, BF16):
        assert torch.equal(tcec.unpack_q4(tcec.pack_q4(w, scale=scale), 64, 128).double(), values(w, 128, scale))


def test_weights_that_have_no_codes():
    w = randn(8, 256, seed=5)
    w[0, 3], w[1, 200], w[2, 10], w[3, :] = float("inf"), float("nan"), -float("inf"), 0.0
    w[4, :128] *= 1e8   # a scale beyond f16
    w[5, :128] = 1e-12  # and one below it
    out = tcec.unpack_q4(tcec.pack_q4(w), 8, 256)
    nan = torch.zeros(8, 256, dtype=torch.bool, device=DEV)
    nan[0, :128] = nan[1, 128:] = nan[2, :128] = nan[4, :128] = True
    assert torch.equal(out.isnan(), nan)
    assert (out[3] == 0).all() and (out[5, :128] == 0).all()
    keep = ~nan.any(1)
    assert torch.equal(out[keep].double(), values(w[keep], 128, F16))
    wide = tcec.unpack_q4(tcec.pack_q4(w, scale=BF16), 8, 256)
    assert wide[4].isfinite().all() and (wide[5, :128] != 0).all()
    # scales below the normal FP32 numbers
    tiny = randn(4, 128, seed=6) * 1e-38
    assert torch.equal(tcec.unpack_q4(tcec.pack_q4(tiny, scale=BF16), 4, 128).double(), values(tiny, 128, BF16))


def with_codes(n, k, group, seed, scale=F16, zeros=True):
    """Random codes, the bytes that hold them, and the values."""
    g = gen(seed)
    count = -(-k // group)
    q = torch.randint(0, 16, (n, k + k % 2), device=DEV, generator=g, dtype=torch.uint8)
    s = (torch.rand(n, count, device=DEV, generator=g) * 0.1 + 0.01).to(scale)
    z = torch.randint(0, 16, (n, count), device=DEV, generator=g, dtype=torch.uint8) if zeros else None
    byte = q[:, 0::2] | q[:, 1::2] << 4
    each = torch.arange(k, device=DEV) // group
    off = z.double()[:, each] if zeros else 8.0
    return byte, s, z, (q[:, :k].double() - off) * s.double()[:, each]


@pytest.mark.parametrize("n,k", SIZES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros,scale", [(True, F16), (False, BF16)])
def test_codes_that_exist_are_laid_out(n, k, group, zeros, scale):
    byte, s, z, w = with_codes(n, k, group, n * k, scale, zeros)
    packed = tcec.pack_q4_codes(byte, s, z, k=k, group=group)
    assert torch.equal(tcec.unpack_q4(packed, n, k, group=group).double(), w)


# ---------------------------------------------------------------- products with them
def product_case(m, n, k, group, dtype, seed, out=None, scale=F16):
    byte, s, z, w = with_codes(n, k, group, seed, scale)
    x = randn(m, k, seed=seed + 1, dtype=dtype)
    packed = tcec.pack_q4_codes(byte, s, z, k=k, group=group)
    exact = x.double() @ w.T
    tol = bound(x.double().abs() @ w.abs().T, exact, out or dtype, k, 3 if dtype == F32 else 1)
    return x, packed, exact, tol


@pytest.mark.parametrize("m", [1, 2, 3, 8, 9, 10, 11, 16, 17, 32, 33, 40, 64, 65, 129, 300])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_products_of_many_token_counts(m, dtype, group):
    x, packed, exact, tol = product_case(m, 136, 416, group, dtype, m)
    check(tcec.gemm_q4(x, packed, 136, group=group), exact, tol)
    tcec.device_status()


@pytest.mark.parametrize("n,k", SIZES + [(64, 4096), (1000, 130), (1031, 2050)])
@pytest.mark.parametrize("m,dtype", [(1, F32), (1, BF16), (5, F16), (20, BF16), (100, BF16), (50, F32), (260, F16)])
def test_products_of_odd_sizes(m, n, k, dtype):
    x, packed, exact, tol = product_case(m, n, k, 64, dtype, m + n)
    check(tcec.gemm_q4(x, packed, n, group=64), exact, tol)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_products_large_enough_for_pairs(group, dtype):
    """17 x 6 tiles of 128 x 256: the last pair of SMs has one row of tiles, the last column of tiles fewer than 128 columns."""
    x, packed, exact, tol = product_case(1350, 2170, 700, group, dtype, 41)
    check(tcec.gemm_q4(x, packed, 2170, group=group), exact, tol)
    tcec.device_status()


@pytest.mark.parametrize("m", [3, 150])
@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F16, F32), (F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("lx", ["rows", "odd", "columns"])
@pytest.mark.parametrize("lc", ["rows", "columns"])
def test_products_of_any_layout_into_a_larger_matrix(m, dtype, out, lx, lc):
    n, k = 200, 300
    x, packed, exact, tol = product_case(m, n, k, 128, dtype, 7, out)
    there = {"rows": lambda: torch.empty(m, k + 8, device=DEV, dtype=dtype)[:, :k], "odd": lambda: torch.empty(m, k + 1, device=DEV, dtype=dtype)[:, 1:],
             "columns": lambda: torch.empty(k, m + 1, device=DEV, dtype=dtype)[:, :m].T}[lx]()
    there.copy_(x)
    whole = torch.full((m + 2, n + 3) if lc == "rows" else (n + 3, m + 2), 7.0, device=DEV, dtype=out)
    c = whole[1:m + 1, 2:n + 2] if lc == "rows" else whole[2:n + 2, 1:m + 1].T
    old = randn(m, n, seed=9, dtype=out)
    c.copy_(old)
    r = tcec.gemm_q4(there, packed, n, c, alpha=0.5, beta=-2.0)
    assert r.data_ptr() == c.data_ptr()
    want = 0.5 * exact - 2.0 * old.double()
    check(c, want, 0.5 * tol + (want.abs() + 2 * old.double().abs() + 0.5 * exact.abs()) * (2.0**-23 + torch.finfo(out).eps / 2))
    edge = whole.clone()
    (edge[1:m + 1, 2:n + 2] if lc == "rows" else edge[2:n + 2, 1:m + 1]).fill_(7.0)
    assert (edge == 7.0).all()  # nothing around it is written


@pytest.mark.parametrize("m", [1, 100])
def test_products_of_nothing(m):
    x, packed, exact, tol = product_case(m, 40, 64, 32, F32, 11)
    c = torch.full((m, 40), float("nan"), device=DEV)
    check(tcec.gemm_q4(x, packed, 40, c, group=32), exact, tol)  # beta 0 does not read C
    c = randn(m, 40, seed=1)
    keep = c.clone()
    assert torch.equal(tcec.gemm_q4(x * float("nan"), packed, 40, c, group=32, alpha=0.0, beta=0.5), 0.5 * keep)
    assert torch.equal(tcec.gemm_q4(x[:, :0], packed[:0], 40, group=32), torch.zeros(m, 40, device=DEV))
    assert tcec.gemm_q4(x[:0], packed, 40, group=32).shape == (0, 40)
    assert tcec.gemm_q4(x, packed[:0], 0, group=32).shape == (m, 0)


@pytest.mark.parametrize("m", [4, 70])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_what_is_not_finite_stays_in_its_row(m, dtype):
    n, k = 64, 256
    x, packed, exact, tol = product_case(m, n, k, 128, dtype, 13)
    clean = tcec.gemm_q4(x, packed, n)
    x[1, 5], x[2, 200] = float("nan"), float("inf")
    got = tcec.gemm_q4(x, packed, n)
    assert got[1].isnan().all() and not got[2].isfinite().any()
    keep = [0, *range(3, m)]
    assert torch.equal(got[keep], clean[keep])
    w = tcec.unpack_q4(packed, n, k)
    w[3, 7] = float("nan")
    poison = tcec.pack_q4(w)  # a column of the result
    x = randn(m, k, seed=2, dtype=dtype)
    bad = tcec.gemm_q4(x, poison, n).isnan()
    assert bad[:, 3].all() and bad.sum() == m


def test_large_and_small_fp32_values():
    """Three bf16 parts hold an FP32 number over its whole range but for the last bits of the very smallest."""
    byte, s, z, w = with_codes(32, 128, 128, 17)
    packed = tcec.pack_q4_codes(byte, s, z, k=128)
    for m in (2, 64):
        x = randn(m, 128, seed=m)
        for scale in (1e34, 1e-25):
            exact = (x * scale).double() @ w.T
            check(tcec.gemm_q4(x * scale, packed, 32), exact, bound((x * scale).double().abs() @ w.abs().T, exact, F32, 128, 3))

# ---------------------------------------------------------------- 8-bit activations
def quantise8(x):
    m, k = x.shape
    blocks = -(-m // 128)
    g = torch.zeros(blocks * 128, k, dtype=torch.float64, device=x.device)
    g[:m] = x.double()
    g = g.reshape(blocks, 128, k)
    s = (g.abs().amax(1) / 127).float().double().clamp(min=2.0**-120)
    return torch.round(g / s[:, None]).reshape(-1, k)[:m], s.repeat_interleave(128, 0)[:m]


@pytest.mark.parametrize("m,k", [(1, 1), (1, 300), (127, 64), (128, 128), (129, 130), (1000, 257)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_activations_go_to_the_nearest_of_255_steps(m, k, dtype):
    x = randn(m, k, seed=m * k, dtype=dtype)
    q, s = quantise8(x)
    got = tcec.unpack_q8(tcec.pack_q8(x), m, k)
    assert torch.equal(got, (q * s).float())
    assert ((got.double() - x.double()).abs() <= s * 0.5001).all()
    assert torch.equal(tcec.unpack_q8(tcec.pack_q8(x), m, k, dtype=BF16), (q * s).float().bfloat16())


@pytest.mark.parametrize("order", ["wide", "odd", "columns"])
def test_activations_of_any_stride(order):
    m, k = 200, 130
    x = randn(m, k, seed=3, dtype=BF16)
    there = {"wide": lambda: torch.empty(m, k + 2, device=DEV, dtype=BF16)[:, :k], "odd": lambda: torch.empty(m, k + 1, device=DEV, dtype=BF16)[:, 1:],
             "columns": lambda: torch.empty(k, m + 3, device=DEV, dtype=BF16)[:, :m].T}[order]()
    there.copy_(x)
    packed = tcec.pack_q8(there)
    assert torch.equal(packed, tcec.pack_q8(x))
    out = torch.empty_strided(there.shape, there.stride(), device=DEV, dtype=BF16)
    assert torch.equal(tcec.unpack_q8(packed, m, k, out=out), tcec.unpack_q8(packed, m, k, dtype=BF16))


def test_activations_at_the_borders_and_beyond():
    x = torch.zeros(256, 64, device=DEV)
    for f in range(64):
        s = float(torch.tensor(0.013 * 1.9**(f - 32), dtype=F32))
        x[:128, f] = (torch.arange(128, device=DEV) - 60).float() * s * 0.5
        x[0, f] = 127.0 * s
        x[64:128, f] = torch.nextafter(x[64:128, f], torch.zeros((), device=DEV))
    x[128:] = 1e-40
    q, s = quantise8(x)
    assert torch.equal(tcec.unpack_q8(tcec.pack_q8(x), 256, 64).double(), (q * s).float().double())
    x[5, 1], x[200, 2], x[130, 3] = float("nan"), float("inf"), -float("inf")
    got = tcec.unpack_q8(tcec.pack_q8(x), 256, 64)
    nan = torch.zeros(256, 64, dtype=torch.bool, device=DEV)
    nan[:128, 1] = nan[128:, 2] = nan[128:, 3] = True
    assert torch.equal(got.isnan(), nan)
    assert torch.equal(got[~nan].double(), (q * s).float().double()[~nan])


# ---------------------------------------------------------------- gradients from them
def gradient_case(m, n, k, dtype, seed, out=None):
    x = randn(m, k, seed=seed)
    dy = randn(m, n, seed=seed + 1, dtype=dtype)
    packed = tcec.pack_q8(x)
    q, s = quantise8(x)
    exact = dy.double().T @ (q * s)
    tol = bound(dy.double().abs().T @ (q * s).abs(), exact, out or dtype, m, 3 if dtype == F32 else 1)
    return dy, packed, exact, tol


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 200, 130), (127, 16, 128), (128, 64, 128), (129, 65, 257), (700, 130, 300), (1030, 8, 1000),
                                   (5000, 20, 140), (300, 1000, 2000), (500, 1350, 2170)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gradients(m, n, k, dtype):
    dy, packed, exact, tol = gradient_case(m, n, k, dtype, m + n)
    check(tcec.wgrad_q8(dy, packed, k), exact, tol)
    tcec.device_status()


@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("ly", ["rows", "odd", "columns"])
@pytest.mark.parametrize("lc", ["rows", "columns"])
def test_gradients_of_any_layout_add_up(dtype, out, ly, lc):
    m, n, k = 260, 72, 150
    dy, packed, exact, tol = gradient_case(m, n, k, dtype, 5, out)
    there = {"rows": lambda: torch.empty(m, n + 8, device=DEV, dtype=dtype)[:, :n], "odd": lambda: torch.empty(m, n + 1, device=DEV, dtype=dtype)[:, 1:],
             "columns": lambda: torch.empty(n, m + 4, device=DEV, dtype=dtype)[:, :m].T}[ly]()
    there.copy_(dy)
    whole = torch.full((n + 2, k + 3) if lc == "rows" else (k + 3, n + 2), 7.0, device=DEV, dtype=out)
    c = whole[1:n + 1, 2:k + 2] if lc == "rows" else whole[2:k + 2, 1:n + 1].T
    old = randn(n, k, seed=9, dtype=out)
    c.copy_(old)
    tcec.wgrad_q8(there, packed, k, c, beta=1.0)
    want = exact + old.double()
    check(c, want, tol + (want.abs() + old.double().abs() + exact.abs()) * (2.0**-23 + torch.finfo(out).eps / 2))
    edge = whole.clone()
    (edge[1:n + 1, 2:k + 2] if lc == "rows" else edge[2:k + 2, 1:n + 1]).fill_(7.0)
    assert (edge == 7.0).all()


def test_gradients_of_nothing():
    dy, packed, exact, tol = gradient_case(130, 20, 40, F32, 5)
    c = randn(20, 40, seed=1)
    keep = c.clone()
    assert torch.equal(tcec.wgrad_q8(dy[:0], packed[:0], 40, c, beta=1.0), keep)  # no tokens: nothing is added
    assert torch.equal(tcec.wgrad_q8(dy[:0], packed[:0], 40), torch.zeros(20, 40, device=DEV))
    assert torch.equal(tcec.wgrad_q8(dy * float("nan"), packed, 40, c, alpha=0.0, beta=1.0), keep)
    assert tcec.wgrad_q8(dy[:, :0], packed, 40).shape == (0, 40)
    dy[3, 4] = float("nan")
    bad = tcec.wgrad_q8(dy, packed, 40).isnan()
    assert bad[4].all() and bad.sum() == 40


# ---------------------------------------------------------------- as they are used
def test_a_layer_is_served_and_trained():
    """A frozen layer in 4 bits with a trained adapter of low rank: y = x W^T + (x A^T) B^T, the input kept in 8 bits for dA."""
    m, n, k, rank = 300, 256, 384, 16
    w, a, b, x = randn(n, k, seed=1) / 20, randn(rank, k, seed=2) / 20, randn(n, rank, seed=3), randn(m, k, seed=4)
    packed = tcec.pack_q4(w)
    kept = tcec.pack_q8(x)
    low = tcec.sgemm(x, a.T)
    y = tcec.gemm_q4(x, packed, n)
    tcec.sgemm(low, b.T, y, beta=1.0)
    dy = randn(m, n, seed=5)
    dlow = tcec.sgemm(dy, b)
    da = tcec.wgrad_q8(dlow, kept, k)
    db = tcec.sgemm(dy.T, low)
    wq, xq = values(w, 128, F16), (lambda t: t[0] * t[1])(quantise8(x))
    low64 = x.double() @ a.double().T
    y64 = x.double() @ wq.T + low64 @ b.double().T
    dlow64 = dy.double() @ b.double()
    for got, want in ((y, y64), (da, dlow64.T @ xq), (db, dy.double().T @ low64)):
        assert (got.double() - want).norm() <= 4e-6 * want.norm()
    # against differences: the loss sum(dy * y) along a direction of A, with the kept input
    d = randn(rank, k, seed=6).double()
    loss = lambda t: (dy.double() * ((xq @ (a.double() + t * d).T) @ b.double().T)).sum()  # noqa: E731
    slope = (loss(1e-3) - loss(-1e-3)) / 2e-3
    # the loss is linear in A, so the difference's own error is its rounding alone
    assert abs((da.double() * d).sum() - slope) <= 1e-5 * (da.double() * d).abs().sum()
    # one token at a time gives the rows of the whole
    for i in (0, 299):
        one = tcec.gemm_q4(x[i:i + 1], packed, n)
        assert (one.double() - x[i:i + 1].double() @ wq.T).norm() <= 4e-6 * (x[i:i + 1].double() @ wq.T).norm()


@pytest.mark.parametrize("m", [2, 90])
def test_calls_are_captured_and_replayed(m):
    n, k = 144, 320
    x, packed, exact, tol = product_case(m, n, k, 128, BF16, 19)
    dy, kept, exact_g, tol_g = gradient_case(m, n, k, BF16, 21)
    c, g = torch.zeros(m, n, device=DEV, dtype=BF16), torch.zeros(n, k, device=DEV, dtype=BF16)
    tcec.gemm_q4(x, packed, n, c)
    tcec.wgrad_q8(dy, kept, k, g)
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        tcec.gemm_q4(x, packed, n, c)
    with torch.cuda.graph(second):
        tcec.wgrad_q8(dy, kept, k, g)
    side = torch.cuda.Stream()
    for _ in range(5):  # both at once: each has a workspace of its own
        c.zero_(), g.zero_()
        side.wait_stream(torch.cuda.current_stream())
        first.replay()
        with torch.cuda.stream(side):
            second.replay()
        torch.cuda.current_stream().wait_stream(side)
        check(c, exact, tol)
        check(g, exact_g, tol_g)
    tcec.device_status()


def test_equal_calls_give_equal_bits_on_any_stream():
    x, packed, exact, tol = product_case(100, 500, 1000, 32, F32, 23)
    dy, kept, _, _ = gradient_case(3000, 40, 300, F32, 25)
    one, grad = tcec.gemm_q4(x, packed, 500, group=32), tcec.wgrad_q8(dy, kept, 300)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append((tcec.gemm_q4(x, packed, 500, group=32), tcec.wgrad_q8(dy, kept, 300)))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, one) and torch.equal(b, grad)


def test_python_refuses():
    x, packed, _, _ = product_case(4, 32, 64, 32, F32, 27)
    good = dict(group=32)
    for call in (
        lambda: tcec.gemm_q4(x, packed[:-16], 32, **good),
        lambda: tcec.gemm_q4(x, packed, 129, **good),
        lambda: tcec.gemm_q4(x, packed, 32, group=48),
        lambda: tcec.gemm_q4(x.double(), packed, 32, **good),
        lambda: tcec.gemm_q4(x[None], packed, 32, **good),
        lambda: tcec.gemm_q4(x[:, ::2], packed, 32, **good),
        lambda: tcec.gemm_q4(x, packed, 32, dtype=F16, **good),
        lambda: tcec.gemm_q4(x, packed, 32, beta=1.0, **good),
        lambda: tcec.gemm_q4(x, packed, 32, torch.empty(4, 31, device=DEV), **good),
        lambda: tcec.gemm_q4(x, packed, 32, torch.empty(4, 32), **good),
        lambda: tcec.gemm_q4(x, packed.cpu(), 32, **good),
        lambda: tcec.pack_q4(x, scale=F32),
        lambda: tcec.pack_q4(x, out=torch.empty(16, dtype=torch.uint8, device=DEV)),
        lambda: tcec.pack_q8(x, out=torch.empty(16, dtype=torch.uint8, device=DEV)),
        lambda: tcec.unpack_q4(packed, 32, 64, group=32, out=torch.empty(32, 63, device=DEV)),
        lambda: tcec.wgrad_q8(x, packed, 64),  # too small for activations
        lambda: tcec.pack_q4_codes(torch.zeros(4, 3, dtype=torch.uint8, device=DEV), torch.ones(4, 1, device=DEV).half(), k=4),
        lambda: tcec.pack_q4_codes(torch.zeros(4, 2, dtype=torch.uint8, device=DEV), torch.ones(4, 2, device=DEV).half(), k=4),
    ):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(tcec.TcecError) as e:  # the result over its own operand
        tcec.gemm_q4(x[:, :32], packed, 32, x[:, :32], group=32)
    assert e.value.status == tcec.ERR_INVALID_ARGUMENT


# ---------------------------------------------------------------- every form of the kernels
@pytest.mark.parametrize("n,k", [(2400, 200), (4810, 130), (8200, 100), (8200, 4100), (9000, 4000), (9600, 300), (9600, 4100)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_few_tokens_of_wide_layers(n, k, group, dtype):
    for m in (1, 2, 5, 8, 10, 12, 16, 24, 32):
        x, packed, exact, tol = product_case(m, n, k, group, dtype, m + n)
        check(tcec.gemm_q4(x, packed, n, group=group), exact, tol)
    tcec.device_status()


@pytest.mark.parametrize("m,n,k", [(40, 1792, 4096), (40, 1921, 4096), (70, 4096, 2050), (40, 4224, 1100), (70, 9400, 1030), (200, 700, 5000),
                                   (600, 4500, 260)])
@pytest.mark.parametrize("dtype,group", [(F32, 32), (F16, 64), (BF16, 128)])
def test_products_divided_among_clusters(m, n, k, dtype, group):
    x, packed, exact, tol = product_case(m, n, k, group, dtype, m + n)
    check(tcec.gemm_q4(x, packed, n, group=group), exact, tol)
    tcec.device_status()


@pytest.mark.parametrize("m", [1, 2, 12, 20, 40])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_without_a_sum_c_is_scaled(m, dtype):
    x, packed, _, _ = product_case(m, 300, 4096, 128, dtype, 31)
    c = randn(m, 300, seed=32, dtype=dtype)
    half = (0.5 * c.double()).to(dtype)
    assert torch.equal(tcec.gemm_q4(x * float("nan"), packed, 300, c.clone(), alpha=0.0, beta=0.5), half)
    assert torch.equal(tcec.gemm_q4(x[:, :0], packed[:0], 300, c.clone(), beta=0.5), half)
    assert (tcec.gemm_q4(x, packed, 300, c.fill_(float("nan")), alpha=0.0) == 0).all()


@pytest.mark.parametrize("m", [1, 2, 5, 9, 10, 24, 60])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tokens_of_any_magnitude(m, dtype):
    """Relative to the largest magnitudes of a token, whatever they are: from 2^-110 (few tokens; more: 2^-90) to 2^100, in a block or in all.

    bound() has an absolute part of 1e-30, so tokens are compared after their results are scaled back, by a power of two.  With one large value
    the rounding of few tokens is relative to scale * (code + zero) * |x|, not to scale * |code - zero| * |x|: the sums of code * x and of x over a
    group are made apart, each rounded to 2^-24 of itself, and the zero point times the second is taken off the first.  Where the code of a value
    2^90 is its zero point the exact term is 0, and 2^-24 * scale * 2 * zero * 2^90 is left of it.
    """
    n, k = 70, 500
    byte, s, z, w = with_codes(n, k, 64, 33)
    packed = tcec.pack_q4_codes(byte, s, z, k=k, group=64)
    base = randn(m, k, seed=m, dtype=dtype)
    for exponent in (-110 if m * (3 if dtype == F32 else 1) <= 32 else -90, -61, -59, 26, 28, 100):
        x = (base.double() * 2.0**exponent).to(dtype)
        exact = base.double() @ w.T
        got = tcec.gemm_q4(x, packed, n, group=64, dtype=F32).double() * 2.0**-exponent
        check(got, exact, bound(base.double().abs() @ w.abs().T, exact, F32, k, 3 if dtype == F32 else 1))
    # a large value in one block of some tokens: these lose what lies far below it, the others nothing
    x = base.clone()
    x[::2, 200] *= 2.0**90
    got = tcec.gemm_q4(x, packed, n, group=64, dtype=F32)
    exact = x.double() @ w.T
    each = torch.arange(k, device=DEV) // 64
    sizes = (torch.stack([byte & 15, byte >> 4], 2).reshape(n, -1)[:, :k].double() + z.double()[:, each]) * s.double()[:, each]
    check(got, exact, bound(x.double().abs() @ sizes.T, exact, F32, k, 3 if dtype == F32 else 1))
    assert torch.equal(got[1::2], tcec.gemm_q4(base, packed, n, group=64, dtype=F32)[1::2])


def test_one_token_that_is_not_finite():
    for dtype in (F32, F16, BF16):
        x, packed, _, _ = product_case(1, 64, 256, 128, dtype, 35)
        x[0, 130] = float("nan")
        assert tcec.gemm_q4(x, packed, 64).isnan().all()
        x[0, 130] = -float("inf")
        assert not tcec.gemm_q4(x, packed, 64).isfinite().any()


@pytest.mark.parametrize("m", [1, 12])
def test_replays_see_new_tokens_and_new_weights(m):
    n, k = 200, 700
    x, packed, _, _ = product_case(m, n, k, 128, BF16, 37)
    c = torch.zeros(m, n, device=DEV, dtype=BF16)
    tcec.gemm_q4(x, packed, n, c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tcec.gemm_q4(x, packed, n, c)
    for seed in (41, 43, 45):
        x2, packed2, exact, tol = product_case(m, n, k, 128, BF16, seed)
        x.copy_(x2), packed.copy_(packed2)
        graph.replay()
        check(c, exact, tol)


def test_calls_of_several_threads_at_once():
    import threading

    cases = [product_case(m, 300, 900, 64, dtype, m) for m, dtype in ((1, F32), (7, BF16), (30, F16), (100, BF16))]
    torch.cuda.synchronize()
    got, streams = [None] * 4, [torch.cuda.Stream() for _ in range(4)]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(50):
                got[i] = tcec.gemm_q4(cases[i][0], cases[i][1], 300, group=64)
        streams[i].synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for c, (_, _, exact, tol) in zip(got, cases):
        check(c, exact, tol)
    tcec.device_status()


def test_packing_and_product_one_after_the_other_without_a_wait():
    """Each call may start before the one before has ended; what it reads has been written all the same."""
    n, k = 1000, 2000
    for i in range(20):
        w = randn(n, k, seed=i, dtype=BF16)
        x = randn(3 + i, k, seed=i + 50, dtype=BF16)
        packed = torch.empty(tcec.q4_bytes(n, k, 128), dtype=torch.uint8, device=DEV)
        kept = torch.empty(tcec.q8_bytes(3 + i, k), dtype=torch.uint8, device=DEV)
        torch.cuda.synchronize()
        y = tcec.gemm_q4(x, tcec.pack_q4(w, out=packed), n)
        g = tcec.wgrad_q8(y, tcec.pack_q8(x, out=kept), k, dtype=F32)
        q, s = quantise8(x)
        wq = values(w, 128, F16)
        exact = x.double() @ wq.T
        check(y, exact, bound(x.double().abs() @ wq.abs().T, exact, BF16, k, 1))
        exact = y.double().T @ (q * s)
        check(g, exact, bound(y.double().abs().T @ (q * s).abs(), exact, F32, 3 + i, 1))


def test_operands_and_result_side_by_side_in_one_matrix():
    x, packed, exact, tol = product_case(6, 96, 160, 32, F32, 51)
    whole = torch.full((6, 300), 7.0, device=DEV)
    whole[:, 10:170] = x
    check(tcec.gemm_q4(whole[:, 10:170], packed, 96, whole[:, 180:276], group=32), exact, tol)
    assert (whole[:, 170:180] == 7.0).all() and (whole[:, 276:] == 7.0).all() and torch.equal(whole[:, 10:170], x)
    for c in (whole[:, 169:265], whole[:, :96]):
        with pytest.raises(tcec.TcecError):
            tcec.gemm_q4(whole[:, 10:170], packed, 96, c, group=32)


def test_with_sms_left_to_others():
    lib = tcec.load()
    x, packed, exact, tol = product_case(40, 300, 4096, 128, BF16, 53)
    y, packed2, exact2, tol2 = product_case(1350, 2170, 300, 128, BF16, 55)
    assert lib.tcec_set_option(b"reserve_sms", 20) == 0
    try:
        check(tcec.gemm_q4(x, packed, 300), exact, tol)
        check(tcec.gemm_q4(y, packed2, 2170), exact2, tol2)
    finally:
        lib.tcec_set_option(b"reserve_sms", 0)


def test_python_and_the_native_binding_agree(monkeypatch):
    x, packed, _, _ = product_case(12, 130, 300, 64, BF16, 57)
    w, dy = randn(130, 300, seed=1), randn(12, 50, seed=2)

    def all_calls():
        p, q = tcec.pack_q4(w, 64), tcec.pack_q8(w)
        c, g = torch.ones(12, 130, device=DEV), torch.ones(300, 50, device=DEV).T
        return [p, q, tcec.unpack_q4(p, 130, 300, 64, BF16), tcec.unpack_q8(q, 130, 300), tcec.gemm_q4(x, packed, 130, group=64),
                tcec.gemm_q4(x, packed, 130, c, group=64, alpha=2.0, beta=-1.0), tcec.wgrad_q8(dy, tcec.pack_q8(w[:12]), 300),
                tcec.wgrad_q8(dy, tcec.pack_q8(w[:12]), 300, g, beta=1.0), tcec.gemm_q4(x, packed, 130, group=64, dtype=F32)]

    assert tcec._binding is not None
    native = all_calls()
    monkeypatch.setattr(tcec, "_binding", None)
    for a, b in zip(native, all_calls()):
        assert a.dtype == b.dtype and a.stride() == b.stride() and torch.equal(a, b)


@pytest.mark.parametrize("m,k", [(1, 2400), (130, 2369), (3000, 1000), (4100, 2700), (700, 9000)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gradients_of_few_columns(m, k, dtype):
    for n in (1, 2, 3, 5, 8, 10, 11, 16, 17, 32, 33):
        dy, packed, exact, tol = gradient_case(m, n, k, dtype, m + n)
        check(tcec.wgrad_q8(dy, packed, k), exact, tol)
        c = randn(n, k, seed=n)
        want = exact - 2.0 * c.double()
        check(tcec.wgrad_q8(dy.T.contiguous().T, packed, k, c, beta=-2.0), want, tol + want.abs() * 2.0**-22 + exact.abs() * 2.0**-22)
    tcec.device_status()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_of_any_magnitude(dtype):
    """As tokens of any magnitude: a column's power of two is of its largest value in a block."""
    m, n, k = 300, 6, 200
    dy, packed, exact, tol = gradient_case(m, n, k, dtype, 61, F32)
    for exponent in (-110 if dtype == BF16 else -90, -61, -59, 26, 28, 100):
        got = tcec.wgrad_q8((dy.double() * 2.0**exponent).to(dtype), packed, k, dtype=F32).double() * 2.0**-exponent
        check(got, exact, tol)
    bad = dy.clone()
    bad[5, 2], bad[200, 4] = float("nan"), float("inf")
    got = tcec.wgrad_q8(bad, packed, k, dtype=F32)
    clean = tcec.wgrad_q8(dy, packed, k, dtype=F32)
    keep = [0, 1, 3, 5]
    assert got[2].isnan().all() and not got[4].isfinite().any() and torch.equal(got[keep], clean[keep])


def test_offsets_beyond_32_bits():
    """Packed weights of 4.6 GB (one tile of rows, repeated), and dense matrices whose lines lie 2^31 elements apart."""
    k, tiles = 65536, 1024
    tile = tcec.pack_q4(randn(128, k, seed=1, dtype=BF16))
    w = tcec.unpack_q4(tile, 128, k).double()
    packed = tile.repeat(tiles)
    for m in (1, 4, 12, 40):
        x = randn(m, k, seed=m, dtype=BF16)
        exact = x.double() @ w.T
        tol = bound(x.double().abs() @ w.abs().T, exact, F32, k, 1)
        got = tcec.gemm_q4(x, packed, 128 * tiles, dtype=F32).reshape(m, tiles, 128)
        for t in (0, 480, 1023):
            check(got[:, t], exact, tol)
        assert torch.equal(got[:, 5], got[:, 1000])
    del packed, got
    features = tcec.pack_q8(randn(40000, 128, seed=2))
    kept = features.repeat(512)
    w = tcec.unpack_q8(features, 40000, 128).double()
    dy = randn(40000, 40, seed=3, dtype=BF16)
    for n in (4, 16, 40):
        exact = dy[:, :n].double().T @ w
        got = tcec.wgrad_q8(dy[:, :n].contiguous(), kept, 128 * 512, dtype=F32).reshape(n, 512, 128)
        check(got[:, 511], exact, bound(dy[:, :n].double().abs().T @ w.abs(), exact, F32, 40000, 1))
        assert torch.equal(got[:, 3], got[:, 500])
    del kept, got
    ld = 2**31 + 8
    store = torch.empty(2 * ld + 256, device=DEV, dtype=BF16)
    far = store.as_strided((3, 256), (ld, 1))
    near = randn(3, 256, seed=4, dtype=BF16)
    far.copy_(near)
    w = tcec.pack_q4(randn(256, 256, seed=5))
    assert torch.equal(tcec.gemm_q4(far, w, 256), tcec.gemm_q4(near, w, 256))
    assert torch.equal(tcec.gemm_q4(far[2:], w, 256), tcec.gemm_q4(near[2:], w, 256))
    assert torch.equal(tcec.pack_q4(far), tcec.pack_q4(near)) and torch.equal(tcec.pack_q8(far), tcec.pack_q8(near))
    q4, q8 = tcec.pack_q4(near), tcec.pack_q8(near)
    assert torch.equal(tcec.unpack_q4(q4, 3, 256, out=far), tcec.unpack_q4(q4, 3, 256, dtype=BF16))
    assert torch.equal(tcec.unpack_q8(q8, 3, 256, out=far), tcec.unpack_q8(q8, 3, 256, dtype=BF16))
    assert torch.equal(tcec.gemm_q4(near, w, 256, far), tcec.gemm_q4(near, w, 256))
    for n in (16, 256):
        far.copy_(near)
        kept = tcec.pack_q8(randn(3, 70, seed=6))
        assert torch.equal(tcec.wgrad_q8(far[:, :n], kept, 70), tcec.wgrad_q8(near[:, :n], kept, 70))
    tcec.device_status()
