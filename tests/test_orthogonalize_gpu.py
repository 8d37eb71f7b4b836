"""The Newton-Schulz orthogonalisation on the GPU against the same iteration in
64 bits.

Bounds, relative to the result's Frobenius norm. The stored result is rounded
once to bf16: at most 2^-8 of every entry. Short side <= 64: everything before
that is fp64 but the last product (fp32, whose factor's entries reach a^steps,
about 485, times the result's: 485 * 2^-24 * (64 + 2) = 1.9e-3 at the worst,
when every rounding adds up). Longer sides: the products' operands are rounded
to fp16, 2^-12 relative to an entry; per step X's product, Q and b Q + c Q^2
carry three such roundings, and an error is carried on by the following steps
within the matrix's own directions with a gain of at most max |p'| = a = 3.45
on the first step it meets and at most 1.9 on average over five (p maps [0, 1]
onto itself up to 1.2): 15 roundings * 2^-12 * 1.9 = 7e-3 if all align, and
(15)^1/2 * 2^-12 * 1.9 = 1.8e-3 as independent ones, to which the bound below
allows twice, as an rms over many entries."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
COEFFS = (3.4445, -4.7750, 2.0315)


def plain(g, steps=5, coeffs=COEFFS, eps=1e-7):
    a, b, c = coeffs
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + eps)
    for _ in range(steps):
        q = x @ x.mT
        x = a * x + (b * q + c * (q @ q)) @ x
    return x.mT if tall else x


def bound(shape):
    return 2.0 ** -8 + (1.9e-3 if min(shape) <= 64 else 3.6e-3)


def rel(o, ref):
    return ((o.double() - ref).norm() / ref.norm()).item()


def gradient(seed, *shape, rank=4, noise=0.1, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    *lead, m, n = shape
    r = lambda *s: torch.randn(*lead, *s, generator=g, device="cuda")
    return ((r(m, rank) @ r(rank, n) + noise * r(m, n)) * 1e-3).to(dtype)


SHAPES = [(1, 1), (1, 8, 8), (3, 16, 4096), (2, 4096, 16), (5, 12, 1000), (2, 1001, 7), (1, 33, 65),
          (2, 64, 2048), (2, 2056, 64), (1, 64, 64), (1, 5, 3), (4, 48, 3001), (1, 65, 65),
          (2, 72, 200), (1, 200, 72), (1, 256, 512), (2, 300, 1000), (1, 1000, 300), (1, 777, 777),
          (1, 1024, 2048), (1, 1500, 520),
          # the SM-pair form of all three products, upright and tall, ragged
          (1, 4096, 4104), (1, 4500, 4100), (3, 2305, 2500),
          # tall rows of 8 bytes, and of no such number
          (3, 1000, 12), (2, 700, 36), (2, 300, 61),
          # few tiles and a long contraction
          (1, 100, 8200), (2, 3001, 130)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize_matches_64_bits(shape, dtype):
    from foundry_trainer_b200 import ops
    for k, kw in enumerate((dict(rank=4, noise=0.1), dict(rank=1, noise=1.0))):
        g = gradient(k, *shape, dtype=dtype, **kw)
        o = ops.orthogonalize(g)
        again = ops.orthogonalize(g)
        torch.cuda.synchronize()
        assert ops.device_status() == 0
        assert o.dtype == BF and o.shape == g.shape
        assert rel(o, plain(g)) <= bound(shape[-2:]), (k, rel(o, plain(g)))
        assert torch.equal(o, again)


@pytest.mark.parametrize("m,n", [(16, 512), (512, 16), (160, 256)])
def test_orthogonalize_scale_zero_and_non_finite(m, n):
    from foundry_trainer_b200 import ops
    g = gradient(9, m, n, dtype=F32)
    ref = ops.orthogonalize(g)
    # the norm is taken in fp64: squares may leave fp32's range. With eps 0 a
    # power of two drops out exactly (an eps of 1e-7 would not: it is 5e-7 of
    # this norm, nothing of the scaled one's)
    ref0 = ops.orthogonalize(g, eps=0.0)
    assert torch.equal(ops.orthogonalize(g * 2.0 ** 90, eps=0.0), ref0)
    assert rel(ops.orthogonalize(g * 2.0 ** -80, eps=0.0), plain(g)) <= bound((m, n))
    assert not ops.orthogonalize(torch.zeros_like(g)).any()
    for v in (float("nan"), float("inf")):
        bad = torch.stack([g, g])
        bad[1, 3, 5] = v
        o = ops.orthogonalize(bad)
        assert torch.equal(o[0], ref)  # the other matrix of the batch is left alone
        assert not torch.isfinite(o[1].float()).all()


@pytest.mark.parametrize("shape", [(24, 640), (640, 24), (96, 320), (320, 96)])
def test_orthogonalize_strides_steps_and_coefficients(shape):
    from foundry_trainer_b200 import ops
    m, n = shape
    big = gradient(5, 3, m, n + 24)
    g = big[:, :, 9:9 + n]  # rows that start anywhere
    assert torch.equal(ops.orthogonalize(g), ops.orthogonalize(g.contiguous()))
    out = torch.zeros(3, m, n + 8, device="cuda", dtype=BF)
    ops.orthogonalize(g, out=out[:, :, :n])
    assert torch.equal(out[:, :, :n], ops.orthogonalize(g)) and not out[:, :, n:].any()
    for steps, co in ((1, COEFFS), (2, (1.5, -0.5, 0.0)), (8, (2.0, -1.5, 0.5))):
        assert rel(ops.orthogonalize(g, steps=steps, coeffs=co), plain(g, steps, co)) <= bound(shape)
    assert ops.orthogonalize(g[:0]).shape == (0, m, n)


def test_orthogonalize_keeps_weak_directions_of_a_thin_factor():
    # singular values from 1 to 1e-4 of the largest: the Gram matrix's
    # eigenvalues span 1e-8, more than fp32 sums would keep
    from foundry_trainer_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(2)
    u = torch.linalg.qr(torch.randn(16, 16, generator=g, device="cuda", dtype=torch.float64))[0]
    v = torch.linalg.qr(torch.randn(2048, 16, generator=g, device="cuda", dtype=torch.float64))[0]
    s = torch.logspace(0, -4, 16, device="cuda", dtype=torch.float64)
    x = ((u * s) @ v.T).float()
    ref = plain(x)
    got = ops.orthogonalize(x).double()
    # along each singular direction, not only in the norm of the whole: the
    # bf16 rounding of the entries, and the last product's, as noise of which
    # one direction sees the share of one
    for i in range(16):
        want = (u[:, i] @ ref @ v[:, i]).item()
        have = (u[:, i] @ got @ v[:, i]).item()
        assert abs(want - have) <= bound((16, 2048)) * max(abs(want), 0.05), (i, want, have)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,n", [(16, 512), (500, 20), (60, 256), (160, 256), (256, 160)])
def test_orthogonalize_at_the_ends_of_the_range(m, n, dtype):
    # norms near the smallest and largest values of the type, without an eps
    from foundry_trainer_b200 import ops
    g = gradient(3, m, n, dtype=dtype)
    for scale in (2.0 ** -122, 2.0 ** -70, 2.0 ** 70, 2.0 ** 126):
        x = (g.float() * scale).to(dtype)
        assert x.isfinite().all() and x.any()
        o = ops.orthogonalize(x, eps=0.0)
        assert rel(o, plain(x, eps=0.0)) <= bound((m, n)), scale
