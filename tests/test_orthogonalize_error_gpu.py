"""The wide form's error as an rms over the result, which X kept as two fp16
parts gives and one part does not.

The result's rounding to bf16: an error uniform over a step of 2^-7 of a value's
power of two, so at most 2^-7 / sqrt(12) = 2.26e-3 of the value as an rms (1.7e-3
over many mantissas). Before it five steps, each with three operands rounded to
fp16: 2^-10 / sqrt(12) = 2.8e-4 each at most, independent, within the matrix's own
directions, where the following steps carry an error with a gain of 1.9 on
average: sqrt(15) 2.8e-4 1.9 = 2.1e-3. Together sqrt(2.26^2 + 2.1^2) e-3 = 3.1e-3.
A rounding of X itself is noise in all directions, of which the steps amplify
those where the matrix has no strength up to 485-fold: the same iteration with
the low part dropped, rounded on the CPU as the kernels round, is off by 5.4e-3
to 1.3e-2 on matrices of falling singular values or of a few strong directions
over noise (1.7e-3 to 1.9e-3 with it; on Gaussian noise 2.2e-3 and 2.4e-3)."""
import pytest
import torch

from tests.test_orthogonalize_gpu import gradient, plain, rel

pytestmark = pytest.mark.gpu

BOUND = 3.1e-3


def falling(seed, batch, m, n):
    """Matrices whose singular values fall from 1 to 1e-4."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = min(m, n)
    q = lambda k: torch.linalg.qr(torch.randn(batch, k, r, generator=g, device="cuda",
                                              dtype=torch.float64))[0]
    s = torch.logspace(0, -4, r, device="cuda", dtype=torch.float64)
    return ((q(m) * s) @ q(n).mT).float()


# narrow tiles (upright, tall, a long contraction split, ragged), and matrices
# that fill the SM pairs in all three products
@pytest.mark.parametrize("batch,m,n", [(1, 128, 2048), (1, 2048, 128), (2, 72, 200), (1, 1000, 204),
                                       (1, 768, 1024), (1, 100, 8200), (2, 1536, 4096),
                                       (2, 4096, 1536)])
def test_weak_directions_of_a_matrix(batch, m, n):
    from foundry_trainer_b200 import ops
    x = falling(m + n, batch, m, n)
    ref = plain(x)
    got = ops.orthogonalize(x)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    for o, r in zip(got, ref):
        assert rel(o, r) <= BOUND, rel(o, r)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,m,n", [(2, 72, 200), (1, 300, 1000), (1, 1000, 300), (1, 1024, 2048),
                                       (2, 1536, 4096)])
def test_rms_error_of_gradients(batch, m, n, dtype):
    from foundry_trainer_b200 import ops
    for k, kw in enumerate((dict(rank=4, noise=0.1), dict(rank=1, noise=1.0))):
        g = gradient(k, batch, m, n, dtype=dtype, **kw)
        assert rel(ops.orthogonalize(g), plain(g)) <= BOUND, (k, rel(ops.orthogonalize(g), plain(g)))


@pytest.mark.parametrize("m,n", [(96, 320), (320, 96), (40, 512)])
def test_coefficients_near_the_range_of_fp16(m, n):
    # One step takes a singular value of 1 to 4.7, where 64 (b Q + c Q^2) is 56700
    # of fp16's 65504, all of it in one entry. Its relative error: the first step's
    # roundings of Q, b Q + c Q^2 and X, 2^-11 each of terms of 2.7 (the sum) and 6.8
    # (|b| + |c|) to 4.7: 1.6e-3, times s p'(s) / p(s) = 5.2 at 4.7; the second's, four
    # of 2^-11; the result's, 2^-8: 1.5e-2 if all align.
    from foundry_trainer_b200 import _lib, ops
    co = (7.4435, -4.7750, 2.0315)
    g = torch.zeros(2, m, n, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(m)
    v = torch.randn(max(m, n), generator=gen, device="cuda")
    u = torch.randn(min(m, n), generator=gen, device="cuda")
    one, spread = (v[None], u[:, None] * v) if m <= n else (v[:, None], v[:, None] * u)
    if m <= n:
        g[0, 7:8] = one
    else:
        g[0, :, 7:8] = one
    g[1] = spread
    ref = plain(g, 2, co)
    got = ops.orthogonalize(g, steps=2, coeffs=co)
    assert torch.isfinite(got).all()
    for o, r in zip(got, ref):
        assert rel(o, r) <= 1.5e-2, rel(o, r)
    if min(m, n) > 64:
        with pytest.raises(_lib.FaError):
            ops.orthogonalize(g, steps=3, coeffs=co)
    else:
        ref = plain(g, 3, co)
        assert rel(ops.orthogonalize(g, steps=3, coeffs=co), ref) <= 5 * 1.5e-2


@pytest.mark.parametrize("shape", [(5, 16, 4096), (3, 1000, 24), (2, 61, 304), (2, 400, 56), (1, 96, 320),
                                   (2, 320, 96), (1, 1536, 2048)])
def test_out_may_be_the_input(shape):
    # nothing reads an element of the input after its place has been written
    from foundry_trainer_b200 import ops
    g = gradient(4, *shape)
    want = ops.orthogonalize(g)
    got = ops.orthogonalize(g, out=g)
    assert got is g and torch.equal(g, want)
