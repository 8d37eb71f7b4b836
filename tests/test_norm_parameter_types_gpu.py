"""The layer norm with parameters of another type than x, in each of the
kernels' forms, with parameter rows that start on their own elements only, and
with rows of x that start anywhere; bounds as in test_block_ops_gpu.py."""
import pytest
import torch

from tests import block_ops_support as sup
from tests.test_block_ops_gpu import BF, F32, _gen, _norm_tols, _rn

pytestmark = pytest.mark.gpu


def check(x, w, b, dy, off, per):
    from foundry_trainer_b200 import ops
    y, stats = ops.layer_norm(x, w, b, unit_offset=off == 1.0)
    dx, dw, db = ops.layer_norm_bwd(x, w, dy, stats, unit_offset=off == 1.0)
    again = ops.layer_norm_bwd(x, w, dy, stats, unit_offset=off == 1.0)
    one = torch.ones(x.shape[-1], device="cuda", dtype=torch.float64)
    wd = w.double() if w is not None else one  # no weight: a gain of 1
    bd = b.double() if b is not None else 0 * one
    if per:
        wd, bd = (t[:, None] if t.dim() == 2 else t for t in (wd, bd))
    gain_off = off if w is not None else 0.0
    x3, dy3 = (t if t.dim() == 3 else t[None] for t in (x, dy))
    ry, h, rstd, _ = sup.norm_ref(x3, wd, bd, 1e-6, gain_off)
    rdx, rdw, rdb = sup.norm_bwd_ref(x3, wd, dy3, 1e-6, gain_off, not per)
    u, ty, tx, th = _norm_tols(x3, wd, dy3, h, rstd, gain_off, x.dtype)
    n = x3.shape[0] * x3.shape[1]
    dims = (1,) if per else (0, 1)
    sup.within(y.view_as(x3), ry, u * ry.abs() + ty + sup.STEP32 * bd.abs(), "y")
    sup.within(dx.view_as(x3), rdx, u * rdx.abs() + tx, "dx")
    assert dw.dtype == F32 and db.dtype == F32
    sup.within(dw, rdw, (dy3.double().abs() * (th + n * sup.STEP32 * h.abs())).sum(dims), "dw")
    sup.within(db, rdb, n * sup.STEP32 * dy3.double().abs().sum(dims), "db")
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("G,R,D,per", [
    (1, 3, 64, False), (3, 17, 64, True), (2, 700, 2048, True), (1, 1300, 520, False),
    (1, 1201, 8200, True), (1, 5, 16384, False), (1, 700, 250, True), (7, 5, 5798, False),
    (2, 33, 1001, True), (1, 3, 16381, False), (1, 1200, 12, False),
    # many groups of few rows, where the form goes by the rows of all groups
    (1300, 1, 1024, True), (400, 3, 2048, True), (1500, 2, 512, False),
])
def test_parameters_of_the_other_type(G, R, D, per, dtype):
    g = _gen(G * 100 + R + D)
    other = F32 if dtype == BF else BF
    x, dy = (_rn(g, G, R, D) * 2 + 0.5).to(dtype), _rn(g, G, R, D, dtype=dtype)
    w, b = (_rn(g, *((G, D) if per else (D,)), std=0.3, dtype=other) for _ in range(2))
    check(x, w, b, dy, 1.0 if per else 0.0, per)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("par", [BF, F32])
@pytest.mark.parametrize("shift", [1, 2, 4])
@pytest.mark.parametrize("D", [2048, 256, 5798])
def test_parameters_that_start_on_any_element(D, shift, par, dtype):
    g = _gen(D + shift)
    x, dy = _rn(g, 2, 611, D, dtype=dtype), _rn(g, 2, 611, D, dtype=dtype)
    both = _rn(g, 2, 2 * D + shift, std=0.3, dtype=par)
    w, b = both[:, shift:].split(D, dim=-1)  # a row stride that 16 bytes do not divide either
    check(x, w, b, dy, 1.0, True)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("R,D", [(40, 320), (1300, 1024), (9, 6000)])
def test_rows_that_start_on_any_element(R, D, dtype):
    g = _gen(R + D)
    x, dy = (_rn(g, R, D + 1, dtype=dtype)[:, 1:] for _ in range(2))
    w = _rn(g, D, std=0.3, dtype=dtype)
    check(x, w, None, dy, 0.0, False)
    check(x, None, None, dy, 0.0, False)
