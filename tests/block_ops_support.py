"""Plain 64-bit forms of the block operators and the error bounds the tests
hold the kernels to (used by the tests only).

Every bound is a sum of roundings: half a step of the stored type per
rounding (u = finfo.eps / 2, relative to the value rounded), and for a sum of
n products in fp32 n steps of 2^-23 relative to the sum of the products'
magnitudes (a full step, not half: the tensor cores cut off rather than round
when they align addends)."""
from __future__ import annotations

import torch

U16 = 2.0 ** -8      # half a bf16 step
STEP32 = 2.0 ** -23  # a full fp32 step


def within(got: torch.Tensor, ref: torch.Tensor, tol: torch.Tensor, what: str) -> None:
    """|got - ref| <= tol element by element; non-finite references must match."""
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape, (what, tuple(got.shape), tuple(ref.shape))
    fin = torch.isfinite(ref)
    assert torch.equal(fin, torch.isfinite(got)), f"{what}: finite in other places"
    off = ((got - ref).abs() - tol)[fin]
    if off.numel():
        worst = off.max().item()
        assert worst <= 0, (f"{what}: over its bound by {worst:.3e} "
                            f"(error {(got - ref).abs()[fin].max().item():.3e})")


def norm_ref(x, w, b, eps, off):
    """(y, h, rstd, mean) in 64 bits; w, b broadcastable over (G, R, D)."""
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    h = (x - mean) * rstd
    return h * (off + w) + b, h, rstd, mean


def norm_bwd_ref(x, w, dy, eps, off, shared):
    _, h, rstd, _ = norm_ref(x, w, 0.0, eps, off)
    t = dy.double() * (off + w)
    dx = rstd * (t - t.mean(-1, keepdim=True) - h * (t * h).mean(-1, keepdim=True))
    dims = (0, 1) if shared else (1,)
    return dx, (dy.double() * h).sum(dims), dy.double().sum(dims)


def lora_ref(x, w, a, b, scale, bias):
    """y and its bound for one adapter (64-bit inputs)."""
    low = scale * (x @ a.T)
    y = x @ w.T + low @ b.T
    if bias is not None:
        y = y + bias
    K, r = x.shape[1], a.shape[0]
    # low: fp32 sum over K, then one rounding
    low_err = U16 * low.abs() + K * STEP32 * abs(scale) * (x.abs() @ a.abs().T)
    tol = (low_err + (r + 1) * STEP32 * low.abs()) @ b.abs().T
    tol = tol + (K + r + 2) * STEP32 * (x.abs() @ w.abs().T)
    if bias is not None:
        tol = tol + STEP32 * bias.abs()
    return y, U16 * (y.abs() + tol) + tol, low, low_err


def lora_bwd_ref(x, w, a, b, dy, scale):
    """((dx, tol), (da, tol), (db, tol)). The factors' gradients multiply the
    inner products as two bf16 numbers: 2^-16 of a value is dropped."""
    N, M, K, r = x.shape[0], w.shape[0], x.shape[1], a.shape[0]
    u = scale * (dy @ b)
    u_sum = M * STEP32 * abs(scale) * (dy.abs() @ b.abs())
    u_err = U16 * u.abs() + u_sum
    low = scale * (x @ a.T)
    low_sum = K * STEP32 * abs(scale) * (x.abs() @ a.abs().T)
    dx = dy @ w + u @ a
    tx = (u_err + (r + 1) * STEP32 * u.abs()) @ a.abs() \
        + (M + r + 2) * STEP32 * (dy.abs() @ w.abs())
    two = U16 * U16 + 2 * N * STEP32  # the remainder's rounding; two sums' steps
    da, ta = u.T @ x, (u_sum + two * u.abs()).T @ x.abs()
    db, tb = dy.T @ low, dy.abs().T @ (low_sum + two * low.abs())
    return tuple((v, U16 * (v.abs() + t) + t) for v, t in ((dx, tx), (da, ta), (db, tb)))
