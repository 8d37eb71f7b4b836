"""Tensor-level calls into the C ABI (PyTorch supplies device memory and streams).

Layouts follow the reference op: (S, H, D) per sequence as in
crates/foundry-spike/src/lib.rs:134, or batched (B, S, H, D). Any strides are
accepted as long as the head dimension is contiguous and the other strides
are 16-byte multiples (the TMA rule); nothing is copied to make inputs
contiguous.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import (FA_DTYPE_BF16, FA_DTYPE_F32, check, fa_matrix_t, fa_rope_t,
                   fa_tensor_t)

ROPE_AXES = (32, 32, 32, 32)  # lib.rs:20
ROPE_THETA = 10000.0          # lib.rs:21


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return FA_DTYPE_BF16
    if t.dtype == torch.float32:
        return FA_DTYPE_F32
    raise TypeError(f"unsupported dtype {t.dtype}: the op computes in bf16 or f32")


def as_bshd(t: torch.Tensor) -> torch.Tensor:
    """(S,H,D) -> (1,S,H,D) view; (B,S,H,D) unchanged."""
    if t.dim() == 3:
        return t.unsqueeze(0)
    if t.dim() == 4:
        return t
    raise ValueError(f"expected (S,H,D) or (B,S,H,D), got shape {tuple(t.shape)}")


def desc(t: torch.Tensor) -> fa_tensor_t:
    t4 = as_bshd(t)
    if not t4.is_cuda:
        raise ValueError("tensor must live on a CUDA device")
    sb, ss, sh, sd = t4.stride()
    return fa_tensor_t(t4.data_ptr(), sb, ss, sh, sd)


def _stream_ptr(stream: Optional[torch.cuda.Stream]) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


@dataclass
class Rope:
    """Axial RoPE descriptor: per-token positions (S, n_axes) and theta.

    Mirrors rope_tables_dtype (lib.rs:77-105); the tables are never
    materialised, the kernels evaluate cos/sin from the positions.
    """
    pos: torch.Tensor              # (S, n_axes) float32 on the device
    axis_dim: int = 32
    theta: float = ROPE_THETA

    def c_struct(self) -> fa_rope_t:
        p = self.pos
        if p.dtype != torch.float32 or not p.is_contiguous() or p.dim() != 2:
            raise ValueError("rope positions must be a contiguous (S, n_axes) float32 tensor")
        return fa_rope_t(p.data_ptr(), p.shape[1], self.axis_dim, self.theta)


def _ref(x):
    return C.byref(x) if x is not None else None


def default_scale(d: int) -> float:
    return 1.0 / math.sqrt(d)  # lib.rs:138


def attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: Optional[float] = None,
             rope: Optional[Rope] = None, out: Optional[torch.Tensor] = None,
             lse: Optional[torch.Tensor] = None, stream=None, saved: Optional[dict] = None):
    """O and fp32 LSE (B, H, S) of softmax(Q K^T * scale) V.

    With `rope` and a `saved` dict, the forward's workspace (rotated q, k and
    their (cos, sin) table) is kept in it for attn_bwd(..., saved=...), which
    then skips the second rotation."""
    q4, k4, v4 = as_bshd(q), as_bshd(k), as_bshd(v)
    B, S, H, D = q4.shape
    if k4.shape != q4.shape or v4.shape != q4.shape:
        raise ValueError("q, k, v must share one shape")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("q, k, v must share one dtype")
    dt = _dtype_code(q)
    if out is None:
        out = torch.empty_like(q)
    if lse is None:
        lse = torch.empty((B, H, S), device=q.device, dtype=torch.float32)
    scale = default_scale(D) if scale is None else float(scale)
    lib = _lib.load()
    rc_rope = rope.c_struct() if rope is not None else None
    ws_bytes = lib.fa_fwd_workspace_bytes(dt, B, S, H, D, _ref(rc_rope))
    ws = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8) if ws_bytes else None
    if saved is not None:
        saved.clear()
        if ws is not None:
            saved.update(ws=ws, shape=(B, S, H, D), dtype=q.dtype)
    dq_, dk_, dv_, do_ = desc(q4), desc(k4), desc(v4), desc(as_bshd(out))
    check(lib.fa_fwd(dt, B, S, H, D, C.byref(dq_), C.byref(dk_), C.byref(dv_), C.byref(do_),
                     lse.data_ptr(), scale, _ref(rc_rope), ws.data_ptr() if ws is not None else None,
                     ws_bytes, _stream_ptr(stream)), "fa_fwd")
    return out, lse


def attn_bwd(q, k, v, o, d_o, lse, *, scale: Optional[float] = None, rope: Optional[Rope] = None,
             deterministic: bool = False, dq=None, dk=None, dv=None, stream=None,
             saved: Optional[dict] = None):
    """dQ, dK, dV of the op (w.r.t. pre-rotation q/k when rope is given).

    `saved`: the dict a matching attn_fwd(..., saved=...) filled; the bf16
    path then reuses the forward's rotated q, k (fa_bwd_saved)."""
    q4 = as_bshd(q)
    B, S, H, D = q4.shape
    dt = _dtype_code(q)
    dq = torch.empty_like(q) if dq is None else dq
    dk = torch.empty_like(k) if dk is None else dk
    dv = torch.empty_like(v) if dv is None else dv
    scale = default_scale(D) if scale is None else float(scale)
    lib = _lib.load()
    rc_rope = rope.c_struct() if rope is not None else None
    if (saved and rope is not None and dt == FA_DTYPE_BF16 and not deterministic
            and saved.get("shape") == (B, S, H, D) and saved.get("dtype") == q.dtype):
        fws = saved["ws"]
        ws_bytes = lib.fa_bwd_saved_workspace_bytes(dt, B, S, H, D)
        ws = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8)
        ds = [desc(x) for x in (v, o, d_o, dq, dk, dv)]
        check(lib.fa_bwd_saved(dt, B, S, H, D, fws.data_ptr(), fws.numel(),
                               *[C.byref(x) for x in ds[:3]], lse.data_ptr(),
                               *[C.byref(x) for x in ds[3:]], scale, C.byref(rc_rope),
                               ws.data_ptr(), ws_bytes, _stream_ptr(stream)), "fa_bwd_saved")
        return dq, dk, dv
    ws_bytes = lib.fa_bwd_workspace_bytes(dt, B, S, H, D, _ref(rc_rope), int(deterministic))
    ws = torch.empty(max(ws_bytes, 1), device=q.device, dtype=torch.uint8)
    ds = [desc(x) for x in (q, k, v, o, d_o, dq, dk, dv)]
    check(lib.fa_bwd(dt, B, S, H, D, *[C.byref(x) for x in ds[:5]], lse.data_ptr(),
                     *[C.byref(x) for x in ds[5:]], scale, _ref(rc_rope), int(deterministic),
                     ws.data_ptr(), ws_bytes, _stream_ptr(stream)), "fa_bwd")
    return dq, dk, dv


def rope_apply(x: torch.Tensor, rope: Rope, *, inverse: bool = False, out=None, stream=None):
    """The reference's apply_rope (lib.rs:122-129) on the device."""
    x4 = as_bshd(x)
    B, S, H, D = x4.shape
    out = torch.empty_like(x) if out is None else out
    r = rope.c_struct()
    dx, dy = desc(x), desc(out)
    check(_lib.load().fa_rope_apply(_dtype_code(x), B, S, H, D, C.byref(dx), C.byref(dy),
                                    C.byref(r), int(inverse), _stream_ptr(stream)),
          "fa_rope_apply")
    return out


NORM_EPS = 1e-6  # lib.rs:26


def qk_norm_rope(x_txt: Optional[torch.Tensor], x_img: Optional[torch.Tensor],
                 w_txt: Optional[torch.Tensor], w_img: Optional[torch.Tensor],
                 rope: Optional[Rope], *, eps: float = NORM_EPS,
                 out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """The joint block's fused q/k prologue (fa_qk_norm_rope_fwd): per stream
    rms_norm with its weight (lib.rs:45-58), apply_rope with the joint
    positions (lib.rs:122-129), written text-then-image into one
    (B, T+I, H, 128) tensor (the cat of lib.rs:363-365). Either stream may
    be None; bf16."""
    xs = [x for x in (x_txt, x_img) if x is not None]
    if not xs:
        raise ValueError("at least one stream is required")
    t4 = as_bshd(x_txt) if x_txt is not None else None
    i4 = as_bshd(x_img) if x_img is not None else None
    B, _, H, D = as_bshd(xs[0]).shape
    T = t4.shape[1] if t4 is not None else 0
    I = i4.shape[1] if i4 is not None else 0
    if out is None:
        out = torch.empty((B, T + I, H, D), device=xs[0].device, dtype=xs[0].dtype)
    r = rope.c_struct() if rope is not None else None
    dt_ = desc(t4) if t4 is not None else None
    di_ = desc(i4) if i4 is not None else None
    do_ = desc(out)
    check(_lib.load().fa_qk_norm_rope_fwd(
        _dtype_code(xs[0]), B, T, I, H, D, _ref(dt_), _ref(di_),
        w_txt.data_ptr() if w_txt is not None else None,
        w_img.data_ptr() if w_img is not None else None, float(eps), _ref(r), C.byref(do_),
        _stream_ptr(stream)), "fa_qk_norm_rope_fwd")
    return out


def qk_norm_rope_bwd(x_txt, x_img, w_txt, w_img, rope: Optional[Rope], dy: torch.Tensor, *,
                     eps: float = NORM_EPS, dw_txt: Optional[torch.Tensor] = None,
                     dw_img: Optional[torch.Tensor] = None, stream=None):
    """Gradients of qk_norm_rope: (dx_txt, dx_img, dw_txt, dw_img). The weight
    gradients are fp32 and ADDED to dw_* when given (zeros otherwise)."""
    t4 = as_bshd(x_txt) if x_txt is not None else None
    i4 = as_bshd(x_img) if x_img is not None else None
    d4 = as_bshd(dy)
    B, S, H, D = d4.shape
    T = t4.shape[1] if t4 is not None else 0
    I = i4.shape[1] if i4 is not None else 0
    dev = dy.device
    dx_t = torch.empty_like(x_txt) if x_txt is not None else None
    dx_i = torch.empty_like(x_img) if x_img is not None else None
    if x_txt is not None and dw_txt is None:
        dw_txt = torch.zeros(D, device=dev, dtype=torch.float32)
    if x_img is not None and dw_img is None:
        dw_img = torch.zeros(D, device=dev, dtype=torch.float32)
    r = rope.c_struct() if rope is not None else None
    ds = [desc(x) if x is not None else None for x in (t4, i4, d4, dx_t, dx_i)]
    check(_lib.load().fa_qk_norm_rope_bwd(
        _dtype_code(dy), B, T, I, H, D, _ref(ds[0]), _ref(ds[1]),
        w_txt.data_ptr() if w_txt is not None else None,
        w_img.data_ptr() if w_img is not None else None, float(eps), _ref(r), C.byref(ds[2]),
        _ref(ds[3]), _ref(ds[4]), dw_txt.data_ptr() if dw_txt is not None else None,
        dw_img.data_ptr() if dw_img is not None else None, _stream_ptr(stream)),
        "fa_qk_norm_rope_bwd")
    return dx_t, dx_i, dw_txt, dw_img


# --------------------------------------------------------- block operators

def _launch(fn, where: str, t: torch.Tensor, stream, temps, *args) -> None:
    """fn(*args, stream) with t's device current, on `stream` or the current
    stream of that device. `temps` are the call's own buffers: on a stream of
    the caller's they are kept until it has passed them."""
    dev = t.get_device()
    if stream is None:
        ptr = torch._C._cuda_getCurrentRawStream(dev)
    else:
        ptr = stream.cuda_stream
        for b in temps:
            if b is not None:
                b.record_stream(stream)
    if dev == torch._C._cuda_getDevice():
        rc = fn(*args, ptr)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, ptr)
    if rc:
        check(rc, where)


def _same_device(ref: torch.Tensor, **tensors) -> None:
    dev = ref.get_device()
    if dev < 0:
        raise ValueError("tensor must live on a CUDA device")
    for name, t in tensors.items():
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{name} is on {t.device}, the first operand on {ref.device}")


def _norm_desc(t: torch.Tensor) -> fa_tensor_t:
    """(rows, D) or (groups, rows, D) as the C ABI's (groups, rows, 1, D)."""
    st = t.stride()
    sd = st[-1] if t.shape[-1] > 1 else 1
    return fa_tensor_t(t.data_ptr(), st[0] if len(st) == 3 else 0, st[-2], 0, sd)


def _norm_params(x: torch.Tensor, weight, bias):
    """Checked (weight, bias, dtype code, stride between groups)."""
    first = weight if weight is not None else bias
    if first is None:
        return None, None, FA_DTYPE_F32, 0
    want = x.shape[-1:] if first.dim() == 1 else (x.shape[0] if x.dim() == 3 else -1, x.shape[-1])
    if first.shape != want or (weight is not None and bias is not None
                               and (bias.shape != want or bias.dtype != first.dtype)):
        raise ValueError("weight and bias must be (D,), or (groups, D) with x (groups, rows, D), "
                         f"and of one dtype: got {[tuple(p.shape) for p in (weight, bias) if p is not None]}"
                         f" for x {tuple(x.shape)}")
    code = _dtype_code(first)
    if first.dim() == 1:
        return (weight.contiguous() if weight is not None else None,
                bias.contiguous() if bias is not None else None, code, 0)
    # two modulation chunks share the stride of their rows; others are copied (D values each)
    ps, unit = first.stride()
    if (ps <= 0 or unit != 1 or x.shape[0] == 1
            or (weight is not None and bias is not None and bias.stride() != (ps, 1))):
        weight, bias = (p.contiguous() if p is not None else None for p in (weight, bias))
        ps = x.shape[-1]
    return weight, bias, code, ps


def _ptr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None else None


def _check_norm_x(x: torch.Tensor) -> Tuple[int, int, int]:
    s = x.shape
    if len(s) == 3:
        return s
    if len(s) != 2:
        raise ValueError(f"expected (rows, D) or (groups, rows, D), got {tuple(s)}")
    return 1, s[0], s[1]


def _check_like(x: torch.Tensor, name: str, t: torch.Tensor) -> None:
    if t.shape != x.shape or t.dtype != x.dtype:
        raise ValueError(f"{name} must have x's shape and dtype")


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, *, unit_offset: bool = False,
               eps: float = NORM_EPS, out: Optional[torch.Tensor] = None, stream=None):
    """Layer norm over the last dimension of x (rows, D) or (groups, rows, D),
    bf16 or f32: y = h * weight + bias, h = (x - mean) / sqrt(var + eps); with
    unit_offset the gain is 1 + weight (the modulation of layer_norm_mod,
    lib.rs:60-71). weight and bias: (D,), or (groups, D) for one pair per
    group; None: no gain or no bias. Returns (y, stats), stats the fp32
    (2, groups * rows) means and reciprocal deviations layer_norm_bwd reads."""
    G, R, D = _check_norm_x(x)
    _same_device(x, weight=weight, bias=bias, out=out)
    dt = _dtype_code(x)
    w, b, pdt, ps = _norm_params(x, weight, bias)
    y = torch.empty_like(x) if out is None else out
    if out is not None:
        _check_like(x, "out", out)
    stats = x.new_empty((2, G * R), dtype=torch.float32)
    _launch(_lib.load().fa_layer_norm_fwd, "fa_layer_norm_fwd", x, stream, (w, b), dt, G, R, D,
            C.byref(_norm_desc(x)), _ptr(w), _ptr(b), pdt, ps, int(unit_offset), float(eps),
            C.byref(_norm_desc(y)), stats.data_ptr())
    return y, stats


def layer_norm_bwd(x: torch.Tensor, weight: Optional[torch.Tensor], dy: torch.Tensor,
                   stats: torch.Tensor, *, unit_offset: bool = False, params: bool = True,
                   stream=None):
    """Gradients of layer_norm: (dx, dweight, dbias), the last two fp32 with
    weight's shape (of a (D,) pair when weight is None), or None with
    params=False. Identical bits across repeats."""
    G, R, D = _check_norm_x(x)
    _check_like(x, "dy", dy)
    _same_device(x, weight=weight, dy=dy, stats=stats)
    if (stats.dtype != torch.float32 or tuple(stats.shape) != (2, G * R)
            or not stats.is_contiguous()):
        raise ValueError("stats must be layer_norm's (2, rows) float32 tensor")
    dt = _dtype_code(x)
    w, _, pdt, ps = _norm_params(x, weight, None)
    dx = torch.empty_like(x)
    lead = () if ps == 0 else (G,)
    dw = torch.empty(lead + (D,), device=x.device, dtype=torch.float32) if params else None
    db = torch.empty_like(dw) if params else None
    lib = _lib.load()
    nb = lib.fa_layer_norm_bwd_workspace_bytes(G, R, D)
    ws = torch.empty(nb, device=x.device, dtype=torch.uint8) if nb else None
    _launch(lib.fa_layer_norm_bwd, "fa_layer_norm_bwd", x, stream, (w, ws), dt, G, R, D,
            C.byref(_norm_desc(x)), _ptr(w), pdt, ps, int(unit_offset), C.byref(_norm_desc(dy)),
            stats.data_ptr(), C.byref(_norm_desc(dx)), _ptr(dw), _ptr(db), _ptr(ws), nb)
    return dx, dw, db


def _matrix(t: torch.Tensor, name: str) -> fa_matrix_t:
    """A 2-D or (batch, rows, cols) tensor for the C ABI."""
    s, st = t.shape, t.stride()
    if s[-1] > 1 and st[-1] != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    # a stride that no element uses may be anything: give it a legal one
    sr = st[-2] if s[-2] > 1 else -(-s[-1] // 8) * 8
    sb = 0
    if len(s) == 3:
        sb = st[0] if s[0] > 1 else s[1] * sr
    return fa_matrix_t(t.data_ptr(), sb, sr)


def _rows2d(t: torch.Tensor, name: str) -> torch.Tensor:
    """(..., K) as one (rows, K) matrix, without a copy."""
    if t.dim() == 2:
        return t
    if t.dim() < 2:
        raise ValueError(f"{name}: expected (..., features), got {tuple(t.shape)}")
    try:
        return t.view(-1, t.shape[-1]) if t.numel() else t.reshape(0, t.shape[-1])
    except RuntimeError:
        raise ValueError(f"{name}: the leading dimensions must be one strided set of rows; "
                         "reshape it first") from None


def _aligned_rows(rows: int, cols: int, like: torch.Tensor) -> torch.Tensor:
    """An uninitialised (rows, cols) bf16 matrix whose rows start on 16 bytes."""
    ld = -(-cols // 8) * 8
    t = torch.empty((rows, ld), device=like.device, dtype=torch.bfloat16)
    return t if ld == cols else t[:, :cols]


def _pad_rank(a: torch.Tensor, b: torch.Tensor):
    """The factors with the rank a multiple of 8 (zero rows of a, columns of b)."""
    p = -a.shape[-2] % 8
    if p:
        a, b = torch.nn.functional.pad(a, (0, 0, 0, p)), torch.nn.functional.pad(b, (0, p))
    return a, b


def _check_lora(x2, w, a, b, bias, stacked: bool) -> None:
    for name, t in (("x", x2), ("w", w), ("a", a), ("b", b), ("bias", bias)):
        if t is not None and t.dtype != torch.bfloat16:
            raise TypeError(f"{name}: the linear with adapters computes in bf16, got {t.dtype}")
    _same_device(x2, w=w, a=a, b=b, bias=bias)
    nd = 3 if stacked else 2
    if w.dim() != 2 or a.dim() != nd or b.dim() != nd:
        raise ValueError("expected w (out, in) and factors a (..., rank, in), b (..., out, rank)")
    K, M = w.shape[1], w.shape[0]
    if x2.shape[1] != K or a.shape[-1] != K or b.shape[-2] != M or a.shape[-2] != b.shape[-1]:
        raise ValueError(f"shapes do not fit: x (..., {x2.shape[1]}), w {tuple(w.shape)}, "
                         f"a {tuple(a.shape)}, b {tuple(b.shape)}")
    if stacked and a.shape[0] != b.shape[0]:
        raise ValueError("a and b must hold as many adapters")
    if bias is not None and (tuple(bias.shape) != (M,) or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous (out,) vector")


def _low_dim(rank: int) -> int:
    return -(-rank // 16) * 16


def lora_linear(x: torch.Tensor, w: torch.Tensor, a: torch.Tensor, b: torch.Tensor, *,
                scale: float = 1.0, bias: Optional[torch.Tensor] = None, stream=None):
    """y = x w^T + bias + scale (x a^T) b^T in one product (the reference's
    linear with LoRA factors, lib.rs:270-287): x (..., in), w (out, in),
    a (rank, in), b (out, rank), bf16, fp32 sums. Rows of x, w and a must
    start on 16 bytes; a rank that is no multiple of 8 costs a padded copy of
    the factors, rank <= 256. Returns (y, low), low = scale x a^T as
    lora_linear_bwd reads it."""
    x2 = _rows2d(x, "x")
    _check_lora(x2, w, a, b, bias, False)
    a, b = _pad_rank(a, b)
    N, K, M, r = x2.shape[0], w.shape[1], w.shape[0], a.shape[0]
    y = _aligned_rows(N, M, x)
    low = torch.empty((N, _low_dim(r)), device=x.device, dtype=torch.bfloat16)
    ms = [_matrix(t, n) for t, n in ((x2, "x"), (w, "w"), (a, "a"), (b, "b"), (y, "y"))]
    _launch(_lib.load().fa_lora_linear_fwd, "fa_lora_linear_fwd", x, stream, (a, b), FA_DTYPE_BF16,
            N, K, M, r, *[C.byref(m) for m in ms[:4]], float(scale), _ptr(bias), C.byref(ms[4]),
            low.data_ptr())
    return y.view(*x.shape[:-1], M) if x.dim() != 2 else y, low


def lora_linear_bwd(x: torch.Tensor, w: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                    dy: torch.Tensor, low: torch.Tensor, *, scale: float = 1.0,
                    need_dx: bool = True, need_factors: bool = True, stream=None):
    """Gradients of lora_linear with w frozen: (dx, da, db) in bf16, each None
    when not needed. `low` is what the forward returned for the same x, a and
    scale. Identical bits across repeats. (The bias's gradient, where it
    trains, is dy summed over its rows.)"""
    x2, dy2 = _rows2d(x, "x"), _rows2d(dy, "dy")
    _check_lora(x2, w, a, b, None, False)
    _same_device(x, dy=dy, low=low)
    if dy2.dtype != torch.bfloat16 or tuple(dy2.shape) != (x2.shape[0], w.shape[0]):
        raise ValueError(f"dy must be bf16 (..., {w.shape[0]}) with x's rows")
    rank = a.shape[0]
    a, b = _pad_rank(a, b)
    N, K, M, r = x2.shape[0], w.shape[1], w.shape[0], a.shape[0]
    if (low.dtype != torch.bfloat16 or tuple(low.shape) != (N, _low_dim(r))
            or not low.is_contiguous()):
        raise ValueError("low must be the tensor lora_linear returned for these rows")
    dx = _aligned_rows(N, K, x) if need_dx else None
    da = torch.empty((r, K), device=x.device, dtype=torch.bfloat16) if need_factors else None
    db = torch.empty((M, r), device=x.device, dtype=torch.bfloat16) if need_factors else None
    lib = _lib.load()
    nb = lib.fa_lora_linear_bwd_workspace_bytes(N, r)
    ws = torch.empty(nb, device=x.device, dtype=torch.uint8) if nb else None
    ms = [_matrix(t, n) for t, n in ((x2, "x"), (w, "w"), (a, "a"), (b, "b"), (dy2, "dy"))]
    mdx = _matrix(dx, "dx") if need_dx else None
    _launch(lib.fa_lora_linear_bwd, "fa_lora_linear_bwd", x, stream, (a, b, ws), FA_DTYPE_BF16, N, K,
            M, r, *[C.byref(m) for m in ms[:4]], float(scale), low.data_ptr(), C.byref(ms[4]),
            _ref(mdx), _ptr(da), _ptr(db), _ptr(ws), nb)
    if need_dx and x.dim() != 2:
        dx = dx.view(*x.shape)
    if need_factors and r != rank:
        da, db = da[:rank], db[:, :rank]
    return dx, da, db


def lora_linear_many(x: torch.Tensor, w: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                     ids: torch.Tensor, scales: torch.Tensor, *,
                     bias: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """lora_linear for rows of many requests at once: a (E, rank, in),
    b (E, out, rank), scales (E,) fp32, ids (rows,) int32 on the device; row i
    uses adapter ids[i], and an id outside [0, E) means w alone. From one
    token to packed prompts; ids in any order. Returns y."""
    x2 = _rows2d(x, "x")
    _check_lora(x2, w, a, b, bias, True)
    _same_device(x, ids=ids, scales=scales)
    if ids.dtype != torch.int32 or tuple(ids.shape) != (x2.shape[0],) or not ids.is_contiguous():
        raise ValueError(f"ids must be a contiguous int32 ({x2.shape[0]},) tensor")
    if (scales.dtype != torch.float32 or tuple(scales.shape) != (a.shape[0],)
            or not scales.is_contiguous()):
        raise ValueError(f"scales must be a contiguous float32 ({a.shape[0]},) tensor")
    a, b = _pad_rank(a, b)
    E, r = a.shape[0], a.shape[1]
    N, K, M = x2.shape[0], w.shape[1], w.shape[0]
    y = _aligned_rows(N, M, x)
    lib = _lib.load()
    nb = lib.fa_lora_linear_many_workspace_bytes(N, r)
    ws = torch.empty(nb, device=x.device, dtype=torch.uint8) if nb else None
    ms = [_matrix(t, n) for t, n in ((x2, "x"), (w, "w"), (a, "a"), (b, "b"), (y, "y"))]
    _launch(lib.fa_lora_linear_many, "fa_lora_linear_many", x, stream, (a, b, ws), FA_DTYPE_BF16, N,
            K, M, r, E, *[C.byref(m) for m in ms[:4]], ids.data_ptr(), scales.data_ptr(),
            _ptr(bias), C.byref(ms[4]), _ptr(ws), nb)
    return y.view(*x.shape[:-1], M) if x.dim() != 2 else y


NS_COEFFS = (3.4445, -4.7750, 2.0315)  # five steps take [0.005, 1] to about [0.7, 1.2]


def orthogonalize(g: torch.Tensor, *, steps: int = 5, coeffs=NS_COEFFS, eps: float = 1e-7,
                  out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of the matrices g (..., m, n), bf16 or
    f32: X = g / (|g|_F + eps), then `steps` times X = a X + (b Q + c Q^2) X
    with Q = X X^T (of the transpose when m > n). Returns bf16, (..., m, n):
    a step's direction, whose singular values the iteration itself leaves
    spread by some 20 percent. Identical bits across repeats."""
    if g.dim() < 2:
        raise ValueError(f"expected (..., m, n), got {tuple(g.shape)}")
    _same_device(g, out=out)
    dt = _dtype_code(g)
    m, n = g.shape[-2:]
    try:
        g3 = g.view(-1, m, n) if g.numel() else g.reshape(-1, m, n)
    except RuntimeError:
        raise ValueError("the leading dimensions must be one strided set of matrices; "
                         "reshape g first") from None
    if n > 1 and g3.stride(-1) != 1:
        raise ValueError("g's last dimension must be contiguous")
    B = g3.shape[0]
    if out is None:
        o3 = _aligned_rows(B * m, n, g).unflatten(0, (B, m))
    else:
        if out.shape != g.shape or out.dtype != torch.bfloat16:
            raise ValueError("out must be bf16 with g's shape")
        o3 = out.view(-1, m, n)
        if n > 1 and o3.stride(-1) != 1:
            raise ValueError("out's last dimension must be contiguous")
    mo = _matrix(o3, "out")
    a, b, c = (float(v) for v in coeffs)
    lib = _lib.load()
    nb = lib.fa_orthogonalize_workspace_bytes(B, m, n, int(steps))
    ws = torch.empty(nb, device=g.device, dtype=torch.uint8) if nb else None
    _launch(lib.fa_orthogonalize, "fa_orthogonalize", g, stream, (ws,), dt, B, m, n, g3.data_ptr(),
            g3.stride(0), g3.stride(1), mo.data, mo.stride_batch, mo.stride_row, int(steps), a, b,
            c, float(eps), _ptr(ws), nb)
    return o3.view(g.shape) if out is None else out


def device_status() -> int:
    """Reads and clears the device status word (0 when no bounded wait expired)."""
    return int(_lib.load().fa_device_status())
