"""The block operators on the GPU against their plain 64-bit forms
(tests/block_ops_support.py holds the bounds): the (modulated) layer norm and
its gradients, the linear with adapters and its gradients, and the same for
rows of many requests."""
import pytest
import torch

from tests import block_ops_support as sup

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rn(g, *shape, std=1.0, dtype=BF):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


# -------------------------------------------------------------- layer norm

def _norm_tols(x, w, dy, h, rstd, off, dtype):
    """Bounds of y, dx, dw, db: the output rounding plus the fp32 arithmetic.
    A row's sums are trees whose longest chain is a thread's share (at most
    64 values) and 10 joins: n = 80 steps; they enter relative to the largest
    magnitude in the row."""
    u = sup.U16 if dtype == BF else 2.0 ** -24
    n = 80 * sup.STEP32
    big = (x.double().abs().amax(-1, keepdim=True) * rstd + 1)  # |x - mean| / sd and mean / sd
    gain = (off + w).abs() if torch.is_tensor(w) else abs(off + w)
    ty = n * big * gain
    t = dy.double().abs() * gain
    tx = n * rstd * big * big * (t + t.amax(-1, keepdim=True))
    return u, ty, tx, n * big


NORM_CASES = [
    # groups, rows, dim, dtype, per-group parameters, unit offset
    (1, 1, 1, F32, False, False),
    (1, 1, 2048, BF, True, True),
    (1, 5, 7, BF, False, False),
    (3, 17, 64, BF, True, True),
    (2, 300, 256, F32, True, True),
    (1, 1000, 1001, F32, False, False),
    (2, 33, 1001, BF, True, True),
    (1, 777, 2056, BF, False, False),
    (4, 129, 4096, BF, True, True),
    (1, 40, 8192, F32, False, False),
    (2, 9, 16384, BF, True, False),
    (1, 3, 16381, F32, False, False),
    (300, 1, 128, BF, True, True),
    (1, 1300, 520, BF, True, True),
    (2, 700, 2048, BF, True, True),
    (1, 1203, 2568, F32, False, False),
    (3, 411, 4104, BF, False, True),
    (1, 1201, 8200, BF, True, True),
    (1, 5, 16384, F32, False, False),
    (1, 1200, 300, F32, True, True),
    # even widths that no 16-byte access divides, in each of their forms
    (2, 600, 26, BF, False, False),
    (1, 700, 250, F32, True, True),
    (1, 1300, 514, BF, False, False),
    (7, 5, 5798, BF, False, True),
    (2, 9, 4098, F32, True, False),
    (2, 20, 8190, BF, True, True),
    (1, 7, 16382, F32, False, False),
]


@pytest.mark.parametrize("G,R,D,dtype,per,unit", NORM_CASES)
def test_layer_norm_and_gradients(G, R, D, dtype, per, unit):
    from foundry_trainer_b200 import ops
    g = _gen(G * 1000 + D)
    x = _rn(g, G, R, D) * 2 + 0.5
    x, dy = x.to(dtype), _rn(g, G, R, D, dtype=dtype)
    w, b = (_rn(g, *((G, D) if per else (D,)), std=0.3, dtype=dtype) for _ in range(2))
    off = 1.0 if unit else 0.0
    y, stats = ops.layer_norm(x, w, b, unit_offset=unit)
    dx, dw, db = ops.layer_norm_bwd(x, w, dy, stats, unit_offset=unit)
    again = ops.layer_norm_bwd(x, w, dy, stats, unit_offset=unit)
    wd, bd = (p.double()[:, None] if per else p.double() for p in (w, b))
    ry, h, rstd, mean = sup.norm_ref(x, wd, bd, 1e-6, off)
    rdx, rdw, rdb = sup.norm_bwd_ref(x, wd, dy, 1e-6, off, not per)
    u, ty, tx, th = _norm_tols(x, wd, dy, h, rstd, off, dtype)
    sup.within(y, ry, u * ry.abs() + ty + sup.STEP32 * bd.abs(), "y")
    sup.within(dx, rdx, u * rdx.abs() + tx, "dx")
    dims = (1,) if per else (0, 1)
    sup.within(dw, rdw, (dy.double().abs() * (th + R * G * sup.STEP32 * h.abs())).sum(dims), "dw")
    sup.within(db, rdb, R * G * sup.STEP32 * dy.double().abs().sum(dims), "db")
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


def test_layer_norm_strides_and_missing_parameters():
    from foundry_trainer_b200 import ops
    g = _gen(3)
    # a stream's slice of a joint tensor, modulation chunks of one linear
    joint, mod = _rn(g, 2, 50, 320), _rn(g, 2, 6 * 320, std=0.2)
    x = joint[:, 13:]
    shift, scale = mod.split(320, dim=-1)[:2]
    y, stats = ops.layer_norm(x, scale, shift, unit_offset=True)
    ref, _ = ops.layer_norm(x.contiguous(), scale.contiguous(), shift.contiguous(),
                            unit_offset=True)
    assert torch.equal(y, ref)
    # rows that start off a 16-byte boundary take the element-wise path
    odd = _rn(g, 40, 321)[:, 1:]
    y1, _ = ops.layer_norm(odd)
    y2, _ = ops.layer_norm(odd.contiguous())
    assert torch.equal(y1, y2) or (y1.float() - y2.float()).abs().max() <= 2 ** -7 * 4
    dy = _rn(g, 2, 37, 320)
    dx, dw, db = ops.layer_norm_bwd(x, None, dy, stats)
    rdx, rdw, rdb = sup.norm_bwd_ref(x, torch.ones(320, device="cuda").double(), dy, 1e-6, 0.0,
                                     True)
    assert dw.shape == (320,)
    sup.within(dx, rdx, sup.U16 * rdx.abs() + 1e-4, "dx")
    sup.within(db, rdb, 74 * sup.STEP32 * dy.double().abs().sum((0, 1)), "db")
    only, none1, none2 = ops.layer_norm_bwd(x, None, dy, stats, params=False)
    assert torch.equal(only, dx) and none1 is None and none2 is None


def test_layer_norm_empty_constant_and_non_finite_rows():
    from foundry_trainer_b200 import ops
    w = torch.ones(64, device="cuda")
    y, stats = ops.layer_norm(torch.empty(0, 64, device="cuda"), w, w)
    assert y.shape == (0, 64) and stats.shape == (2, 0)
    dx, dw, db = ops.layer_norm_bwd(y, w, y, stats)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()
    x = torch.randn(4, 64, device="cuda")
    x[1] = 3.0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    y, _ = ops.layer_norm(x, w, None)
    assert torch.equal(y[1], torch.zeros(64, device="cuda"))  # no variance: h = 0
    assert torch.isfinite(y[:2]).all() and torch.isnan(y[2]).all() and torch.isnan(y[3]).all()


# ---------------------------------------------------------- adapter linears

LORA_CASES = [
    # rows, in, out, rank, bias
    (1, 8, 8, 8, False),
    (1, 4096, 512, 16, True),
    (7, 264, 1000, 4, True),
    (64, 512, 136, 16, False),
    (65, 512, 384, 24, True),
    (200, 1544, 72, 64, False),
    (256, 320, 640, 128, True),
    (257, 320, 640, 16, True),
    (300, 200, 2056, 12, False),
    (777, 1544, 1032, 40, True),
    (1025, 64, 128, 256, False),
    (2304, 640, 1280, 16, False),
    (5000, 2048, 2560, 72, True),
]


def _lora_inputs(g, N, K, M, r, bias, E=None):
    lead = () if E is None else (E,)
    return (_rn(g, N, K), _rn(g, M, K, std=K ** -0.5), _rn(g, *lead, r, K, std=K ** -0.5),
            _rn(g, *lead, M, r, std=0.5), _rn(g, M) if bias else None)


@pytest.mark.parametrize("N,K,M,r,bias", LORA_CASES)
def test_lora_linear_and_gradients(N, K, M, r, bias):
    from foundry_trainer_b200 import ops
    g = _gen(N + K)
    x, w, a, b, bi = _lora_inputs(g, N, K, M, r, bias)
    dy, s = _rn(g, N, M), 1.5
    y, low = ops.lora_linear(x, w, a, b, scale=s, bias=bi)
    got = ops.lora_linear_bwd(x, w, a, b, dy, low, scale=s)
    again = ops.lora_linear_bwd(x, w, a, b, dy, low, scale=s)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    d = [t.double() if t is not None else None for t in (x, w, a, b, bi, dy)]
    ry, ty, _, _ = sup.lora_ref(d[0], d[1], d[2], d[3], s, d[4])
    sup.within(y, ry, ty, "y")
    for name, v, (ref, tol) in zip(("dx", "da", "db"), got,
                                   sup.lora_bwd_ref(d[0], d[1], d[2], d[3], d[5], s)):
        sup.within(v, ref, tol, name)
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    dx, da, db = ops.lora_linear_bwd(x, w, a, b, dy, low, scale=s, need_dx=False)
    assert dx is None and torch.equal(da, got[1]) and torch.equal(db, got[2])
    dx, da, db = ops.lora_linear_bwd(x, w, a, b, dy, low, scale=s, need_factors=False)
    assert torch.equal(dx, got[0]) and da is None and db is None


@pytest.mark.parametrize("N", [40, 600])
def test_lora_linear_strided_rows_and_no_rows(N):
    from foundry_trainer_b200 import ops
    g = _gen(N)
    x, w, a, b, _ = _lora_inputs(g, N, 256, 512, 16, False)
    y, low = ops.lora_linear(x, w, a, b)
    wide = _rn(g, N, 256 + 72)
    wide[:, 40:296] = x
    y2, low2 = ops.lora_linear(wide[:, 40:296].unflatten(0, (2, N // 2)), w, a, b)
    assert y2.shape == (2, N // 2, 512)
    assert torch.equal(y2.flatten(0, 1), y) and torch.equal(low2, low)
    e = x[:0]
    y0, low0 = ops.lora_linear(e, w, a, b)
    dx, da, db = ops.lora_linear_bwd(e, w, a, b, y0, low0)
    assert y0.shape == (0, 512) and dx.shape == (0, 256) and not da.any() and not db.any()


MANY_CASES = [
    # rows, in, out, rank, adapters, ids
    (1, 2048, 512, 16, 4, "one"),
    (3, 264, 136, 8, 1, "random"),
    (64, 1024, 640, 16, 48, "random"),
    (64, 512, 256, 64, 3, "none"),
    (65, 512, 256, 12, 70, "random"),
    (256, 320, 640, 32, 300, "random"),
    (257, 320, 640, 32, 5, "runs"),
    (700, 640, 520, 16, 300, "random"),
    (1500, 512, 768, 128, 9, "runs"),
    (2049, 256, 512, 8, 2, "runs"),
    (600, 256, 256, 16, 4, "none"),
    # more turns of the ring than its slots before the adapters' blocks, more
    # adapters' blocks than slots, several clusters an SM
    (1, 4096, 4096, 16, 4, "one"),
    (8, 4096, 4096, 16, 8, "random"),
    (40, 8192, 128, 64, 40, "random"),
    (64, 4096, 6144, 16, 48, "random"),
    (200, 2048, 3000, 96, 200, "random"),
    # operands built from an adapter's own rows only: pairs and columns, ranks
    # of one and of two K blocks, packed adapters beyond what a warp keeps
    (700, 408, 920, 64, 14, "random"),
    (301, 256, 520, 80, 5, "random"),
    (226, 408, 920, 64, 14, "random"),
    (256, 1024, 512, 32, 100, "random"),
    (250, 512, 384, 12, 37, "random"),
    (129, 264, 256, 16, 3, "runs"),
]


@pytest.mark.parametrize("N,K,M,r,E,kind", MANY_CASES)
def test_lora_linear_many_requests(N, K, M, r, E, kind):
    from foundry_trainer_b200 import ops
    g = _gen(N * 7 + E)
    x, w, a, b, bi = _lora_inputs(g, N, K, M, r, N % 2 == 1, E)
    scales = torch.rand(E, generator=g, device="cuda") + 0.5
    if kind == "one":
        ids = torch.full((N,), E - 1, device="cuda", dtype=torch.int32)
    elif kind == "none":
        ids = torch.tensor([-1, E, -7], device="cuda", dtype=torch.int32).repeat(N)[:N].contiguous()
    else:
        ids = torch.randint(-1, E, (N,), generator=g, device="cuda", dtype=torch.int32)
        if kind == "runs":
            ids = ids[torch.arange(N, device="cuda") // 190].contiguous()
    y = ops.lora_linear_many(x, w, a, b, ids, scales, bias=bi)
    y2 = ops.lora_linear_many(x, w, a, b, ids, scales, bias=bi)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    assert torch.equal(y, y2)
    dbl = lambda t: t.double() if t is not None else None
    for e in ids.unique().tolist():
        rows = ids == e
        if 0 <= e < E:
            ae, be, s = a[e], b[e], scales[e].item()
        else:
            ae, be, s = a[0] * 0, b[0] * 0, 1.0
        ref, tol, _, _ = sup.lora_ref(x[rows].double(), w.double(), ae.double(), be.double(), s,
                                      dbl(bi))
        sup.within(y[rows], ref, tol, f"adapter {e}")


def test_lora_rows_do_not_touch_other_adapters():
    # an unused adapter full of NaN, and NaN rows of another request, stay away
    from foundry_trainer_b200 import ops
    g = _gen(11)
    for N in (48, 200, 600):
        x, w, a, b, _ = _lora_inputs(g, N, 256, 512, 16, False, 3)
        scales = torch.ones(3, device="cuda")
        ids = (torch.arange(N, device="cuda") % 2).to(torch.int32)
        ref = ops.lora_linear_many(x, w, a, b, ids, scales)
        a2, b2 = a.clone(), b.clone()
        a2[2], b2[2] = float("nan"), float("inf")
        assert torch.equal(ops.lora_linear_many(x, w, a2, b2, ids, scales), ref)
        a2[1] = float("nan")
        got = ops.lora_linear_many(x, w, a2, b2, ids, scales)
        even = ids == 0
        want, tol, _, _ = sup.lora_ref(x[even].double(), w.double(), a[0].double(), b[0].double(),
                                       1.0, None)
        sup.within(got[even], want, tol, f"{N} rows beside a broken adapter")
        assert torch.isnan(got[~even]).all()
        # rows without an adapter beside a broken one
        ids[::2] = -1
        got = ops.lora_linear_many(x, w, a2, b2, ids, scales)
        want, tol, _, _ = sup.lora_ref(x[even].double(), w.double(), a[0].double() * 0,
                                       b[0].double() * 0, 1.0, None)
        sup.within(got[even], want, tol, f"{N} rows without an adapter")


@pytest.mark.parametrize("N", [1, 48, 200, 600])
def test_lora_rows_do_not_meet_broken_factors(N):
    # a request whose b is broken in some columns or everywhere, rows without
    # an adapter, and a row that is NaN itself
    from foundry_trainer_b200 import ops
    g = _gen(12)
    x, w, a, b, _ = _lora_inputs(g, N, 256, 512, 12, False, 3)
    scales = torch.ones(3, device="cuda")
    pattern = torch.tensor([0, -1, 1, 0, 2], device="cuda")
    for broken, kinds in (((1,), (0, -1, 2)), ((1, 2), (0, -1))):
        for cols in (slice(None), slice(70, 71)):
            b2 = b.clone()
            for e in broken:
                b2[e, cols] = float("inf")
                b2[e, cols, 0] = float("nan")
            ids = pattern[torch.arange(N, device="cuda") % 5].to(torch.int32)
            x2 = x.clone()
            if N > 10:
                x2[10] = float("nan")
            got = ops.lora_linear_many(x2, w, a, b2, ids, scales)
            for e in kinds:
                rows = ids == e
                if N > 10:
                    assert torch.isnan(got[10]).all()
                    rows[10] = False
                gain = 1.0 if e >= 0 else 0.0
                want, tol, _, _ = sup.lora_ref(x[rows].double(), w.double(), a[max(e, 0)].double(),
                                               b[max(e, 0)].double() * gain, 1.0, None)
                sup.within(got[rows], want, tol, f"{N} rows, adapter {e} beside {broken}")
            for e in broken:
                assert torch.isnan(got[ids == e][:, cols]).all()
    from foundry_trainer_b200 import _lib
    assert _lib.load().fa_device_status() == 0


@pytest.mark.parametrize("N", [40, 300])
def test_lora_linear_with_an_infinity(N):
    # one infinite input: its row of y follows the formula, db gets infinities of
    # its row's signs, not NaN. Its column of da is not finite; infinities there
    # may be NaN, as u = hi + lo is multiplied in two parts: inf hi + inf lo is
    # NaN where the remainder has the other sign.
    from foundry_trainer_b200 import ops
    g = _gen(13)
    x, w, a, b, _ = _lora_inputs(g, N, 128, 264, 12, False)
    dy = torch.randn(N, 264, generator=g, device="cuda").to(BF)
    x[7, 5] = float("inf")
    b[:20] = (w[:20, 5].sign()[:, None] * a[:, 5].sign()) * b[:20].abs()  # of the base's sign
    y, low = ops.lora_linear(x, w, a, b, scale=0.5)
    dx, da, db = ops.lora_linear_bwd(x, w, a, b, dy, low, scale=0.5)
    assert torch.equal(low[7, :12].float(), a[:, 5].float().sign() * float("inf"))
    assert not low[:, 12:16].any() and torch.isfinite(low[7, 16:]).all()
    assert torch.equal(db.float(), dy[7].float().sign()[:, None] * a[:, 5].float().sign()
                       * float("inf"))
    assert not torch.isfinite(da[:, 5]).any()
    assert torch.isfinite(da[:, :5]).all() and torch.isfinite(da[:, 6:]).all()
    assert torch.isfinite(dx).all()
    rest = torch.arange(N, device="cuda") != 7
    assert torch.isfinite(y[rest]).all() and not torch.isfinite(y[7]).any()
    # where base and adapter agree in sign for every rank, y is that infinity
    same = ((a[:, 5].sign() * b.sign()) == w[:, 5].sign()[:, None]).all(1)
    assert same.sum() >= 20
    assert torch.equal(y[7, same].float(), w[same, 5].float().sign() * float("inf"))


def test_lora_linear_without_rows():
    from foundry_trainer_b200 import ops
    g = _gen(14)
    x, w, a, b, _ = _lora_inputs(g, 4, 64, 48, 16, False)
    for shape in ((0, 64), (3, 0, 64), (0, 5, 64)):
        e = x.new_empty(shape)
        y, low = ops.lora_linear(e, w, a, b)
        assert y.shape == (*shape[:-1], 48)
        dx, da, db = ops.lora_linear_bwd(e, w, a, b, y, low)
        assert dx.shape == shape and not da.any() and not db.any()
        ids = torch.zeros(0, device="cuda", dtype=torch.int32)
        y = ops.lora_linear_many(e, w, a[None], b[None], ids, torch.ones(1, device="cuda"))
        assert y.shape == (*shape[:-1], 48)


def test_layer_norm_in_place():
    from foundry_trainer_b200 import ops
    g = _gen(15)
    for shape in ((5, 7), (3, 2048), (4000, 1024), (2, 3000, 514)):
        x = torch.randn(*shape, generator=g, device="cuda").to(BF)
        y, stats = ops.layer_norm(x)
        z, again = ops.layer_norm(x, out=x)
        assert z is x and torch.equal(x, y) and torch.equal(stats, again)


def test_lora_linear_takes_any_rows_of_b():
    # slices whose rows start anywhere, of one matrix and of stacked ones
    from foundry_trainer_b200 import ops
    g = _gen(16)
    E, N, K, M, r = 3, 90, 128, 200, 16
    x, w, a, _, bias = _lora_inputs(g, N, K, M, r, True, E)
    ids = (torch.arange(N, device="cuda") % (E + 1) - 1).to(torch.int32)
    scales = torch.rand(E, generator=g, device="cuda") + 0.5
    dy = _rn(g, N, M)
    big = _rn(g, E, M + 5, 40, std=0.5)
    # a row stride of 16 bytes or not, a first element on 16 bytes or not
    for rows, cols in ((slice(0, M), slice(3, 3 + r)), (slice(1, M + 1), slice(8, 8 + r)),
                       (slice(5, M + 5), slice(0, 12)), (slice(0, M), slice(1, 1 + r))):
        for whole in (big, _rn(g, E, M + 5, 37, std=0.5), big[:, :M + 3].contiguous()[:, :M + 5]):
            b = whole[:, :M][:, :, cols] if rows.stop > whole.shape[1] else whole[:, rows, cols]
            aa = a[:, :b.shape[2]]
            got = ops.lora_linear_many(x, w, aa, b, ids, scales, bias=bias)
            want = ops.lora_linear_many(x, w, aa, b.contiguous(), ids, scales, bias=bias)
            assert torch.equal(got, want)
            y, low = ops.lora_linear(x, w, aa[1], b[1], bias=bias)
            y2, low2 = ops.lora_linear(x, w, aa[1], b[1].contiguous(), bias=bias)
            assert torch.equal(y, y2) and torch.equal(low, low2)
            for p, q in zip(ops.lora_linear_bwd(x, w, aa[1], b[1], dy, low),
                            ops.lora_linear_bwd(x, w, aa[1], b[1].contiguous(), dy, low)):
                assert torch.equal(p, q)
