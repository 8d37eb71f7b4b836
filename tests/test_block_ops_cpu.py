"""Refusals of the block operators, answered without a GPU: the Python entry
points raise before any launch, the C ABI returns a status code; and what the
blocks do without them stays as it was."""
import ctypes as C

import pytest
import torch

from foundry_trainer_b200 import _lib, blocks, ops

BF = torch.bfloat16


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("kw", [
    dict(x=z(8)), dict(x=z(1, 2, 3, 8)),                       # 1 or 4 dimensions
    dict(x=z(4, 8), weight=z(9)), dict(x=z(4, 8), bias=z(7)),  # another width
    dict(x=z(4, 8), weight=z(1, 8)),                           # per group without groups
    dict(x=z(2, 4, 8), weight=z(3, 8)),                        # another number of groups
    dict(x=z(4, 8), weight=z(8), bias=z(8, dtype=torch.float32)),
    dict(x=z(4, 8), out=z(4, 9)), dict(x=z(4, 8), out=z(4, 8, dtype=torch.float32)),
    dict(x=z(4, 8)),                                           # not on a GPU
])
def test_layer_norm_refuses(kw):
    with pytest.raises(ValueError):
        ops.layer_norm(**kw)


def test_layer_norm_refuses_types():
    with pytest.raises(TypeError):
        ops.layer_norm(z(4, 8, dtype=torch.float16))
    with pytest.raises(TypeError):
        ops.layer_norm(z(4, 8), z(8, dtype=torch.float16))
    with pytest.raises(TypeError):
        ops.layer_norm([1.0, 2.0])
    with pytest.raises(ValueError):
        ops.layer_norm_bwd(z(4, 8), None, z(4, 9), z(2, 4, dtype=torch.float32))


@pytest.mark.parametrize("x,w,a,b,bias", [
    (z(4, 16), z(8, 24), z(4, 16), z(8, 4), None),             # in does not fit w
    (z(4, 16), z(8, 16), z(4, 24), z(8, 4), None),             # nor a
    (z(4, 16), z(8, 16), z(4, 16), z(9, 4), None),             # out does not fit b
    (z(4, 16), z(8, 16), z(4, 16), z(8, 5), None),             # two ranks
    (z(4, 16), z(8, 16), z(1, 4, 16), z(1, 8, 4), None),       # stacked factors
    (z(4, 16), z(8, 16), z(4, 16), z(8, 4), z(9)),             # bias of another width
    (z(16), z(8, 16), z(4, 16), z(8, 4), None),                # one dimension
    (z(4, 2, 32).transpose(0, 1)[:, :, :16], z(8, 16), z(4, 16), z(8, 4), None),  # no one stride
    (z(4, 16), z(8, 16), z(4, 16), z(8, 4), None),             # not on a GPU
])
def test_lora_linear_refuses(x, w, a, b, bias):
    with pytest.raises(ValueError):
        ops.lora_linear(x, w, a, b, bias=bias)


def test_lora_linear_refuses_types_and_many_its_ids():
    with pytest.raises(TypeError):
        ops.lora_linear(z(4, 16, dtype=torch.float32), z(8, 16), z(4, 16), z(8, 4))
    with pytest.raises(ValueError):
        ops.lora_linear_many(z(4, 16), z(8, 16), z(3, 4, 16), z(2, 8, 4),
                             torch.zeros(4, dtype=torch.int32), torch.ones(3))
    with pytest.raises(ValueError):
        ops.lora_linear_many(z(4, 16), z(8, 16), z(4, 16), z(8, 4),
                             torch.zeros(4, dtype=torch.int32), torch.ones(3))


def test_orthogonalize_refuses():
    for g in (z(8), z(4, 8)):
        with pytest.raises(ValueError):
            ops.orthogonalize(g)
    with pytest.raises(TypeError):
        ops.orthogonalize(z(4, 8, dtype=torch.float16))
    with pytest.raises(TypeError):
        ops.orthogonalize(z(4, 8), steps=1.5)
    with pytest.raises(ValueError):
        ops.orthogonalize(z(4, 8), coeffs=(1.0, 2.0))


def test_c_abi_layer_norm_validates_without_a_gpu():
    lib = _lib.load()
    t = _lib.fa_tensor_t(4096, 0, 64, 0, 1)
    INV, UNS, ALI, BIG = (_lib.FA_ERR_INVALID_ARG, _lib.FA_ERR_UNSUPPORTED, _lib.FA_ERR_ALIGNMENT,
                          _lib.FA_ERR_TOO_LARGE)

    def fwd(dtype=1, groups=1, rows=4, dim=64, x=t, pdt=1, ps=0, eps=1e-6, y=t, w=None):
        return lib.fa_layer_norm_fwd(dtype, groups, rows, dim, C.byref(x) if x else None, w, None,
                                     pdt, ps, 0, eps, C.byref(y) if y else None, None, None)

    assert fwd(dtype=2) == UNS and fwd(pdt=5) == UNS
    assert fwd(groups=-1) == INV and fwd(rows=-1) == INV and fwd(dim=0) == INV and fwd(ps=-1) == INV
    assert fwd(dim=16385) == BIG and fwd(groups=70000) == BIG
    assert fwd(groups=65535, rows=1 << 20) == BIG
    assert fwd(eps=-1.0) == INV and fwd(eps=float("nan")) == INV
    assert fwd(x=None) == INV and fwd(y=None) == INV
    assert fwd(x=_lib.fa_tensor_t(4097, 0, 64, 0, 1)) == ALI
    assert fwd(x=_lib.fa_tensor_t(4096, 0, 64, 0, 2)) == ALI
    assert fwd(w=4097) == ALI
    assert fwd(rows=0, x=None, y=None) == _lib.FA_OK
    assert lib.fa_layer_norm_bwd(1, 1, 4, 64, C.byref(t), None, 1, 0, 0, C.byref(t), None,
                                 C.byref(t), None, None, None, 0, None) == INV  # no stats
    assert lib.fa_layer_norm_bwd_workspace_bytes(1, 4608, 2048) >= 2 * 2048 * 4
    assert lib.fa_layer_norm_bwd_workspace_bytes(0, 4608, 2048) == 0


def test_c_abi_lora_validates_without_a_gpu():
    lib = _lib.load()
    m = _lib.fa_matrix_t(4096, 0, 64)
    INV, UNS, ALI, BIG = (_lib.FA_ERR_INVALID_ARG, _lib.FA_ERR_UNSUPPORTED, _lib.FA_ERR_ALIGNMENT,
                          _lib.FA_ERR_TOO_LARGE)

    def fwd(dtype=1, rows=4, K=64, M=64, r=16, x=m, scale=1.0, low=4096, bias=None):
        ref = C.byref(x) if x else None
        return lib.fa_lora_linear_fwd(dtype, rows, K, M, r, ref, C.byref(m), C.byref(m), C.byref(m),
                                      scale, bias, C.byref(m), low, None)

    assert fwd(dtype=0) == UNS and fwd(r=257) == UNS
    assert fwd(rows=-1) == INV and fwd(K=0) == INV and fwd(M=0) == INV and fwd(r=0) == INV
    assert fwd(scale=float("inf")) == INV
    assert fwd(K=(1 << 24) + 1) == BIG
    assert fwd(x=None) == INV and fwd(low=None) == INV
    assert fwd(x=_lib.fa_matrix_t(4104, 0, 64)) == ALI and fwd(x=_lib.fa_matrix_t(4096, 0, 60)) == ALI
    assert fwd(x=_lib.fa_matrix_t(4096, 0, -64)) == ALI
    assert fwd(low=4104) == ALI and fwd(bias=4097) == ALI
    assert fwd(rows=0, x=None, low=None) == _lib.FA_OK

    def bwd(da=4096, db=4096, ws=4096, nb=1 << 20, low=4096, dy=m):
        return lib.fa_lora_linear_bwd(1, 4, 64, 64, 16, C.byref(m), C.byref(m), C.byref(m),
                                      C.byref(m), 1.0, low, C.byref(dy) if dy else None, C.byref(m),
                                      da, db, ws, nb, None)

    assert bwd(da=None) == INV and bwd(db=None) == INV  # both or neither
    assert bwd(low=None) == INV and bwd(dy=None) == INV
    assert bwd(ws=None) == _lib.FA_ERR_WORKSPACE and bwd(nb=8) == _lib.FA_ERR_WORKSPACE
    assert bwd(ws=4104) == ALI
    assert lib.fa_lora_linear_bwd_workspace_bytes(10, 12) == 10 * 2 * 16 * 2

    def many(E=3, ids=4096, scales=4096, ws=4096, nb=1 << 20):
        return lib.fa_lora_linear_many(1, 4, 64, 64, 16, E, C.byref(m), C.byref(m), C.byref(m),
                                       C.byref(m), ids, scales, None, C.byref(m), ws, nb, None)

    assert many(E=0) == INV and many(ids=None) == INV and many(scales=None) == INV
    assert many(ids=4098) == ALI and many(ws=None) == _lib.FA_ERR_WORKSPACE
    assert many(nb=16) == _lib.FA_ERR_WORKSPACE
    assert lib.fa_pad_rows(-1, 4, 4096, 4, 4096, 8, None) == INV
    assert lib.fa_pad_rows(1, 4, 4096, 4, 4096, 3, None) == INV
    assert lib.fa_pad_rows(0, 4, None, 4, None, 8, None) == _lib.FA_OK


def test_c_abi_lora_refuses_rows_that_overlap():
    # expanded operands: a row or an adapter stride of zero, or below the width
    lib = _lib.load()
    ALI = _lib.FA_ERR_ALIGNMENT
    M = lambda sr, sb=0: _lib.fa_matrix_t(4096, sb, sr)
    for at in range(5):
        for bad in (0, 56):
            ms = [M(64) for _ in range(5)]
            ms[at] = M(min(bad, 8) if at == 3 else bad)
            rc = lib.fa_lora_linear_fwd(1, 4, 64, 64, 16, *[C.byref(m) for m in ms[:4]], 1.0, None,
                                        C.byref(ms[4]), 4096, None)
            assert rc == ALI, (at, bad)
            rc = lib.fa_lora_linear_bwd(1, 4, 64, 64, 16, *[C.byref(m) for m in ms[:4]], 1.0, 4096,
                                        C.byref(ms[4]), C.byref(M(64)), 4096, 4096, 4096, 1 << 20, None)
            assert rc == ALI, (at, bad)
    for sa, sb in ((0, 1024), (1024, 0)):
        rc = lib.fa_lora_linear_many(1, 4, 64, 64, 16, 3, C.byref(M(64)), C.byref(M(64)),
                                     C.byref(M(64, sa)), C.byref(M(16, sb)), 4096, 4096, None,
                                     C.byref(M(64)), 4096, 1 << 20, None)
        assert rc == ALI


def test_aligned_rows_of_expanded_tensors():
    x = torch.randn(1, 24).to(BF).expand(5, 24)
    y = blocks._aligned(x)
    assert y.stride() == (24, 1) and torch.equal(x, y)
    assert blocks._aligned(y) is y


def test_c_abi_orthogonalize_validates_without_a_gpu():
    lib = _lib.load()

    def go(dtype=1, B=1, m=16, n=64, g=4096, o=4096, orow=64, steps=5, a=1.0, eps=1e-7, ws=4096,
           nb=1 << 30):
        return lib.fa_orthogonalize(dtype, B, m, n, g, m * n, n, o, m * n, orow, steps, a, -1.0, 0.5,
                                    eps, ws, nb, None)

    INV = _lib.FA_ERR_INVALID_ARG
    assert go(dtype=3) == _lib.FA_ERR_UNSUPPORTED
    assert go(B=-1) == INV and go(m=0) == INV and go(n=0) == INV and go(steps=0) == INV
    assert go(steps=65) == _lib.FA_ERR_TOO_LARGE and go(m=1 << 21) == _lib.FA_ERR_TOO_LARGE
    assert go(a=float("nan")) == INV and go(eps=-1.0) == INV
    assert go(g=None) == INV and go(o=None) == INV
    assert go(o=4098) == _lib.FA_ERR_ALIGNMENT and go(orow=63) == _lib.FA_ERR_ALIGNMENT
    assert go(m=128, n=128, orow=128, nb=64) == _lib.FA_ERR_WORKSPACE
    assert go(B=0) == _lib.FA_OK
    assert lib.fa_orthogonalize_workspace_bytes(4, 64, 4096, 5) == 0
    assert lib.fa_orthogonalize_workspace_bytes(1, 128, 256, 5) >= 3 * 128 * 256 * 2


def test_blocks_refuse_the_fused_kernels_on_cpu_and_muon_vectors():
    w = blocks.make_c3_weights(dim=256, heads=2, rank=4, seed=3, dtype=BF)
    k = blocks.FusedKernels()
    x = z(1, 8, 256)
    with pytest.raises(ValueError):
        k.linear(w, "double.img.to_q", x, 1.0)
    with pytest.raises(ValueError):
        k.layer_norm_mod(x, z(256), z(256))
    # a linear without factors is torch's
    assert torch.equal(k.linear(w, "double.img.mlp.fc1", x, 1.0),
                       blocks.linear(w, "double.img.mlp.fc1", x, 1.0))
    with pytest.raises(ValueError):
        blocks.Muon().init([z(4)])
    p = [z(4, 8)]
    with pytest.raises(ValueError):
        blocks.Muon().step(p, p, blocks.Muon().init(p), 1)


def test_fused_linear_refuses_a_trained_weight_and_stacked_gradients():
    w = {"weights/l.weight": z(8, 16).requires_grad_(True), "weights/l.lora_a": z(4, 16),
         "weights/l.lora_b": z(8, 4)}
    with pytest.raises(ValueError, match="must not require"):
        blocks.FusedKernels().linear(w, "l", z(2, 16), 1.0)
    w = {"weights/l.weight": z(8, 16), "weights/l.lora_a": z(3, 4, 16).requires_grad_(True),
         "weights/l.lora_b": z(3, 8, 4)}
    k = blocks.FusedKernels(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="without gradients"):
        k.linear(w, "l", z(2, 5, 16), 1.0)
    with torch.no_grad(), pytest.raises(ValueError, match="one adapter id"):
        k.linear(w, "l", z(3, 5, 16), 1.0)
    with torch.no_grad(), pytest.raises(ValueError, match="one adapter id"):
        blocks.FusedKernels().linear(w, "l", z(2, 5, 16), 1.0)


def test_out_must_not_share_elements():
    with pytest.raises(ValueError, match="share memory"):
        ops.layer_norm(z(4, 8), out=z(1, 8).expand(4, 8))
    with pytest.raises(ValueError, match="share memory"):
        ops.orthogonalize(z(3, 4, 8), out=z(1, 4, 8).expand(3, 4, 8))


def test_c_abi_lora_many_bounds_its_contraction():
    # (what a broken neighbour costs grows with it, under a bounded wait)
    lib = _lib.load()

    def many(K):
        m = _lib.fa_matrix_t(4096, 1 << 30, 1 << 24)
        return lib.fa_lora_linear_many(1, 4, K, 64, 16, 2, C.byref(m), C.byref(m), C.byref(m),
                                       C.byref(m), 4096, 4096, None, C.byref(m), None, 0, None)

    assert many((1 << 20) + 1) == _lib.FA_ERR_TOO_LARGE
    assert many(1 << 20) == _lib.FA_ERR_WORKSPACE  # the next check


def test_c_abi_orthogonalize_refuses_coefficients_beyond_fp16():
    lib = _lib.load()

    def go(m, steps, a, b, c):
        return lib.fa_orthogonalize(0, 1, m, 320, 4096, m * 320, 320, 4096, m * 320, 320, steps, a,
                                    b, c, 1e-7, None, 0, None)

    UNS, WS = _lib.FA_ERR_UNSUPPORTED, _lib.FA_ERR_WORKSPACE  # (the next check)
    default = (3.4445, -4.7750, 2.0315)
    for steps in (1, 5, 64):
        assert go(65, steps, *default) == WS
    # p(1) = 4.7, then 64 (b 4.7^2 + c 4.7^4) = 56700; the last step's result is bf16
    assert go(65, 2, 7.4435, *default[1:]) == WS and go(65, 3, 7.4435, *default[1:]) == UNS
    assert go(65, 2, 7.6435, *default[1:]) == UNS  # 4.9: 67600
    assert go(65, 2, 31.0, 0.0, 0.0) == WS and go(65, 2, 32.0, 0.0, 0.0) == UNS  # Q alone
    assert go(65, 1, 1.0, 1001.0, 0.0) == UNS and go(65, 1, 1.0, 0.0, -1001.0) == UNS
    assert go(65, 1, 0.0, 4004.0, -4004.0) == UNS  # its largest inside: 4004 / 4 at s^2 = 1/2
    assert go(65, 1, 0.0, 3990.0, -3990.0) == WS
    # short sides up to 64 are fp64 throughout
    assert go(64, 3, 32.0, 0.0, 0.0) not in (UNS, WS)


def test_fused_linear_refuses_a_trained_bias_beside_stacked_factors():
    # (its gradient would be missing without a word)
    w = {"weights/l.weight": z(8, 16), "weights/l.lora_a": z(3, 4, 16),
         "weights/l.lora_b": z(3, 8, 4), "weights/l.bias": z(8).requires_grad_(True)}
    k = blocks.FusedKernels(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="without gradients"):
        k.linear(w, "l", z(2, 5, 16), 1.0)


def test_fused_linear_takes_a_trainable_weight_without_gradients():
    # sampling with a model whose weights are parameters: on to the kernel, which
    # here misses its GPU
    w = {"weights/l.weight": z(8, 16).requires_grad_(True), "weights/l.lora_a": z(4, 16),
         "weights/l.lora_b": z(8, 4)}
    for graph_free in (torch.no_grad(), torch.inference_mode()):
        with graph_free, pytest.raises(ValueError, match="CUDA device"):
            blocks.FusedKernels().linear(w, "l", z(2, 16), 1.0)


def test_muon_bounds_what_it_orthogonalises_at_once(monkeypatch):
    # (32 matrices of 4096 x 14336 in one call took 7.5 GB of updates and 13 GB of
    # workspace)
    sizes = []

    def fake(u, **kw):
        sizes.append(u.numel())
        return (u * 0.5).to(BF)

    monkeypatch.setattr(ops, "orthogonalize", fake)
    shapes = [(8, 16)] * 7 + [(16, 8)] * 2 + [(64, 64)]
    g = torch.Generator().manual_seed(1)
    first = [torch.randn(*s, generator=g) for s in shapes]
    grads = [torch.randn(*s, generator=g) for s in shapes]
    results = []
    for most in (None, 300):  # two of the small ones, one large one
        if most:
            monkeypatch.setattr(blocks, "_MUON_ELEMENTS", most)
        p, opt = [t.clone() for t in first], blocks.Muon(weight_decay=0.1)
        state = opt.init(p)
        sizes.clear()
        opt.step(p, grads, state, 1)
        results.append(p + state)
    assert sorted(sizes) == [128, 256, 256, 256, 256, 4096]
    assert all(torch.equal(a, b) for a, b in zip(*results))
