"""The block operators as the blocks use them (blocks.FusedKernels, Muon,
LoraTrainer) on the GPU: the reference's recorded block pair with them inside,
gradients against autograd of the plain form and against differences, streams,
capture, and a batch of requests with an adapter each."""
import pytest
import torch

from foundry_trainer_b200 import attn, blocks
from tests import block_ops_support as sup
from tests import block_support as bs
from tests.test_blocks_cpu import ACTS

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rn(g, *shape, std=1.0, dtype=BF):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


class FusedRun(bs.FixtureRun):
    """The recorded pipeline with FusedKernels in both blocks."""

    kernels = blocks.FusedKernels()

    def forward(self, img, txt, acts=None):
        fx = self.fx
        img2, txt2 = blocks.double_block(self.w, img, txt, self.temb, self.joint, fx.shape,
                                         lora_scale=fx.lora_scale, acts=acts, kernels=self.kernels)
        out = blocks.single_block(self.w, torch.cat([txt2, img2], dim=1), self.temb, self.single,
                                  fx.shape, lora_scale=fx.lora_scale, acts=acts,
                                  kernels=self.kernels)
        t, i = out[:, :self.T], out[:, self.T:]
        if acts is not None:
            acts["output/img"], acts["output/txt"] = i, t
        loss = blocks.mse(i, self.target_img) + blocks.mse(t, self.target_txt)
        if acts is not None:
            acts["loss"] = loss
        return loss


def test_recorded_block_pair_with_the_fused_kernels():
    # the reference's acceptance of its recorded bf16 values (lib.rs:640-667)
    fx = bs.Fixture()
    run = FusedRun(fx, BF, "cuda", lambda p: attn.JointAttention(p.cuda()),
                   lambda p: blocks.SingleAttention(p.cuda()))
    acts, grads = run.grads()
    torch.cuda.synchronize()
    pairs = [(n, acts[n][0], fx.recorded("bf16", n)) for n in ACTS]
    pairs.append(("loss", acts["loss"].reshape(1), fx.recorded("bf16", "loss").reshape(1)))
    for key in fx.z.files:
        if key.startswith("bf16:grad:"):
            name = key[len("bf16:"):].replace(":", "/")
            pairs.append((name, grads[name], fx.recorded("bf16", name)))
    assert len(pairs) == len(ACTS) + 9
    for name, got, want in pairs:
        got = got.detach().float().cpu().reshape(want.shape)
        assert bs.cosine(got, want) >= 0.999 and bs.rel_l2(got, want) <= 2e-2, (
            name, bs.cosine(got, want), bs.rel_l2(got, want))


@pytest.mark.parametrize("lead,per", [((2, 40), False), ((2, 40), True), ((80,), False)])
@pytest.mark.parametrize("dim", [96, 2048, 1001])
def test_layer_norm_mod_gradients_through_autograd(lead, per, dim):
    # fp32: against autograd of the plain form in 64 bits, and the derivative
    # along one direction against a central difference of the kernel's own
    # forward
    g = _gen(dim)
    x = _rn(g, *lead, dim, dtype=F32)
    mod = (lead[0], 1, dim) if per else (dim,)
    shift, scale, dy = _rn(g, *mod, dtype=F32), _rn(g, *mod, std=0.3, dtype=F32), \
        _rn(g, *lead, dim, dtype=F32)
    k = blocks.FusedKernels()
    leaves = [t.clone().requires_grad_(True) for t in (x, shift, scale)]
    y = k.layer_norm_mod(*leaves)
    got = torch.autograd.grad(y, leaves, dy)
    ref = [t.double().requires_grad_(True) for t in (x, shift, scale)]
    c = ref[0] - ref[0].mean(-1, keepdim=True)
    yr = c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-6) * (1 + ref[2]) + ref[1]
    want = torch.autograd.grad(yr, ref, dy.double())
    # sums of n terms in fp32 steps, magnitudes of order |dy| |h| (1 + |scale|) <= 100
    n = x.numel() // dim
    for name, a, b, terms in zip(("dx", "dshift", "dscale"), got, want, (dim, n, n)):
        assert a.shape == b.shape and a.dtype == F32
        tol = (80 + terms ** 0.5 * 8) * sup.STEP32 * (b.abs().max() + 10)
        assert (a.double() - b).abs().max() <= tol, (name, (a.double() - b).abs().max(), tol)
    v = [_rn(g, *t.shape, dtype=F32) for t in (x, shift, scale)]
    h = 2.0 ** -7
    with torch.no_grad():
        up = k.layer_norm_mod(*(t + h * d for t, d in zip((x, shift, scale), v)))
        dn = k.layer_norm_mod(*(t - h * d for t, d in zip((x, shift, scale), v)))
    diff = ((up.double() - dn.double()) / (2 * h) * dy).sum()
    along = sum((a.double() * d).sum() for a, d in zip(got, v))
    # h^2 / 6 times third derivatives of order ten, over y.numel() terms whose
    # signs are independent, and the outputs' rounding over h
    size = (y.numel() ** 0.5) * (10 * h * h / 6 * 10 + 2 ** -22 / h * 10)
    assert abs(diff - along) <= 6 * size, (diff.item(), along.item(), size)


@pytest.mark.parametrize("lead,K,M,r,bias", [((2, 300), 256, 384, 16, False), ((70,), 264, 136, 4, True),
                                             ((3, 5, 9), 128, 100, 12, True)])
def test_fused_linear_gradients_through_autograd(lead, K, M, r, bias):
    g = _gen(K + M)
    w = {"weights/l.weight": _rn(g, M, K, std=K ** -0.5), "weights/l.lora_a": _rn(g, r, K, std=K ** -0.5),
         "weights/l.lora_b": _rn(g, M, r, std=0.5)}
    if bias:
        w["weights/l.bias"] = _rn(g, M)
    x, dy, s = _rn(g, *lead, K), _rn(g, *lead, M), 0.75
    keys = [k for k in w if not k.endswith("weight")]
    leaves = [x.clone().requires_grad_(True)] + [w[k].clone().requires_grad_(True) for k in keys]
    ww = dict(w, **dict(zip(keys, leaves[1:])))
    y = blocks.FusedKernels().linear(ww, "l", leaves[0], s)
    assert y.shape == (*lead, M)
    got = dict(zip(["x"] + keys, torch.autograd.grad(y, leaves, dy)))
    d = [t.double() for t in (x.reshape(-1, K), w["weights/l.weight"], w["weights/l.lora_a"],
                              w["weights/l.lora_b"], dy.reshape(-1, M))]
    ry, ty, _, _ = sup.lora_ref(d[0], d[1], d[2], d[3], s,
                                w["weights/l.bias"].double() if bias else None)
    sup.within(y.detach().reshape(-1, M), ry, ty, "y")
    refs = sup.lora_bwd_ref(*d, s)
    for name, (ref, tol) in zip(("x", "weights/l.lora_a", "weights/l.lora_b"), refs):
        sup.within(got[name].reshape(ref.shape), ref, tol, name)
    if bias:
        ref = d[4].sum(0)
        sup.within(got["weights/l.bias"], ref,
                   sup.U16 * ref.abs() + d[4].shape[0] * sup.STEP32 * d[4].abs().sum(0) * 2, "bias")
    # y is linear in x: <dy, y(x + v) - y(x)> = <dx, v>, up to the outputs'
    # roundings (independent, half a step each: rms 2^-8 / sqrt(3)) and dx's
    v = _rn(g, *lead, K)
    with torch.no_grad():
        moved = (x.float() + v.float()).to(BF)
        y2 = blocks.FusedKernels().linear(w, "l", moved, s)
    step = moved.double() - x.double()
    left = ((y2.double() - y.detach().double()) * dy).sum()
    right = (got["x"].double() * step).sum()
    noise = sup.U16 * ((dy.double() * y2).square().sum() + (dy.double() * y.detach()).square().sum()
                       + (got["x"].double() * step).square().sum()).sqrt()
    assert abs(left - right) <= 6 * noise, (left.item(), right.item(), noise.item())


def _trainer(seed=3, opt=None, kernels=None, T=40, G=8):
    w = blocks.make_c3_weights(dim=256, heads=2, rank=16, seed=seed, device="cuda")
    g = torch.Generator().manual_seed(11)
    for k in w:
        if k.endswith(".lora_b"):
            w[k] = (torch.randn(w[k].shape, generator=g) * 0.02).to(device="cuda", dtype=BF)
    tr = blocks.LoraTrainer(w, blocks.BlockShape(256, 2), blocks.joint_positions(T, G), opt=opt,
                            kernels=kernels)
    mk = lambda *s: torch.randn(*s, generator=g).to(device="cuda", dtype=BF)
    return tr, (mk(1, G * G, 256), mk(1, T, 256), mk(256), mk(1, G * G, 256), mk(1, T, 256))


def test_trainer_with_the_fused_kernels_and_muon():
    # the loss and the factors' gradients agree with torch's norms and linears
    # as two bf16 evaluations of one block do; Muon's steps move every factor by
    # an orthogonalised direction
    plain, batch = _trainer()
    fused, _ = _trainer(opt=blocks.Muon(lr=0.01), kernels=blocks.FusedKernels())
    la, lb = plain.loss(*batch), fused.loss(*batch)
    ga, gb = torch.autograd.grad(la, plain.params), torch.autograd.grad(lb, fused.params)
    assert abs(la.item() - lb.item()) <= 2e-2 * abs(la.item())
    for key, a, b in zip(plain.keys, ga, gb):
        assert b.dtype == BF and bs.cosine(a, b) >= 0.999 and bs.rel_l2(b, a) <= 4e-2, (
            key, bs.cosine(a, b), bs.rel_l2(b, a))
    before = [p.detach().clone() for p in fused.params]
    state = [m.clone() for m in fused.state]
    first = [g.clone() for g in gb]
    fused.step(*batch)
    torch.cuda.synchronize()
    for p, q, m0, m1, g in zip(before, fused.params, state, fused.state, first):
        assert torch.allclose(m1, m0.lerp(g.float(), 0.05), rtol=1e-5, atol=1e-9)
        u = g.double().lerp(m1.double(), 0.95)
        x = u / (u.norm() + 1e-7)
        x = x.mT if x.shape[0] > x.shape[1] else x
        for _ in range(5):
            s = x @ x.mT
            x = 3.4445 * x + (-4.7750 * s + 2.0315 * (s @ s)) @ x
        x = x.mT if u.shape[0] > u.shape[1] else x
        lr = 0.01 * max(1.0, u.shape[0] / u.shape[1]) ** 0.5
        want = p.double() - lr * x
        # the orthogonalised direction's bf16 rounding and the parameter's
        tol = sup.U16 * (want.abs() + 2 * lr * x.abs()) + 1e-2 * lr * x.abs().max()
        assert ((q.double() - want).abs() <= tol).all()
    for _ in range(2):
        assert torch.isfinite(fused.step(*batch))


def test_a_step_on_a_side_stream_and_on_a_given_stream():
    from foundry_trainer_b200 import ops
    g = _gen(1)
    x, w, a, b = _rn(g, 500, 256), _rn(g, 384, 256), _rn(g, 12, 256), _rn(g, 384, 12)
    mod = _rn(g, 2, 256).t().contiguous().t()  # rows that need a copy
    x3 = x.view(2, 250, 256)
    ref = (*ops.lora_linear(x, w, a, b), ops.layer_norm(x3, mod, mod)[0],
           ops.orthogonalize(x[:100]))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for given in (None, side):
        # the inputs are made on the stream that the calls are ordered on
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            x2, m2 = x + 0, mod + 0
        if given is None:
            with torch.cuda.stream(side):
                got = (*ops.lora_linear(x2, w, a, b), ops.layer_norm(x2.view(2, 250, 256), m2, m2)[0],
                       ops.orthogonalize(x2[:100]))
        else:
            got = (*ops.lora_linear(x2, w, a, b, stream=side),
                   ops.layer_norm(x2.view(2, 250, 256), m2, m2, stream=side)[0],
                   ops.orthogonalize(x2[:100], stream=side))
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, ref))


def test_captured_steps_replay_in_turn():
    # forward and backward of the fused block captured twice, replayed in turn.
    # (No eager graph of these leaves may live then: torch ties their gradient
    # nodes to the stream of the first graph and invalidates the capture, with
    # or without these kernels.)
    from foundry_trainer_b200 import ops
    tr, batch = _trainer(kernels=blocks.FusedKernels())
    ref = [g.clone() for g in torch.autograd.grad(tr.loss(*batch), tr.params)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(tr.loss(*batch), tr.params)  # warm up
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(torch.autograd.grad(tr.loss(*batch), tr.params))
        graphs.append(graph)
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    # the attention backward adds dQ in arrival order; the rest repeats exactly
    for o in outs:
        for key, a, b in zip(tr.keys, o, ref):
            assert bs.rel_l2(a, b) <= 1e-2, (key, bs.rel_l2(a, b))


def test_captured_backward_beside_a_living_eager_graph():
    # over aliases of the leaves a capture is sound while an eager graph of the
    # leaves themselves lives; both give the same gradients afterwards
    g = _gen(6)
    w = {"weights/l.weight": _rn(g, 512, 256), "weights/l.lora_a": _rn(g, 16, 256),
         "weights/l.lora_b": _rn(g, 512, 16)}
    x, dy = _rn(g, 300, 256), _rn(g, 300, 512)
    shift, scale = _rn(g, 256), _rn(g, 256)
    leaves = [t.requires_grad_(True) for t in (x, w["weights/l.lora_a"], w["weights/l.lora_b"],
                                               shift, scale)]
    k = blocks.FusedKernels()

    def forward(x, a, b, sh, sc):
        ww = dict(w, **{"weights/l.lora_a": a, "weights/l.lora_b": b})
        return k.linear(ww, "l", k.layer_norm_mod(x, sh, sc), 1.0)

    eager = forward(*leaves)  # lives through the capture
    alias = [t.detach().requires_grad_(True) for t in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = [t.detach().requires_grad_(True) for t in leaves]
        torch.autograd.grad(forward(*warm), warm, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(forward(*alias), alias, dy)
    graph.replay()
    want = torch.autograd.grad(eager, leaves, dy)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_tokens_of_many_requests_follow_their_ids():
    from foundry_trainer_b200 import ops
    g = _gen(9)
    N, K, M, r, E = 24, 512, 640, 16, 6
    x, w, a, b = _rn(g, N, K), _rn(g, M, K), _rn(g, E, r, K), _rn(g, E, M, r)
    ids = torch.zeros(N, device="cuda", dtype=torch.int32)
    scales = torch.ones(E, device="cuda")
    ops.lora_linear_many(x, w, a, b, ids, scales)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.lora_linear_many(x, w, a, b, ids, scales)
    for seed in (1, 2):
        ids.copy_(torch.randint(-1, E, (N,), generator=_gen(seed), device="cuda", dtype=torch.int32))
        x.copy_(_rn(_gen(seed + 5), N, K))
        graph.replay()
        assert torch.equal(y, ops.lora_linear_many(x, w, a, b, ids, scales))


def test_a_batch_of_requests_with_an_adapter_each():
    # stacked factors and one adapter id a sample: each sample as if alone
    # with its own factors (or none)
    tr, (img, txt, temb, _, _) = _trainer()
    E, B = 3, 4
    g = _gen(4)
    stacked, single = dict(tr.w), []
    for key in tr.keys:
        t = tr.w[key].detach()
        stacked[key] = torch.stack([t, _rn(g, *t.shape, std=0.05), _rn(g, *t.shape, std=0.05)])
    stacked = {k: v.detach() for k, v in stacked.items()}
    imgs, txts = _rn(g, B, *img.shape[1:]), _rn(g, B, *txt.shape[1:])
    adapters = torch.tensor([2, -1, 0, 2], device="cuda", dtype=torch.int32)
    att = attn.JointAttention(blocks.joint_positions(40, 8).cuda())
    with torch.no_grad():
        oi, ot = blocks.double_block(stacked, imgs, txts, temb, att, tr.shape, lora_scale=0.5,
                                     kernels=blocks.FusedKernels(adapters))
        for i, e in enumerate(adapters.tolist()):
            w = {k: v[e] if k in tr.keys else v for k, v in stacked.items()
                 if not (e < 0 and k in tr.keys)}
            si, st = blocks.double_block(w, imgs[i:i + 1], txts[i:i + 1], temb, att, tr.shape,
                                         lora_scale=0.5, kernels=blocks.FusedKernels())
            for a, b in ((oi[i:i + 1], si), (ot[i:i + 1], st)):
                assert bs.rel_l2(a, b) <= 1e-2, (i, e, bs.rel_l2(a, b))
    assert E == stacked[tr.keys[0]].shape[0]


def test_fused_linear_of_a_trainable_weight_without_gradients():
    g = _gen(12)
    w = {"weights/l.weight": _rn(g, 256, 128), "weights/l.lora_a": _rn(g, 16, 128),
         "weights/l.lora_b": _rn(g, 256, 16)}
    x = _rn(g, 2, 70, 128)
    want = blocks.FusedKernels().linear(w, "l", x, 0.5)
    w = {k: t.clone().requires_grad_(True) for k, t in w.items()}
    for graph_free in (torch.no_grad(), torch.inference_mode()):
        with graph_free:
            y = blocks.FusedKernels().linear(w, "l", x, 0.5)
        assert torch.equal(y, want) and not y.requires_grad


def test_calls_at_once_on_three_streams():
    # each call repeats its bits, whatever runs beside it: clusters, tensor memory,
    # early starts and workspaces of calls on other streams
    from foundry_trainer_b200 import ops
    g = _gen(14)
    x, w = _rn(g, 900, 1024), _rn(g, 1544, 1024, std=0.03)
    a, b = _rn(g, 5, 12, 1024, std=0.03), _rn(g, 5, 1544, 12)
    dy = _rn(g, 900, 1544)
    ids = torch.randint(-1, 5, (900,), generator=g, device="cuda", dtype=torch.int32)
    scales = torch.ones(5, device="cuda")
    square, thin = _rn(g, 2, 300, 700), _rn(g, 6, 2000, 24)
    norm_w = _rn(g, 1024, std=0.2)

    def train():
        y, low = ops.lora_linear(x, w, a[0], b[0])
        return (y, *ops.lora_linear_bwd(x, w, a[0], b[0], dy, low))

    def serve():
        return tuple(ops.lora_linear_many(x[:n], w, a, b, ids[:n], scales) for n in (1, 60, 200, 900))

    def rest():
        y, stats = ops.layer_norm(x, norm_w, None)
        return (ops.orthogonalize(square), *ops.layer_norm_bwd(x, norm_w, x, stats),
                ops.orthogonalize(thin), y)

    calls = [train, serve, rest]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for turn in range(3):
        got = [[] for _ in calls]
        for _ in range(8):
            for k, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[k].append(calls[(k + turn) % 3]())
        torch.cuda.synchronize()
        assert ops.device_status() == 0
        for k in range(3):
            for one in got[k]:
                assert all(torch.equal(p, q) for p, q in zip(one, want[(k + turn) % 3]))
