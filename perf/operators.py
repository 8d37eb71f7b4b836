"""Measured cases of the block operators: the (modulated) layer norm, the linear
with low-rank adapters, and the Newton-Schulz orthogonalisation of an update.

A case is a dict of plain values. `prepare` makes what a program holds before
the call, `run` makes one pass: with `own` false in plain torch operations in
fp32, with `own` true through foundry_trainer_b200.ops. `exact` is the same
result in fp64, by another route.
"""
import math

import torch

own = False

EPS_NORM = 1e-6
EPS_NS = 1e-7
NS_COEFFS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5

BF16, F32 = "bf16", "f32"
_DT = {BF16: torch.bfloat16, F32: torch.float32}


# ------------------------------------------------------------------- cases

def _ln(name, B, L, D, dtype, mod, train):
    return {"name": name, "op": "layer_norm", "B": B, "L": L, "D": D, "dtype": dtype, "mod": mod,
            "train": train}


def _lora(name, N, K, M, r, bias):
    return {"name": name, "op": "lora_train", "N": N, "K": K, "M": M, "r": r, "bias": bias}


def _many(name, N, K, M, r, E, runs, bias):
    return {"name": name, "op": "lora_many", "N": N, "K": K, "M": M, "r": r, "E": E, "runs": runs,
            "bias": bias}


def _ns(name, batch, m, n, dtype, rank):
    return {"name": name, "op": "orthogonalize", "batch": batch, "m": m, "n": n, "dtype": dtype,
            "rank": rank}


def listed():
    return [
        # one token's modulated norm while sampling: the launch is the cost
        _ln("norm_one_row", 1, 1, 2048, BF16, True, False),
        # one block's norm in a training step: 512 text + 64x64 image tokens
        _ln("norm_block_train", 1, 4608, 2048, BF16, True, True),
        # an affine norm with an odd width and ragged rows, in fp32
        _ln("norm_odd_f32_train", 1, 3001, 1001, F32, False, True),
        # a batch of eight samples, each with its own modulation
        _ln("norm_batch_train", 8, 4608, 4096, BF16, True, True),
        # a square projection of a block with its rank-16 adapter, one step
        _lora("lora_proj_train", 4608, 2560, 2560, 16, False),
        # the same at odd sizes and a rank that is no multiple of eight
        _lora("lora_odd_train", 777, 1544, 2056, 12, True),
        # the wide linear of an MLP over two samples' tokens
        _lora("lora_mlp_train", 9216, 4096, 16384, 32, False),
        # one token of one request
        _many("lora_one_token", 1, 4096, 4096, 16, 4, 1, False),
        # single tokens of many requests, adapters in no order
        _many("lora_tokens", 64, 4096, 6144, 16, 48, 64, True),
        # ragged prompts of several requests packed one behind the other
        _many("lora_prompts", 6000, 4096, 4096, 32, 16, 9, False),
        # the gradients of one block's rank-16 factors, stacked
        _ns("muon_factors", 16, 16, 4096, BF16, 6),
        # the gradient of one full weight matrix
        _ns("muon_matrix", 1, 4096, 8192, F32, 96),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "lora_train", "lora_many", "orthogonalize"])
    if op == "layer_norm":
        B, D = rng.randint(1, 8), _logint(rng, 64, 8192)
        if rng.random() < 0.6:
            D = max(64, D // 64 * 64)
        L = _logint(rng, 1, max(1, min(9000, 36864 * 4096 // (B * D))))
        c = _ln("", B, L, D, rng.choice([BF16, F32]), rng.random() < 0.6, rng.random() < 0.7)
    elif op == "lora_train":
        K, M = 8 * _logint(rng, 32, 1024), 8 * _logint(rng, 32, 1024)
        N = _logint(rng, 1, 12000)
        c = _lora("", N, K, M, rng.choice([4, 8, 12, 16, 24, 32, 48, 64]), rng.random() < 0.5)
    elif op == "lora_many":
        K, M = 8 * _logint(rng, 32, 1024), 8 * _logint(rng, 32, 1024)
        N, E = _logint(rng, 1, 9000), _logint(rng, 1, 64)
        runs = N if N <= 256 and rng.random() < 0.6 else min(N, rng.randint(1, 24))
        c = _many("", N, K, M, rng.choice([8, 12, 16, 32, 64]), E, runs, rng.random() < 0.5)
    else:
        if rng.random() < 0.5:  # factors of adapters, either way up
            r, n, batch = rng.randint(4, 64), 8 * _logint(rng, 16, 1024), rng.randint(1, 32)
            m, n = (r, n) if rng.random() < 0.5 else (n, r)
            rank = rng.randint(1, r)
        else:
            m, n, batch = 8 * _logint(rng, 16, 512), 8 * _logint(rng, 16, 768), rng.randint(1, 2)
            rank = rng.randint(4, 128)
        c = _ns("", batch, m, n, rng.choice([BF16, F32]), rank)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rn(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    s = {"case": case}
    if case["op"] == "layer_norm":
        B, L, D, dt = case["B"], case["L"], case["D"], _DT[case["dtype"]]
        # hidden states of a residual stream: an offset and a few large channels
        x = torch.randn(B, L, D, generator=g, device="cuda")
        x = x * (1 + 4 * (torch.rand(D, generator=g, device="cuda") < 0.02)) + 0.3
        s["x"], s["dy"] = x.to(dt), rn(B, L, D, dtype=dt)
        lead = (B, D) if case["mod"] else (D,)
        s["w"] = rn(*lead, std=0.2, dtype=dt) if case["mod"] else rn(*lead, std=0.1, dtype=dt) + 1
        s["b"] = rn(*lead, std=0.2, dtype=dt)
    elif case["op"] in ("lora_train", "lora_many"):
        N, K, M, r = case["N"], case["K"], case["M"], case["r"]
        s["x"] = rn(N, K)
        s["w"] = rn(M, K, std=0.02)
        s["bias"] = rn(M, std=0.1) if case["bias"] else None
        E = case.get("E", 1)
        s["a"] = rn(E, r, K, std=1 / math.sqrt(K))
        s["b"] = rn(E, M, r, std=0.05)
        if case["op"] == "lora_train":
            s["a"], s["b"], s["scale"] = s["a"][0], s["b"][0], 2.0
            s["dy"] = rn(N, M)
        else:
            s["scale"] = torch.rand(E, generator=g, device="cuda") + 0.5
            # requests of unequal length one behind the other; one in eight has no adapter
            runs = case["runs"]
            ids = torch.randint(0, E, (runs,), generator=g, device="cuda", dtype=torch.int32)
            none = torch.rand(runs, generator=g, device="cuda") < 0.125
            none[0] = False
            ids = torch.where(none, torch.full_like(ids, -1), ids)
            if runs < N:
                cut = torch.rand(N, generator=g, device="cuda").argsort()[:runs - 1] if runs > 1 \
                    else torch.zeros(0, device="cuda", dtype=torch.int64)
                step = torch.zeros(N, device="cuda", dtype=torch.int64)
                step[cut[cut > 0]] = 1
                ids = ids[step.cumsum(0)]
            s["ids"] = ids.contiguous()
    else:
        batch, m, n, k = case["batch"], case["m"], case["n"], case["rank"]
        # a gradient: a few strong directions of falling strength over noise
        fall = 1.0 / torch.arange(1, k + 1, device="cuda").sqrt()
        u = torch.randn(batch, m, k, generator=g, device="cuda") * fall
        v = torch.randn(batch, k, n, generator=g, device="cuda")
        grad = (u @ v + torch.randn(batch, m, n, generator=g, device="cuda")) * 1e-3
        s["g"] = grad.to(_DT[case["dtype"]])
    return s


# ----------------------------------------------------------------- one pass

def _plain_norm(s, case):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    if case["mod"]:
        w, b = 1 + w[:, None], b[:, None]
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS_NORM)
    h = c * rstd
    y = (h * w + b).to(s["x"].dtype)
    if not case["train"]:
        return {"y": y}
    dy = s["dy"].float()
    dh = dy * w
    dx = rstd * (dh - dh.mean(-1, keepdim=True) - h * (dh * h).mean(-1, keepdim=True))
    dims = (1,) if case["mod"] else (0, 1)
    return {"y": y, "dx": dx.to(s["x"].dtype), "dw": (dy * h).sum(dims), "db": dy.sum(dims)}


def _plain_lora_train(s):
    x, w, a, b, dy = (s[k].float() for k in ("x", "w", "a", "b", "dy"))
    low = x @ a.T * s["scale"]
    y = x @ w.T + low @ b.T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    u = dy @ b * s["scale"]
    dx = dy @ w + u @ a
    return {k: v.to(torch.bfloat16) for k, v in
            (("y", y), ("dx", dx), ("da", u.T @ x), ("db", dy.T @ low))}


def _plain_lora_many(s):
    x, w, a, b = (s[k].float() for k in ("x", "w", "a", "b"))
    E, r, K = a.shape
    mine = (s["ids"][:, None] == torch.arange(E, device="cuda")) * s["scale"]
    low = (x @ a.reshape(E * r, K).T).reshape(-1, E, r) * mine[:, :, None]
    y = x @ w.T + low.reshape(-1, E * r) @ b.transpose(1, 2).reshape(E * r, -1)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return {"y": y.to(torch.bfloat16)}


def _plain_orthogonalize(s):
    a, b, c = NS_COEFFS
    x = s["g"].float()
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2) if tall else x
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPS_NS)
    for _ in range(NS_STEPS):
        q = x @ x.transpose(1, 2)
        x = a * x + (b * q + c * (q @ q)) @ x
    return {"o": (x.transpose(1, 2) if tall else x).to(torch.bfloat16)}


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if not own:
        if op == "layer_norm":
            return _plain_norm(s, case)
        if op == "lora_train":
            return _plain_lora_train(s)
        if op == "lora_many":
            return _plain_lora_many(s)
        return _plain_orthogonalize(s)
    from foundry_trainer_b200 import ops
    if op == "layer_norm":
        y, stats = ops.layer_norm(s["x"], s["w"], s["b"], unit_offset=case["mod"], eps=EPS_NORM)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = ops.layer_norm_bwd(s["x"], s["w"], s["dy"], stats, unit_offset=case["mod"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if op == "lora_train":
        y, low = ops.lora_linear(s["x"], s["w"], s["a"], s["b"], scale=s["scale"], bias=s["bias"])
        dx, da, db = ops.lora_linear_bwd(s["x"], s["w"], s["a"], s["b"], s["dy"], low,
                                         scale=s["scale"])
        return {"y": y, "dx": dx, "da": da, "db": db}
    if op == "lora_many":
        return {"y": ops.lora_linear_many(s["x"], s["w"], s["a"], s["b"], s["ids"], s["scale"],
                                          bias=s["bias"])}
    return {"o": ops.orthogonalize(s["g"], steps=NS_STEPS, coeffs=NS_COEFFS, eps=EPS_NS)}


# ------------------------------------------------------------ what it costs

def work(case):
    op = case["op"]
    if op == "layer_norm":
        n, es = case["B"] * case["L"] * case["D"], 4 if case["dtype"] == F32 else 2
        lead = (case["B"] if case["mod"] else 1) * case["D"]
        if not case["train"]:
            return {"bytes": 2 * n * es + 2 * lead * es, "flops": 8 * n}
        return {"bytes": 4 * n * es + 2 * lead * es + 8 * lead, "flops": 22 * n}
    if op == "lora_train":
        N, K, M, r = case["N"], case["K"], case["M"], case["r"]
        return {"bytes": 2 * (2 * N * K + 2 * N * M + M * K + 2 * r * (K + M)),
                "flops": 4 * N * K * M + 6 * N * r * (K + M)}
    if op == "lora_many":
        N, K, M, r = case["N"], case["K"], case["M"], case["r"]
        # adapters that are drawn at least once, on the average over seeds
        used = case["E"] * (1 - (1 - 0.875 / case["E"]) ** case["runs"])
        return {"bytes": 2 * (N * K + N * M + M * K + used * r * (K + M)),
                "flops": 2 * N * (K * M + r * (K + M))}
    b, es = case["batch"], 4 if case["dtype"] == F32 else 2
    m, n = min(case["m"], case["n"]), max(case["m"], case["n"])
    # both Gram products are symmetric: half of their sums suffice. Where one
    # side is short, sums over the long side are needed twice only: the Gram
    # matrix of the input, and the polynomial in it times the input.
    full = NS_STEPS * (m * m * n + m ** 3 + 2 * m * m * n)
    thin = m * m * n + 2 * m * m * n + NS_STEPS * 4 * m ** 3
    return {"bytes": b * m * n * (es + 2), "flops": b * min(full, thin)}


# ----------------------------------------------------------------- in 64 bits

def _exact_norm(s, case):
    x, w, b, dy = (s[k].double() for k in ("x", "w", "b", "dy"))
    if case["mod"]:
        w, b = (w + 1).unsqueeze(1), b.unsqueeze(1)
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    sd = torch.sqrt(var + EPS_NORM)
    out = {"y": (x - mean) / sd * w + b}
    if case["train"]:
        # dx = J^T (w dy) with J = (I - 11^T/D - h h^T/D) / sd
        h, D = (x - mean) / sd, x.shape[-1]
        t = dy * w
        along = torch.einsum("blj,blj->bl", t, h).unsqueeze(-1) / D
        out["dx"] = (t - t.sum(-1, keepdim=True) / D - along * h) / sd
        eq = "blj,blj->bj" if case["mod"] else "blj,blj->j"
        out["dw"], out["db"] = torch.einsum(eq, dy, h), torch.einsum(eq, dy, torch.ones_like(h))
    return out


def _exact_lora(s, case):
    x, w, a, b = (s[k].double() for k in ("x", "w", "a", "b"))
    bias = 0 if s["bias"] is None else s["bias"].double()
    if case["op"] == "lora_train":
        # through the merged weight and its gradient
        merged = w + s["scale"] * (b @ a)
        dy = s["dy"].double()
        grad = dy.T @ x
        return {"y": x @ merged.T + bias, "dx": dy @ merged, "da": s["scale"] * (b.T @ grad),
                "db": s["scale"] * (grad @ a.T)}
    y = torch.empty(x.shape[0], w.shape[0], dtype=torch.float64, device="cuda")
    for e in range(-1, case["E"]):
        rows = (s["ids"] == e).nonzero().squeeze(1)
        if rows.numel():
            merged = w if e < 0 else w + s["scale"][e].double() * (b[e] @ a[e])
            y[rows] = x[rows] @ merged.T
    return {"y": y + bias}


def _exact_orthogonalize(s):
    # X_5 = P X_0 with P the product of the steps' polynomials in the Gram
    # matrix, all of which commute
    a, b, c = NS_COEFFS
    x = s["g"].double()
    wide = x.shape[1] <= x.shape[2]
    x = x if wide else x.mT
    x = x / (torch.linalg.matrix_norm(x)[:, None, None] + EPS_NS)
    q = x @ x.mT
    eye = torch.eye(q.shape[1], dtype=torch.float64, device="cuda")
    p = eye
    for _ in range(NS_STEPS):
        f = a * eye + q @ (b * eye + c * q)
        p, q = f @ p, f @ q @ f
    x = p @ x
    return {"o": x if wide else x.mT}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        return _exact_norm(s, case)
    if case["op"] == "orthogonalize":
        return _exact_orthogonalize(s)
    return _exact_lora(s, case)
