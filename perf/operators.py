"""Measured cases of the fine-tuning operators: low-rank adapters of many requests beside a frozen projection, the norms
around a transformer block fused with its gate and residual scale, and the orthogonalised matrix update.

`run` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at the end) or, with
`own` set, through dreammat_amd.hipops.  `exact` restates the definitions in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
NS_COEFFS = (3.4445, -4.7750, 2.0315)          # quintic Newton-Schulz step: x <- a x + b x^3 + c x^5 on every singular value


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of 16 requests, each with its own adapter: latency and the weight read
        dict(name="adapter_tokens", op="adapter", mode="fwd", type="bf16", requests=16, rows=16, K=1280, N=1280, R=16, E=32, ragged=False, residual=False),
        # prompts of unequal length through the key projection of a cross attention (context 1024 -> 1280); some without adapter
        dict(name="adapter_ragged", op="adapter", mode="fwd", type="f16", requests=24, rows=1851, K=1024, N=1280, R=32, E=9, ragged=True, residual=False),
        # 24 images of the guidance batch (32 x 32 tokens), output projection with its residual
        dict(name="adapter_views", op="adapter", mode="fwd", type="bf16", requests=24, rows=24576, K=640, N=640, R=16, E=9, ragged=False, residual=True),
        # training: batch 4 at 64 x 64 tokens, forward and all gradients
        dict(name="adapter_train", op="adapter", mode="train", type="f16", requests=4, rows=16384, K=320, N=320, R=8, E=4, ragged=False, residual=False),
        # training: the widest projection of a block at 24 images
        dict(name="adapter_train_wide", op="adapter", mode="train", type="bf16", requests=24, rows=24576, K=1280, N=5120, R=64, E=8, ragged=False, residual=False),
        # two encoded prompts: a launch that is all latency
        dict(name="norm_prompts", op="norm", mode="fwd", type="f16", B=2, S=77, C=1024, kind="layer", gate="channel", post=True, pre=True),
        # the guidance batch at 64 x 64 tokens: the widest activation of the nets
        dict(name="norm_views", op="norm", mode="fwd", type="bf16", B=24, S=4096, C=320, kind="layer", gate="item", post=False, pre=True),
        # training, batch 4 at 64 x 64, every parameter
        dict(name="norm_train", op="norm", mode="train", type="bf16", B=4, S=4096, C=640, kind="layer", gate="item", post=True, pre=True),
        # training in 32 bits, RMS norms
        dict(name="norm_train_f32", op="norm", mode="train", type="f32", B=24, S=1024, C=1280, kind="rms", gate="channel", post=True, pre=True),
        # one attention projection of the 64 x 64 level
        dict(name="ortho_one", op="ortho", type="bf16", count=1, m=320, n=320),
        # the attention projections of the 16 x 16 level, one stack
        dict(name="ortho_stack", op="ortho", type="bf16", count=16, m=1280, n=1280),
        # the matrices of one 16 x 16-level transformer block and its 3 x 3 convolution, 32-bit masters
        dict(name="muon_block", op="muon", type="f32", width=1280, context=1024, inner=5120, conv=True),
    ]


def _spread(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["adapter", "adapter", "norm", "ortho", "muon"])
    if op == "adapter":
        mode = rng.choice(["fwd", "train"])
        requests = _spread(rng, 1, 64)
        each = 1 if mode == "fwd" and rng.random() < 0.3 else _spread(rng, 1, 4096)
        rows = min(24576 // requests * requests, requests * each)
        return dict(op=op, mode=mode, type=rng.choice(["bf16", "f16"]), requests=requests, rows=rows, K=_spread(rng, 64, 1280, 8),
                    N=_spread(rng, 64, 5120, 8), R=rng.choice([1, 4, 8, 12, 16, 32, 64]), E=_spread(rng, 1, 9), ragged=rng.random() < 0.5,
                    residual=rng.random() < 0.5)
    if op == "norm":
        C = _spread(rng, 64, 5120, rng.choice([1, 8, 8]))
        tokens = _spread(rng, 1, max(2, 30_000_000 // C))
        B = rng.choice([b for b in (1, 2, 3, 4, 8, 24) if b <= tokens])
        return dict(op=op, mode=rng.choice(["fwd", "train"]), type=rng.choice(["bf16", "f16", "f32"]), B=B, S=max(1, tokens // B), C=C,
                    kind=rng.choice(["layer", "rms"]), gate=rng.choice(["none", "channel", "item"]), post=rng.random() < 0.7, pre=rng.random() < 0.8)
    if op == "ortho":
        m, n = _spread(rng, 16, 1280), _spread(rng, 16, 2560)
        return dict(op=op, type=rng.choice(["bf16", "f16", "f32"]), count=_spread(rng, 1, 8), m=m, n=n)
    return dict(op=op, type="f32", width=_spread(rng, 64, 1280, 8), context=_spread(rng, 64, 1024, 8), inner=_spread(rng, 128, 5120, 8), conv=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _rand(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _muon_shapes(case):
    w, c, i = case["width"], case["context"], case["inner"]
    shapes = [(w, w)] * 6 + [(w, c)] * 2 + [(2 * i, w), (w, i)]
    return shapes + ([(w, w, 3, 3)] if case["conv"] else [])


def _gradient(g, rows, cols, dtype=torch.float32):
    """a gradient-like matrix: rows and columns of unequal size and a few directions that stand out"""
    m = torch.randn(rows, cols, generator=g, device=DEV) * torch.exp(0.5 * torch.randn(rows, 1, generator=g, device=DEV))
    m = m * torch.exp(0.5 * torch.randn(1, cols, generator=g, device=DEV))
    m = m + 0.5 * torch.randn(rows, 4, generator=g, device=DEV) @ torch.randn(4, cols, generator=g, device=DEV)
    return (1e-3 * m).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    t = TYPES[case["type"]]
    s = dict(case=case)
    if case["op"] == "adapter":
        M, K, N, R, E, n = (case[k] for k in ("rows", "K", "N", "R", "E", "requests"))
        s["x"] = _rand(g, M, K, dtype=t)
        s["w"] = _rand(g, N, K, dtype=t, scale=K ** -0.5)
        s["w_t"] = s["w"].t().contiguous()                     # laid out once, as for every frozen layer that is differentiated through
        s["bias"] = _rand(g, N, dtype=t, scale=0.1)
        s["a"] = _rand(g, E, R, K, dtype=t, scale=K ** -0.5)
        s["b"] = _rand(g, E, N, R, dtype=t, scale=0.3 * R ** -0.5)
        s["residual"] = _rand(g, M, N, dtype=t) if case["residual"] else None
        s["ids"] = torch.randint(-1 if n > 4 else 0, E, (n,), generator=g, device=DEV, dtype=torch.int32)
        s["offsets"] = None
        if case["ragged"]:                                      # cut points anywhere (empty requests among them), a tail behind the last
            last = M - M // 50
            cuts = torch.sort(torch.randint(0, last + 1, (n - 1,), generator=g, device=DEV)).values
            s["offsets"] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), last)]).to(torch.int32)
        s["dy"] = _rand(g, M, N, dtype=t) if case["mode"] == "train" else None
    elif case["op"] == "norm":
        B, S, C = case["B"], case["S"], case["C"]
        s["x"] = (_rand(g, B, S, C) * torch.exp(0.5 * _rand(g, C)) + 0.3 * _rand(g, C)).to(t)
        s["h"] = (_rand(g, B, S, C) * torch.exp(0.3 * _rand(g, C))).to(t)
        s["gate"] = {"none": None, "channel": _rand(g, C, dtype=t, scale=0.5), "item": _rand(g, B, C, dtype=t, scale=0.5)}[case["gate"]]
        for k in ("post", "pre"):
            s[k] = ((1 + 0.1 * _rand(g, C)).to(t), _rand(g, C, dtype=t, scale=0.1) if case["kind"] == "layer" else None) if case[k] else None
        if case["mode"] == "train":
            s["dy"] = _rand(g, B, S, C, dtype=t)
            s["dz"] = _rand(g, B, S, C, dtype=t) if case["pre"] else None
    elif case["op"] == "ortho":
        s["g"] = torch.stack([_gradient(g, case["m"], case["n"], t) for _ in range(case["count"])])
    else:
        shapes = _muon_shapes(case)
        flat = [(q[0], math.prod(q[1:])) for q in shapes]
        s["grads"] = [_gradient(g, *f).view(q) for f, q in zip(flat, shapes)]
        s["momenta"] = [_gradient(g, *f).view(q) for f, q in zip(flat, shapes)]
        s["params"] = [_rand(g, *q, scale=0.02) for q in shapes]
    return s


# ------------------------------------------------------------------------------------------------ plain forms
ADAPTER_SCALE, RES_SCALE, EPS = 0.75, 0.9, 1e-5
LR, MOMENTUM, DECAY = 2e-3, 0.95, 0.01


def _row_ids(s, M):
    """adapter of every row; -1 where there is none"""
    ids = s["ids"].long()
    if s["offsets"] is None:
        return ids.repeat_interleave(M // ids.numel(), output_size=M)
    at = torch.searchsorted(s["offsets"].long(), torch.arange(M, device=DEV), right=True) - 1
    return torch.where(at < ids.numel(), ids[at.clamp(max=ids.numel() - 1)], -torch.ones_like(at))


def _adapter_plain(s):
    case, t = s["case"], s["x"].dtype
    M, E, R = case["rows"], case["E"], case["R"]
    x, w = s["x"].float(), s["w"].float()
    a = s["a"].float().reshape(E * R, -1)                       # every adapter's rank rows side by side; a row keeps its own adapter's
    b = s["b"].float().permute(0, 2, 1).reshape(E * R, -1)
    mine = (_row_ids(s, M)[:, None] == torch.arange(E, device=DEV)).float().repeat_interleave(R, dim=1) * ADAPTER_SCALE
    u = (x @ a.t()) * mine
    y = x @ w.t() + s["bias"].float() + u @ b
    y = (y if s["residual"] is None else y + s["residual"].float()).to(t)
    if case["mode"] == "fwd":
        return y
    dy = s["dy"].float()
    du = (dy @ b.t()) * mine
    dx = dy @ w + du @ a
    da = du.t() @ x
    db = u.t() @ dy
    return dict(y=y, dx=dx.to(t), da=da.view(E, R, -1).to(t), db=db.view(E, R, -1).permute(0, 2, 1).to(t))


def _norm(v, kind, affine):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    if affine is None:
        return v
    v = v * affine[0]
    return v if affine[1] is None else v + affine[1]


def _norm_forward(x, h, gate, post, pre, kind):
    n = h if post is None else _norm(h, kind, post)
    if gate is not None:
        n = n * (gate[:, None] if gate.dim() == 2 else gate)
    y = x + RES_SCALE * n
    return (y, _norm(y, kind, pre)) if pre is not None else (y, None)


def _norm_leaves(s):
    return [s["x"], s["h"], s["gate"]] + [v for k in ("post", "pre") for v in (s[k] or (None, None))]


def _norm_plain(s):
    t, train = s["x"].dtype, s["case"]["mode"] == "train"
    v = [None if q is None else q.float() for q in _norm_leaves(s)]
    if train:
        v = [None if q is None else q.detach().requires_grad_() for q in v]
    x, h, gate, pg, pb, qg, qb = v
    with torch.set_grad_enabled(train):
        y, z = _norm_forward(x, h, gate, (pg, pb) if s["post"] else None, (qg, qb) if s["pre"] else None, s["case"]["kind"])
    out = [y.detach().to(t), None if z is None else z.detach().to(t)]
    if train:
        leaves = [q for q in v if q is not None]
        outs, ups = ([y, z], [s["dy"].float(), s["dz"].float()]) if z is not None else ([y], [s["dy"].float()])
        out += [q.to(t) for q in torch.autograd.grad(outs, leaves, ups)]
    return [q for q in out if q is not None]


def _newton_schulz(g, steps=5, eps=1e-7):
    a, b, c = NS_COEFFS
    wide = g.shape[-2] <= g.shape[-1]
    x = g if wide else g.mT
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + eps)
    for _ in range(steps):
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    return x if wide else x.mT


def _muon_plain(s):
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        m.mul_(MOMENTUM).add_(g)
        o = _newton_schulz((g + MOMENTUM * m).flatten(1)).view_as(p)
        rows, cols = p.shape[0], p[0].numel()
        p.mul_(1 - LR * DECAY).sub_(o, alpha=LR * 0.2 * math.sqrt(max(rows, cols)))
    return dict(params=s["params"], momenta=s["momenta"])


# ------------------------------------------------------------------------------------------------ the framework's calls
def _adapter_own(s):
    from dreammat_amd import hipops
    if s["case"]["mode"] == "fwd":
        return hipops.linear_adapted(s["x"], s["w"], s["bias"], s["a"], s["b"], s["ids"], scale=ADAPTER_SCALE, residual=s["residual"], offsets=s["offsets"])
    x, a, b = (s[k].detach().requires_grad_() for k in ("x", "a", "b"))
    y = hipops.linear_adapted_autograd(x, s["w"], s["w_t"], s["bias"], a, b, s["ids"], scale=ADAPTER_SCALE, residual=s["residual"], offsets=s["offsets"])
    dx, da, db = torch.autograd.grad(y, (x, a, b), s["dy"])
    return dict(y=y.detach(), dx=dx, da=da, db=db)


def _norm_own(s):
    from dreammat_amd import hipops
    train = s["case"]["mode"] == "train"
    v = _norm_leaves(s)
    if train:
        v = [None if q is None else q.detach().requires_grad_() for q in v]
    x, h, gate, pg, pb, qg, qb = v
    got = hipops.gated_add_norm(x, h, gate, post=(pg, pb) if s["post"] else None, pre=(qg, qb) if s["pre"] else None, scale=RES_SCALE, eps=EPS,
                                kind=s["case"]["kind"])
    outs = list(got) if isinstance(got, tuple) else [got]
    if not train:
        return outs
    leaves = [q for q in v if q is not None]
    grads = torch.autograd.grad(outs, leaves, [s["dy"], s["dz"]][:len(outs)])
    return [q.detach() for q in outs] + list(grads)


def _muon_own(s):
    from dreammat_amd import hipops
    hipops.muon_step(s["params"], s["grads"], s["momenta"], lr=LR, momentum=MOMENTUM, nesterov=True, weight_decay=DECAY, scale="rms")
    return dict(params=s["params"], momenta=s["momenta"])


def _ortho_own(s):
    from dreammat_amd import hipops
    return hipops.orthogonalize(s["g"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"adapter": _adapter_own, "norm": _norm_own, "ortho": _ortho_own, "muon": _muon_own}[op](state)
    if op == "ortho":
        return _newton_schulz(state["g"].float()).to(state["g"].dtype)
    return {"adapter": _adapter_plain, "norm": _norm_plain, "muon": _muon_plain}[op](state)


# ------------------------------------------------------------------------------------------------ floors
def _ns_flops(m, n, steps=5):
    """X X^T and its square are symmetric: half of each; the last product is whole (m <= n)"""
    m, n = min(m, n), max(m, n)
    return steps * (m * m * n + m * m * m + 2.0 * m * m * n)


def work(case):
    size = torch.empty(0, dtype=TYPES[case["type"]]).element_size()
    if case["op"] == "adapter":
        M, K, N, R = (float(case[k]) for k in ("rows", "K", "N", "R"))
        used = min(case["E"], case["requests"])
        base, low = 2 * M * K * N, 2 * M * R * (K + N)
        read = M * K + K * N + N + used * R * (K + N) + (M * N if case["residual"] else 0)
        if case["mode"] == "fwd":
            return dict(bytes=size * (read + M * N), flops=base + low)
        return dict(bytes=size * (read + M * N + M * N + M * K + case["E"] * R * (K + N)), flops=2 * base + 3 * low)
    if case["op"] == "norm":
        n, C = float(case["B"] * case["S"] * case["C"]), case["C"]
        big = 3 + (1 if case["pre"] else 0)                     # x, h -> y, z
        if case["mode"] == "train":
            big += 3 + (1 if case["pre"] else 0)                # dy, dz -> dx, dh
        return dict(bytes=size * (big * n + 6 * C), flops=0)
    if case["op"] == "ortho":
        return dict(bytes=2.0 * size * case["count"] * case["m"] * case["n"], flops=case["count"] * _ns_flops(case["m"], case["n"]))
    shapes = [(q[0], math.prod(q[1:])) for q in _muon_shapes(case)]
    return dict(bytes=4.0 * 5 * sum(r * c for r, c in shapes), flops=sum(_ns_flops(r, c) for r, c in shapes))


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_adapter(s):
    case = s["case"]
    x, w, bias, a, b = (s[k].double() for k in ("x", "w", "bias", "a", "b"))
    M, E = case["rows"], case["E"]
    y = torch.addmm(bias, x, w.T)
    if s["residual"] is not None:
        y += s["residual"].double()
    starts = (s["offsets"].tolist() if s["offsets"] is not None else [i * (M // case["requests"]) for i in range(case["requests"] + 1)])
    train = case["mode"] == "train"
    if train:
        dy = s["dy"].double()
        dx, da, db = dy @ w, torch.zeros_like(a), torch.zeros_like(b)
    for e, lo, hi in zip(s["ids"].tolist(), starts, starts[1:]):
        if not 0 <= e < E or lo == hi:
            continue
        u = ADAPTER_SCALE * (x[lo:hi] @ a[e].T)
        y[lo:hi] += u @ b[e].T
        if train:
            du = ADAPTER_SCALE * (dy[lo:hi] @ b[e])
            dx[lo:hi] += du @ a[e]
            da[e] += du.T @ x[lo:hi]
            db[e] += dy[lo:hi].T @ u
    return dict(y=y, dx=dx, da=da, db=db) if train else y


def _exact_normed(v, kind):
    mu = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    r = 1 / torch.sqrt(((v - mu) ** 2).mean(-1, keepdim=True) + EPS)
    return (v - mu) * r, r


def _exact_norm_back(d, hat, r, kind):
    """gradient through hat = (v - mean) r or v r"""
    along = (d * hat).mean(-1, keepdim=True) * hat
    return r * (d - along - (d.mean(-1, keepdim=True) if kind == "layer" else 0))


def _exact_norm(s):
    case, kind = s["case"], s["case"]["kind"]
    x, h = s["x"].double(), s["h"].double()
    C = case["C"]
    one, zero = torch.ones(C, device=DEV, dtype=torch.float64), torch.zeros(C, device=DEV, dtype=torch.float64)
    pair = lambda q: (one, zero) if q is None else (q[0].double(), zero if q[1] is None else q[1].double())
    gate = one[None, None] if s["gate"] is None else (s["gate"].double()[:, None] if s["gate"].dim() == 2 else s["gate"].double()[None, None])
    (pg, pb), (qg, qb) = pair(s["post"]), pair(s["pre"])
    hat, r = _exact_normed(h, kind) if s["post"] else (h, None)
    n = hat * pg + pb if s["post"] else h
    y = x + RES_SCALE * gate * n
    yhat, yr = _exact_normed(y, kind)
    out = [y] + ([yhat * qg + qb] if s["pre"] else [])
    if case["mode"] == "fwd":
        return out
    dY = s["dy"].double()
    if s["pre"]:
        dz = s["dz"].double()
        dY = dY + _exact_norm_back(dz * qg, yhat, yr, kind)
    dn = RES_SCALE * gate * dY
    out += [dY, _exact_norm_back(dn * pg, hat, r, kind) if s["post"] else dn]
    if s["gate"] is not None:
        dg = RES_SCALE * (n * dY).sum(1)
        out.append(dg if s["gate"].dim() == 2 else dg.sum(0))
    if s["post"]:
        out += [(dn * hat).sum((0, 1))] + ([dn.sum((0, 1))] if s["post"][1] is not None else [])
    if s["pre"]:
        out += [(dz * yhat).sum((0, 1))] + ([dz.sum((0, 1))] if s["pre"][1] is not None else [])
    return out


def _exact_ortho(g):
    """the same polynomial applied to the matrix on its longer side: x (a I + b G + c G^2), G = x^T x of the smaller side"""
    a, b, c = NS_COEFFS
    g = g.double()
    flip = g.shape[0] < g.shape[1]
    x = g.T if flip else g
    x = x / (torch.linalg.matrix_norm(x) + 1e-7)
    for _ in range(5):
        q = x.T @ x
        x = a * x + b * (x @ q) + c * ((x @ q) @ q)
    return x.T if flip else x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adapter":
        return _exact_adapter(s)
    if case["op"] == "norm":
        return _exact_norm(s)
    if case["op"] == "ortho":
        return torch.stack([_exact_ortho(g) for g in s["g"]])
    params, momenta = [], []
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        m = MOMENTUM * m.double() + g.double()
        o = _exact_ortho((g.double() + MOMENTUM * m).flatten(1)).view_as(p)
        params.append((1 - LR * DECAY) * p.double() - LR * 0.2 * math.sqrt(max(p.shape[0], p[0].numel())) * o)
        momenta.append(m)
    return dict(params=params, momenta=momenta)
