"""GPU parity of the fine-tuning operators (low-rank adapters beside a frozen projection, norms around a block with gate and residual
scale, orthogonalised updates) against their formulas in 64 bits.

Tolerances.  A stored 16-bit or 32-bit number is off by half a step, h = eps(type) / 2 relative.  A sum of n products in fp32 is off by at most
n 2^-23 times the sum of the absolute terms (2^-24 per rounding of product and sum).  The pair form of u keeps 2^-17 of each entry."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"


def rand(g, *shape, dtype=FP, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def gen(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def half(t):
    return torch.finfo(t).eps / 2


def near(got, ref, terms, n, extra=0.0):
    """|got - ref| <= h |ref| + (n 2^-23 + extra) terms, elementwise (terms: the sum of the absolute terms of ref)"""
    tol = half(got.dtype) * ref.abs() * 1.001 + (n * 2.0 ** -23 + extra) * terms + torch.finfo(got.dtype).tiny
    off = (got.double() - ref).abs()
    worst = (off / tol).max().item() if off.numel() else 0.0
    assert torch.isfinite(got.double()).all() and worst <= 1.0, worst


# ------------------------------------------------------------------------------------------------ adapters
def adapter_inputs(seed, dtype, shape, N, R, E, ids, residual=False, bias=True, offsets=None):
    g = gen(seed)
    K = shape[-1]
    return dict(x=rand(g, *shape, dtype=dtype), w=rand(g, N, K, dtype=dtype, scale=K ** -0.5), bias=rand(g, N, dtype=dtype, scale=0.1) if bias else None,
                a=rand(g, E, R, K, dtype=dtype, scale=K ** -0.5), b=rand(g, E, N, R, dtype=dtype, scale=R ** -0.5),
                residual=rand(g, *shape[:-1], N, dtype=dtype) if residual else None, ids=torch.tensor(ids, dtype=torch.int32, device=DEV),
                offsets=None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device=DEV), dy=rand(g, *shape[:-1], N, dtype=dtype))


def row_ids(s, M):
    ids = s["ids"].tolist()
    out = torch.full((M,), -1, dtype=torch.long)
    off = s["offsets"].tolist() if s["offsets"] is not None else [i * (M // len(ids)) for i in range(len(ids) + 1)]
    for e, lo, hi in zip(ids, off, off[1:]):
        out[lo:hi] = e if 0 <= e < s["a"].shape[0] else -1
    return out.to(DEV)


def adapter_reference(s, scale):
    """-> {name: (value, sum of absolute terms)} of y, dx, da, db in 64 bits"""
    x, w, a, b, dy = (s[k].double() for k in ("x", "w", "a", "b", "dy"))
    K, N = x.shape[-1], w.shape[0]
    x, dy = x.reshape(-1, K), dy.reshape(-1, N)
    rid = row_ids(s, x.shape[0])

    def parts(x, w, a, b, dy, extra):
        y = x @ w.T + extra
        dx = dy @ w
        da, db = torch.zeros_like(a), torch.zeros_like(b)
        for e in range(a.shape[0]):
            r = (rid == e).nonzero()[:, 0]
            u, du = abs(scale) * x[r] @ a[e].T, abs(scale) * dy[r] @ b[e]
            y[r] += u @ b[e].T
            dx[r] += du @ a[e]
            da[e] = du.T @ x[r]
            db[e] = dy[r].T @ u
        return y, dx, da, db
    add = (s["bias"].double() if s["bias"] is not None else 0) + (s["residual"].double().reshape(-1, N) if s["residual"] is not None else 0)
    sign = math.copysign(1.0, scale)
    value = parts(x, w, a, b * sign, dy, add)
    value = (value[0], value[1], value[2], value[3] * sign)
    size = parts(x.abs(), w.abs(), a.abs(), b.abs(), dy.abs(), add.abs() if torch.is_tensor(add) else 0)
    return {k: (v, t) for k, v, t in zip(("y", "dx", "da", "db"), value, size)}


def check_adapter(s, scale, train):
    from dreammat_amd import hipops
    ref = adapter_reference(s, scale)
    K, N, R = s["x"].shape[-1], s["w"].shape[0], s["a"].shape[1]
    if not train:
        y = hipops.linear_adapted(s["x"], s["w"], s["bias"], s["a"], s["b"], s["ids"], scale, s["residual"], s["offsets"])
        near(y.reshape(-1, N), *ref["y"], K + 2 * R, 2.0 ** -17)
        return y
    x, a, b = (s[k].detach().requires_grad_() for k in ("x", "a", "b"))
    res = None if s["residual"] is None else s["residual"].detach().requires_grad_()
    y = hipops.linear_adapted_autograd(x, s["w"], s["w"].t().contiguous(), s["bias"], a, b, s["ids"], scale, res, s["offsets"])
    leaves = [x, a, b] + ([res] if res is not None else [])
    grads = torch.autograd.grad(y, leaves, s["dy"])
    M = s["x"].numel() // K
    near(y.detach().reshape(-1, N), *ref["y"], K + 2 * R, 2.0 ** -17)
    near(grads[0].reshape(-1, K), *ref["dx"], N + 2 * R, 2.0 ** -17)
    near(grads[1], *ref["da"], M + N, 2.0 ** -17)
    near(grads[2], *ref["db"], M + K, 2.0 ** -17)
    if res is not None:
        assert torch.equal(grads[3], s["dy"])
    return [y.detach()] + list(grads)


ADAPTER_CASES = [
    # shape of x, N, R, E, ids, residual, bias, offsets
    ((1, 64), 64, 16, 1, [0], False, True, None),                                    # one token
    ((16, 256), 80, 4, 5, [i % 6 - 1 for i in range(16)], True, True, None),          # tokens of 16 requests, some without adapter
    ((31, 72), 136, 16, 3, [2], False, False, None),                                  # odd rows, sizes that end inside a tile
    ((3, 77, 64), 200, 12, 4, [3, -1, 3], True, True, None),                          # prompts; the same adapter twice; rank off 8
    ((2, 130, 320), 320, 8, 2, [1, 0], False, True, None),
    ((4, 64, 40), 48, 1, 2, [0, 1, 2, -5], False, True, None),                        # ids outside the adapters; rank 1
    ((513, 96), 264, 64, 3, [0, 1, 2, 0], True, True, [0, 5, 5, 300, 500]),           # ragged, an empty request, a tail
    ((200, 128), 128, 33, 2, [1, 0], False, True, [20, 100, 180]),                    # rows before the first request
    ((300, 64), 72, 128, 2, [0, 1, 0], False, False, [0, 100, 101, 300]),             # the largest rank
    ((150, 64), 64, 5, 40, [(7 * i) % 40 for i in range(150)], False, True, None),     # a row each, many adapters
    ((1, 640), 1280, 16, 9, [8], False, True, None),
    ((2, 1024, 64), 64, 16, 2, [-1, -1], False, True, None),                          # nobody has an adapter
    ((300, 512), 1024, 33, 8, [7, 0, 1, 2, 9, 3, 4, 5, 6, 1], False, True, [0, 3, 60, 61, 61, 100, 170, 200, 230, 290, 299]),      # wide, few rows each
    ((1500, 64), 64, 4, 1100, [(37 * i) % 1101 for i in range(1500)], False, True, None),      # more than 1024 adapters and requests
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", range(len(ADAPTER_CASES)))
def test_linear_adapted_against_64_bits(case, dtype):
    shape, N, R, E, ids, residual, bias, offsets = ADAPTER_CASES[case]
    s = adapter_inputs(case, dtype, shape, N, R, E, ids, residual, bias, offsets)
    check_adapter(s, 0.75, False)
    check_adapter(s, -1.5, True)


def test_linear_adapted_forward_same_with_and_without_autograd_buffers():
    from dreammat_amd import hipops
    s = adapter_inputs(3, BF, (300, 128), 192, 16, 3, [0, 2, 1], True, True, [0, 100, 130, 290])
    y = hipops.linear_adapted(s["x"], s["w"], s["bias"], s["a"], s["b"], s["ids"], 1.0, s["residual"], s["offsets"])
    z = hipops.linear_adapted_autograd(s["x"], s["w"], s["w"].t().contiguous(), s["bias"], s["a"].requires_grad_(), s["b"], s["ids"], 1.0, s["residual"], s["offsets"])
    assert torch.equal(y, z.detach())


def test_linear_adapted_keeps_other_adapters_infinities_out():
    """an adapter full of infinities and NaN next to a finite one in the same tile, and rows without adapter"""
    from dreammat_amd import hipops
    for rows in (24, 384):                                                   # the single-token path and the tiled one
        s = adapter_inputs(5, BF, (rows, 64), 64, 16, 3, [0, 1, -1, 2], True)
        clean = hipops.linear_adapted(s["x"], s["w"], s["bias"], s["a"], s["b"], s["ids"], 1.0, s["residual"])
        s["a"][1], s["b"][1] = float("inf"), float("nan")
        got = hipops.linear_adapted(s["x"], s["w"], s["bias"], s["a"], s["b"], s["ids"], 1.0, s["residual"])
        q = rows // 4
        mine = torch.ones(rows, dtype=torch.bool, device=DEV)
        mine[q:2 * q] = False
        assert torch.equal(got[mine], clean[mine])
        assert not torch.isfinite(got[q:2 * q].float()).any()


def test_linear_adapted_of_millions_of_single_rows():
    """more rows with an adapter each than one grid has workgroups"""
    from dreammat_amd import hipops
    M = (1 << 22) + 77
    g = gen(11)
    x, w, a, b = rand(g, M, 8, dtype=BF), rand(g, 8, 8, dtype=BF), rand(g, 5, 16, 8, dtype=BF), rand(g, 5, 8, 16, dtype=BF)
    ids = torch.randint(-1, 5, (M,), generator=g, device=DEV, dtype=torch.int32)
    y = hipops.linear_adapted(x, w, None, a, b, ids)
    at = torch.cat([torch.arange(0, 300), torch.arange((1 << 20) - 100, (1 << 20) + 100), torch.arange((1 << 21) - 5, (1 << 21) + 200), torch.arange(M - 300, M)]).to(DEV)
    xs, e = x[at].double(), ids[at].long()
    low = [torch.where((e >= 0)[:, None], torch.matmul(torch.matmul(v.unsqueeze(1), p[e.clamp(min=0)].mT.contiguous()), q[e.clamp(min=0)].mT.contiguous())[:, 0], 0.0)
           for v, p, q in ((xs, a.double(), b.double()), (xs.abs(), a.double().abs(), b.double().abs()))]
    near(y[at], xs @ w.double().T + low[0], xs.abs() @ w.double().abs().T + low[1], 8 + 16 + 16, 2.0 ** -17)


@pytest.mark.parametrize("size", [1e-6, 1e4])
def test_linear_adapted_half_range_of_the_low_rank_factor(size):
    """u = x A^T far outside and far below half's range, B the other way round: the pair keeps its bits (row scales)"""
    s = adapter_inputs(6, HF, (96, 64), 64, 16, 2, [0, 1], False, False)
    s["a"] = (s["a"].float() * (size if size > 1 else size * 100)).to(HF)
    s["b"] = (s["b"].float() / (size if size > 1 else 1)).to(HF)
    check_adapter(s, 1.0, False)
    s["dy"] = (s["dy"].float() * 1e-2).to(HF)
    check_adapter(s, 16.0 if size > 1 else 1024.0, False)


def test_linear_adapted_strided_and_unaligned_inputs():
    from dreammat_amd import hipops
    g = gen(8)
    wide = rand(g, 100, 3 * 64, dtype=BF)
    s = adapter_inputs(8, BF, (100, 64), 64, 16, 2, [0, 1], True)
    off = torch.zeros(64 * 64 + 1, dtype=BF, device=DEV)
    w = off[1:].view(64, 64).copy_(s["w"])                                    # two bytes off a 16-byte boundary
    a = hipops.linear_adapted(wide[:, 64:128], w, s["bias"], s["a"], s["b"].transpose(1, 2).contiguous().transpose(1, 2), s["ids"], 1.0, s["residual"])
    b = hipops.linear_adapted(wide[:, 64:128].contiguous(), s["w"], s["bias"], s["a"], s["b"], s["ids"], 1.0, s["residual"])
    assert torch.equal(a, b)


def test_linear_adapted_same_bits_every_run():
    s = adapter_inputs(9, BF, (4, 500, 64), 128, 16, 3, [2, 0, 2, 1])
    one, two = check_adapter(s, 1.0, True), check_adapter(s, 1.0, True)
    assert all(torch.equal(p, q) for p, q in zip(one, two))


def test_linear_adapted_gradients_only_where_wanted():
    from dreammat_amd import hipops
    s = adapter_inputs(10, BF, (200, 64), 72, 16, 2, [0, 1])
    full = check_adapter(s, 1.0, True)
    for need in ((0,), (1,), (2,), (0, 2), (1, 2)):
        v = [s[k].detach().requires_grad_(i in need) for i, k in enumerate(("x", "a", "b"))]
        y = hipops.linear_adapted_autograd(v[0], s["w"], s["w"].t().contiguous(), s["bias"], v[1], v[2], s["ids"])
        grads = torch.autograd.grad(y, [v[i] for i in need], s["dy"])
        assert all(torch.equal(p, full[1 + i]) for p, i in zip(grads, need))


def test_linear_adapted_empty_batch():
    from dreammat_amd import hipops
    s = adapter_inputs(11, BF, (0, 64), 64, 16, 2, [0, 1])
    assert hipops.linear_adapted(s["x"], s["w"], s["bias"], s["a"], s["b"], s["ids"]).shape == (0, 64)
    a = s["a"].requires_grad_()
    y = hipops.linear_adapted_autograd(s["x"].requires_grad_(), s["w"], s["w"].t().contiguous(), s["bias"], a, s["b"], s["ids"])
    assert not torch.autograd.grad(y.sum(), a)[0].any()


def test_linear_adapted_gradient_against_differences():
    """central differences of a scalar of y along random directions of x, A and B.  The loss is bilinear in (A, B) and linear in x along each
    direction alone, so the difference quotient is exact up to rounding of y: 2 h |dy|.|y| / (2 t) of the quotient"""
    from dreammat_amd import hipops
    s = adapter_inputs(12, HF, (3, 20, 64), 64, 8, 2, [1, 0, 1])
    x, a, b = (s[k].detach().requires_grad_() for k in ("x", "a", "b"))
    y = hipops.linear_adapted_autograd(x, s["w"], s["w"].t().contiguous(), s["bias"], a, b, s["ids"])
    grads = torch.autograd.grad(y, (x, a, b), s["dy"])
    f = lambda x, a, b: hipops.linear_adapted(x, s["w"], s["bias"], a, b, s["ids"])
    for i, v in enumerate((x, a, b)):
        d = torch.sign(rand(gen(20 + i), *v.shape)) * 2.0 ** -3 * v.detach().float().abs().clamp(min=2.0 ** -6)
        up, down = (v.detach().float() + d).to(HF), (v.detach().float() - d).to(HF)
        args = [x.detach(), a.detach(), b.detach()]
        yu, yd = f(*args[:i], up, *args[i + 1:]), f(*args[:i], down, *args[i + 1:])
        quotient = (s["dy"].double() * (yu.double() - yd.double())).sum()
        slope = (grads[i].double() * (up.double() - down.double())).sum()
        tol = half(HF) * (s["dy"].double().abs() * (yu.double().abs() + yd.double().abs())).sum() + half(HF) * (grads[i].double() * (up.double() - down.double())).abs().sum()
        assert (quotient - slope).abs() <= tol


# ------------------------------------------------------------------------------------------------ norms
def norm_inputs(seed, dtype, shape, gate, post, pre):
    g = gen(seed)
    C = shape[-1]
    p = lambda q: None if q is None else tuple(rand(g, C, dtype=dtype, scale=0.2).add_(1 - i) if on else None for i, on in enumerate(q))
    return dict(x=rand(g, *shape, dtype=dtype), h=rand(g, *shape, dtype=dtype).add_(0.25), gate={None: None, "channel": rand(g, C, dtype=dtype), "item": rand(g, shape[0], C, dtype=dtype)}[gate],
                post=p(post), pre=p(pre), dy=rand(g, *shape, dtype=dtype), dz=rand(g, *shape, dtype=dtype))


def norm_formula(x, h, gate, pg, pb, qg, qb, post, pre, scale, eps, kind):
    def norm(v, ga, be):
        mu = v.mean(-1, keepdim=True) if kind == "layer" else 0
        v = (v - mu) / torch.sqrt(((v - mu) ** 2).mean(-1, keepdim=True) + eps)
        v = v if ga is None else v * ga
        return v if be is None else v + be
    n = norm(h, pg, pb) if post else h
    if gate is not None:
        n = n * (gate.view(gate.shape[0], *[1] * (x.dim() - 2), -1) if gate.dim() == 2 and x.dim() > 2 else gate)
    y = x + scale * n
    return (y, norm(y, qg, qb)) if pre else (y,)


def check_norm(s, kind, scale=0.8, eps=1e-5):
    """value and gradients against 64 bits.  Bound of an output of a row: every quantity of a row is a fixed chain of sums of C terms, (4 C + 64)
    2^-23 of the row's largest absolute value where the norm does not amplify (rstd = O(1) here); of a column sum: n rows more"""
    from dreammat_amd import hipops
    post, pre = s["post"] is not None, s["pre"] is not None
    flat = [s["x"], s["h"], s["gate"], *(s["post"] or (None, None)), *(s["pre"] or (None, None))]
    mine = [None if t is None else t.detach().requires_grad_() for t in flat]
    out = hipops.gated_add_norm(*mine[:3], post=tuple(mine[3:5]) if post else None, pre=tuple(mine[5:7]) if pre else None, scale=scale, eps=eps, kind=kind)
    out = out if isinstance(out, tuple) else (out,)
    with torch.no_grad():
        plain = hipops.gated_add_norm(*flat[:3], post=s["post"], pre=s["pre"], scale=scale, eps=eps, kind=kind)
    assert all(torch.equal(p.detach(), q) for p, q in zip(out, plain if pre else (plain,)))
    exact = [None if t is None else t.double().requires_grad_() for t in flat]
    ref = norm_formula(*exact, post, pre, scale, eps, kind)
    ups = [s["dy"], s["dz"]][:len(out)]
    leaves, xleaves = [t for t in mine if t is not None], [t for t in exact if t is not None]
    got = torch.autograd.grad(out, leaves, ups)
    want = torch.autograd.grad(ref, xleaves, [u.double() for u in ups])
    C, rows = s["x"].shape[-1], s["x"].numel() // s["x"].shape[-1]
    for o, r in zip(out, ref):
        near(o.detach(), r.detach(), r.detach().abs().amax(-1, keepdim=True).clamp(min=1), 4 * C + 64)
    for q, r in zip(got, want):
        if q.shape == s["x"].shape:
            near(q, r, r.abs().amax(-1, keepdim=True).clamp(min=1), 4 * C + 64)
        else:
            # a column sum: the rows' terms are O(10) here; their own errors (above) and the sum's
            near(q, r, torch.full_like(r, 10.0 * math.sqrt(rows) + 10.0), 4 * C + 64 + rows)
    return list(out) + list(got)


NORM_CASES = [
    # shape, gate, post (gamma, beta), pre, kind
    ((1, 8), None, (1, 1), (1, 1), "layer"),
    ((1, 1, 64), "item", (1, 1), (1, 1), "layer"),
    ((2, 77, 320), "item", (1, 1), (1, 1), "layer"),
    ((3, 5, 640), "channel", None, (1, 1), "layer"),
    ((50, 1280), None, (1, 0), (1, 0), "rms"),
    ((7, 33, 100), "item", (1, 1), None, "layer"),                         # rows that are not whole 16-byte chunks
    ((13, 1), "channel", (1, 1), None, "rms"),                              # one channel
    ((4, 3, 2, 257), "item", (0, 0), (0, 1), "layer"),                      # norms without gamma
    ((2, 30, 2048), "channel", (1, 1), (1, 1), "layer"),
    ((5, 4096), "item", (1, 1), (1, 1), "rms"),
    ((3, 8192), None, (1, 1), (1, 1), "layer"),
    ((3, 8191), "channel", (1, 1), (1, 1), "layer"),
    ((600, 3, 40), "item", None, None, "layer"),                            # several items per workgroup, no norm at all
    ((2, 1500, 96), "item", (1, 1), (1, 1), "rms"),                         # an item over several workgroups
    ((1100, 136), "item", (1, 1), (1, 1), "layer"),                         # an item per row
]


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("case", range(len(NORM_CASES)))
def test_gated_add_norm_against_64_bits(case, dtype):
    shape, gate, post, pre, kind = NORM_CASES[case]
    check_norm(norm_inputs(case, dtype, shape, gate, post, pre), kind)


def test_gated_add_norm_constant_rows_and_large_means():
    """rows without variance come out as beta (eps decides), a mean of 1000 does not cost the variance its bits"""
    from dreammat_amd import hipops
    h = torch.full((4, 64), 3.0, device=DEV)
    be = rand(gen(1), 64)
    y = hipops.gated_add_norm(torch.zeros_like(h), h, post=(torch.ones(64, device=DEV), be))
    assert torch.equal(y, be.expand_as(y))
    h = rand(gen(2), 8, 640) + 1000.0
    y = hipops.gated_add_norm(torch.zeros_like(h), h, post=(None, None))
    ref = torch.nn.functional.layer_norm(h.double(), (640,))
    # the mean of fp32 numbers near 1000 is off by 640 roundings at most (2^-24 1000 each); rstd = 1
    assert (y - ref).abs().max() <= 2 * 640 * 2.0 ** -24 * 1000


def test_gated_add_norm_infinite_rows_stay_rows():
    from dreammat_amd import hipops
    s = norm_inputs(3, BF, (40, 64), None, (1, 1), (1, 1))
    y, z = hipops.gated_add_norm(s["x"], s["h"], None, s["post"], s["pre"])
    s["h"][7] = float("inf")
    s["x"][9, 3] = float("nan")
    y2, z2 = hipops.gated_add_norm(s["x"], s["h"], None, s["post"], s["pre"])
    keep = torch.ones(40, dtype=torch.bool, device=DEV)
    keep[7] = keep[9] = False
    assert torch.equal(y[keep], y2[keep]) and torch.equal(z[keep], z2[keep])
    assert torch.isnan(z2[7].float()).all() and torch.isnan(z2[9].float()).all()


def test_gated_add_norm_strided_inputs_and_same_bits():
    from dreammat_amd import hipops
    s = norm_inputs(4, BF, (2, 60, 96), "item", (1, 1), (1, 1))
    one = check_norm(s, "layer")
    t = dict(s, x=s["x"].transpose(0, 1).contiguous().transpose(0, 1), h=torch.cat([s["h"], s["h"]], -1)[..., 96:], gate=torch.cat([s["gate"], s["gate"]], -1)[:, 96:])
    two = check_norm(t, "layer")
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    # 2 bytes off a 16-byte boundary: element by element, the same sums in another order
    off = torch.empty(s["x"].numel() + 1, dtype=BF, device=DEV)[1:].view(s["x"].shape).copy_(s["x"])
    check_norm(dict(s, x=off), "layer")


def test_gated_add_norm_one_output_used():
    """only z (or only y) of the two outputs reaches the loss"""
    from dreammat_amd import hipops
    s = norm_inputs(5, FP, (3, 17, 64), "channel", (1, 1), (1, 1))
    x = s["x"].clone().requires_grad_()
    for which in (0, 1):
        out = hipops.gated_add_norm(x, s["h"], s["gate"], s["post"], s["pre"])
        (g,) = torch.autograd.grad(out[which], x, s["dy"])
        xd = s["x"].double().requires_grad_()
        ref = norm_formula(xd, s["h"].double(), s["gate"].double(), *[t.double() for t in s["post"] + s["pre"]], True, True, 1.0, 1e-5, "layer")
        (r,) = torch.autograd.grad(ref[which], xd, s["dy"].double())
        near(g, r, r.abs().amax(-1, keepdim=True).clamp(min=1), 4 * 64 + 64)


def test_gated_add_norm_no_rows():
    from dreammat_amd import hipops
    x = torch.zeros(0, 64, device=DEV, requires_grad=True)
    ga = torch.ones(64, device=DEV, requires_grad=True)
    y, z = hipops.gated_add_norm(x, x.detach(), None, (ga, None), (None, None))
    assert y.shape == z.shape == (0, 64)
    assert not torch.autograd.grad((y.sum() + z.sum()), ga)[0].any()


# ------------------------------------------------------------------------------------------------ orthogonalised updates
def ns_formula(g, steps=5, eps=1e-7):
    a, b, c = 3.4445, -4.7750, 2.0315
    x = g.double()
    flip = x.shape[-2] > x.shape[-1]
    x = x.mT if flip else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        s = x @ x.mT
        x = a * x + (b * s + c * s @ s) @ x
    return x.mT if flip else x


# Three stored matrices per step (X, S, P), each off by 2^-22 (pairs) or 2^-12 (values), and noise that enters at step k is amplified by at most
# a^(6 - k) = 3.4445^(6 - k): 485 141 41 12 3.4 for the five steps.
AMPLIFY = [3.4445 ** k for k in (5, 4, 3, 2, 1)]
NS_TOL = {FP: 3 * 2.0 ** -22 * sum(AMPLIFY), HF: 3 * 2.0 ** -22 * sum(AMPLIFY) + half(HF),
          BF: 3 * (2.0 ** -22 * sum(AMPLIFY[:3]) + 2.0 ** -12 * sum(AMPLIFY[3:])) + half(BF)}


def rel(x, y):
    return ((x.double() - y).norm() / y.norm()).item()


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("shape", [(1, 1), (1, 40), (37, 1), (16, 16), (64, 64), (5, 100, 30), (65, 64), (2, 3, 64, 129), (200, 513), (320, 320), (3, 384, 640), (17, 40, 24)])
def test_orthogonalize_against_64_bits(shape, dtype):
    from dreammat_amd import hipops
    g = rand(gen(sum(shape)), *shape, dtype=dtype, scale=1e-3)
    got, ref = hipops.orthogonalize(g), ns_formula(g)
    assert got.dtype == dtype and got.shape == g.shape
    for p, q in zip(got.reshape(-1, *shape[-2:]), ref.reshape(-1, *shape[-2:])):
        assert rel(p, q) <= NS_TOL[dtype]


@pytest.mark.parametrize("steps", [1, 2, 7])
def test_orthogonalize_step_counts_and_scales(steps):
    from dreammat_amd import hipops
    tol = 3 * 2.0 ** -22 * sum(3.4445 ** k for k in range(1, steps + 1))
    for size in (1e-20, 1.0, 1e30):                                       # |g|^2 leaves fp32's range both ways
        g = rand(gen(steps), 96, 160) * size
        assert rel(hipops.orthogonalize(g, steps=steps, eps=0.0), ns_formula(g, steps, 0.0)) <= tol


def test_orthogonalize_makes_singular_values_near_one_and_handles_zero():
    from dreammat_amd import hipops
    s = torch.linalg.svdvals(hipops.orthogonalize(rand(gen(3), 128, 300)).double())
    # a Gaussian's singular values start above 1e-2 of its norm: 3.4445^5 1e-2 > 0.6, and the quintic keeps (0.6, 1.2) in (0.6, 1.2)
    assert s.min() > 0.6 and s.max() < 1.25
    z = torch.zeros(3, 40, 70, device=DEV, dtype=BF)
    z[1] = 1
    o = hipops.orthogonalize(z)
    assert not o[0].any() and not o[2].any() and torch.isfinite(o.float()).all()
    assert rel(o[1], ns_formula(z[1])) <= NS_TOL[BF]
    z[1, 0, 0] = float("inf")
    o = hipops.orthogonalize(z)
    assert not o[0].any() and not torch.isfinite(o[1].float()).any()


def test_orthogonalize_strided_and_same_bits():
    from dreammat_amd import hipops
    g = rand(gen(4), 100, 60)
    one = hipops.orthogonalize(g)
    assert torch.equal(one, hipops.orthogonalize(torch.cat([g, g], 1)[:, 60:]))
    assert torch.equal(one, hipops.orthogonalize(torch.stack([g, g + 1]))[0])


@pytest.mark.parametrize("gdtype", [FP, BF])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step_against_64_bits(nesterov, gdtype):
    from dreammat_amd import hipops
    g = gen(7)
    shapes = [(64, 64), (40, 24, 3, 3), (64, 64), (128, 30), (24, 200), (64, 64)]
    p, m = ([rand(g, *q, scale=c) for q in shapes] for c in (0.02, 1e-3))
    gr = [rand(g, *q, dtype=gdtype, scale=1e-3) for q in shapes]
    lr, wd, mu = 0.02, 0.1, 0.9
    want = []
    for a, b, c in zip(p, m, gr):
        mm = mu * b.double() + c.double()
        o = ns_formula((c.double() + mu * mm if nesterov else mm).flatten(1)).view(a.shape)
        s = 0.2 * math.sqrt(max(a.shape[0], a[0].numel()))
        want.append((a.double() * (1 - lr * wd) - lr * s * o, mm, lr * s * o))
    versions = [q._version for q in p + m]
    assert hipops.muon_step(p, gr, m, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd) is None
    assert all(q._version > v for q, v in zip(p + m, versions))
    tol = NS_TOL[gdtype if gdtype != BF else BF]
    for a, b, (pa, mm, up) in zip(p, m, want):
        assert (b.double() - mm).abs().max() <= 3 * 2.0 ** -24 * 8e-3
        assert (a.double() - pa).norm() <= tol * up.norm() + 3 * 2.0 ** -24 * pa.norm()


def test_muon_step_groups_of_many_matrices_equal_single_ones():
    from dreammat_amd import hipops
    g = gen(8)
    p, m, gr = ([rand(g, 48, 72, scale=c) for _ in range(19)] for c in (0.02, 1e-3, 1e-3))
    p2, m2 = [q.clone() for q in p], [q.clone() for q in m]
    hipops.muon_step(p, gr, m, lr=0.1, scale="spectral")
    for a, b, c in zip(p2, gr, m2):
        hipops.muon_step([a], [b], [c], lr=0.1, scale="spectral")
    assert all(torch.equal(a, b) for a, b in zip(p + m, p2 + m2))


@pytest.mark.parametrize("shapes", [
    [(192, 5000), (130, 2100), (64, 64)],                                                                # few tiles: the Gram contraction in shares
    [(1024, 1100), (640, 5120), (2560, 300), (1024, 1100), (70, 9000), (1024, 1100), (33, 33)],          # classes of one and of three
    [(320 + 64 * (i % 5), 200 + 37 * i) for i in range(19)],                                             # two groups
    [(1280, 1280)] * 9 + [(1280, 4000)]])                                                                # whole rounds of the largest tiles
def test_muon_step_of_many_shapes_at_once_against_64_bits(shapes):
    from dreammat_amd import hipops
    g = gen(len(shapes))
    p, m = ([rand(g, *q, scale=c) for q in shapes] for c in (0.02, 1e-3))
    gr = [rand(g, *q, scale=1e-3) for q in shapes]
    want = []
    for a, b, c in zip(p, m, gr):
        mm = 0.9 * b.double() + c.double()
        up = 0.1 * 0.2 * max(a.shape) ** 0.5 * ns_formula(c.double() + 0.9 * mm)
        want.append((a.double() * (1 - 0.1 * 0.02) - up, mm, up))
    state = [q.clone() for q in p + m]
    hipops.muon_step(p, gr, m, lr=0.1, momentum=0.9, weight_decay=0.02)
    for a, b, (pa, mm, up) in zip(p, m, want):
        assert (b.double() - mm).abs().max() <= 3 * 2.0 ** -24 * 8e-3
        assert (a.double() - pa).norm() <= NS_TOL[FP] * up.norm() + 3 * 2.0 ** -24 * pa.norm()
    n = len(shapes)
    hipops.muon_step(state[:n], gr, state[n:], lr=0.1, momentum=0.9, weight_decay=0.02)
    assert all(torch.equal(a, b) for a, b in zip(p + m, state))                  # no atomics: the same bits


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("shape", [(128, 320), (640, 320)])
def test_orthogonalize_of_a_few_strong_directions(shape, dtype):
    """three directions a thousand times the others, as gradients have them: the weak ones are what the iteration amplifies most"""
    from dreammat_amd import hipops
    g = gen(9)
    u = (rand(g, shape[0], 3) @ rand(g, 3, shape[1]) + 1e-3 * rand(g, *shape)).to(dtype)
    assert rel(hipops.orthogonalize(u), ns_formula(u)) <= NS_TOL[dtype]


# ------------------------------------------------------------------------------------------------ together
def block(hipops, s, w, wt, leaves, ids):
    """x + gate norm(adapted projection of norm(x)): the three operators as a fine-tuned branch uses them"""
    a, b, gate, pg, qg = leaves
    zeros = torch.zeros_like(s)
    _, z = hipops.gated_add_norm(s, zeros, None, None, (qg, None))
    h = hipops.linear_adapted_autograd(z, w, wt, None, a, b, ids)
    return hipops.gated_add_norm(s, h, gate, (pg, None), None, scale=0.5)


def block_inputs(seed, B=3, S=50, C=128, R=8, E=2, dtype=BF):
    g = gen(seed)
    x, w = rand(g, B, S, C, dtype=dtype), rand(g, C, C, dtype=dtype, scale=C ** -0.5)
    leaves = [rand(g, E, R, C, dtype=dtype, scale=C ** -0.5), rand(g, E, C, R, dtype=dtype, scale=0.3), rand(g, C, dtype=dtype),
              torch.ones(C, device=DEV, dtype=dtype), torch.ones(C, device=DEV, dtype=dtype)]
    return x, w, w.t().contiguous(), [t.requires_grad_() for t in leaves], torch.tensor([0, 1, 0], dtype=torch.int32, device=DEV), rand(g, B, S, C, dtype=dtype)


def test_adapted_gated_block_and_its_update():
    """forward, all gradients against 64-bit autograd, then a Muon step on the adapters' fp32 masters"""
    from dreammat_amd import hipops
    x, w, wt, leaves, ids, dy = block_inputs(1)
    y = block(hipops, x, w, wt, leaves, ids)
    grads = torch.autograd.grad(y, leaves, dy)
    xd, wd = x.double(), w.double()
    a, b, gate, pg, qg = (t.detach().double().requires_grad_() for t in leaves)
    _, z = norm_formula(xd, torch.zeros_like(xd), None, None, None, qg, None, False, True, 1.0, 1e-5, "layer")
    h = z @ wd.T + torch.stack([(z[i] @ a[e].T) @ b[e].T for i, e in enumerate(ids.tolist())])
    (ref,) = norm_formula(xd, h, gate, pg, None, None, None, True, False, 0.5, 1e-5, "layer")
    want = torch.autograd.grad(ref, (a, b, gate, pg, qg), dy.double())
    # bf16 z, h and their gradients each carry half a step; the sums over 150 rows average it: a few half steps of the norm
    assert rel(y.detach(), ref.detach()) <= 4 * half(BF)
    for q, r in zip(grads, want):
        assert rel(q, r) <= 8 * half(BF)
    master = [[t for t in leaf.detach().float()] for leaf in leaves[:2]]
    for leaf, gr, ms in zip(leaves, grads, master):
        before = [t.clone() for t in ms]
        hipops.muon_step(ms, list(gr), [torch.zeros_like(t) for t in ms], lr=0.1, momentum=0.9)
        for e, (p, q) in enumerate(zip(ms, before)):
            step = 0.1 * 0.2 * math.sqrt(max(p.shape)) * ns_formula((1 + 0.9) * gr[e].double())
            assert ((q.double() - p.double()) - step).norm() <= NS_TOL[BF] * step.norm() + 2.0 ** -22 * q.norm()


def test_block_captured_in_a_graph_and_replayed():
    """forward, backward and the update in one captured graph; replays on new inputs match the eager run bit for bit"""
    from dreammat_amd import hipops
    x, w, wt, leaves, ids, dy = block_inputs(2)
    p, m = [leaves[0][0].detach().float().clone()], [torch.zeros(8, 128, device=DEV)]

    def step(x, dy, p, m):
        mine = [t.detach().requires_grad_() for t in leaves]
        y = block(hipops, x, w, wt, mine, ids)
        grads = torch.autograd.grad(y, mine, dy)
        hipops.muon_step(p, [grads[0][0]], m, lr=0.05)
        return [y.detach()] + [g for g in grads]
    sx, sdy, sp, sm = x.clone(), dy.clone(), [p[0].clone()], [m[0].clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(sx, sdy, [sp[0].clone()], [sm[0].clone()])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sx, sdy, sp, sm)
    for k in range(3):
        nx, ndy = rand(gen(30 + k), *x.shape, dtype=BF), rand(gen(40 + k), *x.shape, dtype=BF)
        sx.copy_(nx)
        sdy.copy_(ndy)
        graph.replay()
        torch.cuda.synchronize()
        want = step(nx, ndy, p, m)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert torch.equal(sp[0], p[0]) and torch.equal(sm[0], m[0])


def test_two_captured_graphs_do_not_share_scratch():
    from dreammat_amd import hipops
    g = gen(50)
    ga, gb = rand(g, 100, 140), rand(g, 64, 200)
    graphs, outs = [], []
    for t in (ga, gb):
        hipops.orthogonalize(t)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(hipops.orthogonalize(t))
        graphs.append(graph)
    for order in ((0, 1), (1, 0)):
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], hipops.orthogonalize(ga)) and torch.equal(outs[1], hipops.orthogonalize(gb))


def test_operators_on_a_side_stream():
    from dreammat_amd import hipops
    x, w, wt, leaves, ids, dy = block_inputs(3)
    want = block(hipops, x, w, wt, leaves, ids).detach()
    wo = hipops.orthogonalize(w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x2 = x.clone()
        got, go = block(hipops, x2, w, wt, leaves, ids).detach(), hipops.orthogonalize(w)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(go, wo)


def test_controlnet_trainer_with_orthogonalised_steps():
    """ControlNetTrainer(optimizer="muon"): every matrix master moves by the formula's step (64 bits, from the gradient the trainer used), the others
    by AdamW, the bf16 module holds the rounded masters, and the optimizer's state survives a round trip"""
    from dreammat_amd import controlnet_train as ct
    from dreammat_amd.sd import ARCHS, AutoencoderKLEncoder, UNet2DConditionModel
    torch.manual_seed(0)
    a = ARCHS["tiny"]
    unet, vae = UNet2DConditionModel(a).to(DEV, BF), AutoencoderKLEncoder(a).to(DEV, BF)
    tr = ct.ControlNetTrainer(vae, unet, ct.init_controlnet(unet).to(DEV, BF), lr=1e-3, weight_decay=0.01, max_grad_norm=1e9, optimizer="muon")
    g = gen(60)
    img, cond = rand(g, 2, 3, 64, 64, dtype=BF).clamp(-1, 1), torch.rand(2, 22, 64, 64, generator=g, device=DEV)
    text = rand(g, 2, 77, a.cross_dim, dtype=BF)
    for step in range(2):
        loss = ct.controlnet_training_loss(tr.vae, tr.unet, tr.controlnet, tr.scheduler, img, cond, text, timesteps=torch.tensor([300, 700], device=DEV),
                                           noise=rand(g, 2, 4, 8, 8), posterior_noise=rand(g, 2, 4, 8, 8))
        loss.backward()
        assert torch.isfinite(loss)
        params = tr._params()
        grads = [None if p.grad is None else p.grad.double() for p in params]
        masters = [m.detach().double() for m in tr.master]
        before = [None if m is None else m.double() for m in tr.opt.momenta]
        tr.apply_gradients()
        at = 0
        for p, gr, old, new in zip(params, grads, masters, tr.master):
            assert torch.equal(p, new.to(BF))
            if p.dim() < 2:
                continue
            mom = before[at] if before[at] is not None else torch.zeros_like(gr)
            at += 1
            mom = 0.95 * mom + gr
            u = (gr + 0.95 * mom).flatten(1)
            up = 1e-3 * 0.2 * math.sqrt(max(u.shape)) * ns_formula(u).view(p.shape)
            assert (tr.opt.momenta[at - 1].double() - mom).norm() <= 3 * 2.0 ** -24 * (mom.norm() + gr.norm())
            if not gr.any():
                assert not up.any()
            # (the directions of a real gradient that lie 1e-4 below its norm are amplified in full: the bound of the file's head holds for them too)
            assert (new.detach().double() - (old * (1 - 1e-5) - up)).norm() <= NS_TOL[FP] * up.norm() + 3 * 2.0 ** -24 * old.norm()
    moved = [bool((m.detach() != o.float()).any()) for m, o in zip(tr.master, masters) if m.dim() < 2]
    assert any(moved)
    state = tr.opt.state_dict()
    other = ct.MuonAdamW(tr.master, lr=1e-3)
    other.load_state_dict(state)
    assert all(torch.equal(p, q) for p, q in zip(other.momenta, tr.opt.momenta))


def test_controlnet_launcher_with_orthogonalised_steps(tmp_path):
    from dreammat_amd import controlnet_train as ct
    from tests.test_nets_cpu import _tiny_render_tree
    _tiny_render_tree(tmp_path / "data", tmp_path / "prompts.json")
    tr = ct.main(["--synthetic", "--pretrained_model_name_or_path", "tiny", "--train_data_dir", str(tmp_path / "data"), "--prompt_file",
                  str(tmp_path / "prompts.json"), "--resolution", "64", "--train_batch_size", "2", "--max_train_steps", "2", "--output_dir",
                  str(tmp_path / "out"), "--checkpointing_steps", "2", "--optimizer", "muon"])
    assert tr.global_step == 2 and isinstance(tr.opt, ct.MuonAdamW) and all(torch.isfinite(m).all() for m in tr.master)
