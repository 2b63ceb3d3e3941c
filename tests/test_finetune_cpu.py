"""Refusals of the fine-tuning operators (CPU: every check comes before the first launch) and the size queries of their C entries."""
import pytest
import torch

from dreammat_amd import _lib, hipops

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def adapter(**kw):
    v = dict(x=torch.zeros(4, 6, 64, dtype=BF), w=torch.zeros(72, 64, dtype=BF), bias=torch.zeros(72, dtype=BF), lora_a=torch.zeros(3, 16, 64, dtype=BF),
             lora_b=torch.zeros(3, 72, 16, dtype=BF), ids=torch.zeros(4, dtype=torch.int32))
    v.update(kw)
    return v


BAD_ADAPTER = [
    (TypeError, dict(x=torch.zeros(4, 6, 64))),
    (TypeError, dict(w=torch.zeros(72, 64, dtype=HF))),
    (TypeError, dict(bias=torch.zeros(72))),
    (TypeError, dict(residual=torch.zeros(4, 6, 72, dtype=HF))),
    (ValueError, dict(x=torch.zeros(4, 6, 32, dtype=BF))),
    (ValueError, dict(w=torch.zeros(72 * 64, dtype=BF))),
    (ValueError, dict(lora_b=torch.zeros(3, 72, 8, dtype=BF))),
    (ValueError, dict(lora_b=torch.zeros(2, 72, 16, dtype=BF))),
    (ValueError, dict(lora_a=torch.zeros(3, 129, 64, dtype=BF), lora_b=torch.zeros(3, 72, 129, dtype=BF))),
    (ValueError, dict(lora_a=torch.zeros(3, 0, 64, dtype=BF), lora_b=torch.zeros(3, 72, 0, dtype=BF))),
    (ValueError, dict(lora_a=torch.zeros(0, 16, 64, dtype=BF), lora_b=torch.zeros(0, 72, 16, dtype=BF))),
    (ValueError, dict(w=torch.zeros(70, 64, dtype=BF), bias=None, lora_b=torch.zeros(3, 70, 16, dtype=BF))),
    (ValueError, dict(bias=torch.zeros(64, dtype=BF))),
    (ValueError, dict(ids=torch.zeros(4, dtype=torch.int64))),
    (ValueError, dict(ids=torch.zeros(0, dtype=torch.int32))),
    (ValueError, dict(ids=torch.zeros(2, 2, dtype=torch.int32))),
    (ValueError, dict(ids=torch.zeros(5, dtype=torch.int32))),                       # 24 rows are not 5 equal requests
    (ValueError, dict(offsets=torch.zeros(4, dtype=torch.int32))),
    (ValueError, dict(offsets=torch.zeros(5, dtype=torch.int64))),
    (ValueError, dict(residual=torch.zeros(24, 72, dtype=BF))),
    (_lib.DmError, dict()),                                                          # all right, but on the CPU
]


@pytest.mark.parametrize("case", range(len(BAD_ADAPTER)))
def test_linear_adapted_refuses(case):
    error, change = BAD_ADAPTER[case]
    v = adapter(**change)
    with pytest.raises(error):
        hipops.linear_adapted(**v)
    if v["w"].dim() == 2:
        with pytest.raises(error):
            hipops.linear_adapted_autograd(w_t=v["w"].t().contiguous(), **v)


def test_linear_adapted_autograd_refuses_a_trainable_projection_and_a_foreign_transpose():
    v = adapter()
    with pytest.raises(ValueError):
        hipops.linear_adapted_autograd(w_t=v["w"], **v)
    with pytest.raises(ValueError):
        hipops.linear_adapted_autograd(w_t=v["w"].t().contiguous(), **adapter(w=torch.zeros(72, 64, dtype=BF, requires_grad=True)))
    with pytest.raises(ValueError):
        hipops.linear_adapted_autograd(w_t=v["w"].t().contiguous(), **adapter(bias=torch.zeros(72, dtype=BF, requires_grad=True)))
    with pytest.raises(ValueError, match="trained together"):
        hipops.linear_adapted_autograd(w_t=v["w"].t().contiguous(), **adapter(lora_a=torch.zeros(60001, 1, 64, dtype=BF), lora_b=torch.zeros(60001, 72, 1, dtype=BF)))


ONE = torch.ones(64)
BAD_NORM = [
    (TypeError, dict(x=torch.zeros(3, 64, dtype=torch.float64), h=torch.zeros(3, 64, dtype=torch.float64))),
    (TypeError, dict(h=torch.zeros(2, 3, 64, dtype=BF))),
    (TypeError, dict(post=(ONE.to(BF), None))),
    (TypeError, dict(gate=ONE.to(HF))),
    (ValueError, dict(h=torch.zeros(2, 4, 64))),
    (ValueError, dict(kind="batch")),
    (ValueError, dict(gate=torch.ones(3, 64))),
    (ValueError, dict(gate=torch.ones(2, 1, 64))),
    (ValueError, dict(gate=torch.ones(32))),
    (ValueError, dict(post=ONE)),
    (ValueError, dict(pre=(ONE, torch.ones(32)))),
    (ValueError, dict(pre=(ONE, ONE, ONE))),
    (ValueError, dict(x=torch.zeros(2, 8193), h=torch.zeros(2, 8193))),
    (ValueError, dict(x=torch.zeros(2, 0), h=torch.zeros(2, 0))),
    (ValueError, dict(x=torch.zeros(65001, 1), h=torch.zeros(65001, 1), gate=torch.zeros(65001, 1))),
    (_lib.DmError, dict()),
]


@pytest.mark.parametrize("case", range(len(BAD_NORM)))
def test_gated_add_norm_refuses(case):
    error, change = BAD_NORM[case]
    v = dict(x=torch.zeros(2, 3, 64), h=torch.zeros(2, 3, 64))
    v.update(change)
    with pytest.raises(error):
        hipops.gated_add_norm(**v)


def test_orthogonalize_refuses():
    for error, g, kw in [(ValueError, torch.zeros(4), {}), (ValueError, torch.zeros(4, 4, dtype=torch.float64), {}), (ValueError, torch.zeros(4, 4), dict(steps=0)),
                         (ValueError, torch.zeros(4, 4), dict(steps=65)), (ValueError, torch.empty(1, 1, device="meta").expand(40000, 40000), {}),
                         (_lib.DmError, torch.zeros(4, 4), {})]:
        with pytest.raises(error):
            hipops.orthogonalize(g, **kw)


def test_muon_step_refuses():
    z = lambda *s, **k: torch.zeros(*s, **k)
    p, g, m = z(4, 6), z(4, 6), z(4, 6)
    for error, args, kw in [
            (ValueError, ([p], [g, g], [m]), {}), (ValueError, ([z(4)], [z(4)], [z(4)]), {}), (TypeError, ([p.to(BF)], [g], [m]), {}),
            (TypeError, ([p], [g], [m.to(BF)]), {}), (TypeError, ([p], [g.double()], [m]), {}), (ValueError, ([p], [z(6, 4)], [m]), {}),
            (ValueError, ([p], [g], [z(4, 7)]), {}), (ValueError, ([z(6, 4).t()], [g], [m]), {}), (ValueError, ([p, p], [g, g], [m, z(4, 6)]), {}),
            (ValueError, ([p], [g], [p]), {}), (ValueError, ([p], [g], [m]), dict(steps=0)), (ValueError, ([p], [g], [m]), dict(scale="none")),
            (_lib.DmError, ([p], [g], [m]), {})]:
        with pytest.raises(error):
            hipops.muon_step(*args, lr=0.1, **kw)
    assert not p.any() and not m.any()
    hipops.muon_step([], [], [], lr=0.1)                                              # nothing to do


def test_muon_step_refuses_shared_memory():
    both, g = torch.zeros(80), torch.zeros(4, 6)
    view = lambda lo, *shape: both[lo:lo + 24].view(*(shape or (4, 6)))
    for params, grads, momenta in [([view(0)], [view(0)], [view(40)]), ([view(0)], [view(40)], [view(40)]), ([view(0)], [view(20)], [view(50)]),
                                   ([view(0), view(23, 2, 12)], [g, g.view(2, 12)], [view(50), torch.zeros(2, 12)]), ([view(30)], [g], [view(53)])]:
        with pytest.raises(ValueError, match="share memory"):
            hipops.muon_step(params, grads, momenta, lr=0.1)
    for grads in ([g, g], [view(30), g]):                           # neighbours, and one gradient twice, are fine as far as memory goes
        with pytest.raises(_lib.DmError):
            hipops.muon_step([view(0), torch.zeros(4, 6)], grads, [view(54), torch.zeros(4, 6)], lr=0.1)


def test_c_entries_refuse_before_any_launch():
    L = _lib.lib()
    ARG, WS, UNS = -1, -2, -3
    P = 1 << 12                                                                       # an aligned address that no check dereferences

    def lin(x=P, w=P, b=P, ids=P, offsets=None, n=2, ws=P, wb=1 << 20, y=P, M=4, K=64, N=64, R=16, E=1, res=None):
        return L.dm_linear_adapted_bf16(x, w, None, res, P, b, ids, offsets, n, 1.0, ws, wb, y, M, K, N, R, E, 0, None)
    for kw, rc in [(dict(x=None), ARG), (dict(ids=None), ARG), (dict(n=0), ARG), (dict(n=3), ARG), (dict(E=0), ARG), (dict(R=0), ARG), (dict(K=0), ARG),
                   (dict(w=None), ARG), (dict(b=None), ARG), (dict(y=None), ARG), (dict(ws=None), ARG), (dict(x=P + 2), ARG), (dict(res=P + 2), ARG),
                   (dict(M=-4), ARG), (dict(R=129), UNS), (dict(K=60), UNS), (dict(N=60), UNS), (dict(E=70000), UNS), (dict(wb=16), WS),
                   (dict(R=12, wb=4 * 68 + 64), WS)]:
        assert lin(**kw) == rc, kw
    assert lin(M=0) == 0

    def bwd(x=P, dy=P, wt=P, u=P, ws=P, wb=1 << 30, dx=P, da=P, db=P, M=4, K=64, N=64, R=16, E=1, n=2):
        return L.dm_linear_adapted_bwd_f16(x, dy, wt, P, P, P, None, n, 1.0, u, ws, wb, dx, da, db, M, K, N, R, E, None)
    need = L.dm_linear_adapted_bwd_workspace_bytes(4, 64, 64, 16, 1, 2)
    for kw, rc in [(dict(x=None), ARG), (dict(dy=None), ARG), (dict(wt=None), ARG), (dict(u=None), ARG), (dict(ws=None), ARG), (dict(M=0), ARG), (dict(n=3), ARG),
                   (dict(dx=P + 2), ARG), (dict(K=60), UNS), (dict(R=200), UNS), (dict(wb=need - 1), WS)]:
        assert bwd(**kw) == rc, kw

    def norm(x=P, rows=6, items=0, C=64, gate=None, pre=0, z=None, stats=None):
        return L.dm_gated_add_norm_fwd_f32(x, P, gate, items, 0, None, None, pre, None, None, P, z, stats, rows, C, 1.0, 1e-5, 0, None)
    for kw, rc in [(dict(x=None), ARG), (dict(rows=-1), ARG), (dict(C=0), ARG), (dict(C=8193), UNS), (dict(pre=1), ARG), (dict(stats=P + 4), ARG),
                   (dict(gate=P, items=4), ARG)]:
        assert norm(**kw) == rc, kw
    assert norm(rows=0) == 0
    nbwd = lambda ws, words: L.dm_gated_add_norm_bwd_bf16(P, P, P, 2, 1, P, P, 0, None, P, None, P, P, P, P, P, P, None, None, ws, words, 6, 64, 1.0, 1e-5, 0, None)
    assert nbwd(None, 0) == WS and nbwd(P, 100) == WS

    import ctypes
    ptrs = (ctypes.c_void_p * 1)(P)
    null = (ctypes.c_void_p * 1)(None)
    need = L.dm_orthogonalize_workspace_bytes(1, 8, 8)
    ns = lambda g=ptrs, o=ptrs, count=1, rows=8, cols=8, dt=0, steps=5, ws=P, wb=need: L.dm_orthogonalize(g, o, count, rows, cols, dt, steps, 1e-7, ws, wb, None)
    for kw, rc in [(dict(g=None), ARG), (dict(g=null), ARG), (dict(o=null), ARG), (dict(count=-1), ARG), (dict(rows=0), ARG), (dict(dt=3), ARG), (dict(steps=0), ARG),
                   (dict(ws=P + 16), ARG), (dict(ws=None), ARG), (dict(wb=need - 1), WS), (dict(rows=40000, cols=40000), UNS)]:
        assert ns(**kw) == rc, kw
    assert ns(count=0) == 0
    eight, length = (ctypes.c_int * 1)(8), (ctypes.c_float * 1)(0.1)
    mu = lambda g=ptrs, m=ptrs, p=ptrs, rows=eight, cols=eight, count=1, wb=need: L.dm_muon_step(g, m, p, rows, cols, length, count, 2, 5, 0.9, 1, 1e-7, 1.0, P, wb, None)
    zero, huge = (ctypes.c_int * 1)(0), (ctypes.c_int * 1)(40000)
    for kw, rc in [(dict(m=null), ARG), (dict(p=null), ARG), (dict(g=null), ARG), (dict(m=None), ARG), (dict(rows=None), ARG), (dict(rows=zero), ARG),
                   (dict(rows=huge, cols=huge), UNS), (dict(count=-1), ARG), (dict(wb=need - 1), WS)]:
        assert mu(**kw) == rc, kw
    assert mu(count=0) == 0
    assert L.dm_muon_step_workspace_bytes(eight, eight, 1) == need and L.dm_muon_step_workspace_bytes(zero, eight, 1) == 0


def test_size_queries():
    L = _lib.lib()
    up = lambda v: (v + 255) // 256 * 256
    u = lambda M, r: up(M * (4 * r + 8))                                             # pairs of 16-bit columns (padded rank), a scale and an adapter per row
    assert [L.dm_linear_adapted_workspace_bytes(10, 64, r, 3) for r in (16, 24, 64, 128)] == [u(10, p) for p in (16, 32, 64, 128)]
    assert [L.dm_linear_adapted_workspace_bytes(10, 64, r, 3) for r in (1, 33)] == [u(10, p) + 2 * 3 * 64 * p for p in (16, 64)]      # + B in padded rows
    assert L.dm_linear_adapted_workspace_bytes(0, 64, 16, 1) == L.dm_linear_adapted_workspace_bytes(4, 64, 129, 1) == 0
    # every adapter may end inside an item of 128 rows: full items and one more each
    assert L.dm_linear_adapted_bwd_workspace_bytes(1000, 64, 72, 16, 3, 7) == u(1000, 16) + up(2 * 3 * 64 * 16) + up(2 * 3 * 72 * 16) + up(4 * (8 + 7 + 1000)) + 4 * 10 * 16 * 136
    assert L.dm_orthogonalize_workspace_bytes(40, 65, 10) == 16 * L.dm_orthogonalize_workspace_bytes(1, 65, 10)
    assert L.dm_gated_add_norm_workspace_floats(0, 0, 8) == 0 and L.dm_gated_add_norm_workspace_floats(6, 2, 8) == (5 + 3) * 8


def test_trainer_optimizer_names_and_cpu():
    from dreammat_amd import controlnet_train as ct
    from dreammat_amd.sd import ARCHS, AutoencoderKLEncoder, UNet2DConditionModel
    a = ARCHS["tiny"]
    unet, vae = UNet2DConditionModel(a), AutoencoderKLEncoder(a)
    with pytest.raises(ValueError):
        ct.ControlNetTrainer(vae, unet, optimizer="sgd")
    tr = ct.ControlNetTrainer(vae, unet, optimizer="muon")
    assert len(tr.opt.matrices) + len(tr.opt.adamw.param_groups[0]["params"]) == len(tr._params())
    tr.opt.matrices[0].grad = torch.ones_like(tr.opt.matrices[0])
    with pytest.raises(_lib.DmError):                                                # no CPU form
        tr.opt.step()
    tr.opt.zero_grad()
    assert tr.opt.matrices[0].grad is None
    with pytest.raises(ValueError):
        tr.opt.load_state_dict({"momenta": [], "adamw": None})
    assert isinstance(ct.ControlNetTrainer(vae, unet).opt, torch.optim.AdamW)
