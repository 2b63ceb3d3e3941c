"""GPU: the fine-tuning operators at the borders of their number formats -- the result's type only rounds it, one rank or one row far smaller than
the others keeps its digits, an infinite entry gives what the formula gives.  Tolerances as in test_finetune_gpu.py."""
import pytest
import torch

from tests.test_finetune_gpu import BF, DEV, HF, adapter_inputs, adapter_reference, gen, half, near, rand

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ orthogonalised updates
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("shape", [(320, 320), (3, 64, 200), (2, 200, 72), (65, 63), (16, 1280, 1280)])
def test_orthogonalize_rounds_once(shape, dtype):
    """a 16-bit matrix gives the fp32 result of the same values, rounded: one set of products for all types"""
    from dreammat_amd import hipops
    g = rand(gen(shape[-1]), *shape, dtype=dtype, scale=1e-3)
    assert torch.equal(hipops.orthogonalize(g), hipops.orthogonalize(g.float()).to(dtype))


@pytest.mark.parametrize("gdtype", [BF, HF])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step_of_16_bit_gradients_is_the_fp32_step(nesterov, gdtype):
    """an fp32 parameter does not lose bits to its gradient's type"""
    from dreammat_amd import hipops
    g = gen(7)
    shapes = [(64, 64), (40, 24, 3, 3), (640, 320), (24, 200), (320, 1280)]
    p, m = ([rand(g, *q, scale=c) for q in shapes] for c in (0.02, 1e-3))
    gr = [rand(g, *q, dtype=gdtype, scale=1e-3) for q in shapes]
    p2, m2 = [q.clone() for q in p], [q.clone() for q in m]
    hipops.muon_step(p, gr, m, lr=0.02, nesterov=nesterov)
    hipops.muon_step(p2, [q.float() for q in gr], m2, lr=0.02, nesterov=nesterov)
    assert all(torch.equal(a, b) for a, b in zip(p + m, p2 + m2))


# ------------------------------------------------------------------------------------------------ adapters: unequal ranks and rows
def close(got, ref, terms, n):
    """`near`, down into the subnormals: the floor is half their step"""
    t = got.dtype
    tol = half(t) * ref.abs() * 1.001 + (n * 2.0 ** -23 + 2.0 ** -17) * terms + torch.finfo(t).tiny * half(t)
    worst = ((got.double() - ref).abs() / tol).max().item()
    assert torch.isfinite(got).all() and worst <= 1.0, worst


def check_all(s, scale=1.0):
    """forward and gradients against 64 bits -> the outputs"""
    from dreammat_amd import hipops
    ref = adapter_reference(s, scale)
    K, N, R, M = s["x"].shape[-1], s["w"].shape[0], s["a"].shape[1], s["x"].numel() // s["x"].shape[-1]
    x, a, b = (s[k].detach().requires_grad_() for k in ("x", "a", "b"))
    y = hipops.linear_adapted_autograd(x, s["w"], s["w"].t().contiguous(), s["bias"], a, b, s["ids"], scale, s["residual"], s["offsets"])
    dx, da, db = torch.autograd.grad(y, (x, a, b), s["dy"])
    close(y.detach().reshape(M, N), *ref["y"], K + 2 * R)
    close(dx.reshape(M, K), *ref["dx"], N + 2 * R)
    close(da, *ref["da"], M + N)
    close(db, *ref["db"], M + K)
    return y.detach(), dx, da, db


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows", [96, 12400])
@pytest.mark.parametrize("side", ["a", "b"])
def test_linear_adapted_of_ranks_of_unequal_size(side, rows, dtype):
    """rank r is 2^-r of the first one in A (so in u), or in B (so in du): every rank's gradients keep their digits.  Half: entries down to 2^-22 of
    their row's largest keep 2^-16 of themselves, smaller ones are off by no more than those; a rank of 2^-15 is that far down only where its
    product is 2^-7 of its usual size, and those rows hardly count in its sum."""
    s = adapter_inputs(21, dtype, (rows, 64), 136, 16, 2, [0, 1, 1, 0])
    down = 2.0 ** -torch.arange(16, device=DEV)
    if side == "a":                                      # u = 1 ... 2^-15; dy large, so that the results stay normal halves
        s["a"] = (s["a"].float() * down[None, :, None]).to(dtype)
        s["b"] = (s["b"].float() / 64).to(dtype)
        s["dy"] = (s["dy"].float() * 100).to(dtype)
    else:                                                # du = 0.5 ... 2^-16; x large
        s["b"] = (s["b"].float() * down[None, None, :]).to(dtype)
        s["x"] = (s["x"].float() * 100).to(dtype)
        s["dy"] = (s["dy"].float() / 6).to(dtype)
    check_all(s, 1.0)


@pytest.mark.parametrize("rows", [96, 12400])
def test_linear_adapted_half_of_rows_of_unequal_size(rows):
    """rows of x and of dy from 2^-12 to 2^11 next to each other, in a tile and in a range of the weight gradients (both products of a row are
    then of one size: every row counts)"""
    s = adapter_inputs(22, HF, (rows, 64), 136, 16, 2, [0, 1])
    size = 2.0 ** (torch.arange(rows, device=DEV) % 24 - 12.0)[:, None]
    s["x"] = (s["x"].float() * size).to(HF)
    s["dy"] = (s["dy"].float() * size.flip(0) * 2.0 ** -10).to(HF)
    check_all(s, 1.0)


# ------------------------------------------------------------------------------------------------ adapters: infinite entries
def same_with_infinities(got, ref, terms, n):
    """finite, +inf, -inf and NaN where the formula has them; `near` on the finite ones"""
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf].double(), ref[inf])
    fine = torch.isfinite(ref)
    near(torch.where(fine, got, 0.0), torch.where(fine, ref, 0.0), torch.where(fine, terms, 0.0), n, 2.0 ** -17)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("R", [8, 16, 24, 40, 100])
@pytest.mark.parametrize("rows", [24, 384, 12400])
@pytest.mark.parametrize("where", ["a", "b", "x", "dy"])
def test_linear_adapted_infinite_entry(where, rows, R, dtype):
    """one infinite entry: +-inf where the formula says so, whatever the number of rows, and nothing elsewhere"""
    from dreammat_amd import hipops
    s = adapter_inputs(23, dtype, (rows, 64), 136, R, 3, [0, 1, -1, 2])
    at = {"a": (1, R - 1, 5), "b": (1, 9, R - 1), "x": (rows // 4 + 1, 5), "dy": (rows // 4 + 1, 9)}[where]
    s[where][at] = float("inf")
    ref = {k: (v, t.nan_to_num(0.0, 0.0, 0.0)) for k, (v, t) in adapter_reference(s, 1.0).items()}
    if where == "a":                                     # 0 inf of rows of other adapters is no part of the formula
        assert torch.isinf(ref["y"][0][rows // 4:rows // 2]).all()
    y = hipops.linear_adapted(s["x"], s["w"], s["bias"], s["a"], s["b"], s["ids"])
    same_with_infinities(y, *ref["y"], 64 + 2 * R)
    x, a, b = (s[k].detach().requires_grad_() for k in ("x", "a", "b"))
    y = hipops.linear_adapted_autograd(x, s["w"], s["w"].t().contiguous(), s["bias"], a, b, s["ids"])
    grads = torch.autograd.grad(y, (x, a, b), s["dy"])
    same_with_infinities(y.detach(), *ref["y"], 64 + 2 * R)
    for name, got, n in zip(("dx", "da", "db"), grads, (136 + 2 * R, rows + 136, rows + 64)):
        same_with_infinities(got, *ref[name], n)


# ------------------------------------------------------------------------------------------------ norms
def test_gated_add_norm_refuses_forward_mode():
    """a tangent is refused, not dropped: the operator has a backward pass only"""
    from torch.autograd import forward_ad
    from dreammat_amd import hipops
    x, h = rand(gen(1), 4, 64), rand(gen(2), 4, 64)
    with forward_ad.dual_level():
        for v in ((forward_ad.make_dual(x, h), h), (x, forward_ad.make_dual(h, x))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):
                    hipops.gated_add_norm(*v, pre=(None, None))
        y = hipops.gated_add_norm(x, h)                                # no tangent: as ever
    assert torch.equal(y, hipops.gated_add_norm(x, h))


def test_controlnet_trainer_takes_channels_last_weights():
    """fp32 weights in channels_last: the same step, bit for bit, as from contiguous ones"""
    from dreammat_amd import controlnet_train as ct
    from dreammat_amd.sd import ARCHS, AutoencoderKLEncoder, UNet2DConditionModel
    a = ARCHS["tiny"]
    out = []
    for form in (torch.contiguous_format, torch.channels_last):
        torch.manual_seed(0)
        unet = UNet2DConditionModel(a).to(DEV)
        tr = ct.ControlNetTrainer(AutoencoderKLEncoder(a).to(DEV), unet, ct.init_controlnet(unet).to(DEV, memory_format=form), lr=1e-3, max_grad_norm=1e9,
                                  optimizer="muon")
        for i, p in enumerate(tr._params()):
            p.grad = rand(gen(i), *p.shape).to(memory_format=form if p.dim() == 4 else torch.contiguous_format)
        tr.apply_gradients()
        out.append([p.detach().clone() for p in tr._params()])
    assert all(torch.equal(p, q) for p, q in zip(*out))


def test_linear_adapted_autograd_keeps_the_low_rank_factor_only():
    """ranks off 8: the adapters' padded copy is the forward's scratch, not kept until the backward"""
    from dreammat_amd import _lib
    from dreammat_amd import hipops
    s = adapter_inputs(24, BF, (200, 64), 136, 12, 50, [0, 49])
    y = hipops.linear_adapted_autograd(s["x"], s["w"], s["w"].t().contiguous(), s["bias"], s["a"].requires_grad_(), s["b"], s["ids"])
    kept = [t.untyped_storage().nbytes() for t in y.grad_fn.saved_tensors if t is not None and t.dtype == torch.uint8]
    assert kept == [_lib.lib().dm_linear_adapted_workspace_bytes(200, 136, 16, 50)] == [(200 * 72 + 255) // 256 * 256]
    s = adapter_inputs(24, BF, (200, 64), 136, 12, 50, [0, 49])
    check_all(s, 0.5)


def test_linear_adapted_half_training_step_captured_and_replayed():
    """half, a rank off 8 and rows of every scale in a captured graph: replays on new inputs match the eager step bit for bit"""
    from dreammat_amd import hipops
    s = adapter_inputs(25, HF, (300, 64), 136, 12, 3, [0, -1, 2], True)
    wt = s["w"].t().contiguous()

    def step(x, dy):
        v = [t.detach().requires_grad_() for t in (x, s["a"], s["b"])]
        y = hipops.linear_adapted_autograd(v[0], s["w"], wt, s["bias"], v[1], v[2], s["ids"], 0.5, s["residual"])
        return [y.detach(), *torch.autograd.grad(y, v, dy)]
    x, dy = s["x"].clone(), s["dy"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, dy)
    for k in range(3):
        x.copy_(rand(gen(70 + k), 300, 64) * 8.0 ** (torch.arange(300, device=DEV) % 5 - 2.0)[:, None])
        dy.copy_(rand(gen(80 + k), 300, 136))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step(x, dy)))
