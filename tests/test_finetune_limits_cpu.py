"""Sizes and states of the fine-tuning operators at their limits (CPU: size queries, refusals before any launch, the optimizer's bookkeeping)."""
import pytest
import torch

from dreammat_amd import _lib, hipops


def test_backward_workspace_follows_the_adapters_a_call_can_use():
    """a request has one adapter: stored ones that no request can name cost no partial sums"""
    L = _lib.lib()
    up = lambda v: (v + 255) // 256 * 256
    sizes = lambda E, n: L.dm_linear_adapted_bwd_workspace_bytes(24576, 1280, 5120, 64, E, n)
    # 24576 rows in items of 1216, and every used adapter may end inside one
    fixed = lambda E, n: up(24576 * (4 * 64 + 8)) + up(2 * E * 1280 * 64) + up(2 * E * 5120 * 64) + up(4 * (2 * (E + 1) + n + 24576))
    assert sizes(8, 24) == fixed(8, 24) + 4 * (20 + 8) * 64 * 6400
    assert sizes(1000, 24) == fixed(1000, 24) + 4 * (20 + 24) * 64 * 6400
    # .. and the entry takes that much (one byte less is refused, before any launch)
    P = 1 << 12
    bwd = lambda wb: L.dm_linear_adapted_bwd_bf16(P, P, P, P, P, P, None, 24, 1.0, P, P, wb, P, P, P, 24576, 1280, 5120, 64, 1000, None)
    assert bwd(sizes(1000, 24) - 1) == -2
    # as many adapters as an id can name, one request: 64 K adapters of one row range each were refused
    assert L.dm_linear_adapted_bwd_bf16(P, P, P, P, P, P, None, 1, 1.0, P, P, 16, P, P, P, 128 * 70000, 64, 64, 16, 65535, None) == -2


def test_adapters_refuse_more_rows_than_a_grid_holds():
    """2^30 rows would take grids of 2^32 threads"""
    BF, rows = torch.bfloat16, 1 << 30
    x, w = torch.zeros(1, 8, dtype=BF).expand(rows, 8), torch.zeros(8, 8, dtype=BF)
    args = (torch.zeros(1, 16, 8, dtype=BF), torch.zeros(1, 8, 16, dtype=BF), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="rows"):
        hipops.linear_adapted(x, w, None, *args)
    with pytest.raises(ValueError, match="rows"):
        hipops.linear_adapted_autograd(x, w, w, None, *args)
    L, P = _lib.lib(), 1 << 12
    assert L.dm_linear_adapted_bf16(P, P, None, None, P, P, P, None, 1, 1.0, P, 1 << 50, P, rows, 8, 8, 16, 1, 0, None) == -3
    assert L.dm_linear_adapted_bwd_bf16(P, P, P, P, P, P, None, 1, 1.0, P, P, 1 << 50, P, P, P, rows, 8, 8, 16, 1, None) == -3


def test_muon_state_brings_its_learning_rate_to_both_halves():
    """a restored state sets rate and decay of the matrices as torch's AdamW sets those of the rest: one rate for both"""
    from dreammat_amd.controlnet_train import MuonAdamW
    params = [torch.nn.Parameter(torch.zeros(4, 6)), torch.nn.Parameter(torch.zeros(4))]
    a, b = MuonAdamW(params, lr=1e-3, weight_decay=0.1, momentum=0.9), MuonAdamW(params, lr=1e-5)
    b.load_state_dict(a.state_dict())
    assert (b.lr, b.weight_decay, b.momentum) == (1e-3, 0.1, 0.9)
    assert all(g["lr"] == b.lr and g["weight_decay"] == b.weight_decay for g in b.adamw.param_groups)
    # a state without them (saved before it held them) leaves the matrices' own
    c = MuonAdamW(params, lr=1e-5)
    c.load_state_dict({"momenta": [None], "adamw": c.adamw.state_dict()})
    assert c.lr == 1e-5


def test_muon_state_of_other_shapes_is_refused():
    from dreammat_amd.controlnet_train import MuonAdamW
    one, other = (MuonAdamW([torch.nn.Parameter(torch.zeros(*s))], lr=1e-3) for s in ((4, 6), (6, 4)))
    one.momenta[0] = torch.ones(4, 6)
    with pytest.raises(ValueError, match="other parameters"):
        other.load_state_dict(one.state_dict())
    assert other.momenta == [None]


def test_trainer_steps_matrices_of_any_memory_format():
    """fp32 weights that are not contiguous (channels_last) get contiguous masters: the step takes no others"""
    from dreammat_amd import controlnet_train as ct
    from dreammat_amd.sd import ARCHS, AutoencoderKLEncoder, UNet2DConditionModel
    a = ARCHS["tiny"]
    unet = UNet2DConditionModel(a)
    net = ct.init_controlnet(unet).to(memory_format=torch.channels_last)
    tr = ct.ControlNetTrainer(AutoencoderKLEncoder(a), unet, net, optimizer="muon")
    assert any(not p.is_contiguous() for p in tr._params()) and all(p.is_contiguous() for p in tr.opt.matrices)
    assert ct.ControlNetTrainer(AutoencoderKLEncoder(a), unet, net).master is None
