"""GPU: the fine-tuning operators at the borders of their number formats -- the result's type only rounds it, one rank or one row far smaller than
the others keeps its digits, an infinite entry gives what the formula gives.  Tolerances as in test_finetune_gpu.py."""
import math

import pytest
import torch

from tests.test_finetune_gpu import BF, DEV, FP, HF, adapter_inputs, adapter_reference, gen, near, ns_formula, rand, rel

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
