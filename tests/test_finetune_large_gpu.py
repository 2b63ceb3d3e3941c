"""GPU: the fine-tuning operators at the sizes that pick their larger kernels -- tiles of 128 and 256, the rings of LDS stages past their first
round, workgroups that walk over several groups of rows -- against 64 bits, off the multiples of every tile.  Tolerances as in test_finetune_gpu.py."""
import math

import pytest
import torch

from tests.test_finetune_gpu import BF, DEV, FP, HF, NS_TOL, adapter_inputs, check_adapter, check_norm, gen, norm_inputs, ns_formula, rand, rel

pytestmark = pytest.mark.gpu


def cuts(rows, n, seed):
    """n ragged requests, an empty one among them, rows in front and behind; many shorter than a tile"""
    g = torch.Generator().manual_seed(seed)
    at = torch.randint(3, rows - 40, (n + 1,), generator=g).sort().values
    at[2] = at[1]
    return at.tolist()


LARGE_ADAPTERS = [
    # rows, K, N, R, E, ids (None: ragged over 60 requests), residual
    (8200, 200, 328, 12, 5, None, True),             # 32 rows per workgroup of x A^T; 128 tile
    (9001, 328, 136, 33, 3, [2], False),             # .. rank 64 padded; 64 tiles in the three-stage ring forward, 128 back
    (8320, 72, 264, 128, 4, None, False),            # .. the largest rank
    (8192, 136, 200, 16, 2, [0, -1, 1, 0], True),    # .. whole tiles, one without adapter
    (12301, 328, 712, 16, 7, None, True),            # x A^T through the ring of stages, mixed 128 tiles
    (12416, 136, 72, 64, 3, [0, 2, -1, 1], False),   # .. K shorter than the ring
    (12300, 520, 328, 128, 2, [1, 0, 1], True),      # .. R 128: two K steps of values, two of rests
    (12345, 64, 1032, 32, 60, None, False),          # .. one K step, adapters 60
    (13000, 648, 200, 1, 4, None, False),            # .. rank 1
    (1500, 704, 1096, 24, 3, None, True),            # 64 tiles in the three-stage ring, eleven K steps
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", range(len(LARGE_ADAPTERS)))
def test_linear_adapted_large(case, dtype):
    rows, K, N, R, E, ids, residual = LARGE_ADAPTERS[case]
    offsets = None
    if ids is None:
        offsets, ids = cuts(rows, 60, case), [(7 * i) % (E + 1) - 1 for i in range(60)]
    s = adapter_inputs(100 + case, dtype, (rows, K), N, R, E, ids, residual, True, offsets)
    check_adapter(s, 0.75, False)
    check_adapter(s, -1.5, True)


@pytest.mark.parametrize("rows", [8500, 12500])
@pytest.mark.parametrize("size", [1e-3, 1e2])
def test_linear_adapted_large_half_rows_of_every_scale(rows, size):
    """half: rows whose factor needs another power of two than their neighbours', tiles of one adapter and mixed ones"""
    for offsets in (None, cuts(rows, 60, 5)):
        ids = [0, 1] if offsets is None else [i % 4 - 1 for i in range(60)]
        s = adapter_inputs(7, HF, (rows, 136), 328, 16, 3, ids, True, True, offsets)
        s["x"] = (s["x"].float() * 4.0 ** (torch.arange(rows, device=DEV) % 5 - 2.0)[:, None]).to(HF)
        s["a"], s["b"] = (s["a"].float() * size).to(HF), (s["b"].float() / size).clamp(-6e4, 6e4).to(HF)
        s["dy"] = (s["dy"].float() * 1e-3).to(HF)
        check_adapter(s, 1.0, False)
        check_adapter(s, 0.5, True)


def test_linear_adapted_gradients_of_many_stored_adapters():
    """more stored adapters than requests, R off 8 and on it: the row ranges follow the adapters that are used, the others get zeros"""
    for E, rows, ids, R in ((3000, 1500, [2999, 7, 7, -1, 0], 4), (500, 12400, [499, 0], 16), (900, 8200, None, 12)):
        offsets = None
        if ids is None:
            offsets, ids = cuts(rows, 60, 9), [(53 * i) % (E + 1) - 1 for i in range(60)]
        s = adapter_inputs(31, BF, (rows, 72), 136, R, E, ids, False, True, offsets)
        _, _, da, db = check_adapter(s, 0.5, True)
        unused = [e for e in range(E) if e not in ids]
        assert not da[unused].any() and not db[unused].any()


LARGE_NORMS = [
    # shape, gate, post, pre, kind, type
    ((3, 5001, 320), "item", (1, 1), (1, 1), "layer", BF),          # rows of a quarter wave: two workgroups per CU, gates change inside a workgroup
    ((2, 4099, 640), "item", (1, 1), (1, 1), "layer", HF),          # half a wave
    ((5, 1601, 640), "channel", None, (1, 1), "layer", BF),
    ((2, 2501, 1024), "item", (1, 1), (1, 1), "rms", BF),           # a wave
    ((3, 1501, 1280), "item", (1, 1), (1, 1), "rms", FP),           # a workgroup of 256, backward 512
    ((2, 1301, 2048), "channel", (1, 1), (1, 1), "layer", HF),
    ((3, 801, 100), "item", (1, 1), (1, 1), "layer", BF),           # element by element, several rows per workgroup
    ((2, 1301, 1001), "channel", (1, 1), (1, 1), "rms", FP),        # .. a workgroup per row
    ((7, 161, 8192), "item", (1, 1), (1, 1), "layer", BF),          # the widest rows, two per workgroup
    ((1201, 5001), "channel", (1, 0), (1, 1), "layer", HF),
    ((4000, 5, 64), "item", (1, 1), (1, 1), "layer", FP),           # items shorter than a row group
]


@pytest.mark.parametrize("case", range(len(LARGE_NORMS)))
def test_gated_add_norm_large(case):
    shape, gate, post, pre, kind, dtype = LARGE_NORMS[case]
    check_norm(norm_inputs(200 + case, dtype, shape, gate, post, pre), kind)


# tiles that the products X X^T | S S^T | P X take
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("shape", [
    (16, 1280, 1280),        # 256
    (12, 1100, 1300),        # 256, sides off the tile
    (12, 1300, 1100),        # .. turned
    (10, 500, 700),          # 64 in the four-stage ring
    (16, 640, 640),          # 64 | 64 | 128
    (8, 900, 700),           # 64 | 64 | 128, turned, off the tile
    (3, 1279, 1281),         # 128 in shares | 64 | 128, rows that are no whole chunks
    (8, 250, 4090)])         # 64 in shares | 64 | 256
def test_orthogonalize_large(shape, dtype):
    from dreammat_amd import hipops
    g = rand(gen(sum(shape)), *shape, dtype=dtype, scale=1e-3)
    got, ref = hipops.orthogonalize(g), ns_formula(g)
    for p, q in zip(got, ref):
        assert torch.isfinite(p.float()).all() and rel(p, q) <= NS_TOL[dtype]
