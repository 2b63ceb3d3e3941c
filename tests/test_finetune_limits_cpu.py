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
