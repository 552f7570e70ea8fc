"""How many rows a weight gradient's fp32 sums run over, from the workspace that ppo_qk_rotary_bwd asks for (on the CPU, which plans for 256 compute units)."""

from __future__ import annotations

import ctypes

import pytest


@pytest.mark.parametrize("type_", [0, 1])
@pytest.mark.parametrize("q_heads,kv_heads", [(16, 8), (64, 64), (1024, 8), (4096, 4096)])
@pytest.mark.parametrize("head_dim,lanes", [((64, 64), (8, 4)), ((128, 128), (16, 8)), ((512, 512), (64, 32)), ((510, 126), (64, 64)), ((2, 2), (1, 1))])
def test_sums_are_of_512_rows_at_most(head_dim, lanes, q_heads, kv_heads, type_):
    from tt_rsl_rl_amd import _lib as L

    dim, rotary = head_dim
    at_once = 256 // lanes[type_]  # rows that a block's lanes hold, each of which they add to the last one they held
    for tokens in (1, 1000, 1 << 16, 1 << 20, (1 << 24) + 1):
        args = L.QkRotaryArgs(tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=dim, rotary_dim=rotary, type=type_, weight_type=type_)
        sums = (L.load().ppo_qk_rotary_bwd_workspace_bytes(ctypes.byref(args)) - 256) // (2 * dim * 4)  # of queries and of keys
        # a block is a tile of up to 64 tokens of a group of heads; one whose tile and group are not whole has fewer rows than the mean of whole ones
        tile = min(64, 4096 // max(1, rotary // 2))
        least = min(tile, at_once)
        while tile > least and -(-tokens // tile) < 4 * 256:
            tile = max(least, tile // 2)
        groups, left = divmod(sums, -(-tokens // tile))
        assert left == 0 and groups >= 1
        group = -(-(q_heads + kv_heads) // groups)
        assert -(-min(tile, tokens) * group // at_once) <= 512
