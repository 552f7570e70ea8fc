"""decay_attention_fwd and _bwd at the ends of their rows, pieces and sequences; inputs, forms and bars of tests/test_gpu_decay_attention.py."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_decay_attention import _case, _check_backward, _check_forward, _ops, _to
from tests.test_gpu_token_ops import F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("dk,dv", [(68, 100), (124, 68), (76, 124), (92, 84), (116, 108), (64, 100), (100, 128)])
def test_fp32_heads_of_an_odd_number_of_pieces(cuda, dk, dv, states):
    """Blocks enough for 128 columns each, where a lane has two pieces of 16 bytes, of which the last lane's second may lie past the head: heads four
    elements and tokens eight more apart than they are wide, and what lies between them stays as it was."""
    ops = _ops()
    s = _case(dk, [450, 1, 199], 8, 8, dk, dv, F32, states)
    d = _to(s, cuda)
    n, stores = 650, []

    def spaced(dim):
        store = torch.full((n, 8 * (dim + 4) + 8), 9.0, device=cuda)
        stores.append((store, dim))
        return store[:, 4 : 4 + 8 * (dim + 4)].unflatten(1, (8, dim + 4))[..., :dim]

    out, last = spaced(dv), torch.empty_like(d["s0"]) if states else None
    ops.decay_attention_fwd(d["q"], d["k"], d["v"], d["ld"], out, scale=0.2, cu_seqlens=d["cu"], initial_state=d.get("s0"), final_state=last)
    grads, first = [spaced(dk), spaced(dk), spaced(dv)], torch.empty_like(d["s0"]) if states else None
    ops.decay_attention_bwd(d["g"], d["q"], d["k"], d["v"], d["ld"], *grads, scale=0.2, cu_seqlens=d["cu"], initial_state=d.get("s0"),
                            d_final_state=d.get("g1"), d_initial_state=first)
    for store, dim in stores:
        between = torch.ones_like(store, dtype=torch.bool)
        between[:, 4 : 4 + 8 * (dim + 4)].unflatten(1, (8, dim + 4))[..., :dim] = False
        assert bool((store[between] == 9).all())
    _check_forward(s, out, last, 0.2)
    _check_backward(s, (*grads, first), 0.2)
