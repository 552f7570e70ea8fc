"""decay_attention_fwd and _bwd at the ends of their rows, pieces and sequences; inputs, forms and bars of tests/test_gpu_decay_attention.py."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_decay_attention import _backward, _case, _check_backward, _check_forward, _forward, _ops, _to
from tests.test_gpu_token_ops import BF16, F16, F32

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


def _rows_equal(got, want, rows, what):
    """The same bits (but for a zero's sign) in the rows named."""
    for name, x, y in zip(("d_q", "d_k", "d_v") if len(got) == 3 else ("out",), got, want):
        assert torch.equal(x[rows], y[rows]), f"{what}: {name}"


@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dk,dv", [(16, 16), (128, 128), (24, 40), (20, 36)])
def test_what_lies_outside_the_sequences_is_not_seen(cuda, dk, dv, dtype, states):
    """NaN before the first sequence and behind the last one, in tokens that share a piece with theirs."""
    ops = _ops()
    for before, lengths, behind in ((0, [120], 5), (5, [40, 23], 0), (3, [30], 30), (40, [100, 1, 60], 77)):
        s = _case(dk + before, [before] + lengths + [behind], 4, 2, dk, dv, dtype, False)
        s["cu"] = s["cu"][1:-1]
        if states:
            s["s0"], s["g1"] = torch.randn(2, len(lengths), 2, dk, dv, generator=torch.Generator().manual_seed(3))
        clean = _to(s, cuda)
        lo, hi = before, before + sum(lengths)
        nan = {k: v.clone() for k, v in clean.items()}
        for x in ("q", "k", "v", "g"):
            nan[x][:lo], nan[x][hi:] = float("nan"), float("nan")
        want, want_last = _forward(ops, clean, 0.4)
        out, last = _forward(ops, nan, 0.4)
        _rows_equal((out,), (want,), slice(lo, hi), f"{before}, {lengths}, {behind}")
        *wants, want_first = _backward(ops, clean, 0.4)
        *grads, first = _backward(ops, nan, 0.4)
        _rows_equal(grads, wants, slice(lo, hi), f"{before}, {lengths}, {behind}")
        if states:
            assert torch.equal(last, want_last) and torch.equal(first, want_first)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("dk,dv", [(16, 16), (128, 128), (20, 36)])
def test_a_value_that_is_not_finite_at_a_pieces_end(cuda, dk, dv, dtype, states, value):
    """In a sequence's last token a key or value is seen by that token alone, in its first one a query or a gradient of an output by that one's going back."""
    ops = _ops()
    for lengths in ([1], [33], [40, 23], [3, 60, 200], [100, 27, 500]):
        s = _case(sum(lengths), lengths, 2, 1, dk, dv, dtype, states)
        clean = _to(s, cuda)
        want, want_last = _forward(ops, clean, 0.4)
        *wants, want_first = _backward(ops, clean, 0.4)
        starts = s["cu"].tolist()
        for b in range(len(lengths)):
            for which, token in (("k", starts[b + 1] - 1), ("v", starts[b + 1] - 1), ("q", starts[b]), ("g", starts[b])):
                d = {k: v.clone() for k, v in clean.items()}
                d[which][token, 0, 5] = value
                what = f"{lengths}, {which} of token {token}"
                others = torch.ones(sum(lengths), dtype=torch.bool, device=cuda)
                others[token] = False
                out, last = _forward(ops, d, 0.4)
                *grads, first = _backward(ops, d, 0.4)
                _rows_equal((out,), (want,), others, what)
                _rows_equal(grads, wants, others, what)
                if which in "kv":
                    assert not bool(out[token].isfinite().all()), what
                if states:
                    apart = [i for i in range(len(lengths)) if i != b]
                    assert torch.equal(last[apart], want_last[apart]) and torch.equal(first[apart], want_first[apart]), what


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kv_heads,dk,dv,lengths,huge", [(520, 16, 16, [150, 30, 170], [1]), (520, 12, 20, [100, 150], [0]), (2, 16, 16, [10, 10, 160, 10, 7], [0, 1, 3, 4]),
                                                         (520, 32, 128, [9, 200], [0])])
def test_a_sequence_whose_state_overflows(cuda, kv_heads, dk, dv, lengths, huge, dtype):
    """Its products leave fp32's range: the sequences before and behind it are as they are without it.  (Heads enough for one block to go through all tokens.)"""
    ops = _ops()
    s = _case(11, lengths, kv_heads, kv_heads, dk, dv, dtype, False)
    s["ld"] = s["ld"].clamp(max=-0.01)
    d = _to(s, cuda)
    starts, overflown = s["cu"].tolist(), torch.zeros(sum(lengths), dtype=torch.bool)
    for b in huge:
        overflown[starts[b] : starts[b + 1]] = True
    for x in ("q", "k", "v", "g"):
        d[x][overflown] *= 1e25
        s[x][overflown] = 0
    out, _ = _forward(ops, d, 0.5)
    grads = _backward(ops, d, 0.5)
    assert not bool(out[overflown].isfinite().all())
    for x in (out, *grads[:3]):
        x[overflown] = 0
    _check_forward(s, out, None, 0.5)
    _check_backward(s, grads, 0.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_value_that_is_not_finite_where_the_decays_powers_vanish(cuda, dtype):
    """It reaches its sequence's end all the same, as 0 times what is not finite does: nowhere between does an output look right."""
    ops = _ops()
    s = _case(14, [300, 20], 2, 2, 16, 16, dtype, False)
    clean = _to(s, cuda)
    clean["ld"].copy_(torch.tensor([-4.0, -float("inf")]))
    want, _ = _forward(ops, clean, 0.5)
    *wants, _ = _backward(ops, clean, 0.5)
    d = {k: v.clone() for k, v in clean.items()}
    d["k"][10, :, 3] = float("inf")
    out, _ = _forward(ops, d, 0.5)
    assert torch.equal(out[:10], want[:10]) and torch.equal(out[300:], want[300:])
    assert not bool(out[10:300].isfinite().any())
    d = {k: v.clone() for k, v in clean.items()}
    d["g"][290, :, 3] = float("inf")
    _, d_k, d_v, _ = _backward(ops, d, 0.5)
    assert torch.equal(d_k[291:], wants[1][291:]) and torch.equal(d_v[291:], wants[2][291:])
    assert not bool(d_k[:291].isfinite().any()) and not bool(d_v[:291, :, 3].isfinite().any())
