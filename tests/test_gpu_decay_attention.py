"""decay_attention_fwd, _bwd and _step against the 64-bit forms of tests/token_layer_reference.py.

Bars.  u is the rounding of the output's type, U = 2^-24 that of fp32; sizes are the same sums over magnitudes.  A query-key product is off
by dk U; the decay's powers by 2 U each, and a state passes one of them a chunk; a sum over a chunk (64 tokens at most) adds 64 U and the
state n / 16 more over n tokens: E = (dk + dv + 160 + n / 8) U.  bf16 takes a state and the chunk's matrix as two parts of 8 bits,
which leave 2^-17 of them, into outputs and gradients (not into states: three parts, 2^-24, in E)."""

from __future__ import annotations

import math

import pytest
import torch

from tests import token_layer_reference as ref
from tests.test_gpu_token_ops import BF16, F16, F32, HALF, TINY, U, _gen, _inside

pytestmark = pytest.mark.gpu

LEFT = {F32: 0.0, BF16: 2.0**-16, F16: 0.0}


def _ops():
    from tt_rsl_rl_amd import _lib, ops

    _lib.load()
    return ops


def _fading(heads):
    return torch.log1p(-torch.exp2(-torch.linspace(1.0, 9.0, heads, dtype=torch.float64))).float()


def _case(seed, lengths, q_heads, kv_heads, dk, dv, dtype, states=True):
    g, n = _gen(seed), sum(lengths)
    r = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    s = dict(q=r(n, q_heads, dk).to(dtype), k=r(n, kv_heads, dk).to(dtype), v=r(n, kv_heads, dv).to(dtype), g=r(n, q_heads, dv).to(dtype),
             ld=_fading(kv_heads), cu=torch.tensor([0] + list(lengths)).cumsum(0))
    if states:
        s["s0"], s["g1"] = 2 * r(len(lengths), kv_heads, dk, dv), 2 * r(len(lengths), kv_heads, dk, dv)
    return s


def _to(s, cuda):
    return {k: v.to(cuda) for k, v in s.items()}


def _forward(ops, d, scale, cu=True):
    out = torch.empty(*d["q"].shape[:2], d["v"].shape[2], dtype=d["q"].dtype, device=d["q"].device)
    last = torch.empty_like(d["s0"]) if "s0" in d else None
    ops.decay_attention_fwd(d["q"], d["k"], d["v"], d["ld"], out, scale=scale, cu_seqlens=d["cu"] if cu else None, initial_state=d.get("s0"),
                            final_state=last)
    return out, last


def _backward(ops, d, scale, cu=True):
    outs = [torch.empty_like(d[x]) for x in ("q", "k", "v")]
    first = torch.empty_like(d["s0"]) if "s0" in d else None
    ops.decay_attention_bwd(d["g"], d["q"], d["k"], d["v"], d["ld"], *outs, scale=scale, cu_seqlens=d["cu"] if cu else None,
                            initial_state=d.get("s0"), d_final_state=d.get("g1"), d_initial_state=first)
    return (*outs, first)


def _error(s):
    longest = int((s["cu"][1:] - s["cu"][:-1]).max())
    return (s["q"].shape[2] + s["v"].shape[2] + 160 + longest / 8) * U


def _abs(s):
    return {k: v.abs() if k not in ("ld", "cu") else v for k, v in s.items()}


def _check_forward(s, out, last, scale, what=""):
    dtype, m = s["q"].dtype, _abs(s)
    want, want_last = ref.decay_attention(s["q"], s["k"], s["v"], s["ld"], scale, s["cu"], s.get("s0"))
    size, size_last = ref.decay_attention(m["q"], m["k"], m["v"], s["ld"], abs(scale), s["cu"], m.get("s0"))
    E = _error(s)
    _inside(out, want, (E + LEFT[dtype]) * size + 1.01 * HALF[dtype] * want.abs() + TINY[dtype], what + "out")
    if last is not None:
        _inside(last, want_last, E * size_last + 1e-37, what + "final state")


def _check_backward(s, got, scale, what=""):
    dtype, m = s["q"].dtype, _abs(s)
    want = ref.decay_attention_grad(s["g"], s["q"], s["k"], s["v"], s["ld"], scale, s["cu"], s.get("s0"), s.get("g1"))
    size = ref.decay_attention_grad(m["g"], m["q"], m["k"], m["v"], s["ld"], abs(scale), s["cu"], m.get("s0"), m.get("g1"))
    E = (s["q"].shape[1] // s["k"].shape[1]) * _error(s)
    for name, x, w, z in zip(("d_q", "d_k", "d_v"), got, want, size):
        _inside(x, w, (E + LEFT[dtype]) * z + 1.01 * HALF[dtype] * w.abs() + TINY[dtype], what + name)
    if got[3] is not None:
        _inside(got[3], want[3], E * size[3] + 1e-37, what + "d_initial")


LENGTHS = [[1], [2], [63], [64], [65], [31], [33], [200], [1, 1, 1], [5, 0, 64, 1, 130, 0], [0, 0, 7], [3] * 60, [700], [64, 128, 64], [500, 1, 300]]
HEADS = [(1, 1, 16, 16), (4, 2, 128, 128), (3, 3, 40, 72), (2, 1, 1, 3), (6, 2, 65, 128), (2, 2, 128, 64), (1, 1, 7, 100)]


@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: "-".join(map(str, x[:6])))
def test_lengths(cuda, lengths, dtype, states):
    ops = _ops()
    s = _case(len(lengths) + sum(lengths), lengths, 4, 2, 24, 40, dtype, states)
    d = _to(s, cuda)
    _check_forward(s, *_forward(ops, d, 0.3), 0.3)
    _check_backward(s, _backward(ops, d, 0.3), 0.3)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("q_heads,kv_heads,dk,dv", HEADS)
def test_heads(cuda, q_heads, kv_heads, dk, dv, dtype):
    ops = _ops()
    s = _case(dk + dv, [70, 3, 129], q_heads, kv_heads, dk, dv, dtype)
    s["cu"] = s["cu"].to(torch.int32)
    d = _to(s, cuda)
    _check_forward(s, *_forward(ops, d, dk**-0.5), dk**-0.5)
    _check_backward(s, _backward(ops, d, dk**-0.5), dk**-0.5)
    a, b = _backward(ops, d, 0.7), _backward(ops, d, 0.7)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long(cuda, dtype, states):
    """Cut into segments, whose states are made first and handed on; sequences begin and end inside them and on their borders."""
    ops = _ops()
    s = _case(3, [2048, 1, 700, 2347, 1024], 2, 1, 48, 32, dtype, states)
    d = _to(s, cuda)
    _check_forward(s, *_forward(ops, d, 0.2), 0.2)
    _check_backward(s, _backward(ops, d, 0.2), 0.2)


def test_one_sequence_without_cu_seqlens(cuda):
    ops = _ops()
    s = _case(4, [1500], 2, 2, 32, 32, BF16)
    d = _to(s, cuda)
    for x, y in zip(_forward(ops, d, 0.5) + _backward(ops, d, 0.5), _forward(ops, d, 0.5, cu=False) + _backward(ops, d, 0.5, cu=False)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decays(cuda, dtype):
    """None (plain sums), all at once (-inf: each token alone), and fast ones, whose powers vanish."""
    ops = _ops()
    s = _case(5, [150, 40], 3, 3, 16, 16, dtype)
    s["ld"] = torch.tensor([0.0, -math.inf, -30.0])
    d = _to(s, cuda)
    _check_forward(s, *_forward(ops, d, 0.5), 0.5)
    _check_backward(s, _backward(ops, d, 0.5), 0.5)


def test_tokens_outside_the_sequences(cuda):
    """Before the first and behind the last, NaN in the inputs: outputs there stay as they were, and the others do not see them."""
    ops = _ops()
    s = _case(6, [90, 25], 2, 1, 20, 36, BF16)
    inside = _to(s, cuda)
    want = _forward(ops, inside, 0.4) + _backward(ops, inside, 0.4)
    around = lambda x: torch.cat([torch.full_like(x[:7], math.nan), x, torch.full_like(x[:50], math.nan)])  # noqa: E731
    d = {k: around(v) if k in ("q", "k", "v", "g") else v for k, v in inside.items()}
    d["cu"] = inside["cu"] + 7
    out = torch.full((172, 2, 36), 5.0, dtype=BF16, device=cuda)
    last = torch.empty_like(d["s0"])
    ops.decay_attention_fwd(d["q"], d["k"], d["v"], d["ld"], out, scale=0.4, cu_seqlens=d["cu"], initial_state=d["s0"], final_state=last)
    outs = [torch.full_like(d[x], 5.0) for x in ("q", "k", "v")]
    first = torch.empty_like(d["s0"])
    ops.decay_attention_bwd(d["g"], d["q"], d["k"], d["v"], d["ld"], *outs, scale=0.4, cu_seqlens=d["cu"], initial_state=d["s0"],
                            d_final_state=d["g1"], d_initial_state=first)
    s["cu"] = s["cu"] + 7
    for x in (out, *outs):
        assert bool((x[:7] == 5).all()) and bool((x[122:] == 5).all())
    host = {k: torch.cat([torch.zeros_like(v[:7]), v, torch.zeros_like(v[:50])]) if k in ("q", "k", "v", "g") else v for k, v in s.items()}
    blank = lambda x: torch.cat([torch.zeros_like(x[:7]), x[7:122], torch.zeros_like(x[122:])])  # noqa: E731
    _check_forward(host, blank(out), last, 0.4)
    _check_backward(host, (*map(blank, outs), first), 0.4)
    assert want[1].shape == last.shape


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_values_that_are_not_finite_stay_in_their_head_and_sequence(cuda, dtype, which):
    """NaN from the token on in its own head, none elsewhere (a query's: its own row)."""
    ops = _ops()
    s = _case(7, [50, 40, 90], 2, 2, 16, 16, dtype)
    clean = _to(s, cuda)
    want, want_last = _forward(ops, clean, 0.5)
    d = {k: v.clone() for k, v in clean.items()}
    d[which][60, 1, 3] = math.inf
    d[which][61, 1, 2] = math.nan
    out, last = _forward(ops, d, 0.5)
    hit = torch.zeros(180, dtype=torch.bool)
    hit[60 if which != "q" else 61:90 if which != "q" else 62] = True
    row = out[:, 1].isnan().all(-1).cpu()
    assert bool(row[hit].all())
    touched = torch.zeros(180, 2, dtype=torch.bool, device=cuda)
    touched[60:90 if which != "q" else 62, 1] = True
    assert torch.equal(out[~touched], want[~touched])
    keep = torch.ones(3, 2, dtype=torch.bool, device=cuda)
    if which != "q":
        keep[1, 1] = False
        assert bool(last[1, 1].isnan().all())
    assert torch.equal(last[keep], want_last[keep])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views(cuda, dtype):
    """Columns of one buffer off any alignment, heads before tokens, a key shared by a stride of 0."""
    ops = _ops()
    s = _case(8, [100, 30], 4, 2, 24, 16, dtype)
    d = _to(s, cuda)
    want, want_last = _forward(ops, d, 0.5)
    wants = _backward(ops, d, 0.5)
    n, row = 130, 4 * 24 + 2 * 24 + 2 * 16 + 3
    buf = torch.zeros(n * row + 1, dtype=dtype, device=cuda)[1:].view(n, row)
    v = dict(d)
    v["q"], v["k"], v["v"] = buf[:, :96].unflatten(1, (4, 24)), buf[:, 96:144].unflatten(1, (2, 24)), buf[:, 145:177].unflatten(1, (2, 16))
    for x in ("q", "k", "v"):
        v[x].copy_(d[x])
    v["g"] = d["g"].transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty(4, n, 16, dtype=dtype, device=cuda).transpose(0, 1)
    last = d["s0"].clone()
    ops.decay_attention_fwd(v["q"], v["k"], v["v"], v["ld"], out, scale=0.5, cu_seqlens=v["cu"], initial_state=last, final_state=last)
    assert torch.equal(out, want) and torch.equal(last, want_last)
    grads = torch.full_like(buf, 9.0)
    outs = grads[:, :96].unflatten(1, (4, 24)), grads[:, 96:144].unflatten(1, (2, 24)), grads[:, 145:177].unflatten(1, (2, 16))
    first = d["g1"].clone()
    ops.decay_attention_bwd(v["g"], v["q"], v["k"], v["v"], v["ld"], *outs, scale=0.5, cu_seqlens=v["cu"], initial_state=v["s0"],
                            d_final_state=first, d_initial_state=first)
    for x, y in zip((*outs, first), wants):
        assert torch.equal(x, y)
    assert bool((grads[:, 144] == 9).all()) and bool((grads[:, 177:] == 9).all())
    one = d["k"][:, :1].expand(n, 2, 24)
    a, b = torch.empty_like(want), torch.empty_like(want)
    ops.decay_attention_fwd(d["q"], one, d["v"], d["ld"], a, cu_seqlens=d["cu"])
    ops.decay_attention_fwd(d["q"], one.contiguous(), d["v"], d["ld"], b, cu_seqlens=d["cu"])
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_states_in_place_over_many_segments(cuda, dtype):
    """The block that ends a sequence is another one than that which began it, and may be done first."""
    ops = _ops()
    s = _case(12, [5000, 0, 3000, 2500], 2, 1, 32, 24, dtype)
    d = _to(s, cuda)
    want, want_last = _forward(ops, d, 0.1)
    wants = _backward(ops, d, 0.1)
    for _ in range(5):
        out, state = torch.empty_like(want), d["s0"].clone()
        ops.decay_attention_fwd(d["q"], d["k"], d["v"], d["ld"], out, scale=0.1, cu_seqlens=d["cu"], initial_state=state, final_state=state)
        assert torch.equal(out, want) and torch.equal(state, want_last)
        outs, state = [torch.empty_like(d[x]) for x in ("q", "k", "v")], d["g1"].clone()
        ops.decay_attention_bwd(d["g"], d["q"], d["k"], d["v"], d["ld"], *outs, scale=0.1, cu_seqlens=d["cu"], initial_state=d["s0"], d_final_state=state,
                                d_initial_state=state)
        for x, y in zip((*outs, state), wants):
            assert torch.equal(x, y)


def test_no_tokens(cuda):
    ops = _ops()
    s = _case(9, [0, 0], 2, 1, 8, 8, F32)
    d = _to(s, cuda)
    out, last = _forward(ops, d, 1.0)
    assert out.numel() == 0 and torch.equal(last, d["s0"])
    assert torch.equal(_backward(ops, d, 1.0)[3], d["g1"])


# ---- single tokens ----

STEPS = [(1, 1, 1, 16, 16), (8, 4, 2, 128, 128), (3, 6, 3, 40, 72), (5, 2, 1, 1, 3), (700, 4, 4, 64, 64), (9, 8, 1, 128, 65), (2, 1, 1, 127, 128),
         (1100, 2, 2, 128, 128)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,q_heads,kv_heads,dk,dv", STEPS)
def test_step(cuda, rows, q_heads, kv_heads, dk, dv, dtype):
    ops = _ops()
    s = _case(rows + dk, [rows], q_heads, kv_heads, dk, dv, dtype, False)
    g = _gen(rows)
    state = torch.randn(rows + 3, kv_heads, dk, dv, generator=g)
    slots = torch.randperm(rows + 3, generator=g)[:rows]
    fresh = torch.rand(rows, generator=g) < 0.3
    if rows > 2:
        slots[1], slots[2] = -1, rows + 3
    state[int(slots[0])] = math.nan if bool(fresh[0]) else state[int(slots[0])]
    for slot_type in (torch.int64, torch.int32):
        got = state.to(cuda)
        out = torch.empty(rows, q_heads, dv, dtype=dtype, device=cuda)
        d = _to(s, cuda)
        ops.decay_attention_step(d["q"], d["k"], d["v"], d["ld"], got, out, scale=0.6, slots=slots.to(slot_type).to(cuda), fresh=fresh.to(cuda))
        want, after = ref.decay_step(s["q"], s["k"], s["v"], s["ld"], state, 0.6, slots, fresh)
        size, size_after = ref.decay_step(s["q"].abs(), s["k"].abs(), s["v"].abs(), s["ld"], state.abs(), 0.6, slots, fresh)
        _inside(got, after, 4 * U * size_after, "state")
        _inside(out, want, (dk + 8) * U * size + 1.01 * HALF[dtype] * want.abs() + TINY[dtype], "out")


def test_step_is_the_prompts_recurrence(cuda):
    """Tokens one at a time give what the prompt gives, to their bars."""
    ops = _ops()
    s = _case(10, [40, 40, 40], 4, 2, 32, 24, F32)
    d = _to(s, cuda)
    state = d["s0"].clone()
    out = torch.empty(3, 40, 4, 24, device=cuda)
    by = {x: d[x].view(3, 40, *d[x].shape[1:]) for x in ("q", "k", "v")}
    for t in range(40):
        ops.decay_attention_step(by["q"][:, t], by["k"][:, t], by["v"][:, t], d["ld"], state, out[:, t], scale=0.5)
    _check_forward(s, out.flatten(0, 1), state, 0.5, "steps: ")


# Blocks enough for 128 columns each on 256 compute units, query heads together; and fewer, with 64 columns and a query head or a few each.
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("q_heads,kv_heads,dk,dv,lengths", [(8, 4, 128, 128, [1900, 3, 1300, 64, 700]), (4, 4, 40, 128, [2600]), (4, 4, 99, 77, [1000, 1500]),
                                                            (8, 1, 128, 104, [700, 90]), (12, 2, 30, 128, [400]), (6, 1, 77, 101, [65, 65])])
def test_shares_of_blocks(cuda, q_heads, kv_heads, dk, dv, lengths, dtype):
    ops = _ops()
    for states in (True, False):
        s = _case(dk, lengths, q_heads, kv_heads, dk, dv, dtype, states)
        d = _to(s, cuda)
        _check_forward(s, *_forward(ops, d, 0.2), 0.2)
        _check_backward(s, _backward(ops, d, 0.2), 0.2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_that_are_not_finite_in_wide_heads(cuda, dtype):
    """A block may have half of a head's columns: an infinite key reaches all of them, an infinite value its own at least; no other token, head or sequence."""
    ops = _ops()
    s = _case(9, [50, 40, 90], 2, 2, 128, 128, dtype)
    clean = _to(s, cuda)
    want, want_last = _forward(ops, clean, 0.5)
    for which in ("k", "v"):
        d = {k: v.clone() for k, v in clean.items()}
        d[which][60, 1, 100] = math.inf
        out, last = _forward(ops, d, 0.5)
        columns = slice(None) if which == "k" else slice(100, 101)
        assert not bool(out[60:90, 1, columns].isfinite().any()) and not bool(last[1, 1, 100 if which == "k" else slice(None), columns].isfinite().any())
        touched = torch.zeros(180, 2, dtype=torch.bool, device=cuda)
        touched[60:90, 1] = True
        assert torch.equal(out[~touched], want[~touched])
        keep = torch.ones(3, 2, dtype=torch.bool, device=cuda)
        keep[1, 1] = False
        assert torch.equal(last[keep], want_last[keep])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths", [[1], [40], [20, 11], [64, 0, 3, 60]])
def test_states_in_place_with_query_heads_apart(cuda, dtype, lengths):
    """Query heads of a head may be blocks of their own, which all read the state that one of them replaces."""
    ops = _ops()
    s = _case(13, lengths, 16, 2, 128, 128, dtype)
    d = _to(s, cuda)
    want, want_last = _forward(ops, d, 0.1)
    wants = _backward(ops, d, 0.1)
    for _ in range(5):
        state, grad, out = d["s0"].clone(), d["g1"].clone(), torch.empty_like(want)
        ops.decay_attention_fwd(d["q"], d["k"], d["v"], d["ld"], out, scale=0.1, cu_seqlens=d["cu"], initial_state=state, final_state=state)
        assert torch.equal(out, want) and torch.equal(state, want_last)
        grads = [torch.empty_like(d[x]) for x in ("q", "k", "v")]
        ops.decay_attention_bwd(d["g"], d["q"], d["k"], d["v"], d["ld"], *grads, scale=0.1, cu_seqlens=d["cu"], initial_state=d["s0"],
                                d_final_state=grad, d_initial_state=grad)
        assert all(torch.equal(a, b) for a, b in zip((*grads, grad), wants))
