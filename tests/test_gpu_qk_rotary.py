"""qk_norm_rotary_fwd and _bwd against the 64-bit forms of tests/token_layer_reference.py.

Bars.  u is the rounding of the output's type, U = 2^-24 that of fp32.  A row's mean of squares is off by at most (D + 4) U, its inverse
root by half of that and 3 U more; sine and cosine come from an angle that is off by 2^-25 turns (4 U in radians) and, for far positions,
by 2^-51 of the angle, and are themselves off by 2 U; products and sums add 8.  So results are off by (D / 2 + 24) U + 2^-51 |angle| of the sizes they are made
of.  Weight gradients add the roundings of their sums: up to 64 tokens of all heads in fp32, the rest in fp64."""

from __future__ import annotations

import pytest
import torch

from tests import token_layer_reference as ref
from tests.test_gpu_token_ops import BF16, F16, F32, HALF, TINY, U, _gen, _inside

pytestmark = pytest.mark.gpu


def _ops():
    from tt_rsl_rl_amd import _lib, ops

    _lib.load()
    return ops


def _case(seed, tokens, q_heads, kv_heads, dim, rotary, dtype, weight_type=None, per_head=False, far=5000):
    g = _gen(seed)
    s = dict(q=torch.randn(tokens, q_heads, dim, generator=g).to(dtype), k=(3 * torch.randn(tokens, kv_heads, dim, generator=g)).to(dtype))
    shape = lambda h: (h, dim) if per_head else (dim,)  # noqa: E731
    s["wq"], s["wk"] = (torch.randn(*shape(h), generator=g).to(weight_type or dtype) for h in (q_heads, kv_heads))
    s["pos"] = torch.randint(-far, far, (tokens,), generator=g)
    s["freqs"] = _ops().rotary_frequencies(rotary)
    s["gq"], s["gk"] = torch.randn(tokens, q_heads, dim, generator=g).to(dtype), torch.randn(tokens, kv_heads, dim, generator=g).to(dtype)
    return s


def _bound(dim, far):
    return (dim / 2 + 24) * U + far * 2.0**-51


CASES = [(1, 1, 1, 2, 2), (1, 4, 2, 128, 128), (3, 2, 1, 6, 4), (8, 16, 4, 128, 128), (130, 3, 3, 80, 40), (77, 5, 1, 96, 96), (64, 2, 2, 512, 512),
         (33, 2, 1, 510, 254), (257, 8, 2, 64, 32), (1000, 6, 2, 48, 48), (40, 70, 10, 34, 2), (2100, 4, 4, 256, 128)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rotary", CASES)
def test_forward(cuda, tokens, q_heads, kv_heads, dim, rotary, dtype, interleaved):
    ops = _ops()
    s = _case(tokens + dim, tokens, q_heads, kv_heads, dim, rotary, dtype, per_head=dim == 96)
    d = {k: v.to(cuda) for k, v in s.items()}
    q, k = torch.empty_like(d["q"]), torch.empty_like(d["k"])
    ops.qk_norm_rotary_fwd(d["q"], d["k"], d["wq"], d["wk"], d["pos"], d["freqs"], q, k, eps=1e-5, interleaved=interleaved)
    for got, x, w in ((q, s["q"], s["wq"]), (k, s["k"], s["wk"])):
        want, before = ref.qk_rotary(x, w, s["pos"], s["freqs"], 1e-5, interleaved)
        _inside(got, want, _bound(dim, 5000) * ref.pair_size(before, s["freqs"], interleaved) + 1.01 * HALF[dtype] * want.abs() + TINY[dtype], "turned")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("dtype,weight_type", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16)])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rotary", CASES)
def test_backward(cuda, tokens, q_heads, kv_heads, dim, rotary, dtype, weight_type, per_head, interleaved):
    ops = _ops()
    s = _case(tokens + dim + 1, tokens, q_heads, kv_heads, dim, rotary, dtype, weight_type, per_head)
    d = {k: v.to(cuda) for k, v in s.items()}
    out = [torch.empty_like(d[k]) for k in ("q", "k", "wq", "wk")]
    ops.qk_norm_rotary_bwd(d["gq"], d["gk"], d["q"], d["k"], d["wq"], d["wk"], d["pos"], d["freqs"], *out, eps=1e-5, interleaved=interleaved)
    again = [torch.empty_like(o) for o in out]
    ops.qk_norm_rotary_bwd(d["gq"], d["gk"], d["q"], d["k"], d["wq"], d["wk"], d["pos"], d["freqs"], *again, eps=1e-5, interleaved=interleaved)
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    for got_x, got_w, x, w, g in ((out[0], out[2], s["q"], s["wq"], s["gq"]), (out[1], out[3], s["k"], s["wk"], s["gk"])):
        dx, dw, x_size, w_size = ref.qk_rotary_grad(g, x, w, s["pos"], s["freqs"], 1e-5, interleaved)
        E = _bound(dim, 5000)
        _inside(got_x, dx, (2 * E + 20 * U) * x_size + 1.01 * HALF[dtype] * dx.abs() + TINY[dtype], "d_x")
        n = min(tokens, 64) * (1 if per_head else x.shape[1])
        _inside(got_w, dw, (E + n * U) * w_size + 1.01 * HALF[weight_type] * dw.abs() + TINY[weight_type], "d_weight")


@pytest.mark.parametrize("positions", [torch.int64, torch.int32])
def test_far_positions(cuda, positions):
    """Angles far past what fp32 resolves: 2^30 turns less a few."""
    ops = _ops()
    s = _case(5, 50, 2, 1, 64, 64, F32)
    s["pos"] = (2**30 - torch.arange(50) * 7919).to(positions)
    d = {k: v.to(cuda) for k, v in s.items()}
    q, k = torch.empty_like(d["q"]), torch.empty_like(d["k"])
    ops.qk_norm_rotary_fwd(d["q"], d["k"], d["wq"], d["wk"], d["pos"], d["freqs"], q, k)
    want, before = ref.qk_rotary(s["q"], s["wq"], s["pos"], s["freqs"], 1e-6, False)
    _inside(q, want, _bound(64, 2.0**30) * ref.pair_size(before, s["freqs"], False) + 1.01 * U * want.abs(), "far")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_and_in_place(cuda, dtype):
    """Columns of one projection's output, off any alignment, heads before tokens; in place; nothing else is written."""
    ops = _ops()
    s = _case(9, 37, 4, 2, 24, 24, dtype)
    d = {k: v.to(cuda) for k, v in s.items()}
    want_q, want_k = torch.empty_like(d["q"]), torch.empty_like(d["k"])
    ops.qk_norm_rotary_fwd(d["q"], d["k"], d["wq"], d["wk"], d["pos"], d["freqs"], want_q, want_k)
    row = 8 * 24 + 3
    both = torch.full((37 * row + 1,), 7.0, dtype=dtype, device=cuda)[1:].view(37, row)
    q, k = both[:, 1:97].unflatten(1, (4, 24)), both[:, 97:145].unflatten(1, (2, 24))
    q.copy_(d["q"])
    k.copy_(d["k"])
    ops.qk_norm_rotary_fwd(q, k, d["wq"], d["wk"], d["pos"], d["freqs"], q, k)
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    assert bool((both[:, 0] == 7).all()) and bool((both[:, 145:] == 7).all())
    hq, hk = torch.empty(4, 37, 24, dtype=dtype, device=cuda), torch.empty(2, 37, 24, dtype=dtype, device=cuda)  # heads before tokens
    ops.qk_norm_rotary_fwd(d["q"], d["k"], d["wq"], d["wk"], d["pos"], d["freqs"], hq.transpose(0, 1), hk.transpose(0, 1))
    assert torch.equal(hq.transpose(0, 1), want_q) and torch.equal(hk.transpose(0, 1), want_k)
    outs = [torch.empty_like(d[k]) for k in ("q", "k", "wq", "wk")]
    ops.qk_norm_rotary_bwd(d["gq"], d["gk"], d["q"], d["k"], d["wq"], d["wk"], d["pos"], d["freqs"], *outs)
    for over_q, over_k in ((d["gq"].clone(), d["gk"].clone()),):  # the gradient in the place of the one that comes in
        ws = [torch.empty_like(d["wq"]), torch.empty_like(d["wk"])]
        ops.qk_norm_rotary_bwd(over_q, over_k, d["q"], d["k"], d["wq"], d["wk"], d["pos"], d["freqs"], over_q, over_k, *ws)
        assert torch.equal(over_q, outs[0]) and torch.equal(over_k, outs[1]) and torch.equal(ws[0], outs[2])
    shared = d["k"][:, :1].expand(37, 2, 24)  # one key for both heads: a stride of 0
    a, b = torch.empty_like(d["k"]), torch.empty_like(d["k"])
    ops.qk_norm_rotary_fwd(d["q"], shared, d["wq"], d["wk"], d["pos"], d["freqs"], want_q, a)
    ops.qk_norm_rotary_fwd(d["q"], shared.contiguous(), d["wq"], d["wk"], d["pos"], d["freqs"], want_q, b)
    assert torch.equal(a, b)


def test_rows_stay_apart(cuda):
    """A row of zeros, of NaN, of infinities: its own results and no others."""
    ops = _ops()
    s = _case(11, 40, 3, 1, 64, 64, BF16)
    d = {k: v.to(cuda) for k, v in s.items()}
    want_q, want_k = torch.empty_like(d["q"]), torch.empty_like(d["k"])
    ops.qk_norm_rotary_fwd(d["q"], d["k"], d["wq"], d["wk"], d["pos"], d["freqs"], want_q, want_k)
    d["q"][3, 1], d["q"][5, 0, 7], d["q"][6, 2, 0] = 0.0, float("nan"), float("inf")
    q, k = torch.empty_like(d["q"]), torch.empty_like(d["k"])
    ops.qk_norm_rotary_fwd(d["q"], d["k"], d["wq"], d["wk"], d["pos"], d["freqs"], q, k)
    assert bool((q[3, 1] == 0).all()) and bool(q[5, 0].isnan().all())
    q[3, 1], q[5, 0], q[6, 2] = want_q[3, 1], want_q[5, 0], want_q[6, 2]
    assert torch.equal(q, want_q) and torch.equal(k, want_k)


def test_no_tokens(cuda):
    ops = _ops()
    s = _case(1, 4, 2, 1, 16, 8, F32)
    d = {k: v.to(cuda) for k, v in s.items()}
    none = {k: d[k][:0] for k in ("q", "k", "gq", "gk", "pos")}
    ops.qk_norm_rotary_fwd(none["q"], none["k"], d["wq"], d["wk"], none["pos"], d["freqs"], none["q"], none["k"])
    dwq, dwk = torch.ones_like(d["wq"]), torch.ones_like(d["wk"])
    ops.qk_norm_rotary_bwd(none["gq"], none["gk"], none["q"], none["k"], d["wq"], d["wk"], none["pos"], d["freqs"], none["gq"], none["gk"], dwq, dwk)
    assert not bool(dwq.any()) and not bool(dwk.any())
