"""linear_log_probs and linear_cross_entropy against the 64-bit form of tests/token_layer_reference.py.

Bars.  u is the rounding of the operands' type, U = 2^-24 that of fp32.  A logit is a sum of dim products in fp32: off by (dim + 8) U of the
sum of magnitudes X (fp32 operands: three parts of 8 bits leave 2^-24 of each and products of parts below 2^-23 are left out, 8 U more).
Over the temperature that is dz; probabilities are off by 2 dz + E, E = U (4 max|z| + vocab / 256 + 64) as for logits in memory, relative;
logp and entropy by dz + E, times 1 + max|z| for the entropy.  d = p - [token] is rounded once to the operands' type (u of it, or a
2^-25th of 2^-14 for fp16, U for fp32) and summed over vocab (rows) in fp32: the gradients are off by the sums of |errors of d| times the other
factor, vocab (rows + 64) U of the sum of magnitudes, and u of the value."""

from __future__ import annotations

import math

import pytest
import torch

from tests import token_layer_reference as ref
from tests.test_gpu_token_ops import BF16, F16, F32, HALF, TINY, U, _gen, _inside

pytestmark = pytest.mark.gpu


def _ops():
    from tt_rsl_rl_amd import _lib, ops

    _lib.load()
    return ops


def _case(seed, rows, vocab, dim, dtype, masked=0.3, gain=1.5):
    g = _gen(seed)
    w = (gain / math.sqrt(dim) * torch.randn(vocab, dim, generator=g)).to(dtype)
    tok = torch.randint(0, vocab, (rows,), generator=g)
    h = (torch.randn(rows, dim, generator=g) + w[tok].float()).to(dtype)
    mask = torch.rand(rows, generator=g) >= masked
    if rows > 5:
        tok[1], tok[4] = -1, vocab
    return dict(h=h, w=w, tok=tok, mask=mask)


def _run(ops, d, temperature=1.0, denom=None, mask=True, grads=(True, True)):
    dh = torch.full_like(d["h"], 3.0) if grads[0] else None
    dw = torch.full_like(d["w"], 3.0) if grads[1] else None
    stats, lp, ent = (torch.full((n,), 3.0, device=d["h"].device) for n in (4, d["h"].shape[0], d["h"].shape[0]))
    ops.linear_cross_entropy(d["h"], d["w"], d["tok"], dh, dw, stats, logp=lp, entropy=ent, mask=d["mask"] if mask else None, temperature=temperature,
                             denom=denom)
    return dict(d_hidden=dh, d_weight=dw, stats=stats, logp=lp, entropy=ent)


def _within(got, want, bound, what):
    _inside(got, want, bound.cpu(), what)


def _check(s, got, temperature=1.0, denom=None, mask=True):
    dtype, (rows, dim), vocab = s["h"].dtype, s["h"].shape, s["w"].shape[0]
    want = ref.linear_cross_entropy(s["h"], s["w"], s["tok"], s["mask"] if mask else None, temperature, denom)
    h, w = s["h"].double(), s["w"].double()
    z = (h @ w.t()) / temperature
    X = (h.abs() @ w.abs().t()).amax(1)
    dz = (dim + 8 + (8 if dtype == F32 else 0)) * U * X / temperature
    E = U * (4 * (z - z.amax(1, keepdim=True)).abs().clamp(max=110).amax(1) + vocab / 256 + 64)
    zmax = (z - z.amax(1, keepdim=True)).abs().clamp(max=110).amax(1)
    counts = want["logp"] != 0
    at = torch.where(counts | (want["entropy"] != 0), 2 * dz + E, torch.zeros_like(E))
    _within(got["logp"], want["logp"], at + U * want["logp"].abs(), "logp")
    _within(got["entropy"], want["entropy"], at * (2 + zmax), "entropy")
    n = float(want["stats"][2]) if denom is None else denom
    _within(got["stats"][:1], want["stats"][:1], (at + U * want["logp"].abs()).sum()[None] / max(n, 1e-30) + 2 * U * want["stats"][:1].abs(), "loss")
    _within(got["stats"][1:2], want["stats"][1:2], (at * (2 + zmax)).sum()[None] / max(n, 1e-30) + 2 * U * want["stats"][1:2].abs(), "mean entropy")
    assert float(got["stats"][2]) == float(want["stats"][2]) and float(got["stats"][3]) == 0.0
    k = 1.0 / (max(n, 1.0) if denom is None else n) / temperature
    p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
    small = 2.0**-25 / 16384 if dtype == F16 else 0.0
    off = torch.where((want["d"] != 0).any(1)[:, None], p * (2 * dz + E)[:, None] + 1.01 * HALF[dtype] * want["d"].abs() + small, torch.zeros_like(p))
    safe = torch.where((want["d"] != 0).any(1)[:, None], h, torch.zeros_like(h))
    if got["d_hidden"] is not None:
        bound = k * (off @ w.abs() + (vocab + 64) * U * (want["d"].abs() @ w.abs()))
        _within(got["d_hidden"], want["d_hidden"], bound + (1.01 * HALF[dtype] + 4 * U) * want["d_hidden"].abs() + TINY[dtype], "d_hidden")
    if got["d_weight"] is not None:
        bound = k * (off.t() @ safe.abs() + (rows + 64) * U * (want["d"].abs().t() @ safe.abs()))
        _within(got["d_weight"], want["d_weight"], bound + (1.01 * HALF[dtype] + 4 * U) * want["d_weight"].abs() + TINY[dtype], "d_weight")


SIZES = [(1, 1, 1), (1, 7, 3), (2, 255, 64), (8, 1000, 128), (33, 256, 65), (32, 257, 8), (100, 513, 200), (129, 2049, 64), (300, 1000, 40), (700, 515, 77),
         (5, 33000, 8), (64, 5001, 128), (260, 300, 320)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocab,dim", SIZES)
def test_loss_and_gradients(cuda, rows, vocab, dim, dtype):
    ops = _ops()
    s = _case(rows + vocab, rows, vocab, dim, dtype)
    d = {k: v.to(cuda) for k, v in s.items()}
    got = _run(ops, d, temperature=0.8)
    _check(s, got, temperature=0.8)
    again = _run(ops, d, temperature=0.8)
    assert all(torch.equal(got[k], again[k]) for k in got)
    lp, ent = torch.empty(rows, device=cuda), torch.empty(rows, device=cuda)
    ops.linear_log_probs(d["h"], d["w"], d["tok"], lp, ent, mask=d["mask"], temperature=0.8)
    assert torch.equal(lp, got["logp"]) and torch.equal(ent, got["entropy"])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_options(cuda, dtype):
    """No mask, int32 tokens, a given denominator; one gradient at a time; the same as both."""
    ops = _ops()
    s = _case(1, 90, 700, 72, dtype)
    s["tok"] = s["tok"].to(torch.int32)
    d = {k: v.to(cuda) for k, v in s.items()}
    got = _run(ops, d, 1.7, denom=33.5, mask=False)
    _check(s, got, 1.7, denom=33.5, mask=False)
    one, other = _run(ops, d, 1.7, 33.5, False, (True, False)), _run(ops, d, 1.7, 33.5, False, (False, True))
    assert torch.equal(one["d_hidden"], got["d_hidden"]) and torch.equal(other["d_weight"], got["d_weight"])
    assert torch.equal(_run(ops, d, 1.7, 33.5, False, (False, False))["stats"], got["stats"])
    lp = torch.empty(90, device=cuda)
    ops.linear_log_probs(d["h"], d["w"], d["tok"], lp, temperature=1.7)
    assert torch.equal(lp, got["logp"])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views(cuda, dtype):
    """Rows apart and off their alignment; nothing outside the outputs' columns is written."""
    ops = _ops()
    s = _case(2, 40, 300, 64, dtype)
    d = {k: v.to(cuda) for k, v in s.items()}
    want = _run(ops, d)
    h = torch.zeros(40 * 71 + 1, dtype=dtype, device=cuda)[1:].view(40, 71)[:, 3:67].copy_(d["h"])
    w = torch.zeros(300 * 69 + 1, dtype=dtype, device=cuda)[1:].view(300, 69)[:, 1:65].copy_(d["w"])
    dh, dw = torch.full((40, 67), 9.0, dtype=dtype, device=cuda), torch.full((300, 70), 9.0, dtype=dtype, device=cuda)
    stats = torch.empty(4, device=cuda)
    ops.linear_cross_entropy(h, w, d["tok"], dh[:, 1:65], dw[:, 3:67], stats, mask=d["mask"])
    assert torch.equal(dh[:, 1:65], want["d_hidden"]) and torch.equal(dw[:, 3:67], want["d_weight"]) and torch.equal(stats, want["stats"])
    assert bool((dh[:, 0] == 9).all()) and bool((dh[:, 65:] == 9).all()) and bool((dw[:, :3] == 9).all()) and bool((dw[:, 67:] == 9).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows", [0, 1, 40, 200])
def test_no_row_counts(cuda, rows, dtype):
    ops = _ops()
    s = _case(3, rows, 600, 64, dtype)
    d = {k: v.to(cuda) for k, v in s.items()}
    d["mask"].zero_()
    d["h"].fill_(math.nan)  # not read
    got = _run(ops, d)
    for k, x in got.items():
        assert not bool(x.any()), k


def test_rows_that_do_not_count_are_not_read(cuda):
    ops = _ops()
    s = _case(4, 150, 400, 64, BF16)
    d = {k: v.to(cuda) for k, v in s.items()}
    want = _run(ops, d)
    out = ~(d["mask"] & (d["tok"] >= 0) & (d["tok"] < 400))
    d["h"][out] = math.nan
    got = _run(ops, d)
    assert all(torch.equal(got[k], want[k]) for k in got)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_peaked_and_far_logits(cuda, dtype):
    """Rows whose probability is all at one token, and logits of some hundreds."""
    ops = _ops()
    s = _case(5, 60, 500, 64, dtype, gain=1.5)
    s["h"][:20] = (40 * s["h"][:20].float()).to(dtype)
    d = {k: v.to(cuda) for k, v in s.items()}
    _check(s, _run(ops, d))


# On 256 compute units and tiles of 256 x 256 (fp32: 128 rows): fewer than half a round of d_hidden's tiles, cut along the columns; more, some of whose columns go
# to the units left over, one and two of them and in two pieces of the vocabulary; a whole round and some more.
@pytest.mark.parametrize("dtype,rows,vocab,dim", [(BF16, 2500, 1500, 2304), (BF16, 4200, 1500, 2304), (F16, 4200, 1300, 2300), (F32, 2100, 1500, 2304),
                                                  (BF16, 5900, 40000, 2304), (BF16, 9000, 1500, 2304), (F32, 4500, 1025, 2100)])
def test_many_tiles(cuda, dtype, rows, vocab, dim):
    ops = _ops()
    d = {k: v.to(cuda) for k, v in _case(rows, rows, vocab, dim, dtype, masked=0.02).items()}
    got = _run(ops, d)
    _check(d, got)
    again = _run(ops, d)
    assert all(torch.equal(got[k], again[k]) for k in got)
