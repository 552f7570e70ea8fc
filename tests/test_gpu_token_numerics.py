"""Values of the token loss where fp32 loses them easily: logits far from zero, and a policy close to its reference.  The bars
are those of tests/test_gpu_token_ops.py, which go by how far logits lie below their row's largest and by nothing else."""

from __future__ import annotations

import math

import pytest
import torch

from tests import token_reference as ref
from tests.test_gpu_token_ops import BF16, F16, F32, HALF, INF, TINY, U, _gen, _inside, _loss_error, _ops

pytestmark = pytest.mark.gpu

T, KL, ENT, CLIP = 0.8, 0.1, 0.02, (0.2, 0.3)


def _check(cuda, x, tok, seed=0):
    """Log-probabilities, entropy, stats and gradient of the logits against the 64-bit form, and log-probabilities alone."""
    ops, g, dtype, (rows, vocab) = _ops(), _gen(seed), x.dtype, x.shape
    at = torch.arange(rows)
    z = x.double() / T
    lp = torch.log_softmax(z, 1)[at, tok]
    step = (0.2 * torch.randn(rows, generator=g, dtype=torch.float64)).clamp(-0.15, 0.15)  # (inside the clip range)
    old, refs = (lp - step).float(), (lp + 0.3 * torch.randn(rows, generator=g).double()).float()
    adv = torch.randn(rows, generator=g)
    want = ref.token_loss(x, tok, old, adv, refs, None, CLIP, KL, ENT, T)
    d = lambda t: t.to(cuda)  # noqa: E731
    dx = torch.full((rows, vocab), 5.0, dtype=dtype, device=cuda)
    got_lp, h, stats = (torch.full((n,), 5.0, device=cuda) for n in (rows, rows, 8))
    print(f"loss {dtype} {rows} x {vocab}", flush=True)
    ops.token_ppo_loss(d(x), d(tok), d(old), d(adv), dx, stats, ref_logp=d(refs), logp=got_lp, entropy=h, clip_param=CLIP, kl_coef=KL,
                       entropy_coef=ENT, temperature=T)
    e = _loss_error(x, vocab, T)
    _inside(got_lp, want["logp"], e * (1 + want["logp"].abs()), "logp")
    _inside(h, want["entropy"], e * (1 + want["entropy"].abs()), "entropy")
    size = (1 + float(adv.abs().max())) * 2.5 * (1 + float(want["entropy"].abs().max())) * 8
    _inside(stats[:6], want["stats"], size * e + 2 * U * want["stats"].abs(), "stats")
    row = want["d_logits"].abs().amax(1, keepdim=True) + size / rows
    _inside(dx, want["d_logits"], e * row + 1.01 * HALF[dtype] * want["d_logits"].abs() + TINY[dtype], "d_logits")
    ops.token_log_probs(d(x), d(tok), got_lp, h, temperature=T)
    _inside(got_lp, want["logp"], e * (1 + want["logp"].abs()), "logp alone")
    _inside(h, want["entropy"], e * (1 + want["entropy"].abs()), "entropy alone")


# one wave a row, several, parts of a row, rows too wide for the registers
WIDTHS = [(7, 3), (9, 50), (70, 1000), (66, 9000), (5, 50021), (66, 20011)]
WIDE = [(66, F32, 110003), (66, BF16, 210005)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocab", WIDTHS)
def test_common_offset(cuda, dtype, rows, vocab):
    """The same number added to all logits of a row changes nothing but their rounding."""
    g = _gen(rows + vocab)
    offsets = torch.tensor([1e2, -1e3, 1e4, -3e4, 6e4, -6e4] + ([1e5, -1e6, 1e6, -3e6] if dtype != F16 else []))
    x = (torch.randn(rows, vocab, generator=g) * 2 + offsets[torch.arange(rows) % len(offsets)][:, None]).to(dtype)
    near = x.double() >= x.double().amax(1, keepdim=True) - 8  # (a token of probability 0 has no ratio)
    _check(cuda, x, torch.where(near, torch.rand(rows, vocab, generator=g), -1.0).argmax(1))


def _masked(rows, vocab, dtype):
    """Rows masked by finite values: all of a row, its first half, all but a few columns, all but one."""
    g = _gen(rows * 3 + vocab)
    lows = [-1e4, -65504.0] if dtype == F16 else [-1e4, -65504.0, -1e6, -1e9, -1e10, -1e12, -1e15, -1e30, torch.finfo(dtype).min]
    x = torch.randn(rows, vocab, generator=g) * 2
    tok = torch.randint(0, vocab, (rows,), generator=g)
    for r in range(rows):
        low, kind = lows[r % len(lows)], (r // len(lows)) % 4 if rows > 4 * len(lows) else (r + vocab) % 4
        keep = torch.zeros(vocab, dtype=torch.bool)
        if kind == 1:
            keep[vocab // 2:] = True
        elif kind == 2:
            keep[torch.randint(0, vocab, (5,), generator=g)] = True
        elif kind == 3:
            keep[vocab - 1] = True
        x[r, ~keep] = low
        if bool(keep.any()):
            at = keep.nonzero()[:, 0]
            tok[r] = at[int(torch.randint(0, len(at), (1,), generator=g))]
    return x.to(dtype), tok


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocab", WIDTHS)
def test_masks_of_finite_values(cuda, dtype, rows, vocab):
    _check(cuda, *_masked(rows, vocab, dtype))


@pytest.mark.parametrize("rows,dtype,vocab", WIDE)
def test_wide_rows(cuda, rows, dtype, vocab):
    x, tok = _masked(rows, vocab, dtype)
    x[::7] = (torch.randn(len(x[::7]), vocab, generator=_gen(1)) * 2 + 1e4).to(dtype)
    _check(cuda, x, tok)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(12, 40), (12, 3001), (12, 40000), (70, 17001)])
def test_large_logits_next_to_each_other(cuda, dtype, rows, vocab):
    """Logits whose neighbours in the type lie far apart: the largest ones share the row, the next lower value has none."""
    g = _gen(vocab)
    base = torch.tensor([1e7, 1e8, 1e9, -1e9, 1e10, -1e10, 1e13, -1e13, 1e20, -1e20, 1e36, -1e36])[torch.arange(rows) % 12].to(dtype)
    down = torch.nextafter(base, torch.full_like(base, -INF))
    low = torch.nextafter(down, torch.full_like(base, -INF))
    x = torch.stack([base, down, low], 1).gather(1, torch.randint(0, 3, (rows, vocab), generator=g))
    x[:, vocab // 2] = base
    tok = torch.full((rows,), vocab // 2)
    tok[::5] = torch.randint(0, vocab, (len(tok[::5]),), generator=g)
    near = x[torch.arange(rows), tok] == base  # (a token of probability 0 has no ratio)
    tok[~near] = vocab // 2
    _check(cuda, x, tok)


@pytest.mark.parametrize("vocab", [1000, 20011, 50021])
def test_infinite_logits_beside_masks(cuda, vocab):
    """+inf makes a row's results NaN, also where the rest of it is masked; the other rows keep theirs."""
    ops = _ops()
    x = torch.randn(66, vocab, generator=_gen(vocab))
    x[3, :] = -1e10
    x[3, vocab // 3] = INF
    x[4, : vocab // 2] = -1e10
    lp, h = torch.empty(66, device=cuda), torch.empty(66, device=cuda)
    tok = torch.full((66,), vocab - 1)
    ops.token_log_probs(x.to(cuda), tok.to(cuda), lp, h)
    bad = torch.isnan(h).cpu()
    assert bad.nonzero()[:, 0].tolist() == [3]
    want = torch.log_softmax(x.double(), 1)[:, vocab - 1]
    err = (lp.cpu().double() - want).abs()[~bad]
    assert float(err.max()) < _loss_error(x[:3], vocab, 1.0) * (1 + float(want[~bad].abs().max()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [50, 9000, 16384, 20011, 50021, 65536, 100003, 131072, 140001])
def test_means_are_of_the_returned_values(cuda, dtype, vocab):
    """One row that counts among others: its means are the logp and entropy that the call returns, to the bit, also where a row's
    parts are joined by several blocks and its means by another."""
    ops, g, rows = _ops(), _gen(vocab), 40
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).to(cuda)
    tok = torch.randint(0, vocab, (rows,), generator=g).to(cuda)
    zero, lp, h, stats = torch.zeros(rows, device=cuda), torch.empty(rows, device=cuda), torch.empty(rows, device=cuda), torch.empty(8, device=cuda)
    for r in range(0, rows, 3):
        mask = torch.zeros(rows, dtype=torch.bool, device=cuda)
        mask[r] = True
        ops.token_ppo_loss(x, tok, zero, zero, torch.empty_like(x), stats, logp=lp, entropy=h, mask=mask)
        assert (float(stats[5]), float(stats[3])) == (-float(lp[r]), float(h[r]))


def _near_reference(cuda, vocab, sizes):
    """logp as the loss itself computes it, and a reference that lies d from it, exactly."""
    ops, g, rows = _ops(), _gen(vocab), len(sizes)
    x = (torch.randn(rows, vocab, generator=g)).to(cuda)
    tok = torch.randint(0, vocab, (rows,), generator=g).to(cuda)
    lp, stats, zero = torch.empty(rows, device=cuda), torch.empty(8, device=cuda), torch.zeros(rows, device=cuda)
    ops.token_ppo_loss(x, tok, zero, zero, torch.empty_like(x), stats, logp=lp)
    refs = (lp.double() + sizes.to(cuda).double()).float()
    return x, tok, lp, refs, refs.double() - lp.double()  # (fp32's own difference is exact: they lie within a factor of 2)


@pytest.mark.parametrize("vocab", [64, 700, 20011])
@pytest.mark.parametrize("size", [1e-6, 1e-5, 1e-4, 1e-3, 1e-2, 0.2, 0.3, 0.9])
def test_kl_near_the_reference(cuda, vocab, size):
    """k = exp(d) - d - 1 to 16 U of itself and never negative (a polynomial: 8 operations; exp - 1 less d: U |exp(d) - 1| / k, 9 U
    from d = 0.25 on), its derivative 1 - exp(d) to 8 U, the mean to two roundings more."""
    ops, rows = _ops(), 48
    sizes = size * (1 + torch.rand(rows, generator=_gen(5))) * torch.where(torch.arange(rows) % 2 == 0, 1.0, -1.0)
    x, tok, lp, refs, d = _near_reference(cuda, vocab, sizes)
    dx, stats, zero = torch.empty_like(x), torch.empty(8, device=cuda), torch.zeros(rows, device=cuda)
    ops.token_ppo_loss(x, tok, lp, zero, dx, stats, ref_logp=refs, kl_coef=1.0)
    # exp(d) - d - 1 in 64 bits, by its series where that is the closer one
    k = torch.where(d.abs() < 1e-2, d * d * (0.5 + d * (1 / 6 + d * (1 / 24 + d * (1 / 120 + d / 720)))), torch.expm1(d) - d)
    assert abs(float(stats[2]) - float(k.mean())) <= 18 * U * float(k.mean())
    assert float(stats[0]) == float(stats[2])
    p = torch.softmax(x.double(), 1)
    at = torch.arange(rows, device=cuda)
    g = -torch.expm1(d)[:, None]
    want = -g * p
    want[at, tok] += g[:, 0]
    e = _loss_error(x.cpu(), vocab, 1.0)
    _inside(dx, want / rows, (e * (p + torch.nn.functional.one_hot(tok, vocab)) * g.abs() + 16 * U * g.abs() * p.amax(1, keepdim=True)).cpu()
            / rows * 2, "d_logits")
    # every row by itself: none is negative
    for r in range(0, rows, 7):
        one = slice(r, r + 1)
        ops.token_ppo_loss(x[one], tok[one], lp[one], zero[one], None, stats, ref_logp=refs[one], kl_coef=1.0)
        assert float(stats[2]) > 0.0


@pytest.mark.parametrize("vocab", [64, 20011])
def test_kl_that_is_only_reported(cuda, vocab):
    """kl_coef = 0 with a reference so far off that k is infinite: the loss and its gradient are those without a reference."""
    ops, g, rows = _ops(), _gen(vocab), 9
    x = torch.randn(rows, vocab, generator=g).to(cuda)
    tok, adv = torch.randint(0, vocab, (rows,), generator=g).to(cuda), torch.randn(rows, generator=g).to(cuda)
    old, refs = torch.full((rows,), -math.log(vocab), device=cuda), torch.full((rows,), 100.0, device=cuda)
    out = []
    for reference in (None, refs):
        dx, stats = torch.empty_like(x), torch.empty(8, device=cuda)
        ops.token_ppo_loss(x, tok, old, adv, dx, stats, ref_logp=reference, entropy_coef=0.01)
        out.append((dx, stats))
    assert torch.equal(out[0][0], out[1][0]) and bool(torch.isfinite(out[1][0]).all())
    assert float(out[1][1][2]) == INF and float(out[0][1][2]) == 0.0
    keep = [0, 1, 3, 4, 5, 6, 7]
    assert torch.equal(out[0][1][keep], out[1][1][keep])
