"""The token operators (embedding, token log-probabilities and loss, AdamW over many tensors) against the 64-bit forms of
tests/token_reference.py.

Bars.  u is the rounding of the output's type (2^-24, 2^-8, 2^-11 of the value: significands of 24, 8 and 11
bits), U = 2^-24 that of fp32.
  lookup     one product: U + u of the value.
  gradient   a sum of n terms in fp32: (n + 2) U of the sum of magnitudes, + u of the value.
  loss       z = (x - max) c has two roundings, so exp and log of it are off by 4 U max|z| or less; the sums run over at most
             vocab / 256 + 16 terms in a row: E = U (4 max|z| + vocab / 256 + 64) relative for probabilities, absolute for
             logp and H / (1 + H), with max|z| over the logits that count for anything (z > -110).  The loss' terms carry
             exp(logp - old): (1 + |A|) (1 + ratio) E; gradients E of their row's largest scale, + u of the value.
  AdamW      ten operations on values below the state's magnitude: 16 U of |value| + |change| for p, 4 U for m and v (3e-6
             where a clip coefficient, rounded twice, enters).
"""

from __future__ import annotations

import math

import pytest
import torch

from tests import token_reference as ref

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0**-25}  # half the smallest step near zero
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")


def _ops():
    from tt_rsl_rl_amd import _lib, ops

    _lib.load()
    return ops


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _zipf(n, vocab, g):
    return ((torch.rand(n, generator=g, dtype=torch.float64) * math.log(vocab + 1)).exp() - 1).long().clamp(0, vocab - 1)


def _inside(got, want, bound, what):
    got, want = got.detach().double().cpu(), want.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    over = ((got - want).abs() - bound).nan_to_num(nan=-1.0)
    assert bool((over <= 0).all()), f"{what}: {float(over.max()):.3g} past the bound at {int(over.argmax())}"


# ---- embedding ----


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("count,vocab,dim", [(1, 1, 1), (1, 7, 3), (3, 11, 8), (8, 1000, 64), (130, 513, 515), (1021, 300, 1024),
                                             (33, 50, 4099)])
def test_embedding_lookup(cuda, dtype, count, vocab, dim):
    ops, g = _ops(), _gen(count + dim)
    table = torch.randn(vocab, dim, generator=g).to(dtype)
    tok = torch.randint(0, vocab, (count,), generator=g)
    for i, bad in enumerate((-100, vocab, 2**40)):
        if count > 4 * i + 4:
            tok[4 * i + 2] = bad
    out = torch.full((count, dim), 7.0, dtype=dtype, device=cuda)
    ops.embedding_fwd(tok.to(cuda), table.to(cuda), out, scale=1.7)
    want = ref.embedding(tok, table, 1.7)
    _inside(out, want, (U + HALF[dtype]) * 1.01 * want.abs() + TINY[dtype], "lookup")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embedding_lookup_of_views(cuda, dtype):
    """Rows apart, off their alignment, 2-D int32 tokens; nothing outside the output's columns is written."""
    ops, g = _ops(), _gen(3)
    store = torch.randn(40 * 37 + 1, generator=g).to(dtype)
    dev = store.to(cuda)
    table = dev[1:].view(40, 37)[:, 2:31]
    tok = torch.randint(-1, 41, (5, 9), generator=g, dtype=torch.int32)
    full = torch.full((45, 33), 5.0, dtype=dtype, device=cuda)
    ops.embedding_fwd(tok.to(cuda), table, full[:, 1:30], scale=0.5)
    want = ref.embedding(tok, store[1:].view(40, 37)[:, 2:31], 0.5)
    assert torch.equal(full[:, 1:30].cpu().double(), want)  # a half is exact
    assert bool((full[:, 0] == 5).all()) and bool((full[:, 30:] == 5).all())
    ops.embedding_fwd(tok[:0].to(cuda), table, full[:0, 1:30])


GRADS = [(1, 1, 1), (1, 3, 5), (31, 2, 7), (64, 5, 3), (500, 1, 16), (4096, 300, 40), (4097, 300, 40), (20000, 10, 33),
         (5003, 10007, 515), (9000, 70000, 24), (3000, 1_100_000, 2), (10000, 513, 257)]


def _grad_case(count, vocab, dim, dtype, seed=0):
    g = _gen(seed + count + vocab)
    tok = _zipf(count, vocab, g)
    if count > 20:
        tok[5], tok[17], tok[count // 2] = -100, vocab, vocab - 1
    return tok, torch.randn(count, dim, generator=g).to(dtype)


def _grad_bound(tok, d, vocab, scale, out_dtype, extra=0.0):
    want, size = ref.embedding_grad(tok, d, vocab, scale)
    n = torch.bincount(tok[(tok >= 0) & (tok < vocab)], minlength=vocab).double()[:, None]
    return want, (n + 3) * U * (size + extra) + 1.01 * HALF[out_dtype] * (want.abs() + extra) + TINY[out_dtype]


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("count,vocab,dim", GRADS)
def test_embedding_gradient(cuda, dtype, out, count, vocab, dim):
    ops = _ops()
    tok, d = _grad_case(count, vocab, dim, dtype)
    got = torch.full((vocab, dim), 9.0, dtype=out, device=cuda)
    ops.embedding_bwd(tok.to(cuda), d.to(cuda), got, scale=1.3)
    want, bound = _grad_bound(tok, d, vocab, 1.3, out)
    _inside(got, want, bound, "gradient")
    again = torch.empty_like(got)
    ops.embedding_bwd(tok.to(cuda), d.to(cuda), again, scale=1.3)
    assert torch.equal(got, again), "the same call gives the same bits"


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dim,most", [(24, 2000), (1100, 6000), (1100, 60000), (4100, 40000)])
def test_embedding_gradient_of_runs(cuda, dim, most, accumulate):
    """Tokens that occur 0, 1, 7, 8, 9, ... times, so that runs of the sorted tokens end on, before and behind every boundary the
    kernels cut them at; small whole numbers, whose sums are exact in fp32."""
    ops, g = _ops(), _gen(dim + most)
    lens = torch.tensor([0, 1, 2, 3, 7, 8, 9, 10, 15, 16, 17, 23, 24, 25, 31, 32, 33, 39, 40, 41, 64, 300, 900])
    lens = lens[torch.randint(0, len(lens), (4000,), generator=g)]
    lens = lens[: int((lens.cumsum(0) <= most).sum())]
    tok = torch.repeat_interleave(torch.arange(len(lens)), lens)
    tok = tok[torch.randperm(len(tok), generator=g)]
    d = torch.randint(-3, 4, (len(tok), dim), generator=g).to(BF16)
    start = torch.randint(-3, 4, (len(lens), dim), generator=g).float()
    got = start.to(cuda)
    ops.embedding_bwd(tok.to(cuda), d.to(cuda), got, scale=2.0, accumulate=accumulate)
    want = torch.zeros(len(lens), dim).index_add(0, tok, d.float()) * 2.0 + (start if accumulate else 0.0)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("count,vocab,dim,out", [(1, 4, 3, F32), (700, 90, 37, BF16), (9001, 40, 130, F32)])
def test_embedding_gradient_accumulates(cuda, count, vocab, dim, out):
    ops = _ops()
    tok, d = _grad_case(count, vocab, dim, BF16, seed=5)
    start = torch.randn(vocab, dim, generator=_gen(9)).to(out)
    got = start.to(cuda)
    ops.embedding_bwd(tok.to(cuda).int(), d.to(cuda), got, scale=0.7, accumulate=True)
    want, bound = _grad_bound(tok, d, vocab, 0.7, out, extra=start.double().abs())
    _inside(got, want + start.double(), bound, "accumulated gradient")
    empty = torch.bincount(tok[(tok >= 0) & (tok < vocab)], minlength=vocab) == 0
    assert torch.equal(got.cpu()[empty], start[empty])


def test_embedding_gradient_of_views_and_of_no_tokens(cuda):
    ops, g = _ops(), _gen(11)
    tok = torch.randint(0, 30, (333,), generator=g)
    d = torch.randn(333 * 50 + 3, generator=g)
    dev = d.to(cuda)
    full = torch.full((30, 41), 3.0, device=cuda)
    ops.embedding_bwd(tok.to(cuda), dev[3:].view(333, 50)[:, 1:40], full[:, 1:40], scale=2.0)
    want, bound = _grad_bound(tok, d[3:].view(333, 50)[:, 1:40], 30, 2.0, F32)
    _inside(full[:, 1:40], want, bound, "gradient of views")
    assert bool((full[:, 0] == 3).all()) and bool((full[:, 40:] == 3).all())
    none = torch.zeros(0, dtype=torch.int64, device=cuda)
    ops.embedding_bwd(none, dev[:0].view(0, 39), full[:, 1:40], accumulate=True)
    _inside(full[:, 1:40], want, bound, "nothing added")
    ops.embedding_bwd(none, dev[:0].view(0, 39), full[:, 1:40])
    assert bool((full[:, 1:40] == 0).all()) and bool((full[:, 0] == 3).all())
    ops.embedding_bwd(torch.full((100,), -1, device=cuda), dev[:3900].view(100, 39), full[:, 1:40])
    assert bool((full[:, 1:40] == 0).all())


def test_embedding_past_32_bits(cuda):
    ops = _ops()
    vocab, dim = 600_000, 4096  # 2.46e9 elements
    table = torch.zeros(vocab, dim, dtype=BF16, device=cuda)
    table[-3:] = torch.arange(1, 4, device=cuda)[:, None].to(BF16)
    tok = torch.tensor([vocab - 1, 5, vocab - 3], device=cuda)
    out = torch.empty(3, dim, dtype=BF16, device=cuda)
    ops.embedding_fwd(tok, table, out, scale=2.0)
    assert out.float().mean(1).tolist() == [6.0, 0.0, 2.0]
    ops.embedding_bwd(tok, out, table)
    assert table[-3:].float().mean(1).tolist() == [2.0, 0.0, 6.0] and float(table[5:].float().abs().amax(1)[: vocab - 8].max()) == 0.0


# ---- log-probabilities and loss ----


def _loss_case(rows, vocab, dtype, masked, banned, seed=0, temperature=1.0):
    g = _gen(seed + rows * 7 + vocab)
    x = (torch.randn(rows, vocab, generator=g) * 2).to(dtype)
    tok = torch.randint(0, vocab, (rows,), generator=g)
    at = torch.arange(rows)
    if banned and vocab > 2:
        keep = x[at, tok].clone()
        x[:, torch.rand(vocab, generator=g) < 0.4] = -INF
        x[at, tok] = keep
    x[at, tok] += 3
    lp = torch.log_softmax(x.double() / temperature, 1)[at, tok]
    step = 0.2 * torch.randn(rows, generator=g, dtype=torch.float64)
    for end in (math.log(0.8), math.log(1.3)):  # the clip's ends: their sides are not left to roundings
        step = torch.where((step - end).abs() < 1e-3, torch.full_like(step, end + 1e-3), step)
    mask = torch.rand(rows, generator=g) >= masked if masked else None
    return x, tok, (lp - step).float(), torch.randn(rows, generator=g), (lp + 0.3 * torch.randn(rows, generator=g).double()).float(), mask


def _loss_error(x, vocab, temperature):
    z = (x.double() - x.double().amax(1, keepdim=True)) / temperature
    top = float(torch.where(z > -110, -z, torch.zeros_like(z)).nan_to_num(0.0).max())
    return U * (4 * top / math.log(2) + vocab / 256 + 64)


MANY = [(129, 7), (130, 600), (129, 3001), (131, 9000), (129, 20001), (130, 40000), (129, 70001), (129, 131072), (129, 140001)]
SHAPES = [(1, 1), (1, 2), (2, 5), (3, 64), (5, 1000), (64, 257), (9, 4096), (4, 32000), (3, 50021), (2, 131072), (300, 77)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("masked,banned", [(0.0, False), (0.4, True)])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_token_loss(cuda, dtype, masked, banned, rows, vocab):
    ops = _ops()
    T, kl, ent, clip = 0.8, 0.1, 0.02, (0.2, 0.3)
    x, tok, old, adv, refs, mask = _loss_case(rows, vocab, dtype, masked, banned, temperature=T)
    want = ref.token_loss(x, tok, old, adv, refs, mask, clip, kl, ent, T)
    d = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    dx = torch.full((rows, vocab), 5.0, dtype=dtype, device=cuda)
    lp, h, stats = (torch.full((n,), 5.0, device=cuda) for n in (rows, rows, 8))
    ops.token_ppo_loss(d(x), d(tok), d(old), d(adv), dx, stats, ref_logp=d(refs), logp=lp, entropy=h, mask=d(mask), clip_param=clip,
                       kl_coef=kl, entropy_coef=ent, temperature=T)
    e = _loss_error(x, vocab, T)
    _inside(lp, want["logp"], e * (1 + want["logp"].abs()), "logp")
    _inside(h, want["entropy"], e * (1 + want["entropy"].abs()), "entropy")
    a, ratio = float(adv.abs().max()), float((want["logp"] - old.double()).exp().max())
    size = (1 + a) * (1 + ratio) * (1 + float(want["entropy"].abs().max())) * 8
    _inside(stats[:6], want["stats"], size * e + 2 * U * want["stats"].abs(), "stats")
    n = int(ref.rows_that_count(tok, vocab, mask).sum())
    assert float(stats[6]) == n
    row = want["d_logits"].abs().amax(1, keepdim=True) + size / max(1, n)
    _inside(dx, want["d_logits"], e * row + 1.01 * HALF[dtype] * want["d_logits"].abs() + TINY[dtype], "d_logits")
    lp2, h2 = torch.empty_like(lp), torch.empty_like(h)
    ops.token_log_probs(d(x), d(tok.int()), lp2, h2, mask=d(mask), temperature=T)
    _inside(lp2, want["logp"], e * (1 + want["logp"].abs()), "logp alone")
    _inside(h2, want["entropy"], e * (1 + want["entropy"].abs()), "entropy alone")
    # the same bits again, in place, without the outputs that may be left out
    y, s2 = d(x).clone(), torch.empty_like(stats)
    ops.token_ppo_loss(y, d(tok), d(old), d(adv), y, s2, ref_logp=d(refs), mask=d(mask), clip_param=clip, kl_coef=kl, entropy_coef=ent,
                       temperature=T)
    assert torch.equal(y, dx) and torch.equal(s2, stats)
    ops.token_ppo_loss(d(x), d(tok), d(old), d(adv), None, s2, ref_logp=d(refs), mask=d(mask), clip_param=clip, kl_coef=kl,
                       entropy_coef=ent, temperature=T)
    _inside(s2[:6], want["stats"], size * e + 2 * U * want["stats"].abs(), "stats without gradient")
    ops.token_log_probs(d(x), d(tok), lp2, temperature=T)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", MANY)
def test_token_loss_of_many_rows(cuda, dtype, rows, vocab):
    """More rows than a row each is worth cutting into parts."""
    test_token_loss(cuda, dtype, 0.6, True, rows, vocab)


@pytest.mark.parametrize("rows", [2049, 5000])
def test_token_loss_counts_many_rows(cuda, rows):
    """So many rows that a launch of its own counts them."""
    test_token_loss(cuda, F32, 0.4, False, rows, 30)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [37, 4100, 70001])
def test_token_loss_of_views_and_odd_rows(cuda, dtype, vocab):
    """Logits in rows apart and off their alignment; rows that do not count hold NaN, and their gradient is 0."""
    ops = _ops()
    rows, pad = 12, 5
    x, tok, old, adv, refs, _ = _loss_case(rows, vocab, dtype, 0.0, False, seed=4)
    mask = torch.ones(rows, dtype=torch.uint8)
    mask[3] = 0
    tok[5], tok[6] = -100, vocab
    x[7] = -INF                                                   # no distribution
    x[8] = torch.finfo(dtype).min                                 # uniform: every logit is the type's lowest value
    x[9, : vocab // 2] = torch.finfo(dtype).min                   # a mask of the lowest value
    tok[9] = vocab - 1
    old[8] = refs[8] = -math.log(vocab)
    old[9] = refs[9] = torch.log_softmax(x[9].double(), 0)[vocab - 1].float()
    want = ref.token_loss(x, tok, old, adv, refs, mask, (0.2, 0.2), 0.1, 0.02)
    for r in (3, 5, 6):
        x[r] = float("nan")
        old[r] = adv[r] = refs[r] = float("nan")
    store = torch.zeros(rows * (vocab + pad) + 1, dtype=dtype)
    store[1:].view(rows, -1)[:, 2: 2 + vocab] = x
    dev, out = store.to(cuda), torch.full_like(store, 3.0, device=cuda)
    view = lambda s: s[1:].view(rows, vocab + pad)[:, 2: 2 + vocab]  # noqa: E731
    lp, h, stats = torch.empty(rows, device=cuda), torch.empty(rows, device=cuda), torch.empty(8, device=cuda)
    ops.token_ppo_loss(view(dev), tok.to(cuda), old.to(cuda), adv.to(cuda), view(out), stats, ref_logp=refs.to(cuda), logp=lp, entropy=h,
                       mask=mask.to(cuda), kl_coef=0.1, entropy_coef=0.02)
    e = _loss_error(torch.where(x.isnan(), torch.zeros_like(x), x), vocab, 1.0)
    _inside(lp, want["logp"], e * (1 + want["logp"].abs()), "logp")
    _inside(h, want["entropy"], e * (1 + want["entropy"].abs()), "entropy")
    assert float(stats[6]) == 9.0
    row = want["d_logits"].abs().amax(1, keepdim=True) + 40.0 / 9
    _inside(view(out), want["d_logits"], e * row + 1.01 * HALF[dtype] * want["d_logits"].abs() + 1e-38, "d_logits")
    assert bool((view(out)[[3, 5, 6, 7]] == 0).all())
    edge = out.clone()
    view(edge).fill_(3.0)
    assert bool((edge == 3).all()), "nothing outside the rows is written"


def test_token_loss_with_no_row_that_counts(cuda):
    ops = _ops()
    x = torch.full((4, 50), float("nan"), device=cuda)
    dx, stats, lp, v = torch.ones_like(x), torch.ones(8, device=cuda), torch.ones(4, device=cuda), torch.full((4,), float("nan"), device=cuda)
    ops.token_ppo_loss(x, torch.zeros(4, dtype=torch.int64, device=cuda), v, v, dx, stats, logp=lp, mask=torch.zeros(4, dtype=torch.bool, device=cuda))
    assert float(dx.abs().max()) == 0 and float(stats.abs().max()) == 0 and float(lp.abs().max()) == 0
    stats.fill_(1.0)
    ops.token_ppo_loss(x[:0], torch.zeros(0, dtype=torch.int64, device=cuda), v[:0], v[:0], dx[:0], stats)
    assert float(stats.abs().max()) == 0


@pytest.mark.parametrize("vocab", [100, 40000])
def test_token_loss_nan_stays_in_its_row(cuda, vocab):
    ops = _ops()
    x, tok, old, adv, refs, _ = _loss_case(6, vocab, F32, 0.0, False, seed=8)
    want = ref.token_loss(x, tok, old, adv, refs, None, (0.2, 0.2), 0.1, 0.02)
    x[2, vocab // 3] = float("nan")
    x[4] = -INF
    x[4, vocab - 1] = float("nan")
    lp, h, stats, dx = torch.empty(6, device=cuda), torch.empty(6, device=cuda), torch.empty(8, device=cuda), torch.empty(6, vocab, device=cuda)
    ops.token_ppo_loss(x.to(cuda), tok.to(cuda), old.to(cuda), adv.to(cuda), dx, stats, ref_logp=refs.to(cuda), logp=lp, entropy=h, kl_coef=0.1,
                       entropy_coef=0.02)
    for r in range(6):
        if r in (2, 4):
            assert math.isnan(float(lp[r])) and math.isnan(float(h[r])) and bool(dx[r].isnan().any())
        else:
            assert abs(float(lp[r]) - float(want["logp"][r])) < 1e-4 and not bool(dx[r].isnan().any())
    assert math.isnan(float(stats[0]))


def test_token_loss_denominator_adds_up(cuda):
    """Two halves of a batch with the whole one's row count: losses and gradients of the whole."""
    ops = _ops()
    x, tok, old, adv, refs, mask = _loss_case(64, 900, F32, 0.4, False, seed=2)
    n = float(mask.sum())
    want = ref.token_loss(x, tok, old, adv, refs, mask, (0.2, 0.2), 0.1, 0.02)
    got, total = [], torch.zeros(8, device=cuda)
    for i in (0, 32):
        j = slice(i, i + 32)
        dx, stats = torch.empty(32, 900, device=cuda), torch.empty(8, device=cuda)
        ops.token_ppo_loss(x[j].to(cuda), tok[j].to(cuda), old[j].to(cuda), adv[j].to(cuda), dx, stats, ref_logp=refs[j].to(cuda),
                           mask=mask[j].to(cuda), kl_coef=0.1, entropy_coef=0.02, denom=n)
        got.append(dx)
        total += stats
    e = _loss_error(x, 900, 1.0)
    _inside(torch.cat(got), want["d_logits"], e * (want["d_logits"].abs().amax(1, keepdim=True) + 40 / n) + 1e-38, "d_logits")
    _inside(total[:6], want["stats"], 40 * e, "stats")


def test_token_loss_against_differences(cuda):
    """The gradient against central differences of the loss the kernel itself reports (h^2 / 6 and U / h of 1: under 1e-4)."""
    ops = _ops()
    x, tok, old, adv, refs, _ = _loss_case(3, 9, F32, 0.0, False, seed=6)
    d = [t.to(cuda) for t in (tok, old, adv, refs)]
    dx, stats = torch.empty(3, 9, device=cuda), torch.empty(8, device=cuda)

    def loss(y):
        ops.token_ppo_loss(y.to(cuda), d[0], d[1], d[2], dx, stats, ref_logp=d[3], kl_coef=0.2, entropy_coef=0.1)
        return float(stats[0])

    loss(x)
    grad, h = dx.cpu().clone(), 2.0**-6
    for r in range(3):
        for j in range(9):
            up, down = x.clone(), x.clone()
            up[r, j] += h
            down[r, j] -= h
            assert abs((loss(up) - loss(down)) / (2 * h) - float(grad[r, j])) < 1e-3


def test_token_log_probs_past_32_bits(cuda):
    ops = _ops()
    rows, vocab = 17000, 131072  # 2.2e9 logits
    x = torch.zeros(rows, vocab, dtype=BF16, device=cuda)
    x[-1, 7] = 4.0
    tok = torch.full((rows,), 7, device=cuda)
    lp, h = torch.empty(rows, device=cuda), torch.empty(rows, device=cuda)
    ops.token_log_probs(x, tok, lp, h)
    want = 4.0 - math.log(math.exp(4.0) + vocab - 1)
    assert abs(float(lp[-1]) - want) < 1e-4 and float((lp[:-1] + math.log(vocab)).abs().max()) < 1e-4
    stats = torch.empty(8, device=cuda)
    ops.token_ppo_loss(x, tok, lp, torch.ones(rows, device=cuda), x, stats)
    p = 1 / (math.exp(4.0) + vocab - 1)
    assert abs(float(x[-1, 7]) * rows + 1 - p * math.exp(4.0)) < 0.01 and abs(float(x[-1, 8]) * rows / p - 1) < 0.01


# ---- AdamW ----

SIZES = [1, 3, 4, 255, 256, 257, 1000, 1024, 1025, 5003]


def _adamw_case(sizes, cuda, param, master, grad, seed=0):
    g = _gen(seed)
    p = [torch.randn(n, generator=g) * 0.1 for n in sizes]
    gr = [(torch.randn(n, generator=g) * 0.01).to(grad) for n in sizes]
    m = [torch.randn(n, generator=g) * 1e-3 for n in sizes]
    v = [(torch.randn(n, generator=g) * 1e-3) ** 2 for n in sizes]
    d = lambda ts: [t.to(cuda) for t in ts]  # noqa: E731
    return p, gr, m, v, d([t.to(param) for t in p]), d(gr), d(m), d(v), d(p) if master else None


def _coef(gr, max_norm):
    total = math.sqrt(sum(float(t.double().square().sum()) for t in gr))
    return total, min(1.0, max_norm / (total + 1e-6)) if max_norm else 1.0


@pytest.mark.parametrize("param,master,grad", [(F32, False, F32), (BF16, False, BF16), (BF16, False, F32), (BF16, True, BF16),
                                               (BF16, True, F32)])
@pytest.mark.parametrize("max_norm", [None, 0.05, 100.0])
@pytest.mark.parametrize("repeat", [1, 18])
def test_adamw(cuda, param, master, grad, max_norm, repeat):
    ops = _ops()
    sizes = SIZES * repeat  # 180 tensors: more than a launch takes
    p, gr, m, v, dp, dg, dm, dv, dmaster = _adamw_case(sizes, cuda, param, master, grad)
    lr = [1e-3 * (1 + i % 3) for i in range(len(sizes))]
    wd = [0.1 * (i % 2) for i in range(len(sizes))]
    norm = torch.empty(2, device=cuda)
    ops.adamw_step(dp, dg, dm, dv, step=3, lr=lr, beta1=0.9, beta2=0.99, weight_decay=wd, max_grad_norm=max_norm, masters=dmaster,
                   norm_out=norm)
    total, c = _coef(gr, max_norm)
    assert abs(float(norm[0]) - total) <= 2 * U * total and abs(float(norm[1]) - c) <= 8 * U
    clip = 3e-6 if max_norm else 0.0
    for i, n in enumerate(sizes):
        start = p[i].to(param) if not master else p[i]
        wp, wm, wv = ref.adamw(start, gr[i], m[i], v[i], 3, lr[i], 0.9, 0.99, 1e-8, wd[i], c)
        sm = m[i].double().abs() + gr[i].double().abs()
        sv = v[i].double() + gr[i].double() ** 2
        _inside(dm[i], wm, (4 * U + clip) * sm, f"m {n}")
        _inside(dv[i], wv, (4 * U + clip) * sv, f"v {n}")
        near = (16 * U + clip) * (start.double().abs() + (wp - start.double()).abs()) + 20 * U * lr[i] * sm / (wv.sqrt() + 1e-9) + 1e-12
        if master:
            _inside(dmaster[i], wp, near, f"master {n}")
            assert torch.equal(dp[i], dmaster[i].to(BF16))
        else:
            _inside(dp[i], wp, near + 1.01 * HALF[param] * wp.abs(), f"p {n}")
        assert torch.equal(dg[i].cpu(), gr[i])


def test_adamw_of_unaligned_views_and_empty_tensors(cuda):
    ops = _ops()
    sizes = [5, 0, 300, 1027]
    p, gr, m, v, *_ = _adamw_case(sizes, cuda, BF16, True, BF16, seed=3)
    p = [t.to(BF16).float() for t in p]

    def place(ts, dtype):
        flat = torch.full((sum(sizes) + len(sizes) + 1,), 7.0, dtype=dtype, device=cuda)
        out, at = [], 1
        for t in ts:
            out.append(flat[at:at + t.numel()])
            out[-1].copy_(t)
            at += t.numel() + 1
        return flat, out

    flats, views = zip(*[place(ts, dt) for ts, dt in ((p, BF16), (gr, BF16), (m, F32), (v, F32), (p, F32))])
    ops.adamw_step(list(views[0]), list(views[1]), list(views[2]), list(views[3]), step=1, lr=1e-2, masters=list(views[4]))
    for i, n in enumerate(sizes):
        wp, wm, wv = ref.adamw(p[i], gr[i], m[i], v[i], 1, 1e-2, 0.9, 0.999, 1e-8, 1e-2)
        _inside(views[2][i], wm, 4 * U * (m[i].double().abs() + gr[i].double().abs()), "m")
        _inside(views[4][i], wp, 64 * U * (p[i].double().abs() + (wp - p[i].double()).abs() + 1e-2), "master")
        assert torch.equal(views[0][i], views[4][i].to(BF16))
    for flat in flats:
        at = 0
        for n in sizes:
            assert float(flat[at]) == 7.0
            at += n + 1
        assert float(flat[at]) == 7.0


@pytest.mark.parametrize("param,master,grad", [(F32, False, F32), (BF16, False, BF16), (BF16, True, BF16)])
def test_adamw_states_in_8_bits(cuda, param, master, grad):
    """From the zero state, three steps: what is stored stands for the exact moments of the stored ones to within half a code
    (|m|: scale (q/127)^2, so half a step is sqrt(scale |m|) / 127 + scale / 127^2; v: 4 v^(3/4) scale^(1/4) / 510 and the
    last code's floor), and parameters step by the moments before they are rounded."""
    ops = _ops()
    sizes = [1, 4, 255, 256, 257, 1023, 1025, 5003]
    p, gr, _, _, dp, dg, _, _, dmaster = _adamw_case(sizes, cuda, param, master, grad, seed=4)
    qm = [torch.zeros(n, dtype=torch.int8, device=cuda) for n in sizes]
    qv = [torch.zeros(n, dtype=torch.uint8, device=cuda) for n in sizes]
    sm = [torch.zeros(-(-n // 256), device=cuda) for n in sizes]
    sv = [torch.zeros(-(-n // 256), device=cuda) for n in sizes]
    for step in (1, 2, 3):
        before = [(ref.decode_m(a.cpu(), b.cpu()), ref.decode_v(c.cpu(), d.cpu())) for a, b, c, d in zip(qm, sm, qv, sv)]
        starts = [t.clone().cpu() for t in (dmaster or dp)]
        ops.adamw_step(dp, dg, qm, qv, step=step, lr=1e-3, weight_decay=0.1, max_grad_norm=0.2, masters=dmaster, scales=(sm, sv))
        _, c = _coef(gr, 0.2)
        for i, n in enumerate(sizes):
            m, v = before[i]
            wp, wm, wv = ref.adamw(starts[i], gr[i], m, v, step, 1e-3, 0.9, 0.999, 1e-8, 0.1, c)
            top_m = ref._blocks(wm.abs()).amax(1).repeat_interleave(256)[:n]
            top_v = ref._blocks(wv).amax(1).repeat_interleave(256)[:n]
            _inside(sm[i], ref._blocks(wm.abs()).amax(1), 4e-6 * ref._blocks(wm.abs()).amax(1), "m scale")
            _inside(sv[i], ref._blocks(wv).amax(1), 4e-6 * ref._blocks(wv).amax(1), "v scale")
            got_m, got_v = ref.decode_m(qm[i].cpu(), sm[i].cpu()), ref.decode_v(qv[i].cpu(), sv[i].cpu())
            _inside(got_m, wm, 1.01 * (torch.sqrt(top_m * wm.abs()) / 127 + top_m / 127**2) + 1e-5 * top_m, "m")
            root = (wv / top_v.clamp(min=1e-300)) ** 0.25  # codes are even in the fourth root
            _inside(got_v, wv, 1.01 * top_v * ((root + 1 / 255) ** 4 - root**4) + 1e-5 * wv, "v")
            assert bool(((got_v > 0) | (wv == 0)).all())
            s = starts[i].double()
            near = 1e-5 * (wp - s).abs() + 32 * U * s.abs() + 1e-9
            _inside((dmaster or dp)[i], wp, near + (1.01 * HALF[param] * wp.abs() if not master else 0), "p")


def test_adamw_8_bit_block_with_a_value_that_is_not_finite(cuda):
    ops = _ops()
    n = 700
    p, g = torch.zeros(n, device=cuda), torch.full((n,), 0.01, device=cuda)
    g[300] = INF
    qm, qv = torch.zeros(n, dtype=torch.int8, device=cuda), torch.zeros(n, dtype=torch.uint8, device=cuda)
    sm, sv = torch.zeros(3, device=cuda), torch.zeros(3, device=cuda)
    ops.adamw_step([p], [g], [qm], [qv], step=1, lr=1e-3, scales=([sm], [sv]))
    assert torch.isnan(sm).tolist() == [False, True, False] and torch.isnan(sv).tolist() == [False, True, False]
    assert bool(torch.isfinite(p[:256]).all()) and bool(torch.isfinite(p[512:]).all()) and not bool(torch.isfinite(p[300]))


def test_adamw_past_32_bits(cuda):
    ops = _ops()
    n = (1 << 31) + 1000
    p, g = torch.zeros(n, dtype=BF16, device=cuda), torch.zeros(n, dtype=BF16, device=cuda)
    g[-5:] = 1.0
    qm, qv = torch.zeros(n, dtype=torch.int8, device=cuda), torch.zeros(n, dtype=torch.uint8, device=cuda)
    blocks = -(-n // 256)
    sm, sv, norm = torch.zeros(blocks, device=cuda), torch.zeros(blocks, device=cuda), torch.empty(2, device=cuda)
    ops.adamw_step([p], [g], [qm], [qv], step=1, lr=0.5, weight_decay=0.0, scales=([sm], [sv]), norm_out=norm)
    assert float(norm[0]) == pytest.approx(math.sqrt(5.0), rel=1e-6)
    assert p[-5:].float().tolist() == [-0.5] * 5 and float(p[-1000:-5].abs().max()) == 0.0 and int(qm[-1]) == 127


def test_adamw_refusals_on_the_gpu(cuda):
    ops = _ops()
    x, h = torch.zeros(8, device=cuda), torch.zeros(8, dtype=BF16, device=cuda)
    q, u, s = torch.zeros(8, dtype=torch.int8, device=cuda), torch.zeros(8, dtype=torch.uint8, device=cuda), torch.zeros(1, device=cuda)
    bad = [([x], [h], [x], [x], {}), ([x], [x[:4]], [x], [x], {}), ([x], [x], [q], [u], {}), ([x], [x], [q], [x], dict(scales=([s], [s]))),
           ([x], [x], [q], [u], dict(scales=([s[:0]], [s]))), ([x], [x], [x], [x], dict(masters=[x])), ([x.double()], [x], [x], [x], {}),
           ([x.view(2, 4).t()], [x.view(2, 4).t()], [x], [x], {}), ([x], [x], [x], [x], dict(norm_out=torch.zeros(3, device=cuda))),
           ([x], [x], [x], [x], dict(max_grad_norm=0.0)), ([x], [x], [x], [x], dict(lr=[1e-3, 1e-3]))]
    for p, g, m, v, more in bad:
        with pytest.raises(ValueError, match="adamw_step"):
            ops.adamw_step(p, g, m, v, step=1, **{"lr": 1e-3, **more})
    t = torch.zeros(3, dtype=torch.int64, device=cuda)
    m3 = torch.zeros(3, 5, device=cuda)
    for call in (lambda: ops.embedding_fwd(t.float(), m3, m3), lambda: ops.embedding_fwd(t, m3.double(), m3), lambda: ops.embedding_fwd(t, m3, m3[:2]),
                 lambda: ops.embedding_fwd(t, m3.t(), m3), lambda: ops.embedding_bwd(t, m3, m3.to(BF16)),
                 lambda: ops.embedding_fwd(t, m3, m3.to(BF16)), lambda: ops.embedding_fwd(t, m3, m3[:1].expand(3, 5)),
                 lambda: ops.token_log_probs(m3, t[:2], None), lambda: ops.token_log_probs(m3, t, m3[0]),
                 lambda: ops.token_log_probs(m3, t, None, mask=t), lambda: ops.token_log_probs(m3, t, m3[:, 0], temperature=0.0),
                 lambda: ops.token_ppo_loss(m3, t, s, s, m3, torch.zeros(8, device=cuda))):
        with pytest.raises(ValueError):
            call()


# ---- streams and graphs ----


def _all_ops(ops, s):
    ops.embedding_fwd(s["tok"], s["table"], s["y"], scale=0.5, )
    ops.embedding_bwd(s["tok"], s["y"], s["dt"], scale=0.5, ws=s["ws"][0])
    ops.token_ppo_loss(s["x"], s["tok"], s["old"], s["adv"], s["dx"], s["stats"], mask=s["mask"], kl_coef=0.1, ref_logp=s["old"],
                       logp=s["lp"], ws=s["ws"][1])
    ops.adamw_step([s["table"]], [s["dt"]], [s["m"]], [s["v"]], step=5, lr=1e-2, max_grad_norm=0.5, ws=s["ws"][2])


def _all_state(cuda, ops, rows=6000, vocab=700, dim=96):
    g = torch.Generator(device=cuda).manual_seed(0)
    r = lambda *n: torch.randn(*n, generator=g, device=cuda)  # noqa: E731
    s = dict(tok=torch.randint(0, vocab, (rows,), generator=g, device=cuda), table=r(vocab, dim), y=torch.zeros(rows, dim, device=cuda),
             dt=torch.zeros(vocab, dim, device=cuda), x=r(rows, vocab), old=-6 + 0.1 * r(rows), adv=r(rows), dx=torch.zeros(rows, vocab, device=cuda),
             stats=torch.zeros(8, device=cuda), lp=torch.zeros(rows, device=cuda), mask=r(rows) > 0, m=torch.zeros(vocab, dim, device=cuda),
             v=torch.zeros(vocab, dim, device=cuda), ws=[ops.Workspace(cuda) for _ in range(3)])
    return s


OUT = ("table", "y", "dt", "dx", "stats", "lp", "m", "v")


def test_on_another_stream(cuda):
    ops = _ops()
    a, b = _all_state(cuda, ops), _all_state(cuda, ops)
    for _ in range(3):
        _all_ops(ops, a)
    other = torch.cuda.Stream()
    big = torch.ones(4096, 4096, device=cuda)
    for _ in range(20):
        big = torch.mm(big, big).clamp_(-1.0, 1.0)
    b["x"].add_(big[0, 0] * 0)  # the inputs come late on their own stream
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        for _ in range(3):
            _all_ops(ops, b)
    torch.cuda.current_stream().wait_stream(other)
    for k in OUT:
        assert torch.equal(a[k], b[k]), k


def test_in_a_graph(cuda):
    ops = _ops()
    a, b = _all_state(cuda, ops), _all_state(cuda, ops)
    warm = _all_state(cuda, ops)
    warm["ws"] = b["ws"]
    _all_ops(ops, warm)  # the workspaces grow before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _all_ops(ops, b)
    for _ in range(4):
        _all_ops(ops, a)
        graph.replay()
        torch.cuda.synchronize()
        for k in OUT:
            assert torch.equal(a[k], b[k]), k
