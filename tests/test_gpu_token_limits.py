"""The token operators where a call is so large that its launches have to be laid out for it: more than 2^32 threads."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_token_ops import BF16, F32, U, _loss_error, _ops

pytestmark = pytest.mark.gpu


def _log_probs(x, tok):
    """logp and entropy in 64 bits, on the GPU, a part at a time."""
    out = []
    for y, t in zip(x.split(1 << 22), tok.split(1 << 22)):
        logs = torch.log_softmax(y.double(), 1)
        out.append((logs.gather(1, t[:, None])[:, 0], -(logs.exp() * logs).sum(1)))
    return [torch.cat(p) for p in zip(*out)]


@pytest.mark.parametrize("rows,vocab,dtype", [((1 << 20) - 1, 2, F32), ((1 << 20) + 1, 5, BF16), ((1 << 22) + 5, 4, BF16), ((1 << 22) + 5, 3, F32),
                                              ((1 << 26) + 3, 8, BF16)])
def test_many_rows_of_a_small_vocabulary(cuda, rows, vocab, dtype):
    """On both sides of the rows that a launch holds along one axis, with 1,024 threads to a row (a row narrower than 16 bytes) and
    with 64."""
    ops, g = _ops(), torch.Generator(device=cuda).manual_seed(rows)
    x = torch.randn(rows, vocab, generator=g, device=cuda, dtype=dtype)
    tok = torch.randint(0, vocab, (rows,), generator=g, device=cuda)
    want, entropy = _log_probs(x, tok)
    lp, h = torch.full((rows,), 9.0, device=cuda), torch.full((rows,), 9.0, device=cuda)
    print(f"log-probabilities {rows} x {vocab}", flush=True)
    ops.token_log_probs(x, tok, lp, h)
    e = _loss_error(x[:100_000].cpu(), vocab, 1.0) * 4  # (the largest of all rows' |z| is below four times that of some)
    assert float(((lp - want).abs() - e * (1 + want.abs())).max()) <= 0 and float(((h - entropy).abs() - 2 * e).max()) <= 0
    if rows > 1 << 23:
        return
    print(f"loss {rows} x {vocab}", flush=True)
    adv, dx, stats = torch.randn(rows, generator=g, device=cuda), torch.full_like(x, 9.0), torch.empty(8, device=cuda)
    ops.token_ppo_loss(x, tok, want.float(), adv, dx, stats, denom=1.0)
    p = torch.softmax(x.double(), 1)
    d = adv[:, None] * (p - torch.nn.functional.one_hot(tok, vocab))
    assert float((dx - d).abs().sub(e * (1 + adv.abs())[:, None] * 4 + (2.0**-8 if dtype == BF16 else U) * 1.01 * d.abs()).max()) <= 0
    assert abs(float(stats[3]) - float(entropy.sum())) <= 2 * e * rows


def test_adamw_of_more_elements_than_a_launch_takes(cuda):
    """2^34 and more elements in tensors that a launch would take together; their gradient is one and the same tensor."""
    ops = _ops()
    n, tensors = 1 << 32, 5
    zeros = lambda k, dtype: [torch.zeros(k, dtype=dtype, device=cuda) for _ in range(tensors)]  # noqa: E731
    p, m, v = zeros(n, BF16), zeros(n, torch.int8), zeros(n, torch.uint8)
    sm, sv = zeros(n // 256, F32), zeros(n // 256, F32)
    g = torch.ones(n, dtype=BF16, device=cuda)
    print("AdamW of 2.1e10 elements", flush=True)
    ops.adamw_step(p, [g] * tensors, m, v, step=1, lr=0.5, weight_decay=0.0, scales=(sm, sv))
    for t in p:
        assert float(t.min()) == -0.5 and float(t.max()) == -0.5
    for t in m:
        assert int(t.min()) == 127
    del p, m, v, sm, sv, g
    torch.cuda.empty_cache()


@pytest.mark.parametrize("count,dim", [((1 << 22) + 3, 1025), ((1 << 26) + 5, 1025)])
def test_lookup_of_many_rows(cuda, count, dim):
    """On both sides of what a launch holds along one axis: 2^20 blocks of 4 rows, and 2^32 threads."""
    ops, vocab = _ops(), 251
    if torch.cuda.mem_get_info()[0] < 2.2 * count * dim + (8 << 30):
        pytest.skip("not enough memory")
    table = torch.arange(vocab, device=cuda, dtype=F32)[:, None].to(BF16).expand(vocab, dim).contiguous()
    tok = (torch.arange(count, device=cuda) % 263 - 1).int()  # (some outside of the vocabulary)
    out = torch.empty(count, dim, dtype=BF16, device=cuda)
    print(f"lookup {count} x {dim}", flush=True)
    ops.embedding_fwd(tok, table, out, scale=0.5)
    for i in range(0, count, 1 << 24):
        t = tok[i:i + (1 << 24)]
        want = torch.where((t >= 0) & (t < vocab), t * 0.5, 0.0)
        for c in (0, 500, dim - 1):
            assert torch.equal(out[i:i + (1 << 24), c].float(), want)
    del out, tok
    torch.cuda.empty_cache()
