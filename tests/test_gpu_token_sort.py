"""The embedding's gradient where its tokens go through the tiled sort (more than 12,288 of them): one to four passes of 5 to 9 bits,
both token types, tables in rows apart, runs over every unit's length, in a graph.  Summands are small whole numbers, whose sums are
exact in fp32 in any order."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_token_ops import BF16, F16, F32, _ops

pytestmark = pytest.mark.gpu


def _tokens(count, vocab, cuda, seed=0):
    """Half of them spread over the vocabulary, half over few tokens, some that are none."""
    g = torch.Generator(device=cuda).manual_seed(seed + count)
    few = torch.randint(0, vocab, (97,), generator=g, device=cuda)
    tok = torch.where(torch.rand(count, generator=g, device=cuda) < 0.5, torch.randint(0, vocab, (count,), generator=g, device=cuda),
                      few[torch.randint(0, 97, (count,), generator=g, device=cuda)])
    tok[0], tok[count // 3], tok[-1] = vocab - 1, -100, 0
    tok[count // 5] = vocab
    return tok


def _summands(count, dim, cuda, dtype, seed=0):
    return torch.randint(-3, 4, (count, dim), generator=torch.Generator(device=cuda).manual_seed(seed + dim), device=cuda).to(dtype)


def _want(tok, d, vocab, scale, start=None):
    ok = (tok >= 0) & (tok < vocab)
    out = torch.zeros(vocab, d.shape[1], device=d.device).index_add_(0, tok[ok].long(), d[ok].float() * scale)
    return out if start is None else out + start.float()


# bits of the keys (0 .. vocab): 4 (one pass), 9 (one), 10 (two of 5), 18 (two of 9), 19 (three of 7), 27 (three of 9), 29 (four of 8)
VOCABS = [(10, 33), (511, 24), (513, 130), (200_003, 24), (300_007, 9), ((1 << 26) + 7, 1), ((1 << 28) + 5, 1)]


@pytest.mark.parametrize("token_type", [torch.int64, torch.int32])
@pytest.mark.parametrize("count", [12_289, 20_480, 100_003])
@pytest.mark.parametrize("vocab,dim", VOCABS)
def test_passes(cuda, vocab, dim, count, token_type):
    ops = _ops()
    tok, d = _tokens(count, vocab, cuda), _summands(count, dim, cuda, BF16)
    tok = tok.to(token_type)
    got = torch.full((vocab, dim), 9.0, dtype=F32 if vocab < 1 << 20 else BF16, device=cuda)
    print(f"gradient of {count} tokens, {vocab} x {dim}", flush=True)
    ops.embedding_bwd(tok, d, got, scale=2.0)
    want = _want(tok, d, vocab, 2.0)
    assert torch.equal(got, want.to(got.dtype))
    del want
    again = torch.full_like(got, 7.0)
    ops.embedding_bwd(tok, d, again, scale=2.0)
    assert torch.equal(got, again)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype,out,pad", [(F32, F32, 3), (BF16, F32, 1), (F16, F16, 5), (BF16, BF16, 40_000)])
@pytest.mark.parametrize("count,vocab,dim", [(13_001, 700, 40), (30_011, 60_003, 33), (20_002, 300_007, 5)])
def test_tables_in_rows_apart(cuda, count, vocab, dim, dtype, out, pad, accumulate):
    """Nothing beside the columns is written by the sums or by the zeros, whichever launch's blocks write them."""
    if vocab * (dim + pad) > 1 << 30:
        pad = 11
    ops = _ops()
    tok, d = _tokens(count, vocab, cuda, seed=3), _summands(count, dim + 4, cuda, dtype)[:, 1: 1 + dim]
    full = torch.full((vocab, dim + pad), 3.0, dtype=out, device=cuda)
    table = full[:, 1: 1 + dim]
    ops.embedding_bwd(tok, d, table, accumulate=accumulate)
    assert torch.equal(table, _want(tok, d, vocab, 1.0, start=torch.full_like(table, 3.0) if accumulate else None).to(out))
    assert bool((full[:, 0] == 3).all()) and bool((full[:, 1 + dim:] == 3).all())


@pytest.mark.parametrize("count,dim", [(50_000, 24), (100_000, 24), (200_000, 24), (70_001, 600), (40_000, 2050)])
def test_units_of_every_length(cuda, count, dim):
    """Units of 8, 16 and 32 positions (as the count and the width ask for), with runs that end on, before and behind every boundary
    and one so long that the boundaries it crosses are looked for 64 times 64 at once."""
    ops, g = _ops(), torch.Generator().manual_seed(count + dim)
    lens = torch.tensor([1, 2, 3, 7, 8, 9, 10, 15, 16, 17, 23, 24, 25, 31, 32, 33, 39, 40, 41, 64, 127, 128, 129, 300, 900])
    lens = lens[torch.randint(0, len(lens), (count // 20,), generator=g)]
    lens = lens[: int((lens.cumsum(0) <= count // 3).sum())]
    lens = torch.cat([lens[:50], torch.tensor([0, count - int(lens.sum())]), lens[50:]])
    tok = torch.repeat_interleave(torch.arange(len(lens)), lens)
    tok = tok[torch.randperm(len(tok), generator=g)].to(cuda)
    assert len(tok) == count
    d = _summands(count, dim, cuda, BF16)
    got = torch.full((len(lens), dim), 5.0, device=cuda)
    ops.embedding_bwd(tok, d, got, scale=0.5)
    assert torch.equal(got, _want(tok, d, len(lens), 0.5))


def test_in_a_graph(cuda):
    ops, count, vocab, dim = _ops(), 40_009, 70_001, 40
    ws = ops.Workspace(cuda)
    tok, d = _tokens(count, vocab, cuda), _summands(count, dim, cuda, BF16)
    got = torch.empty(vocab, dim, device=cuda)
    ops.embedding_bwd(tok, d, got, ws=ws)  # the workspace grows before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.embedding_bwd(tok, d, got, ws=ws)
    for i in range(4):
        tok.copy_(_tokens(count, vocab, cuda, seed=i))
        d.copy_(_summands(count, dim, cuda, BF16, seed=i))
        got.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, _want(tok, d, vocab, 1.0)), i
