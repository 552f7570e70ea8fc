"""A policy over sequences of tokens, taught by demonstrations on one GPU and then run token by token:

    tokens -> TokenEmbedding -> DecayMixer layers -> linear_cross_entropy under the embedding's own size of head, no logits in memory
    -> AdamW;   then prompts through forward(), and each further token through step() on the layers' states

The task: repeat a sequence's first tokens in their order, again and again.  Run it with

    python examples/sequence_policy.py [iterations]
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch
import torch.nn as nn

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from tt_rsl_rl_amd import ops  # noqa: E402
from tt_rsl_rl_amd.tokens import AdamW, DecayMixer, TokenEmbedding, linear_cross_entropy  # noqa: E402


class SequencePolicy(nn.Module):
    def __init__(self, vocab: int, dim: int, layers: int, heads: int, kv_heads: int, head_dim: int, device, dtype) -> None:
        super().__init__()
        self.embed = TokenEmbedding(vocab, dim, device=device, dtype=dtype)
        self.norms = nn.ModuleList(nn.LayerNorm(dim, device=device, dtype=dtype) for _ in range(layers + 1))
        self.mixers = nn.ModuleList(DecayMixer(dim, heads, kv_heads, head_dim, device=device, dtype=dtype) for _ in range(layers))
        self.bodies = nn.ModuleList(nn.Sequential(nn.Linear(dim, 2 * dim, device=device, dtype=dtype), nn.ELU(),
                                                  nn.Linear(2 * dim, dim, device=device, dtype=dtype)) for _ in range(layers))
        self.head = nn.Parameter(torch.randn(vocab, dim, device=device).mul_(dim**-0.5).to(dtype))

    def forward(self, tokens, positions, cu_seqlens, states=None, want_states=False):
        """Tokens of sequences one after another -> what the head is given, and the layers' states after each sequence (None unless wanted)."""
        x, after = self.embed(tokens), []
        for i, (mixer, body) in enumerate(zip(self.mixers, self.bodies)):
            mixed, state = mixer(self.norms[i](x), positions, cu_seqlens, None if states is None else states[i], want_states)
            after.append(state)
            x = x + mixed
            x = x + body(x)
        return self.norms[-1](x), after

    @torch.no_grad()
    def step(self, tokens, positions, states, slots=None, fresh=None):
        """One token of each sequence, on the states in place."""
        x = self.embed(tokens)
        for i, (mixer, body) in enumerate(zip(self.mixers, self.bodies)):
            x = x + mixer.step(self.norms[i](x), positions, states[i], slots, fresh)
            x = x + body(x)
        return self.norms[-1](x)


def batch(sequences: int, vocab: int, period: int, longest: int, device, generator):
    """Packed sequences of many lengths, each its first tokens over and over."""
    lengths = torch.randint(2 * period, longest + 1, (sequences,), generator=generator)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)])
    positions = torch.cat([torch.arange(n) for n in lengths.tolist()])
    first = torch.randint(0, vocab, (sequences, period), generator=generator)
    tokens = torch.cat([first[i][torch.arange(n) % period] for i, n in enumerate(lengths.tolist())])
    return tokens.to(device), positions.to(device), cu.to(torch.int32).to(device)


def loss_of(policy, tokens, positions, cu, period):
    """Each token's successor in its sequence; the first ones cannot be known and do not count."""
    following = tokens.roll(-1)
    following[cu[1:].long() - 1] = -1
    mask = positions >= period - 1
    hidden, _ = policy(tokens, positions, cu)
    return linear_cross_entropy(hidden, policy.head, following, mask=mask)


@torch.no_grad()
def correct(policy, vocab: int, period: int, sequences: int, steps: int, device, generator) -> float:
    """Prompts of one period at once, then each further token by itself: the share of greedy tokens that go on as the prompt did."""
    prompts = torch.randint(0, vocab, (sequences, period), generator=generator).to(device)
    cu = torch.arange(0, (sequences + 1) * period, period, dtype=torch.int32, device=device)
    hidden, states = policy(prompts.flatten(), torch.arange(period, device=device).repeat(sequences), cu, want_states=True)
    hidden = hidden.view(sequences, period, -1)[:, -1]
    hits = 0
    for t in range(steps):
        token = (hidden.float() @ policy.head.float().t()).argmax(-1)
        hits += int((token == prompts[:, t % period]).sum())
        token = prompts[:, t % period].contiguous()
        logp = torch.empty(sequences, device=device)
        ops.linear_log_probs(hidden.contiguous(), policy.head.detach(), token, logp)  # (what a rollout would store)
        hidden = policy.step(token, torch.full((sequences,), period + t, device=device), states)
    return hits / (sequences * steps)


def train(iterations: int = 150, sequences: int = 64, vocab: int = 61, dim: int = 128, layers: int = 2, heads: int = 4, kv_heads: int = 2, head_dim: int = 32,
          period: int = 5, longest: int = 40, lr: float = 3e-3, seed: int = 0, log=None) -> list[float]:
    device = torch.device("cuda", torch.cuda.current_device())
    torch.manual_seed(seed)
    generator = torch.Generator().manual_seed(seed)
    policy = SequencePolicy(vocab, dim, layers, heads, kv_heads, head_dim, device, torch.bfloat16)
    optimizer = AdamW(policy.parameters(), lr=lr, max_grad_norm=1.0, weight_decay=0.0)
    history = []
    for it in range(iterations):
        loss = loss_of(policy, *batch(sequences, vocab, period, longest, device, generator), period)
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        history.append(float(loss.detach()))
        if log is not None and it % 10 == 0:
            log(f"iteration {it:3d}  loss {history[-1]:.3f}  greedy tokens right {correct(policy, vocab, period, 64, 10, device, generator):.2f}")
    return history


if __name__ == "__main__":
    train(int(sys.argv[1]) if len(sys.argv) > 1 else 150, log=lambda line: print(line, flush=True))
