"""A policy over tokens trained with PPO on one GPU, from lookup to optimiser step:

    tokens -> TokenEmbedding -> torch layers -> logits -> ops.token_log_probs        (the rollout, and the reference policy)
    ops.gae, ops.adv_normalize -> ops.token_ppo_loss -> logits.backward(d_logits)    (the update)
    -> AdamW (fp32 masters, 8-bit states, clip by the global norm)

The task: each step shows two tokens, and the answer that is rewarded is a fixed function of them.  Run it with

    python examples/token_policy.py [iterations]
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
from tt_rsl_rl_amd.tokens import AdamW, TokenEmbedding  # noqa: E402


class TokenPolicy(nn.Module):
    def __init__(self, vocab: int, dim: int, context: int, hidden: int, device, dtype) -> None:
        super().__init__()
        self.embed = TokenEmbedding(vocab, dim, scale=dim**0.5, device=device, dtype=dtype)
        self.body = nn.Sequential(nn.Linear(context * dim, hidden, device=device, dtype=dtype), nn.ELU(),
                                  nn.Linear(hidden, vocab, device=device, dtype=dtype))

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:  # [rows, context] -> [rows, vocab]
        return self.body(self.embed(tokens).flatten(1))


def train(iterations: int = 60, envs: int = 1024, steps: int = 8, vocab: int = 32, dim: int = 64, hidden: int = 256, epochs: int = 4,
          mini_batches: int = 4, lr: float = 2e-3, kl_coef: float = 0.001, entropy_coef: float = 0.005, state_bits: int = 8, seed: int = 0,
          log=None) -> list[float]:
    """The mean reward of each iteration's rollout (chance: 1 / vocab)."""
    device = torch.device("cuda", torch.cuda.current_device())
    torch.manual_seed(seed)
    policy = TokenPolicy(vocab, dim, 2, hidden, device, torch.bfloat16)
    reference = TokenPolicy(vocab, dim, 2, hidden, device, torch.bfloat16)
    reference.load_state_dict(policy.state_dict())
    matrices = [p for p in policy.parameters() if p.dim() > 1]
    vectors = [p for p in policy.parameters() if p.dim() == 1]
    optimizer = AdamW([dict(params=matrices, weight_decay=0.01), dict(params=vectors, weight_decay=0.0)], lr=lr, max_grad_norm=1.0,
                      state_bits=state_bits)
    answer = torch.randperm(vocab, device=device)
    rows, batch, ws = envs * steps, envs * steps // mini_batches, ops.Workspace(device)
    f32 = dict(dtype=torch.float32, device=device)
    logp, ref_logp, stats = torch.empty(rows, **f32), torch.empty(rows, **f32), torch.empty(8, **f32)
    rewards, values, returns, advantages = (torch.zeros(steps, envs, **f32) for _ in range(4))
    dones, last = torch.ones(steps, envs, dtype=torch.uint8, device=device), torch.zeros(envs, **f32)
    history = []
    for it in range(iterations):
        with torch.no_grad():  # the rollout: one token per environment and step, rewarded at once
            prompts = torch.randint(0, vocab, (rows, 2), device=device)
            logits = policy(prompts)
            actions = torch.multinomial(torch.softmax(logits.float(), -1), 1)[:, 0]
            ops.token_log_probs(logits, actions, logp, ws=ws)
            ops.token_log_probs(reference(prompts), actions, ref_logp, ws=ws)
            rewards.copy_((actions == answer[(prompts[:, 0] + prompts[:, 1]) % 8]).view(steps, envs))
            values.fill_(0.0)
            ops.gae(rewards, values, dones, last, returns, advantages, 0.99, 0.95)
            ops.adv_normalize(advantages, advantages, rows, ws=ws)
        for _ in range(epochs):
            for index in torch.randperm(rows, device=device).split(batch):
                logits = policy(prompts[index])
                d_logits = torch.empty_like(logits)
                ops.token_ppo_loss(logits.detach(), actions[index], logp[index], advantages.view(-1)[index], d_logits, stats,
                                   ref_logp=ref_logp[index], clip_param=0.2, kl_coef=kl_coef, entropy_coef=entropy_coef, ws=ws)
                optimizer.zero_grad(set_to_none=True)
                logits.backward(d_logits)
                optimizer.step()
        history.append(float(rewards.mean()))
        if log is not None:
            loss, surrogate, kl, entropy, clipped = stats[:5].tolist()
            log(f"iteration {it:3d}  reward {history[-1]:.3f}  loss {loss:+.4f}  surrogate {surrogate:+.4f}  kl {kl:.4f}  "
                f"entropy {entropy:.3f}  clipped {clipped:.2f}  gradient norm {float(optimizer.norm[0]):.3f}")
    return history


if __name__ == "__main__":
    train(int(sys.argv[1]) if len(sys.argv) > 1 else 60, log=lambda line: print(line, flush=True))
