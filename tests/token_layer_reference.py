"""Plain 64-bit forms of the operators between a token policy's embedding and its logits, on the CPU: what the tests of their kernels
compare with, checked themselves in tests/test_token_layer_reference.py.  Each returns its results and, where a rounding bound is in terms of
them, the same sums over magnitudes."""

from __future__ import annotations

import torch


# ---- queries and keys, normed and turned ----


def turn(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, interleaved: bool, back: bool = False) -> torch.Tensor:
    x, r = x.double().clone(), 2 * freqs.numel()
    angle = (positions.double()[:, None] * freqs.double()[None, :])[:, None, :]
    cos, sin = torch.cos(angle), -torch.sin(angle) if back else torch.sin(angle)
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., first].clone(), x[..., second].clone()
    x[..., first], x[..., second] = a * cos - b * sin, b * cos + a * sin
    return x


def pair_size(x: torch.Tensor, freqs: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """|a| + |b| of the pair that each element is turned with; |x| of the others."""
    x, r = x.double().abs().clone(), 2 * freqs.numel()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    both = x[..., first] + x[..., second]
    x[..., first], x[..., second] = both, both
    return x


def qk_rotary(x, weight, positions, freqs, eps, interleaved):
    """(turned, its value before the turn)."""
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    return turn(y, positions, freqs, interleaved), y


def qk_rotary_grad(g, x, weight, positions, freqs, eps, interleaved):
    """d_x, d_weight and the magnitudes that they are summed from."""
    x, w = x.double(), weight.double()
    size = pair_size(g, freqs, interleaved)
    g = turn(g, positions, freqs, interleaved, back=True)
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x * r
    d_x = r * (g * w - n * (g * w * n).mean(-1, keepdim=True))
    over = 0 if weight.dim() == 2 else (0, 1)
    x_size = r * (size * w.abs() + n.abs() * (size * w.abs() * n.abs()).mean(-1, keepdim=True))
    return d_x, (g * n).sum(over), x_size, (size * n.abs()).sum(over)


# ---- linear attention with a decay for each head ----


def spans(tokens: int, cu) -> list[tuple[int, int]]:
    if cu is None:
        return [(0, tokens)]
    cu = [int(c) for c in cu]
    return [(min(max(a, 0), tokens), min(max(b, 0), tokens)) for a, b in zip(cu, cu[1:])]


def _fade(n: int, log_decay: torch.Tensor) -> torch.Tensor:
    """decay^(i - j), i >= j, else 0: [heads, n, n]."""
    apart = torch.arange(n, dtype=torch.float64)[:, None] - torch.arange(n, dtype=torch.float64)[None, :]
    power = torch.where(apart == 0, torch.zeros((), dtype=torch.float64), apart.clamp(min=0) * log_decay.double()[:, None, None])
    return torch.where(apart >= 0, torch.exp(power), torch.zeros((), dtype=torch.float64))


def _powers(n: int, log_decay: torch.Tensor, first: int) -> torch.Tensor:
    """decay^first, decay^(first + 1) .. : [heads, n]."""
    at = torch.arange(first, first + n, dtype=torch.float64)
    return torch.where(at == 0, torch.ones((), dtype=torch.float64), torch.exp(torch.where(at == 0, torch.zeros_like(at), at) * log_decay.double()[:, None]))


def decay_attention(q, k, v, log_decay, scale=1.0, cu=None, initial=None):
    """out (0 where a token is in no sequence) and final states, every token against all before it."""
    q, k, v = q.double(), k.double(), v.double()
    group, heads = q.shape[1] // k.shape[1], k.shape[1]
    out = torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64)
    finals = []
    for b, (i, j) in enumerate(spans(q.shape[0], cu)):
        s0 = initial[b].double() if initial is not None else torch.zeros(heads, k.shape[2], v.shape[2], dtype=torch.float64)
        n = max(0, j - i)
        if n == 0:
            finals.append(s0)
            continue
        qh, kh, vh = (x[i:j].transpose(0, 1) for x in (q, k, v))
        of = torch.arange(q.shape[1]) // group
        p = (qh @ kh[of].transpose(1, 2)) * _fade(n, log_decay)[of] * scale
        o = p @ vh[of] + scale * _powers(n, log_decay, 1)[of][:, :, None] * (qh @ s0[of])
        out = torch.cat([out[:i], o.transpose(0, 1), out[j:]])
        left = _powers(n, log_decay, 0).flip(1)
        whole = torch.exp(log_decay.double() * n)
        finals.append(whole[:, None, None] * s0 + (kh * left[:, :, None]).transpose(1, 2) @ vh)
    return out, torch.stack(finals)


def decay_attention_grad(d_out, q, k, v, log_decay, scale=1.0, cu=None, initial=None, d_final=None):
    """d_q, d_k, d_v and d_initial by the formulas."""
    g, q, k, v = d_out.double(), q.double(), k.double(), v.double()
    group, heads = q.shape[1] // k.shape[1], k.shape[1]
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    firsts = []
    zero = torch.zeros(heads, k.shape[2], v.shape[2], dtype=torch.float64)
    of = torch.arange(q.shape[1]) // group
    shared = lambda x: x.view(heads, group, *x.shape[1:]).sum(1)  # noqa: E731
    for b, (i, j) in enumerate(spans(q.shape[0], cu)):
        s0 = initial[b].double() if initial is not None else zero
        s1 = d_final[b].double() if d_final is not None else zero
        n = max(0, j - i)
        if n == 0:
            firsts.append(s1)
            continue
        qh, kh, vh, gh = (x[i:j].transpose(0, 1) for x in (q, k, v, g))
        fade = _fade(n, log_decay)[of] * scale
        p, gp = (qh @ kh[of].transpose(1, 2)) * fade, (gh @ vh[of].transpose(1, 2)) * fade
        since, left = _powers(n, log_decay, 1), _powers(n, log_decay, 0).flip(1)
        dq[i:j] = (gp @ kh[of] + scale * since[of][:, :, None] * (gh @ s0[of].transpose(1, 2))).transpose(0, 1)
        dk[i:j] = (shared(gp.transpose(1, 2) @ qh) + left[:, :, None] * (vh @ s1.transpose(1, 2))).transpose(0, 1)
        dv[i:j] = (shared(p.transpose(1, 2) @ gh) + left[:, :, None] * (kh @ s1)).transpose(0, 1)
        firsts.append(torch.exp(log_decay.double() * n)[:, None, None] * s1 + scale * shared((qh * since[of][:, :, None]).transpose(1, 2) @ gh))
    return dq, dk, dv, torch.stack(firsts)


def decay_step(q, k, v, log_decay, state, scale=1.0, slots=None, fresh=None):
    """out and the states after one token of each row."""
    state = state.double().clone()
    group = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64)
    for r in range(q.shape[0]):
        slot = r if slots is None else int(slots[r])
        if not 0 <= slot < state.shape[0]:
            continue
        before = torch.zeros_like(state[slot]) if fresh is not None and bool(fresh[r]) else torch.exp(log_decay.double())[:, None, None] * state[slot]
        state[slot] = before + k[r].double()[:, :, None] * v[r].double()[:, None, :]
        out[r] = scale * (q[r].double()[:, None, :] @ state[slot].repeat_interleave(group, 0))[:, 0]
    return out, state


# ---- cross entropy under a head ----


def linear_cross_entropy(hidden, weight, tokens, mask=None, temperature=1.0, denom=None):
    rows, vocab = hidden.shape[0], weight.shape[0]
    counts = (tokens >= 0) & (tokens < vocab)
    if mask is not None:
        counts &= mask != 0
    n = float(denom) if denom is not None else max(1.0, float(counts.sum()))
    h, w = hidden.double(), weight.double()
    zeros = lambda *sizes: torch.zeros(*sizes, dtype=torch.float64, device=hidden.device)  # noqa: E731
    out = {"logp": zeros(rows), "entropy": zeros(rows), "d": zeros(rows, vocab)}
    at = counts.nonzero()[:, 0]
    z = (h[at] @ w.t()) / temperature
    z = z - z.amax(1, keepdim=True)
    p = torch.exp(z) / torch.exp(z).sum(1, keepdim=True)
    logs = z - torch.log(torch.exp(z).sum(1, keepdim=True))
    t = tokens[at].long()
    out["logp"][at] = logs[torch.arange(len(at), device=t.device), t]
    out["entropy"][at] = -(p * logs).sum(1)
    d = p.clone()
    d[torch.arange(len(at), device=t.device), t] -= 1.0
    out["d"][at] = d
    safe = torch.where(counts[:, None], h, torch.zeros_like(h))
    out["d_hidden"] = out["d"] @ w / (n * temperature)
    out["d_weight"] = out["d"].t() @ safe / (n * temperature)
    out["stats"] = torch.tensor([-float(out["logp"].sum()) / n, float(out["entropy"].sum()) / n, float(denom) if denom is not None else float(counts.sum()), 0.0],
                                dtype=torch.float64, device=hidden.device)
    return out
