"""The operators between the two ends of a policy that acts in tokens, and of the loss that it is taught with before rewards
train it, as cases to time.  One pass is one call of ``tt_rsl_rl_amd.ops``:

    qk       ``qk_norm_rotary_fwd``: each head's query and key normed and turned by its token's position
    qkgrad   ``qk_norm_rotary_bwd``: the gradients of queries, keys and the norms' weights
    mix      ``decay_attention_fwd``: linear attention whose past fades by a factor for each head, over packed sequences
    mixgrad  ``decay_attention_bwd``: its gradients
    step     ``decay_attention_step``: the same one token at a time, on the states of running sequences
    xent     ``linear_cross_entropy``: the cross entropy of tokens under a head as wide as the vocabulary, with the gradients
             of its input and weight, or (``grad`` false) ``linear_log_probs``: log-probabilities and entropies alone

Tokens follow 1 / rank (a vocabulary sorted by frequency), masked rows stand for prompts and padding, queries and keys are
columns of one projection's output.  With ``own`` false the same results come from elementary torch operations.
"""

from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS, BASE, TEMPERATURE = 1e-6, 10000.0, 1.25
CHUNK = 256  # tokens that the plain form of the attention takes together


def listed():
    return [
        # a token for each of eight running sequences, at positions far apart: what a deployed policy does at every step
        dict(name="qk_8", kind="qk", tokens=8, q_heads=16, kv_heads=4, dim=128, rotary=128, pairs="halves", far=100_000, type="bf16",
             per_head=False),
        # a mini-batch of sequences
        dict(name="qk_16k", kind="qk", tokens=16384, q_heads=16, kv_heads=8, dim=128, rotary=128, pairs="halves", far=4096, type="bf16",
             per_head=False),
        # a small fp32 model's, a part of each head turned, neighbours paired, a weight for each head, an odd number of tokens
        dict(name="qkgrad_4099_odd", kind="qkgrad", tokens=4099, q_heads=6, kv_heads=2, dim=80, rotary=40, pairs="neighbours", far=4099,
             type="f32", per_head=True),
        # a large mini-batch
        dict(name="qkgrad_32k", kind="qkgrad", tokens=32768, q_heads=16, kv_heads=8, dim=128, rotary=128, pairs="halves", far=32768,
             type="bf16", per_head=False),
        # a few short episodes of a small fp32 model whose states come from before and go on after
        dict(name="mix_577_odd", kind="mix", tokens=577, seqs=5, q_heads=6, kv_heads=3, dk=40, dv=72, type="f32", states=True),
        # one long prompt
        dict(name="mix_64k", kind="mix", tokens=65536, seqs=1, q_heads=16, kv_heads=16, dk=128, dv=128, type="bf16", states=True),
        # a mini-batch of episodes of many lengths
        dict(name="mixgrad_32k", kind="mixgrad", tokens=32768, seqs=48, q_heads=16, kv_heads=8, dk=128, dv=128, type="bf16", states=False),
        # a token for each of eight running sequences
        dict(name="step_8", kind="step", seqs=8, slots=64, q_heads=16, kv_heads=4, dk=128, dv=128, type="bf16"),
        # one for each of many environments
        dict(name="step_1k", kind="step", seqs=1024, slots=1024, q_heads=16, kv_heads=8, dk=128, dv=128, type="bf16"),
        # log-probabilities of a few running sequences' tokens under a large vocabulary
        dict(name="xent_8_logp", kind="xent", rows=8, vocab=131072, dim=1024, type="bf16", masked=0.0, grad=False),
        # a short fp32 micro-batch, odd vocabulary and width
        dict(name="xent_257_odd", kind="xent", rows=257, vocab=50021, dim=515, type="f32", masked=0.25, grad=True),
        # a mini-batch of demonstrations, a large vocabulary
        dict(name="xent_8k_128k", kind="xent", rows=8192, vocab=131072, dim=2048, type="bf16", masked=0.25, grad=True),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
    return kv * rng.choice([1, 1, 2, 3, 4]), kv


def draw(rng):
    kind = rng.choice(["qk", "qkgrad", "mix", "mix", "mixgrad", "mixgrad", "step", "xent", "xent", "xent"])
    t = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind == "xent":
        d, v = _spread(rng, 32, 4096), _spread(rng, 1000, 131072)
        if rng.random() < 0.5:  # half of the widths as models have them, the others odd or even as they come
            d, v = -(-d // 64) * 64, -(-v // 64) * 64
        grad = rng.random() < 0.7
        most = (1 << 38) // (v * d) if t == "f32" else (1 << 41) // (v * d)
        return dict(kind=kind, rows=max(1, min(_spread(rng, 1, 16384), most)), vocab=v, dim=d, type=t,
                    masked=rng.choice([0.0, 0.25, 0.6]), grad=grad)
    q_heads, kv_heads = _heads(rng)
    if kind in ("qk", "qkgrad"):
        dim = rng.choice([64, 128, 128, 256, 2 * _spread(rng, 4, 128)])
        rotary = dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2)
        tokens = min(_spread(rng, 1, 65536), (1 << 27) // ((q_heads + kv_heads) * dim))
        return dict(kind=kind, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, dim=dim, rotary=rotary,
                    pairs=rng.choice(["halves", "halves", "neighbours"]), far=_spread(rng, 16, 1 << 20), type=t,
                    per_head=rng.random() < 0.3)
    dk, dv = (rng.choice([64, 128, 128, _spread(rng, 8, 128)]) for _ in range(2))
    if kind == "step":
        seqs, kv_heads = _spread(rng, 1, 1024), min(kv_heads, 8)
        return dict(kind=kind, seqs=seqs, slots=seqs + rng.choice([0, 0, 7]), q_heads=kv_heads * rng.choice([1, 2, 4]),
                    kv_heads=kv_heads, dk=dk, dv=dv, type=t)
    tokens = min(_spread(rng, 1, 65536), (1 << 25 if t == "f32" else 1 << 26) // (q_heads * 128))
    return dict(kind=kind, tokens=tokens, seqs=min(_spread(rng, 1, 128), tokens), q_heads=q_heads, kv_heads=kv_heads, dk=dk, dv=dv,
                type=t, states=rng.random() < 0.5)


def _lengths(case):
    """Tokens of each sequence, spread over a decade and more, the same for the same case."""
    rng, n, total = random.Random(case["seqs"] * 1_000_003 + case["tokens"]), case["seqs"], case["tokens"]
    w = [math.exp(rng.uniform(0.0, 3.0)) for _ in range(n)]
    s = [int(total * x / sum(w)) for x in w]
    s[-1] += total - sum(s)
    return s


def _tokens(n, vocab, g):
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp_(0, vocab - 1)


def _fading(heads):
    """Heads that look back over 16 to some thousand tokens."""
    reach = torch.exp2(torch.linspace(4.0, 12.0, heads, dtype=torch.float64))
    return torch.log1p(-1.0 / reach).float().cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, dtype=torch.float32: torch.randn(*shape, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    empty = lambda *shape, dtype=torch.float32: torch.empty(*shape, device="cuda", dtype=dtype)  # noqa: E731
    s, t, kind = dict(case), TYPES[case["type"]], case["kind"]
    if kind == "xent":
        r, v, d = case["rows"], case["vocab"], case["dim"]
        w = normal(v, d, dtype=t).mul_(2.0 / math.sqrt(d))
        tok = _tokens(r, v, g)
        h = normal(r, d).add_(w[tok].float(), alpha=1.5).to(t)
        s.update(w=w, h=h, tok=tok, valid=None, lp=empty(r))
        if case["masked"] > 0:
            s["valid"] = torch.rand(r, generator=g, device="cuda") >= case["masked"]
        if case["grad"]:
            s.update(dh=torch.empty_like(h), dw=torch.empty_like(w), stats=torch.zeros(4, device="cuda"))
        else:
            s["ent"] = empty(r)
        return s
    hq, hk = case["q_heads"], case["kv_heads"]
    if kind in ("qk", "qkgrad"):
        n, d = case["tokens"], case["dim"]
        both = normal(n, (hq + 2 * hk) * d, dtype=t)  # queries, keys and values side by side, as a projection leaves them
        s["q"], s["k"] = both[:, :hq * d].view(n, hq, d), both[:, hq * d:(hq + hk) * d].view(n, hk, d)
        weight = lambda h: normal(*((h, d) if case["per_head"] else (d,))).mul_(0.2).add_(1.0).to(t)  # noqa: E731
        s["wq"], s["wk"] = weight(hq), weight(hk)
        s["pos"] = torch.randint(0, case["far"], (n,), generator=g, device="cuda")
        s["freqs"] = BASE ** (torch.arange(0, case["rotary"], 2, dtype=torch.float64, device="cuda") / -case["rotary"])
        s["yq"], s["yk"] = empty(n, hq, d, dtype=t), empty(n, hk, d, dtype=t)
        if kind == "qkgrad":
            s["gq"], s["gk"] = normal(n, hq, d, dtype=t), normal(n, hk, d, dtype=t)
            s["dwq"], s["dwk"] = torch.empty_like(s["wq"]), torch.empty_like(s["wk"])
        return s
    dk, dv = case["dk"], case["dv"]
    s["log_decay"], s["scale"] = _fading(hk), dk**-0.5
    if kind == "step":
        n = case["seqs"]
        s["slot"] = torch.randperm(case["slots"], generator=g, device="cuda")[:n].to(torch.int32)
        s["fresh"] = torch.rand(n, generator=g, device="cuda") < 0.1  # episodes that begin
        s["state"] = normal(case["slots"], hk, dk, dv).mul_(3.0)
    else:
        n = case["tokens"]
        s["lengths"] = _lengths(case)
        s["cu"] = torch.tensor([0] + s["lengths"], device="cuda").cumsum(0).to(torch.int32)
        s["s0"] = normal(case["seqs"], hk, dk, dv).mul_(3.0) if case["states"] else None
        s["s1"] = torch.empty_like(s["s0"]) if case["states"] else None
    s["q"], s["k"], s["v"] = normal(n, hq, dk, dtype=t), normal(n, hk, dk, dtype=t), normal(n, hk, dv, dtype=t)
    if kind == "mixgrad":
        s["g"], s["g1"] = normal(n, hq, dv, dtype=t), normal(case["seqs"], hk, dk, dv) if case["states"] else None
        s.update(dq=torch.empty_like(s["q"]), dk_=torch.empty_like(s["k"]), dv_=torch.empty_like(s["v"]))
    else:
        s["o"] = empty(n, hq, dv, dtype=t)
    return s


def run(s):
    return _own(s) if own else _PLAIN[s["kind"]](s)


def _own(s):
    from tt_rsl_rl_amd import ops

    kind = s["kind"]
    if kind == "qk":
        ops.qk_norm_rotary_fwd(s["q"], s["k"], s["wq"], s["wk"], s["pos"], s["freqs"], s["yq"], s["yk"], eps=EPS,
                               interleaved=s["pairs"] == "neighbours")
        return {"q": s["yq"], "k": s["yk"]}
    if kind == "qkgrad":
        ops.qk_norm_rotary_bwd(s["gq"], s["gk"], s["q"], s["k"], s["wq"], s["wk"], s["pos"], s["freqs"], s["yq"], s["yk"], s["dwq"],
                               s["dwk"], eps=EPS, interleaved=s["pairs"] == "neighbours")
        return {"dq": s["yq"], "dk": s["yk"], "dwq": s["dwq"], "dwk": s["dwk"]}
    if kind == "mix":
        ops.decay_attention_fwd(s["q"], s["k"], s["v"], s["log_decay"], s["o"], scale=s["scale"], cu_seqlens=s["cu"],
                                initial_state=s["s0"], final_state=s["s1"])
        return {"o": s["o"], "state": s["s1"]}
    if kind == "mixgrad":
        ops.decay_attention_bwd(s["g"], s["q"], s["k"], s["v"], s["log_decay"], s["dq"], s["dk_"], s["dv_"], scale=s["scale"],
                                cu_seqlens=s["cu"], initial_state=s["s0"], d_final_state=s["g1"], d_initial_state=s["s1"])
        return {"dq": s["dq"], "dk": s["dk_"], "dv": s["dv_"], "dstate": s["s1"]}
    if kind == "step":
        ops.decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["o"], scale=s["scale"], slots=s["slot"],
                                 fresh=s["fresh"])
        return {"o": s["o"], "state": s["state"]}
    if s["grad"]:
        ops.linear_cross_entropy(s["h"], s["w"], s["tok"], s["dh"], s["dw"], s["stats"], logp=s["lp"], mask=s["valid"],
                                 temperature=TEMPERATURE)
        return {"dh": s["dh"], "dw": s["dw"], "loss": s["stats"][:1], "lp": s["lp"]}
    ops.linear_log_probs(s["h"], s["w"], s["tok"], s["lp"], s["ent"], mask=s["valid"], temperature=TEMPERATURE)
    return {"lp": s["lp"], "h": s["ent"]}


# ---- the plain forms ----


def _turned(x, s, back):
    """x [tokens, heads, dim] turned by its tokens' angles, or back."""
    angle = (s["pos"].double()[:, None] * s["freqs"])[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if back:
        sin = -sin
    r = s["rotary"]
    if s["pairs"] == "halves":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., r:]], -1)


def _qk(s):
    def one(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        return _turned(x * w.float(), s, False).to(w.dtype)

    return {"q": one(s["q"], s["wq"]), "k": one(s["k"], s["wk"])}


def _qkgrad(s):
    def one(x, w, g):
        x, g = x.float(), _turned(g.float(), s, True)
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n = x * rstd
        gw = g * w.float()
        dx = rstd * (gw - n * (gw * n).mean(-1, keepdim=True))
        dw = (g * n).sum(0) if w.dim() == 2 else (g * n).sum((0, 1))
        return dx.to(w.dtype), dw.to(w.dtype)

    (dq, dwq), (dk, dwk) = one(s["q"], s["wq"], s["gq"]), one(s["k"], s["wk"], s["gk"])
    return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


def _sequences(s):
    at = 0
    for i, n in enumerate(s["lengths"]):
        yield i, at, at + n
        at += n


def _by_head(x, i, j):
    return x[i:j].transpose(0, 1).float()


def _fades(s, c):
    """decay^(i - j) for i >= j of c tokens, else 0; decay^(i + 1); decay^(c - 1 - j); decay^c: each [kv_heads, ...]."""
    at = torch.arange(c, device="cuda", dtype=torch.float64)
    ld = s["log_decay"].double()[:, None]
    apart = at[:, None] - at[None, :]
    inside = torch.where(apart >= 0, torch.exp(apart.clamp(min=0) * ld[:, :, None]), torch.zeros_like(apart))
    return inside.float(), torch.exp(ld * (at + 1)).float(), torch.exp(ld * (c - 1 - at)).float(), torch.exp(ld * c).float()[:, :, None]


def _mix(s):
    """Chunks of tokens one after another: inside a chunk by the matrix of query-key products, what lies before by the state."""
    hq, hk, group = s["q_heads"], s["kv_heads"], s["q_heads"] // s["kv_heads"]
    out = torch.empty_like(s["o"])
    last = torch.empty_like(s["s1"]) if s["states"] else None
    fades = {}
    for b, start, end in _sequences(s):
        state = s["s0"][b] if s["states"] else torch.zeros(hk, s["dk"], s["dv"], device="cuda")
        for i in range(start, end, CHUNK):
            j = min(i + CHUNK, end)
            if j - i not in fades:
                fades[j - i] = _fades(s, j - i)
            inside, begun, left, whole = fades[j - i]
            q = (_by_head(s["q"], i, j) * s["scale"]).view(hk, group, j - i, s["dk"])
            k, v = _by_head(s["k"], i, j), _by_head(s["v"], i, j)
            p = torch.matmul(q, k.transpose(1, 2).contiguous()[:, None]) * inside[:, None]
            o = torch.matmul(p, v[:, None]) + torch.matmul(q, state[:, None]) * begun[:, None, :, None]
            out[i:j] = o.reshape(hq, j - i, s["dv"]).transpose(0, 1).to(out.dtype)
            state = state * whole + torch.matmul((k * left[:, :, None]).transpose(1, 2).contiguous(), v)
        if s["states"]:
            last[b] = state
    return {"o": out, "state": last}


def _mixgrad(s):
    """Once through each sequence for the states and the queries' gradient, once back for the others."""
    hq, hk, group = s["q_heads"], s["kv_heads"], s["q_heads"] // s["kv_heads"]
    dq, dk, dv = torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["v"])
    first = torch.empty_like(s["s1"]) if s["states"] else None
    fades = {}
    for b, start, end in _sequences(s):
        state = s["s0"][b] if s["states"] else torch.zeros(hk, s["dk"], s["dv"], device="cuda")
        spans = [(i, min(i + CHUNK, end)) for i in range(start, end, CHUNK)]
        for i, j in spans:
            if j - i not in fades:
                fades[j - i] = _fades(s, j - i)
            inside, begun, left, whole = fades[j - i]
            k, v = _by_head(s["k"], i, j), _by_head(s["v"], i, j)
            g = (_by_head(s["g"], i, j) * s["scale"]).view(hk, group, j - i, s["dv"])
            gp = torch.matmul(g, v.transpose(1, 2).contiguous()[:, None]) * inside[:, None]
            d = torch.matmul(gp, k[:, None]) + torch.matmul(g, state.transpose(1, 2).contiguous()[:, None]) * begun[:, None, :, None]
            dq[i:j] = d.reshape(hq, j - i, s["dk"]).transpose(0, 1).to(dq.dtype)
            state = state * whole + torch.matmul((k * left[:, :, None]).transpose(1, 2).contiguous(), v)
        back = s["g1"][b] if s["states"] else torch.zeros(hk, s["dk"], s["dv"], device="cuda")
        for i, j in reversed(spans):
            inside, begun, left, whole = fades[j - i]
            k, v = _by_head(s["k"], i, j), _by_head(s["v"], i, j)
            q = _by_head(s["q"], i, j).view(hk, group, j - i, s["dk"])
            g = (_by_head(s["g"], i, j) * s["scale"]).view(hk, group, j - i, s["dv"])
            p = torch.matmul(q, k.transpose(1, 2).contiguous()[:, None]) * inside[:, None]
            gp = torch.matmul(g, v.transpose(1, 2).contiguous()[:, None]) * inside[:, None]
            dk_ = torch.matmul(gp.transpose(2, 3).contiguous(), q).sum(1) + torch.matmul(v, back.transpose(1, 2).contiguous()) * left[:, :, None]
            dv_ = torch.matmul(p.transpose(2, 3).contiguous(), g).sum(1) + torch.matmul(k, back) * left[:, :, None]
            dk[i:j], dv[i:j] = dk_.transpose(0, 1).to(dk.dtype), dv_.transpose(0, 1).to(dv.dtype)
            back = back * whole + torch.matmul((q * begun[:, None, :, None]).transpose(2, 3).contiguous(), g).sum(1)
        if s["states"]:
            first[b] = back
    return {"dq": dq, "dk": dk, "dv": dv, "dstate": first}


def _step(s):
    slot, group = s["slot"].long(), s["q_heads"] // s["kv_heads"]
    before = torch.where(s["fresh"][:, None, None, None], torch.zeros((), device="cuda"), s["state"][slot])
    state = before * torch.exp(s["log_decay"].double()).float()[:, None, None] + s["k"].float()[..., None] * s["v"].float()[..., None, :]
    q = (s["q"].float() * s["scale"]).view(-1, s["kv_heads"], group, s["dk"])
    o = (q[..., None] * state[:, :, None]).sum(-2).view(s["o"].shape) if len(slot) < 64 else torch.matmul(q, state).view(s["o"].shape)
    s["state"][slot] = state
    return {"o": o.to(s["o"].dtype), "state": s["state"]}


def _xent(s):
    r, kept = s["rows"], s["valid"]
    h, w = s["h"].float(), s["w"].float()
    z = torch.matmul(h, w.t()) * (1.0 / TEMPERATURE)
    z -= z.amax(1, keepdim=True)
    at = z.gather(1, s["tok"][:, None])[:, 0]
    e = torch.exp(z)
    total = e.sum(1)
    zero = torch.zeros(r, device="cuda")
    lp = at - torch.log(total)
    if kept is not None:
        lp = torch.where(kept, lp, zero)
    if not s["grad"]:
        ent = torch.log(total) - (e * z).sum(1) / total
        return {"lp": lp, "h": ent if kept is None else torch.where(kept, ent, zero)}
    n = float(r) if kept is None else kept.sum().clamp(min=1).float()
    del z
    e /= total[:, None]
    e[torch.arange(r, device="cuda"), s["tok"]] -= 1.0
    e *= 1.0 / (n * TEMPERATURE)
    if kept is not None:
        e *= kept[:, None]
    return {"dh": torch.matmul(e, w).to(s["h"].dtype), "dw": torch.matmul(e.t(), h).to(s["w"].dtype), "loss": (-lp.sum() / n)[None], "lp": lp}


_PLAIN = {"qk": _qk, "qkgrad": _qkgrad, "mix": _mix, "mixgrad": _mixgrad, "step": _step, "xent": _xent}


def work(case):
    kind, e = case["kind"], SIZE[case["type"]]
    if kind == "xent":
        r, v, d = case["rows"], case["vocab"], case["dim"]
        kept = r * (1 - case["masked"])  # masked rows need no products
        if case["grad"]:
            return {"bytes": (kept + r + 2 * v) * d * e + r * 13, "flops": 6 * kept * v * d}
        return {"bytes": (kept + v) * d * e + r * 17, "flops": 2 * kept * v * d}
    hq, hk = case["q_heads"], case["kv_heads"]
    if kind in ("qk", "qkgrad"):
        n, d = case["tokens"], case["dim"]
        x = n * (hq + hk) * d
        weights = (hq + hk if case["per_head"] else 2) * d * e
        if kind == "qk":
            return {"bytes": 2 * x * e + n * 8 + weights, "flops": 7 * x}
        return {"bytes": 3 * x * e + n * 8 + 2 * weights, "flops": 14 * x}
    dk, dv = case["dk"], case["dv"]
    if kind == "step":
        n = case["seqs"]
        return {"bytes": n * (2 * hk * dk * dv * 4 + (hq * (dk + dv) + hk * (dk + dv)) * e + 5), "flops": n * dk * dv * (3 * hk + 2 * hq)}
    n = case["tokens"]
    states = 2 * case["seqs"] * hk * dk * dv * 4 if case["states"] else 0
    qkvo = n * (hq * (dk + dv) + hk * (dk + dv)) * e
    once = n * dk * dv * (2 * hk + 2 * hq)  # each token into the state, and the state's answer to each query
    if kind == "mix":
        return {"bytes": qkvo + states, "flops": once}
    return {"bytes": qkvo + n * (hq * dk + hk * (dk + dv)) * e + 1.5 * states, "flops": 3 * once}


# ---- the definitions in 64 bits ----


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("qk", "qkgrad"):
        out = {}
        for name, x, w, g in (("q", s["q"], s["wq"], s.get("gq")), ("k", s["k"], s["wk"], s.get("gk"))):
            parts = [_exact_turned(s, i, x, w, g) for i in range(0, case["tokens"], 4096)]
            if kind == "qk":
                out[name] = torch.cat([p[0] for p in parts])
            else:
                out["d" + name], out["dw" + name] = torch.cat([p[0] for p in parts]), sum(p[1] for p in parts)
        return out
    if kind in ("mix", "mixgrad"):
        return _exact_mix(s)
    if kind == "step":
        state = s["state"].double()
        decay, group = torch.exp(s["log_decay"].double()), case["q_heads"] // case["kv_heads"]
        o = torch.empty(s["o"].shape, dtype=torch.float64, device="cuda")
        for n, slot in enumerate(s["slot"].tolist()):
            if bool(s["fresh"][n]):
                state[slot] = 0
            state[slot] = decay[:, None, None] * state[slot] + s["k"][n].double()[:, :, None] * s["v"][n].double()[:, None, :]
            o[n] = case["dk"] ** -0.5 * torch.matmul(s["q"][n].double()[:, None, :], state[slot].repeat_interleave(group, 0))[:, 0]
        return {"o": o, "state": state}
    keep = torch.ones(case["rows"], dtype=torch.bool, device="cuda") if s["valid"] is None else s["valid"]
    n, w = max(1, int(keep.sum())), s["w"].double()
    lp, ent, dh = (torch.zeros(*shape, dtype=torch.float64, device="cuda") for shape in ((case["rows"],), (case["rows"],), s["h"].shape))
    dw = torch.zeros_like(w) if case["grad"] else None
    for rows in keep.nonzero()[:, 0].split(1024):
        h, tok = s["h"][rows].double(), s["tok"][rows]
        logs = torch.log_softmax(torch.matmul(h, w.t()) / TEMPERATURE, dim=1)
        lp[rows] = logs[torch.arange(len(rows), device="cuda"), tok]
        p = logs.exp()
        ent[rows] = -(p * logs).sum(1)
        if case["grad"]:
            p[torch.arange(len(rows), device="cuda"), tok] -= 1
            dh[rows] = torch.matmul(p, w) / (n * TEMPERATURE)
            dw += torch.matmul(p.t(), h) / (n * TEMPERATURE)
    return {"dh": dh, "dw": dw, "loss": -lp.sum()[None] / n, "lp": lp} if case["grad"] else {"lp": lp, "h": ent}


def _exact_turned(s, i, x, w, g):
    """Tokens i to i + 4095, each pair of a head as a complex number; the gradients by autograd."""
    r, d = s["rotary"], s["dim"]
    x = x[i:i + 4096].double().requires_grad_(g is not None)
    w = w.double().requires_grad_(g is not None)
    y = x / torch.sqrt((x**2).sum(-1, keepdim=True) / d + EPS) * w
    if s["pairs"] == "halves":
        pairs = torch.complex(y[..., :r // 2], y[..., r // 2:r])
    else:
        pairs = torch.complex(y[..., 0:r:2], y[..., 1:r:2])
    angle = s["pos"][i:i + 4096].double()[:, None, None] * s["freqs"]
    pairs = pairs * torch.polar(torch.ones_like(angle), angle)
    if s["pairs"] == "halves":
        y = torch.cat([pairs.real, pairs.imag, y[..., r:]], -1)
    else:
        y = torch.cat([torch.view_as_real(pairs).flatten(-2), y[..., r:]], -1)
    if g is None:
        return (y,)
    return torch.autograd.grad(y, (x, w), g[i:i + 4096].double())


def _exact_mix(s):
    """Each output as the sum over all tokens before it, blocks of queries against everything they see; None if that is long."""
    hk, group, scale, ld = s["kv_heads"], s["q_heads"] // s["kv_heads"], s["dk"] ** -0.5, s["log_decay"].double()
    if sum(n * n for n in s["lengths"]) * s["q_heads"] * (s["dk"] + s["dv"]) * (1 if s["kind"] == "mix" else 3) > 4e13:
        return None
    grad = s["kind"] == "mixgrad"
    zeros = lambda x: torch.zeros(x.shape, dtype=torch.float64, device="cuda") if x is not None else None  # noqa: E731
    out, last = (None, None) if grad else (zeros(s["o"]), zeros(s["s1"]))
    dq, dk, dv, first = (zeros(s["q"]), zeros(s["k"]), zeros(s["v"]), zeros(s["s1"])) if grad else (None, None, None, None)
    for b, start, end in _sequences(s):
        at = torch.arange(start, end, device="cuda", dtype=torch.float64)
        for h in range(hk):
            k, v = s["k"][start:end, h].double(), s["v"][start:end, h].double()
            if s["states"]:
                after, before = torch.exp(ld[h] * (end - 1 - at))[:, None], torch.exp(ld[h] * (at - start + 1))[:, None]
                whole = torch.exp(ld[h] * (end - start))
                if grad:
                    first[b, h] = whole * s["g1"][b, h].double()
                    dk[start:end, h] += after * torch.matmul(v, s["g1"][b, h].double().t())
                    dv[start:end, h] += after * torch.matmul(k, s["g1"][b, h].double())
                else:
                    last[b, h] = whole * s["s0"][b, h].double() + torch.matmul((after * k).t(), v)
            for f in range(h * group, (h + 1) * group):
                for i in range(start, end, 2048):
                    j = min(i + 2048, end)
                    apart = at[i - start:j - start, None] - at[None, :j - start]
                    fade = torch.where(apart >= 0, torch.exp(ld[h] * apart.clamp(min=0)), torch.zeros_like(apart)) * scale
                    q, kk, vv = s["q"][i:j, f].double(), k[:j - start], v[:j - start]
                    if grad:
                        g = s["g"][i:j, f].double()
                        gp = torch.matmul(g, vv.t()) * fade
                        dq[i:j, f] = torch.matmul(gp, kk)
                        dk[start:j, h] += torch.matmul(gp.t(), q)
                        dv[start:j, h] += torch.matmul((torch.matmul(q, kk.t()) * fade).t(), g)
                        if s["states"]:
                            dq[i:j, f] += scale * before[i - start:j - start] * torch.matmul(g, s["s0"][b, h].double().t())
                            first[b, h] += scale * torch.matmul((before[i - start:j - start] * q).t(), g)
                    else:
                        out[i:j, f] = torch.matmul(torch.matmul(q, kk.t()) * fade, vv)
                        if s["states"]:
                            out[i:j, f] += scale * before[i - start:j - start] * torch.matmul(q, s["s0"][b, h].double())
    return {"dq": dq, "dk": dk, "dv": dv, "dstate": first} if grad else {"o": out, "state": last}
