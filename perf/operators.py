"""The operators of a policy that acts in tokens, as cases to time: the two ends of its network, which are as wide as the
vocabulary, and the optimiser of its many tensors.  One pass is one call of ``tt_rsl_rl_amd.ops``:

    embed   ``embedding_fwd``: rows of a table looked up by token, scaled
    egrad   ``embedding_bwd``: the table's gradient, each token's rows summed in fp32 (``into`` = added to what is there)
    logp    ``token_log_probs``: log-probability and entropy of each row's token, as a rollout stores them
    loss    ``token_ppo_loss``: clipped policy loss with a KL term to a reference and an entropy bonus, and the gradient of
            the logits
    adamw   ``adamw_step``: clip by the global norm and AdamW over a list of tensors, states in 32 bits or in 8

Tokens follow 1 / rank (a vocabulary sorted by frequency), logits are normal with the taken token raised, masked rows
stand for prompts and padding.  With ``own`` false the same results come from elementary torch operations.
"""

from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
CLIP, KL, ENTROPY, TEMPERATURE, SCALE = 0.2, 0.05, 0.01, 0.9, 0.5
BETA1, BETA2, EPS, DECAY, LR, MAX_NORM, STEP = 0.9, 0.999, 1e-8, 0.01, 1e-4, 1.0, 1000
BLOCK = 256  # elements that share a scale where AdamW's states are held in 8 bits
HUMANOID = [(29,), (512, 96), (512,), (256, 512), (256,), (128, 256), (128,), (29, 128), (29,),
            (512, 99), (512,), (256, 512), (256,), (128, 256), (128,), (1, 128), (1,)]


def listed():
    return [
        # one token for each of eight running sequences: what a deployed policy looks up at every step
        dict(name="embed_8", kind="embed", tokens=8, vocab=32000, dim=1024, type="bf16"),
        # a mini-batch of whole sequences
        dict(name="embed_16k", kind="embed", tokens=16384, vocab=65536, dim=2048, type="bf16"),
        # a small fp32 model of odd width on a mini-batch of odd length
        dict(name="egrad_5003_odd", kind="egrad", tokens=5003, vocab=10007, dim=515, type="f32", out="f32", into=False),
        # a large mini-batch, bf16 gradients into an fp32 table
        dict(name="egrad_128k", kind="egrad", tokens=131072, vocab=65536, dim=1024, type="bf16", out="f32", into=False),
        # the log-probabilities of a deployed policy's own tokens, a few rows of a large vocabulary
        dict(name="logp_8", kind="logp", rows=8, vocab=131072, type="bf16", masked=0.0, banned=False),
        # those of a rollout under the reference policy
        dict(name="logp_8k", kind="logp", rows=8192, vocab=32000, type="bf16", masked=0.25, banned=False),
        # a short micro-batch, fp32 logits, odd vocabulary, tokens that are not allowed at -inf
        dict(name="loss_257_odd", kind="loss", rows=257, vocab=50021, type="f32", masked=0.25, banned=True),
        # a mini-batch of a small vocabulary
        dict(name="loss_4k", kind="loss", rows=4096, vocab=32000, type="bf16", masked=0.25, banned=False),
        # one of a large vocabulary
        dict(name="loss_8k_128k", kind="loss", rows=8192, vocab=131072, type="bf16", masked=0.25, banned=False),
        # actor and critic of the humanoid workload, as separate tensors
        dict(name="adamw_humanoid", kind="adamw", shapes="humanoid", tensors=len(HUMANOID),
             total=sum(math.prod(s) for s in HUMANOID), param="f32", master=False, grad="f32", bits=32, clip=True),
        # a bf16 model of 150 tensors with fp32 masters
        dict(name="adamw_60m", kind="adamw", shapes="drawn", tensors=150, total=60_000_000, param="bf16", master=True,
             grad="bf16", bits=32, clip=True),
        # a large one whose states are held in 8 bits
        dict(name="adamw_250m_8bit", kind="adamw", shapes="drawn", tensors=40, total=250_000_000, param="bf16", master=True,
             grad="bf16", bits=8, clip=True),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embed", "egrad", "egrad", "logp", "loss", "loss", "adamw", "adamw"])
    if kind in ("embed", "egrad"):
        c = dict(kind=kind, vocab=_spread(rng, 500, 131072), dim=_spread(rng, 32, 4096), type=rng.choice(["f32", "bf16", "f16"]))
        if rng.random() < 0.5:  # half of the widths as models have them, the others odd or even as they come
            c["dim"] = -(-c["dim"] // 64) * 64
        c["vocab"] = min(c["vocab"], (1 << 28) // c["dim"])
        c["tokens"] = min(_spread(rng, 1, 262144), (1 << 28) // c["dim"])
        if kind == "egrad":
            c.update(out=rng.choice(["f32", c["type"]]), into=rng.random() < 0.3)
        return c
    if kind in ("logp", "loss"):
        t = rng.choice(["f32", "bf16", "bf16", "f16"])
        v = _spread(rng, 1000, 131072)
        if rng.random() < 0.5:
            v = -(-v // 64) * 64
        return dict(kind=kind, rows=min(_spread(rng, 1, 16384), (1 << 30) // (v * SIZE[t] // 2)), vocab=v, type=t,
                    masked=rng.choice([0.0, 0.25, 0.6]), banned=rng.random() < 0.3)
    total = _spread(rng, 20_000, 250_000_000)
    p = rng.choice(["f32", "bf16"])
    return dict(kind="adamw", shapes="drawn", tensors=min(_spread(rng, 1, 200), total // 100), total=total, param=p,
                master=p == "bf16" and rng.random() < 0.7, grad=rng.choice(["f32", p]), bits=rng.choice([32, 8]),
                clip=rng.random() < 0.7)


def _sizes(case):
    """Elements of each tensor: the humanoid models', or sizes spread over two decades, the same for the same case."""
    if case["shapes"] == "humanoid":
        return [math.prod(s) for s in HUMANOID]
    rng, n, total = random.Random(case["tensors"] * 1_000_003 + case["total"]), case["tensors"], case["total"]
    w = [math.exp(rng.uniform(0.0, 4.6)) for _ in range(n)]
    s = [max(1, int(total * x / sum(w))) for x in w]
    s[0] += max(0, total - sum(s))
    return s


def _tokens(n, vocab, g):
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp_(0, vocab - 1)


def _distinct(n, vocab):
    """How many different tokens n draws are expected to hold."""
    k = torch.arange(1, vocab + 1, dtype=torch.float64)
    return float((1 - torch.exp(n * torch.log1p(-torch.log((k + 1) / k) / math.log(vocab + 1)))).sum())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, dtype=torch.float32: torch.randn(*shape, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    s = dict(case)
    if case["kind"] in ("embed", "egrad"):
        m, v, d, t = case["tokens"], case["vocab"], case["dim"], TYPES[case["type"]]
        s["tok"] = _tokens(m, v, g)
        if case["kind"] == "embed":
            s["table"], s["y"] = normal(v, d, dtype=t), torch.empty(m, d, dtype=t, device="cuda")
        else:
            s["dy"] = normal(m, d, dtype=t)
            o = TYPES[case["out"]]
            s["dt"] = normal(v, d, dtype=o) if case["into"] else torch.zeros(v, d, dtype=o, device="cuda")
        return s
    if case["kind"] in ("logp", "loss"):
        r, v = case["rows"], case["vocab"]
        x = normal(r, v, dtype=TYPES[case["type"]]).mul_(2)
        tok = _tokens(r, v, g)
        rows = torch.arange(r, device="cuda")
        if case["banned"]:  # a third of the vocabulary, not the taken tokens
            taken = x[rows, tok].clone()
            x.masked_fill_((torch.rand(v, generator=g, device="cuda") < 0.33)[None, :], -math.inf)
            x[rows, tok] = taken
        x[rows, tok] += 6
        s.update(x=x, tok=tok, valid=None, lp=torch.empty(r, device="cuda"), h=torch.empty(r, device="cuda"))
        if case["masked"] > 0:
            s["valid"] = torch.rand(r, generator=g, device="cuda") >= case["masked"]
        if case["kind"] == "loss":
            lp = torch.cat([torch.log_softmax(p.float() / TEMPERATURE, -1).gather(1, q[:, None])[:, 0]
                            for p, q in zip(x.split(1024), tok.split(1024))])
            # the policy has moved since the rollout; the sides of the clip range's ends are not left to roundings
            step = 0.15 * normal(r)
            for end in (math.log(1 - CLIP), math.log(1 + CLIP)):
                step = torch.where((step - end).abs() < 1e-3, torch.full_like(step, end + 1e-3), step)
            s.update(old=lp - step, ref=lp + 0.3 * normal(r), adv=normal(r), dx=torch.empty_like(x),
                     stats=torch.zeros(8, device="cuda"))
        return s
    sizes = _sizes(case)
    room = [-(-n // BLOCK) * BLOCK for n in sizes]  # each tensor starts on a scale's boundary of the flat buffers
    at = [sum(room[:i]) for i in range(len(room))]
    flat = sum(room)
    used = torch.zeros(flat, dtype=torch.bool, device="cuda")
    for a, n in zip(at, sizes):
        used[a:a + n] = True
    views = lambda f, each=1: [f[a // each:a // each + -(-n // each)] for a, n in zip(at, sizes)]  # noqa: E731
    p = normal(flat).mul_(0.02).mul_(used)
    m, u = normal(flat).mul_(1e-3).mul_(used), normal(flat).mul_(1e-3).square_().mul_(used)
    s["p"] = p.to(TYPES[case["param"]])
    s["g"] = normal(flat).mul_(2e-3).mul_(used).to(TYPES[case["grad"]])
    s["master"] = p if case["master"] else None
    if case["bits"] == 8:
        s["sm"], s["su"] = m.view(-1, BLOCK).abs().amax(1), u.view(-1, BLOCK).amax(1)
        s["m"], s["u"] = _code_m(m, s["sm"]), _code_u(u, s["su"])
    else:
        s.update(m=m, u=u, sm=None, su=None)
    s["lists"] = {k: views(s[k]) if s[k] is not None else None for k in ("p", "g", "m", "u", "master")}
    s["lists"].update({k: views(s[k], BLOCK) if s[k] is not None else None for k in ("sm", "su")})
    return s


# States in 8 bits: m = sign * scale * (|q| / 127)^2 and u = scale * (q / 255)^4, q >= 1 wherever u > 0 (a second moment
# that fell to zero would leave its parameter a step of m / eps).  Powers place the codes densely near zero.


def _code_m(m, scale):
    r = m.abs().view(-1, BLOCK) / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]
    return torch.copysign(torch.round(torch.sqrt(r) * 127.0), m.view(-1, BLOCK)).to(torch.int8).view(-1)


def _code_u(u, scale):
    r = u.view(-1, BLOCK) / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]
    q = torch.round(torch.sqrt(torch.sqrt(r)) * 255.0)
    return torch.where(u.view(-1, BLOCK) > 0, q.clamp(min=1.0), q).to(torch.uint8).view(-1)


def _value_m(q, scale):
    f = q.to(scale.dtype).view(-1, BLOCK)
    return (f.sign() * scale[:, None] * (f.abs() * (1.0 / 127.0)).square()).view(-1)


def _value_u(q, scale):
    return (scale[:, None] * (q.to(scale.dtype).view(-1, BLOCK) * (1.0 / 255.0)).square().square()).view(-1)


def run(s):
    return _own(s) if own else _PLAIN[s["kind"]](s)


def _own(s):
    from tt_rsl_rl_amd import ops

    kind = s["kind"]
    if kind == "embed":
        ops.embedding_fwd(s["tok"], s["table"], s["y"], scale=SCALE)
        return s["y"]
    if kind == "egrad":
        ops.embedding_bwd(s["tok"], s["dy"], s["dt"], scale=SCALE, accumulate=s["into"])
        return s["dt"]
    if kind == "logp":
        ops.token_log_probs(s["x"], s["tok"], s["lp"], s["h"], mask=s["valid"], temperature=TEMPERATURE)
        return {"lp": s["lp"], "h": s["h"]}
    if kind == "loss":
        ops.token_ppo_loss(s["x"], s["tok"], s["old"], s["adv"], s["dx"], s["stats"], ref_logp=s["ref"], logp=s["lp"],
                           entropy=s["h"], mask=s["valid"], clip_param=CLIP, kl_coef=KL, entropy_coef=ENTROPY,
                           temperature=TEMPERATURE)
        return {"dx": s["dx"], "lp": s["lp"], "h": s["h"], "stats": s["stats"][:6]}
    f = s["lists"]
    ops.adamw_step(f["p"], f["g"], f["m"], f["u"], step=STEP, lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS, weight_decay=DECAY,
                   max_grad_norm=MAX_NORM if s["clip"] else None, masters=f["master"], scales=(f["sm"], f["su"]) if s["bits"] == 8 else None)
    return _states(s)


def _states(s):
    out = {"p": s["p"], "master": s["master"]}
    if s["bits"] == 8:
        out.update(m=_value_m(s["m"], s["sm"]), u=_value_u(s["u"], s["su"]))
    else:
        out.update(m=s["m"], u=s["u"])
    return out


# ---- the plain forms ----


def _embed(s):
    return (s["table"][s["tok"]].float() * SCALE).to(s["table"].dtype)


def _egrad(s):
    start = s["dt"].float() if s["into"] else torch.zeros(s["dt"].shape, device="cuda")
    got = start.index_add(0, s["tok"], s["dy"].float() * SCALE)
    if s["into"]:
        s["dt"].copy_(got)
        return s["dt"]
    return got.to(s["dt"].dtype)


def _rows(s):
    """Scaled logits less their row's largest, their exponentials and sums, the token's log-probability, the entropy."""
    z = s["x"].float() * (1.0 / TEMPERATURE)
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1)
    log_total = torch.log(total)
    lp = z.gather(1, s["tok"][:, None])[:, 0] - log_total
    h = log_total - torch.where(e > 0, e * z, torch.zeros_like(z)).sum(1) / total
    return z, e, total, log_total, lp, h


def _kept(s, v):
    return v if s["valid"] is None else torch.where(s["valid"], v, torch.zeros_like(v))


def _logp(s):
    *_, lp, h = _rows(s)
    return {"lp": _kept(s, lp), "h": _kept(s, h)}


def _loss(s):
    z, e, total, log_total, lp, h = _rows(s)
    n = float(s["rows"]) if s["valid"] is None else s["valid"].sum().clamp(min=1).float()
    ratio = torch.exp(lp - s["old"])
    clipped = ratio.clamp(1 - CLIP, 1 + CLIP)
    first, second = -s["adv"] * ratio, -s["adv"] * clipped
    d = s["ref"] - lp
    kl = torch.exp(d) - d - 1
    mean = lambda v: _kept(s, v).sum() / n  # noqa: E731
    surrogate, kl_mean, h_mean = mean(torch.maximum(first, second)), mean(kl), mean(h)
    loss = surrogate + KL * kl_mean - ENTROPY * h_mean
    stats = torch.stack([loss, surrogate, kl_mean, h_mean, mean((ratio != clipped).float()), mean(s["old"] - lp)])
    c = torch.where(first >= second, first, torch.zeros_like(first)) + KL * (1 - torch.exp(d))
    p = e / total[:, None]
    dx = -c[:, None] * p + ENTROPY * torch.where(e > 0, p * (z - log_total[:, None] + h[:, None]), torch.zeros_like(p))
    dx[torch.arange(s["rows"], device="cuda"), s["tok"]] += c
    dx = _kept(s, dx.t()).t() if s["valid"] is not None else dx
    return {"dx": (dx * (1.0 / (n * TEMPERATURE))).to(s["x"].dtype), "lp": _kept(s, lp), "h": _kept(s, h), "stats": stats}


def _adamw(s):
    g = s["g"].float()
    if s["clip"]:
        total = torch.sqrt(g.double().square().sum()).float()
        g = g * torch.clamp(MAX_NORM / (total + 1e-6), max=1.0)
    m, u = (_value_m(s["m"], s["sm"]), _value_u(s["u"], s["su"])) if s["bits"] == 8 else (s["m"], s["u"])
    m = m + (1 - BETA1) * (g - m)
    u = u * BETA2 + ((1 - BETA2) * g) * g
    p = (s["p"].float() if s["master"] is None else s["master"]) * (1 - LR * DECAY)
    p = p + (-(LR / (1 - BETA1**STEP)) * m) / (torch.sqrt(u) / math.sqrt(1 - BETA2**STEP) + EPS)
    if s["bits"] == 8:
        s["sm"].copy_(m.view(-1, BLOCK).abs().amax(1))
        s["su"].copy_(u.view(-1, BLOCK).amax(1))
        m, u = _code_m(m, s["sm"]), _code_u(u, s["su"])
    s["m"].copy_(m)
    s["u"].copy_(u)
    s["p"].copy_(p)
    if s["master"] is not None:
        s["master"].copy_(p)
    return _states(s)


_PLAIN = {"embed": _embed, "egrad": _egrad, "logp": _logp, "loss": _loss, "adamw": _adamw}


def work(case):
    kind = case["kind"]
    if kind in ("embed", "egrad"):
        m, d, e = case["tokens"], case["dim"], SIZE[case["type"]]
        rows = _distinct(m, case["vocab"])
        if kind == "embed":
            return {"bytes": m * 8 + (rows + m) * d * e, "flops": m * d}
        o = SIZE[case["out"]]
        return {"bytes": m * (8 + d * e) + (2 * rows if case["into"] else case["vocab"]) * d * o, "flops": m * d}
    if kind in ("logp", "loss"):
        r, v, e = case["rows"], case["vocab"], SIZE[case["type"]]
        kept = r * (1 - case["masked"])  # masked rows are not read
        if kind == "logp":
            return {"bytes": kept * v * e + r * 16, "flops": 5 * kept * v}
        return {"bytes": (kept + r) * v * e + r * 32, "flops": 12 * kept * v}
    n = sum(_sizes(case))
    p = 8 + (2 if case["master"] else 0) if case["param"] == "f32" or case["master"] else 4
    return {"bytes": n * (p + SIZE[case["grad"]] + (4 + 16 / BLOCK if case["bits"] == 8 else 16)), "flops": 15 * n}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "embed":
        return torch.index_select(s["table"], 0, s["tok"]).double().mul(SCALE)
    if kind == "egrad":
        sums = torch.zeros(s["dt"].shape, dtype=torch.float64, device="cuda").index_add_(0, s["tok"], s["dy"].double())
        return s["dt"].double() * (1.0 if case["into"] else 0.0) + SCALE * sums
    if kind in ("logp", "loss"):
        parts = [_exact_rows(s, i, min(i + 1024, case["rows"])) for i in range(0, case["rows"], 1024)]
        out = {k: torch.cat([p[k] for p in parts]) for k in parts[0] if k != "sums"}
        if kind == "loss":
            surr, kl, h, outside, moved = sum(p["sums"] for p in parts).unbind()
            out["stats"] = torch.stack([surr + KL * kl - ENTROPY * h, surr, kl, h, outside, moved])
        return out
    # AdamW as published, bias-corrected moments; run() is called three times on one state where passes are compared, the
    # exact values are those of one call
    g = s["g"].double()
    if case["clip"]:
        g = g * min(1.0, MAX_NORM / (float(torch.linalg.vector_norm(g)) + 1e-6))
    m0 = s["m"].double() if case["bits"] == 32 else _value_m(s["m"], s["sm"].double())
    u0 = s["u"].double() if case["bits"] == 32 else _value_u(s["u"], s["su"].double())
    m1, u1 = BETA1 * m0 + (1 - BETA1) * g, BETA2 * u0 + (1 - BETA2) * g**2
    p = (s["p"] if s["master"] is None else s["master"]).double()
    m_hat, u_hat = m1 / (1 - BETA1**STEP), u1 / (1 - BETA2**STEP)
    p = p - LR * DECAY * p - LR * m_hat / (u_hat.sqrt() + EPS)
    if case["bits"] == 8:  # what the codes stand for depends on the last bit before they are rounded
        m1 = u1 = None
    return {"p": p, "master": p if case["master"] else None, "m": m1, "u": u1}


def _exact_rows(s, i, j):
    """exact() of rows i to j - 1: a row's terms and gradient depend on no other row but by the number of rows that count."""
    keep = torch.ones(j - i, dtype=torch.bool, device="cuda") if s["valid"] is None else s["valid"][i:j]
    x = s["x"][i:j][keep].double().requires_grad_(s["kind"] == "loss")
    logs = torch.log_softmax(x / TEMPERATURE, dim=1)
    lp = logs[torch.arange(len(logs), device="cuda"), s["tok"][i:j][keep]]
    probs = logs.exp()
    h = -(probs * torch.where(probs > 0, logs, torch.zeros_like(logs))).sum(dim=1)

    def full(v):
        out = torch.zeros(j - i, *v.shape[1:], dtype=torch.float64, device="cuda")
        out[keep] = v.detach()
        return out

    if s["kind"] == "logp":
        return {"lp": full(lp), "h": full(h)}
    n = s["rows"] if s["valid"] is None else max(1, int(s["valid"].sum()))
    old, ref, adv = (s[k][i:j][keep].double() for k in ("old", "ref", "adv"))
    ratio = (lp - old).exp()
    surr = -torch.min(adv * ratio, adv * ratio.clip(1 - CLIP, 1 + CLIP))
    kl = torch.expm1(ref - lp) - (ref - lp)
    ((surr + KL * kl - ENTROPY * h).sum() / n).backward()
    sums = [v.detach().sum() / n for v in (surr, kl, h, ((ratio - 1).abs() > CLIP).double(), old - lp)]
    return {"dx": full(x.grad), "lp": full(lp), "h": full(h), "sums": torch.stack(sums)}
