"""The modules and functions of tt_rsl_rl_amd.tokens between embedding and logits under autograd, all operators together as a policy uses them,
on another stream, in captured graphs, and the example."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

from tests import token_layer_reference as ref
from tests.test_gpu_token_ops import BF16, F32, U

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


def _policy(cuda, dtype=BF16, seed=0):
    spec = importlib.util.spec_from_file_location("sequence_policy", ROOT / "examples" / "sequence_policy.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(seed)
    return example, example.SequencePolicy(50, 64, 2, 4, 2, 16, cuda, dtype)


def _tokens(cuda, lengths, vocab=50, seed=1):
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, vocab, (sum(lengths),), generator=g)
    positions = torch.cat([torch.arange(n) for n in lengths])
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
    return tokens.to(cuda), positions.to(cuda), cu.to(cuda)


def test_qk_norm_rotary_gradient(cuda):
    """fp32, against the formula and against differences of the 64-bit form."""
    from tt_rsl_rl_amd.tokens import QkNormRotary

    g = torch.Generator().manual_seed(0)
    layer = QkNormRotary(32, rotary=16, interleaved=True, device=cuda)
    q, k = torch.randn(20, 4, 32, generator=g), torch.randn(20, 2, 32, generator=g)
    pos = torch.randint(0, 999, (20,), generator=g)
    dq, dk = torch.randn(20, 4, 32, generator=g), torch.randn(20, 2, 32, generator=g)
    a, b = q.to(cuda).requires_grad_(), k.to(cuda).requires_grad_()
    torch.autograd.backward(layer(a, b, pos.to(cuda)), (dq.to(cuda), dk.to(cuda)))
    freqs, ones = layer._freqs.cpu(), torch.ones(32)
    for got, got_w, x, d in ((a.grad, layer.q_weight.grad, q, dq), (b.grad, layer.k_weight.grad, k, dk)):
        want, want_w, size, size_w = ref.qk_rotary_grad(d, x, ones, pos, freqs, 1e-6, True)
        assert bool(((got.cpu().double() - want).abs() <= 120 * U * size + 1e-30).all())
        assert bool(((got_w.cpu().double() - want_w).abs() <= 200 * U * size_w).all())
    step, at = 1e-5, (3, 1, 5)
    moved = q.double().clone()
    moved[at] += step
    difference = ((ref.qk_rotary(moved, ones, pos, freqs, 1e-6, True)[0] - ref.qk_rotary(q, ones, pos, freqs, 1e-6, True)[0]) * dq.double()).sum() / step
    assert abs(float(a.grad[at]) - float(difference)) < 1e-3


def test_decay_attention_gradient(cuda):
    """fp32, states in and out, against autograd through the 64-bit form and differences of it."""
    from tt_rsl_rl_amd.tokens import decay_attention

    g = torch.Generator().manual_seed(3)
    cu = torch.tensor([0, 30, 30, 75])
    host = dict(q=torch.randn(75, 4, 24, generator=g), k=torch.randn(75, 2, 24, generator=g), v=torch.randn(75, 2, 40, generator=g),
                s=torch.randn(3, 2, 24, 40, generator=g))
    ld = torch.log(torch.tensor([0.9, 0.99]))
    do, ds = torch.randn(75, 4, 40, generator=g), torch.randn(3, 2, 24, 40, generator=g)
    dev = {k: v.to(cuda).requires_grad_() for k, v in host.items()}
    out, final = decay_attention(dev["q"], dev["k"], dev["v"], ld.to(cuda), 0.3, cu.to(cuda), dev["s"], want_state=True)
    torch.autograd.backward((out, final), (do.to(cuda), ds.to(cuda)))
    exact = {k: v.double().requires_grad_() for k, v in host.items()}
    torch.autograd.backward(ref.decay_attention(exact["q"], exact["k"], exact["v"], ld, 0.3, cu, exact["s"]), (do.double(), ds.double()))
    for k in host:
        assert (dev[k].grad.cpu().double() - exact[k].grad).abs().max() < 2e-5 * (1 + exact[k].grad.abs().max()), k
    # the output alone, without states
    dev = {k: v.to(cuda).requires_grad_() for k, v in host.items() if k != "s"}
    out, final = decay_attention(dev["q"], dev["k"], dev["v"], ld.to(cuda), 0.3, cu.to(cuda))
    assert final is None
    out.sum().backward()  # a gradient that is a broadcast scalar
    moved = {k: v.double().clone() for k, v in host.items()}
    value = lambda: float(ref.decay_attention(moved["q"], moved["k"], moved["v"], ld, 0.3, cu)[0].sum())  # noqa: E731
    before, step = value(), 1e-5
    moved["k"][33, 1, 7] += step
    assert abs((value() - before) / step - float(dev["k"].grad[33, 1, 7])) < 1e-3
    with pytest.raises(ValueError, match="constant"):
        decay_attention(dev["q"], dev["k"], dev["v"], ld.to(cuda).requires_grad_())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_cross_entropy_gradient(cuda, dtype):
    from tt_rsl_rl_amd.tokens import linear_cross_entropy

    g = torch.Generator().manual_seed(4)
    h, w = torch.randn(4, 9, 48, generator=g).to(dtype), (torch.randn(77, 48, generator=g) * 0.2).to(dtype)
    tok = torch.randint(0, 77, (4, 9), generator=g)
    tok[0, 3] = -1
    mask = torch.rand(4, 9, generator=g) < 0.8
    a, b = h.to(cuda).requires_grad_(), w.to(cuda).requires_grad_()
    loss = linear_cross_entropy(a, b, tok.to(cuda), mask.to(cuda), temperature=1.3)
    (loss * 0.3).backward()
    x, y = h.double().requires_grad_(), w.double().requires_grad_()
    keep = mask.flatten() & (tok.flatten() >= 0)
    want = torch.nn.functional.cross_entropy(x.flatten(0, 1)[keep] @ y.t() / 1.3, tok.flatten()[keep])
    (want * 0.3).backward()
    bar = 1e-5 if dtype == F32 else 2e-2
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5
    assert (a.grad.cpu().double() - x.grad).abs().max() < bar * x.grad.abs().max() and (b.grad.cpu().double() - y.grad).abs().max() < bar * y.grad.abs().max()
    only = w.to(cuda).requires_grad_()
    linear_cross_entropy(h.to(cuda), only, tok.to(cuda), mask.to(cuda), temperature=1.3).backward()
    assert (b.grad / 0.3 - only.grad).abs().max() < bar * only.grad.abs().max()


def test_prompt_and_steps_agree(cuda):
    """The layers' states after a prompt, then single tokens, against the whole sequence at once; sequences that begin anew in a slot."""
    example, policy = _policy(cuda, F32)
    lengths = [17, 9, 30]
    tokens, positions, cu = _tokens(cuda, lengths)
    with torch.no_grad():
        whole, _ = policy(tokens, positions, cu)
        bounds = cu.tolist()
        cut = [8, 3, 29]
        parts = [slice(a, a + n) for a, n in zip(bounds, cut)]
        short = torch.tensor([0] + cut).cumsum(0).to(torch.int32).to(cuda)
        _, states = policy(torch.cat([tokens[s] for s in parts]), torch.cat([positions[s] for s in parts]), short, want_states=True)
        slots = torch.tensor([0, 1, 2], device=cuda)
        for t in range(1):
            at = torch.tensor([bounds[i] + cut[i] + t for i in range(3)], device=cuda)
            hidden = policy.step(tokens[at], positions[at], states, slots)
            assert (hidden - whole[at]).abs().max() < 1e-4
        # sequence 1 begins again, in slot 2, from whatever is there
        first = torch.tensor([bounds[1]], device=cuda)
        hidden = policy.step(tokens[first], positions[first], states, torch.tensor([2], device=cuda), torch.ones(1, dtype=torch.bool, device=cuda))
        assert (hidden - whole[first]).abs().max() < 1e-4


def test_training_step_together(cuda):
    """Embedding, mixers, loss, optimiser: gradients of every parameter against the same policy in 64 bits on the CPU, then a step."""
    from tt_rsl_rl_amd.tokens import AdamW

    example, policy = _policy(cuda, F32)
    tokens, positions, cu = _tokens(cuda, [25, 1, 14, 33])
    loss = example.loss_of(policy, tokens, positions, cu, period=2)
    loss.backward()
    params = {n: p.detach().cpu().double().requires_grad_() for n, p in policy.named_parameters()}

    def exact():
        x = params["embed.weight"][tokens.cpu()]
        for i in range(2):
            y = torch.nn.functional.layer_norm(x, (64,), params[f"norms.{i}.weight"], params[f"norms.{i}.bias"])
            heads = (y @ params[f"mixers.{i}.project.weight"].t()).unflatten(-1, (-1, 16))
            mixer = policy.mixers[i]
            q = ref.qk_rotary(heads[:, :4], params[f"mixers.{i}.turn.q_weight"], positions.cpu(), mixer.turn._freqs.cpu(), 1e-6, False)[0]
            k = ref.qk_rotary(heads[:, 4:6], params[f"mixers.{i}.turn.k_weight"], positions.cpu(), mixer.turn._freqs.cpu(), 1e-6, False)[0]
            out = ref.decay_attention(q, k, heads[:, 6:], mixer.log_decay.cpu(), mixer.scale, cu.cpu())[0]
            x = x + out.flatten(1) @ params[f"mixers.{i}.back.weight"].t()
            body = torch.nn.functional.elu(x @ params[f"bodies.{i}.0.weight"].t() + params[f"bodies.{i}.0.bias"])
            x = x + body @ params[f"bodies.{i}.2.weight"].t() + params[f"bodies.{i}.2.bias"]
        x = torch.nn.functional.layer_norm(x, (64,), params["norms.2.weight"], params["norms.2.bias"])
        following = tokens.cpu().roll(-1)
        following[cu.cpu()[1:].long() - 1] = -1
        keep = (positions.cpu() >= 1) & (following >= 0)
        return torch.nn.functional.cross_entropy(x[keep] @ params["head"].t(), following[keep])

    want = exact()
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5 * abs(float(want.detach()))
    for name, p in policy.named_parameters():
        g = params[name].grad
        assert (p.grad.cpu().double() - g).abs().max() < 1e-4 * g.abs().max() + 1e-8, name
    before = policy.head.detach().clone()
    AdamW(policy.parameters(), lr=1e-2, max_grad_norm=1.0).step()
    assert not torch.equal(before, policy.head)


def _all_ops(cuda, seed=0):
    """One call of every operator, on inputs of its own; returns (inputs, run, outputs)."""
    from tt_rsl_rl_amd import ops

    g = torch.Generator(device=cuda).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda).to(BF16)  # noqa: E731
    n, cu = 3000, torch.tensor([0, 1000, 1001, 2900], device=cuda)
    i = dict(q=r(n, 4, 64), k=r(n, 2, 64), v=r(n, 2, 64), g=r(n, 4, 64), pos=torch.randint(0, 5000, (n,), generator=g, device=cuda), h=r(700, 128), w=r(900, 128),
             tok=torch.randint(0, 900, (700,), generator=g, device=cuda), s0=torch.randn(3, 2, 64, 64, generator=g, device=cuda))
    wq, freqs, ld = torch.ones(64, device=cuda, dtype=BF16), ops.rotary_frequencies(64, device=cuda), torch.tensor([-0.05, -0.002], device=cuda)
    e = torch.empty_like
    o = dict(yq=e(i["q"]), yk=e(i["k"]), dwq=e(wq), dwk=e(wq), gq=e(i["q"]), gk=e(i["k"]), out=e(i["g"]), s1=e(i["s0"]), dq=e(i["q"]), dk=e(i["k"]), dv=e(i["v"]),
             ds=e(i["s0"]), step=e(i["q"][:3]), state=e(i["s0"]), dh=e(i["h"]), dw=e(i["w"]), stats=torch.empty(4, device=cuda), lp=torch.empty(700, device=cuda),
             lp2=torch.empty(700, device=cuda))
    workspaces = [ops.Workspace(cuda) for _ in range(5)]

    def run():
        ops.qk_norm_rotary_fwd(i["q"], i["k"], wq, wq, i["pos"], freqs, o["yq"], o["yk"])
        ops.qk_norm_rotary_bwd(i["g"], i["k"], i["q"], i["k"], wq, wq, i["pos"], freqs, o["gq"], o["gk"], o["dwq"], o["dwk"], ws=workspaces[0])
        ops.decay_attention_fwd(o["yq"], o["yk"], i["v"], ld, o["out"], 0.1, cu, i["s0"], o["s1"], ws=workspaces[1])
        ops.decay_attention_bwd(i["g"], o["yq"], o["yk"], i["v"], ld, o["dq"], o["dk"], o["dv"], 0.1, cu, i["s0"], o["s1"], o["ds"], ws=workspaces[2])
        o["state"].copy_(o["s1"])
        ops.decay_attention_step(o["yq"][:3], o["yk"][:3], i["v"][:3], ld, o["state"], o["step"], 0.1)
        ops.linear_cross_entropy(i["h"], i["w"], i["tok"], o["dh"], o["dw"], o["stats"], logp=o["lp"], ws=workspaces[3])
        ops.linear_log_probs(i["h"], i["w"], i["tok"], o["lp2"], ws=workspaces[4])

    return i, run, o


def test_on_another_stream(cuda):
    """Inputs become right on it, late, and nothing orders another stream behind it."""
    inputs, run, want = _all_ops(cuda)
    run()
    late, run_late, got = _all_ops(cuda)
    right = {k: t.clone() for k, t in late.items()}
    for t in late.values():
        t.copy_(t.flip(0))
    for t in got.values():
        t.zero_()
    big, other = torch.ones(4096, 4096, device=cuda), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        for _ in range(40):
            big = torch.mm(big, big).clamp_(-1.0, 1.0)
        for k, t in late.items():
            t.copy_(right[k])
        run_late()
    torch.cuda.synchronize()
    written = slice(0, 2900)  # (tokens past the last sequence are left alone)
    for k in want:
        a, b = (want[k][written], got[k][written]) if k in ("out", "dq", "dk", "dv") else (want[k], got[k])
        assert torch.equal(a, b), k


def test_in_a_graph(cuda):
    """Captured, then replayed with other inputs, eager work between the replays: the same bits as eager calls; two graphs with workspaces of their
    own."""
    inputs, run, out = _all_ops(cuda)
    run()  # (workspaces are there)
    torch.cuda.synchronize()
    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            with torch.cuda.graph(graph, stream=side):
                run()
        graphs.append(graph)
    fresh, eager, want = _all_ops(cuda, seed=5)
    for t in out.values():
        t.zero_()
    for t in want.values():
        t.zero_()
    for replay in range(4):
        for k in inputs:
            if k in ("q", "k", "v", "g", "h"):
                fresh[k].add_(0.25 * replay)
            inputs[k].copy_(fresh[k])
        eager()
        torch.cuda.synchronize()
        graphs[replay % 2].replay()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(out[k], want[k]), (replay, k)
        torch.randn(1000, device=cuda).sum().item()


def test_outputs_are_marked_as_written(cuda):
    inputs, run, out = _all_ops(cuda)
    before = {k: t._version for k, t in out.items()}
    run()
    for k, t in out.items():
        assert t._version > before[k], k
    assert all(t._version == 0 for k, t in inputs.items())


def test_example_runs_and_its_gradients_are_finite(cuda):
    example, policy = _policy(cuda)
    history = example.train(iterations=3, sequences=8, dim=64, head_dim=16)
    assert len(history) == 3 and all(x == x and x < 100 for x in history)
    g = torch.Generator().manual_seed(0)
    tokens, positions, cu = example.batch(6, 50, 4, 20, cuda, g)
    example.loss_of(policy, tokens, positions, cu, 4).backward()
    for name, p in policy.named_parameters():
        assert p.grad is not None and bool(p.grad.isfinite().all()), name
    assert 0.0 <= example.correct(policy, 50, 4, 5, 3, cuda, g) <= 1.0
