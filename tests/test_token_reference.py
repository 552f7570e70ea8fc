"""The plain forms of the token operators against autograd and central differences, and the entry points' refusals: nothing
here needs a GPU (the library checks its arguments before any HIP call)."""

from __future__ import annotations

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from tests import token_reference as ref

ROOT = Path(__file__).resolve().parent.parent
INF = float("inf")


def _problem(rows=7, vocab=11, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, dtype=torch.float64) * 2
    tok = torch.randint(0, vocab, (rows,), generator=g)
    lp = torch.log_softmax(x, 1)[torch.arange(rows), tok]
    old = lp - 0.4 * torch.randn(rows, generator=g, dtype=torch.float64)
    return x, tok, old, torch.randn(rows, generator=g, dtype=torch.float64), lp + 0.3 * torch.randn(rows, generator=g, dtype=torch.float64)


def _loss(x, tok, old, adv, reference, keep, n, temperature, kl, ent, clip):
    logs = torch.log_softmax(x / temperature, 1)
    lp = logs[torch.arange(len(tok)), tok.clamp(min=0)]
    p = logs.exp()
    h = -torch.where(p > 0, p * logs, torch.zeros_like(p)).sum(1)
    ratio = torch.exp(lp - old)
    s = torch.maximum(-adv * ratio, -adv * ratio.clamp(1 - clip[0], 1 + clip[1]))
    d = reference - lp
    return torch.where(keep, s + kl * (torch.exp(d) - d - 1) - ent * h, torch.zeros_like(s)).sum() / n


@pytest.mark.parametrize("kl,ent,temperature", [(0.0, 0.0, 1.0), (0.3, 0.0, 0.7), (0.1, 0.2, 1.6)])
def test_loss_gradient_against_autograd_and_differences(kl, ent, temperature):
    x, tok, old, adv, reference = _problem()
    mask = torch.tensor([1, 1, 0, 1, 1, 1, 0], dtype=torch.bool)
    tok[4] = -100
    keep = ref.rows_that_count(tok, x.shape[1], mask)
    n, clip = float(keep.sum()), (0.2, 0.3)
    got = ref.token_loss(x, tok, old, adv, reference, mask, clip, kl, ent, temperature)
    y = x.clone().requires_grad_()
    loss = _loss(y, tok, old, adv, reference, keep, n, temperature, kl, ent, clip)
    loss.backward()
    assert abs(float(loss) - float(got["stats"][0])) < 1e-12
    assert (y.grad - got["d_logits"]).abs().max() < 1e-12
    h = 1e-5
    for r in range(x.shape[0]):
        for j in range(0, x.shape[1], 3):
            up, down = x.clone(), x.clone()
            up[r, j] += h
            down[r, j] -= h
            f = [float(_loss(q, tok, old, adv, reference, keep, n, temperature, kl, ent, clip)) for q in (up, down)]
            assert abs((f[0] - f[1]) / (2 * h) - float(got["d_logits"][r, j])) < 1e-8  # h^2 and 1e-16 / h


def test_loss_of_forbidden_tokens_and_empty_rows():
    x, tok, old, adv, reference = _problem()
    x[0, :] = -INF                    # no distribution
    x[1, (tok[1] + 1) % 11] = -INF    # a token that is not allowed
    got = ref.token_loss(x, tok, old, adv, reference, None, kl_coef=0.1, entropy_coef=0.1)
    assert torch.isfinite(got["d_logits"]).all() and torch.isfinite(got["stats"]).all()
    assert got["d_logits"][0].abs().max() == 0 and got["logp"][0] == 0
    assert got["d_logits"][1, (tok[1] + 1) % 11] == 0
    none = ref.token_loss(x, tok, old, adv, reference, torch.zeros(7, dtype=torch.bool))
    assert none["stats"].abs().max() == 0 and none["d_logits"].abs().max() == 0


def test_embedding_gradient_against_autograd():
    g = torch.Generator().manual_seed(1)
    table = torch.randn(9, 5, generator=g, dtype=torch.float64, requires_grad=True)
    tok = torch.tensor([3, 3, 0, 8, -1, 3, 9])
    ok = (tok >= 0) & (tok < 9)
    d = torch.randn(7, 5, generator=g, dtype=torch.float64)
    y = table[tok.clamp(0, 8)] * 1.5 * ok[:, None]
    y.backward(d)
    assert (ref.embedding(tok, table.detach(), 1.5) - y.detach()).abs().max() < 1e-14
    assert (ref.embedding_grad(tok, d, 9, 1.5)[0] - table.grad).abs().max() < 1e-14


def test_adamw_against_torch():
    g = torch.Generator().manual_seed(2)
    p = torch.randn(50, generator=g, dtype=torch.float64)
    q = torch.nn.Parameter(p.clone())
    opt = torch.optim.AdamW([q], lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    m = v = torch.zeros(50, dtype=torch.float64)
    for step in range(1, 4):
        q.grad = torch.randn(50, generator=g, dtype=torch.float64)
        p, m, v = ref.adamw(p, q.grad, m, v, step, 3e-3, 0.9, 0.99, 1e-8, 0.1)
        opt.step()
    assert (p - q.detach()).abs().max() < 1e-12


def test_entry_points_refuse_bad_arguments():
    from tt_rsl_rl_amd import _lib as L

    lib = L.load()

    def emb(**more):
        d = dict(tokens=64, src=64, ld_src=8, dst=64, ld_dst=8, count=4, vocab=10, dim=8, token_type=0, src_type=0, dst_type=0,
                 scale=1.0)
        return ctypes.byref(L.EmbeddingArgs(**{**d, **more}))

    for more, what in [(dict(count=-1), "count"), (dict(vocab=0), "vocab"), (dict(dim=0), "dim"), (dict(src_type=3), "src_type"),
                       (dict(dst_type=1), "dst_type"), (dict(token_type=2), "token_type"), (dict(ld_src=7), "leading"),
                       (dict(ld_dst=7), "leading"), (dict(src=None), "null"), (dict(dst=None), "null"), (dict(src=66), "aligned"),
                       (dict(tokens=68), "aligned"), (dict(count=2**31), "count")]:
        with pytest.raises(ValueError, match=what):
            L.call("ppo_embedding_fwd", emb(**more), None)
        with pytest.raises(ValueError, match=what):
            L.call("ppo_embedding_bwd", emb(**{**more, **({"src_type": 0, "dst_type": 2} if "dst_type" in more else {})}), 256,
                   1 << 20, None)
    with pytest.raises(ValueError, match="null arguments"):
        L.call("ppo_embedding_fwd", None, None)
    with pytest.raises(ValueError, match="workspace"):
        L.call("ppo_embedding_bwd", emb(), None, 0, None)
    with pytest.raises(ValueError, match="workspace"):
        L.call("ppo_embedding_bwd", emb(), 256, lib.ppo_embedding_bwd_workspace_bytes(4, 10, 8) - 1, None)
    assert lib.ppo_embedding_bwd_workspace_bytes(-1, 10, 8) == 0

    def loss(**more):
        d = dict(logits=64, ld_logits=10, tokens=64, old_logp=64, advantages=64, d_logits=64, ld_d_logits=10, stats=64, rows=4,
                 vocab=10, clip_low=0.2, clip_high=0.2, temperature=1.0)
        return ctypes.byref(L.TokenLossArgs(**{**d, **more}))

    for more, what in [(dict(rows=-1), "rows"), (dict(vocab=0), "vocab"), (dict(type=3), "type"), (dict(token_type=5), "token_type"),
                       (dict(temperature=0.0), "temperature"), (dict(temperature=math.nan), "temperature"),
                       (dict(ld_logits=9), "leading"), (dict(ld_d_logits=9), "leading"), (dict(logits=None), "null"),
                       (dict(tokens=None), "null"), (dict(stats=None), "null"), (dict(old_logp=None), "null"),
                       (dict(advantages=None), "null"), (dict(clip_low=-0.1), "clip"), (dict(denom=-1.0), "denom"),
                       (dict(logits=66), "aligned"), (dict(ld_d_logits=12), "in place")]:
        with pytest.raises(ValueError, match=what):
            L.call("ppo_token_ppo_loss", loss(**more), 256, 1 << 20, None)
    with pytest.raises(ValueError, match="workspace"):
        L.call("ppo_token_ppo_loss", loss(), 256, 8, None)
    with pytest.raises(ValueError, match="temperature"):
        L.call("ppo_token_log_probs", loss(temperature=-1.0), 256, 1 << 20, None)

    def adamw(**more):
        d = dict(param=64, grad=64, exp_avg=64, exp_avg_sq=64, count=8, lr=1e-3, weight_decay=0.0, bc1=0.1, bc2_sqrt=0.03, state_bits=32)
        return ctypes.cast(ctypes.pointer(L.AdamwTensor(**{**d, **more})), ctypes.c_void_p)

    step = lambda t, *more: L.call("ppo_adamw_step", t, 1, *(more or (1.0, 0.9, 0.999, 1e-8)), None, 256, 1 << 20, None)  # noqa: E731
    for more, what in [(dict(count=-1), "elements"), (dict(param_type=2), "param_type"), (dict(grad_type=1), "gradient"),
                       (dict(state_bits=16), "state_bits"), (dict(master=64), "master"), (dict(grad=None), "null"),
                       (dict(state_bits=8), "null"), (dict(param=66), "aligned")]:
        with pytest.raises(ValueError, match=what):
            step(adamw(**more))
    with pytest.raises(ValueError, match="beta1"):
        step(adamw(), 1.0, 1.0, 0.999, 1e-8)
    with pytest.raises(ValueError, match="corrections"):
        step(adamw(bc1=0.0))
    with pytest.raises(ValueError, match="workspace"):
        L.call("ppo_adamw_step", adamw(), 1, 1.0, 0.9, 0.999, 1e-8, None, None, 0, None)
    with pytest.raises(ValueError, match="tensors"):
        L.call("ppo_adamw_step", None, 0, 1.0, 0.9, 0.999, 1e-8, None, None, 0, None)


def test_tensors_on_the_cpu_are_refused():
    from tt_rsl_rl_amd import ops

    t, x, v = torch.zeros(2, dtype=torch.int64), torch.zeros(2, 4), torch.zeros(2)
    for call in (lambda: ops.embedding_fwd(t, x, x), lambda: ops.embedding_bwd(t, x, x), lambda: ops.token_log_probs(x, t, v),
                 lambda: ops.token_ppo_loss(x, t, v, v, x, torch.zeros(8)),
                 lambda: ops.adamw_step([x], [x], [x], [x], step=1, lr=1e-3)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="grads for"):
        ops.adamw_step([x], [], [x], [x], step=1, lr=1e-3)
    with pytest.raises(ValueError, match="step"):
        ops.adamw_step([x], [x], [x], [x], step=0, lr=1e-3)
    ops.adamw_step([], [], [], [], step=1, lr=1e-3)


def test_adamw_table_refuses_what_is_no_list_of_tensors():
    from tt_rsl_rl_amd import ops

    x = torch.zeros(2, 4)
    for call, what in ((lambda: ops.adamw_step([x], [None], [x], [x], step=1, lr=1e-3), r"grads\[0\]"),
                       (lambda: ops.adamw_step([1.0], [x], [x], [x], step=1, lr=1e-3), r"params\[0\]"),
                       (lambda: ops.adamw_step([x], [x], [x], [x], step=[1, 2], lr=1e-3), "step for"),
                       (lambda: ops.adamw_step([x], [x], [x], [x], step=[0], lr=1e-3), "step of tensor 0"),
                       (lambda: ops.adamw_step([x], [x], [x], [x], step=1, lr=[1e-3, 1e-3]), "lr for"),
                       (lambda: ops.adamw_step([x], [x], [x], [x], step=1, lr=1e-3, masters=[]), "masters for"),
                       (lambda: ops.adamw_step([x], [x], [x], [x], step=1, lr=1e-3, scales=([], [])), "scales for")):
        with pytest.raises(ValueError, match=what):
            call()
    with pytest.raises(TypeError):
        ops.adamw_step([x], [x], [x], [x], step="one", lr=1e-3)
    with pytest.raises(TypeError):
        ops.adamw_step([x], 3, [x], [x], step=1, lr=1e-3)


STRUCTS = {
    "ppo_embedding_args": ("EmbeddingArgs", ["tokens", "src", "ld_src", "dst", "ld_dst", "count", "vocab", "dim", "token_type", "src_type",
                                             "dst_type", "scale", "accumulate"]),
    "ppo_token_loss_args": ("TokenLossArgs", ["logits", "ld_logits", "tokens", "mask", "old_logp", "ref_logp", "advantages", "d_logits",
                                              "ld_d_logits", "logp", "entropy", "stats", "rows", "vocab", "clip_low", "clip_high", "kl_coef",
                                              "entropy_coef", "temperature", "denom", "type", "token_type"]),
    "ppo_adamw_tensor": ("AdamwTensor", ["param", "grad", "master", "exp_avg", "exp_avg_sq", "m_scale", "v_scale", "count", "lr", "weight_decay",
                                         "bc1", "bc2_sqrt", "param_type", "grad_type", "state_bits", "reserved"]),
}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layouts_match_the_c_compiler(tmp_path):
    from tt_rsl_rl_amd import _lib

    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "ppo_hip.h"}"', "int main(void) {"]
    for cname, (_, fields) in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        lines += [f'printf("%zu\\n", offsetof({cname}, {f}));' for f in fields]
    for macro in ("PPO_ADAMW_BLOCK", "PPO_TYPE_F32", "PPO_TYPE_BF16", "PPO_TYPE_F16", "PPO_TOKENS_I64", "PPO_TOKENS_I32"):
        lines.append(f'printf("%d\\n", (int){macro});')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    want = []
    for pyname, fields in STRUCTS.values():
        cls = getattr(_lib, pyname)
        want += [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fields]
    assert got == want + [_lib.ADAMW_BLOCK, _lib.TYPE_F32, _lib.TYPE_BF16, _lib.TYPE_F16, _lib.TOKENS_I64, _lib.TOKENS_I32]
