"""The 64-bit forms of tests/token_layer_reference.py against autograd and differences, and what the operators refuse, all on the CPU."""

from __future__ import annotations

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from tests import token_layer_reference as ref

ROOT = Path(__file__).resolve().parent.parent
M = 1 << 24  # memory of an operand's own


def _randn(seed, *shapes):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g, dtype=torch.float64) for s in shapes]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("per_head", [False, True])
def test_qk_rotary(interleaved, per_head):
    x, g, w = _randn(0, (7, 3, 12), (7, 3, 12), (3, 12) if per_head else (12,))
    pos, freqs = torch.arange(7) * 3 - 5, 10000.0 ** (torch.arange(0, 8, 2, dtype=torch.float64) / -8)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    y, before = ref.qk_rotary(a, b, pos, freqs, 1e-5, interleaved)
    y.backward(g)
    dx, dw, x_size, w_size = ref.qk_rotary_grad(g, x, w, pos, freqs, 1e-5, interleaved)
    assert torch.allclose(a.grad, dx, rtol=1e-12, atol=1e-13) and torch.allclose(b.grad, dw, rtol=1e-12, atol=1e-13)
    assert bool((dx.abs() <= x_size * (1 + 1e-12)).all()) and bool((dw.abs() <= w_size * (1 + 1e-12)).all())
    assert torch.allclose(y.pow(2).sum(-1), before.pow(2).sum(-1))  # a turn keeps lengths
    one, _ = ref.qk_rotary(x[:1], torch.ones(12), torch.tensor([0]), freqs, 0.0, interleaved)
    assert torch.allclose(one, x[:1] / x[:1].pow(2).mean(-1, keepdim=True).sqrt())


def test_decay_attention_is_the_recurrence():
    q, k, v, s0, g, g1 = _randn(1, (20, 4, 5), (20, 2, 5), (20, 2, 6), (4, 2, 5, 6), (20, 4, 6), (4, 2, 5, 6))
    ld, cu = torch.tensor([math.log(0.8), -math.inf], dtype=torch.float64), torch.tensor([0, 9, 9, 10, 18])
    out, last = ref.decay_attention(q, k, v, ld, 0.7, cu, s0)
    for b in range(4):
        state = s0[b:b + 1].clone()
        for t in range(int(cu[b]), int(cu[b + 1])):
            o, state = ref.decay_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], ld, state, 0.7)
            assert torch.allclose(o[0], out[t])
        assert torch.allclose(state[0], last[b])
    assert not bool(out[18:].any())
    leaves = [x.clone().requires_grad_() for x in (q, k, v, s0)]
    torch.autograd.backward(ref.decay_attention(*leaves[:3], ld, 0.7, cu, leaves[3]), (g, g1))
    for leaf, want in zip(leaves, ref.decay_attention_grad(g, q, k, v, ld, 0.7, cu, s0, g1)):
        assert torch.allclose(leaf.grad, want, rtol=1e-11, atol=1e-12)
    step, moved = 1e-6, v.clone()
    moved[3, 0, 2] += step
    value = lambda x: (ref.decay_attention(q, k, x, ld, 0.7, cu, s0)[0] * g).sum() + (ref.decay_attention(q, k, x, ld, 0.7, cu, s0)[1] * g1).sum()  # noqa: E731
    assert abs(float((value(moved) - value(v)) / step) - float(leaves[2].grad[3, 0, 2])) < 1e-6


def test_decay_step_rows_of_padding_and_fresh_ones():
    q, k, v, s = _randn(2, (4, 2, 3), (4, 2, 3), (4, 2, 3), (3, 2, 3, 3))
    out, after = ref.decay_step(q, k, v, torch.zeros(2), s, 1.0, torch.tensor([2, -1, 0, 3]), torch.tensor([False, False, True, False]))
    assert torch.equal(after[1], s[1]) and not bool(out[1].any()) and not bool(out[3].any())
    assert torch.equal(after[0], k[2][:, :, None] * v[2][:, None, :])


def test_linear_cross_entropy():
    h, w = _randn(3, (10, 6), (13, 6))
    tok, mask = torch.tensor([0, 5, -1, 12, 3, 13, 7, 1, 2, 2]), torch.tensor([1, 1, 1, 1, 0, 1, 1, 1, 1, 1])
    got = ref.linear_cross_entropy(h, w, tok, mask, 0.7)
    keep = torch.tensor([0, 1, 3, 6, 7, 8, 9])
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = torch.nn.functional.cross_entropy(a[keep] @ b.t() / 0.7, tok[keep])
    loss.backward()
    assert torch.allclose(got["stats"][0], loss) and float(got["stats"][2]) == 7.0
    assert torch.allclose(got["d_hidden"], a.grad) and torch.allclose(got["d_weight"], b.grad)
    step, moved = 1e-6, w.clone()
    moved[12, 3] += step
    assert abs(float((ref.linear_cross_entropy(h, moved, tok, mask, 0.7)["stats"][0] - loss) / step) - float(b.grad[12, 3])) < 1e-6


STRUCTS = {
    "ppo_head_view": ("HeadView", ["data", "token_stride", "head_stride"]),
    "ppo_qk_rotary_args": ("QkRotaryArgs", ["q", "k", "q_out", "k_out", "d_q", "d_k", "q_weight", "k_weight", "d_q_weight", "d_k_weight", "positions", "freqs",
                                            "tokens", "eps", "q_heads", "kv_heads", "head_dim", "rotary_dim", "type", "weight_type", "position_type",
                                            "interleaved", "weight_per_head"]),
    "ppo_decay_attention_args": ("DecayAttentionArgs", ["q", "k", "v", "out", "d_q", "d_k", "d_v", "log_decay", "cu_seqlens", "initial_state", "final_state",
                                                        "d_final_state", "d_initial_state", "tokens", "sequences", "scale", "q_heads", "kv_heads", "key_dim",
                                                        "value_dim", "type", "cu_type"]),
    "ppo_decay_step_args": ("DecayStepArgs", ["q", "k", "v", "out", "log_decay", "states", "slots", "fresh", "rows", "num_slots", "scale", "q_heads", "kv_heads",
                                              "key_dim", "value_dim", "type", "slot_type"]),
    "ppo_linear_loss_args": ("LinearLossArgs", ["hidden", "ld_hidden", "weight", "ld_weight", "tokens", "mask", "d_hidden", "ld_d_hidden", "d_weight",
                                                "ld_d_weight", "logp", "entropy", "stats", "rows", "vocab", "dim", "temperature", "denom", "type",
                                                "token_type"]),
}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layouts_match_the_c_compiler(tmp_path):
    from tt_rsl_rl_amd import _lib

    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "ppo_hip.h"}"', "int main(void) {"]
    for cname, (_, fields) in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        lines += [f'printf("%zu\\n", offsetof({cname}, {f}));' for f in fields]
    lines += ['printf("%d\\n", PPO_QK_MAX_DIM);', 'printf("%d\\n", PPO_DECAY_MAX_DIM);']
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    want = []
    for pyname, fields in STRUCTS.values():
        cls = getattr(_lib, pyname)
        want += [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fields]
    assert got == want + [_lib.QK_MAX_DIM, _lib.DECAY_MAX_DIM]


# ---- refusals: before any HIP call; addresses are numbers, nothing is read from them ----


def _view(at, token, head):
    from tt_rsl_rl_amd import _lib as L

    return L.HeadView(at * M if at is not None else None, token, head)


def _qk(entry="ppo_qk_rotary_fwd", **more):
    from tt_rsl_rl_amd import _lib as L

    d = dict(q=_view(1, 32, 8), k=_view(2, 16, 8), q_out=_view(3, 32, 8), k_out=_view(4, 16, 8), d_q=_view(5, 32, 8), d_k=_view(6, 16, 8), q_weight=7 * M,
             k_weight=8 * M, d_q_weight=9 * M, d_k_weight=10 * M, positions=11 * M, freqs=12 * M, tokens=5, eps=1e-6, q_heads=4, kv_heads=2, head_dim=8,
             rotary_dim=8)
    args = ctypes.byref(L.QkRotaryArgs(**{**d, **more}))
    L.call(entry, *((args, None) if entry.endswith("fwd") else (args, 13 * M, 1 << 23, None)))


@pytest.mark.parametrize("entry", ["ppo_qk_rotary_fwd", "ppo_qk_rotary_bwd"])
def test_qk_rotary_refusals(entry):
    for more, what in [(dict(tokens=-1), "tokens"), (dict(q_heads=0), "q_heads"), (dict(head_dim=7), "head_dim"), (dict(head_dim=514), "head_dim"),
                       (dict(rotary_dim=3), "rotary_dim"), (dict(rotary_dim=10), "rotary_dim"), (dict(rotary_dim=0), "rotary_dim"), (dict(type=3), "type"),
                       (dict(weight_type=1), "weight_type"), (dict(position_type=7), "position_type"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"),
                       (dict(q_weight=None), "null"), (dict(freqs=None), "null"), (dict(positions=None), "null"), (dict(q=_view(None, 32, 8)), "null"),
                       (dict(freqs=12 * M + 4), "aligned"), (dict(k_weight=8 * M + 2), "aligned"), (dict(q=_view(1, -32, 8)), "strides")]:
        with pytest.raises(ValueError, match=what):
            _qk(entry, **more)
    out = {"ppo_qk_rotary_fwd": ("q_out", "k_out"), "ppo_qk_rotary_bwd": ("d_q", "d_k")}[entry]
    for more in ({out[0]: _view(3, 8, 8)}, {out[0]: _view(3, 32, 4)}):
        with pytest.raises(ValueError, match="rows of"):
            _qk(entry, **more)
    for at in (2, 7, 8, 11, 12) + ((3, 4, 9, 10) if entry.endswith("bwd") else (4,)):
        if entry.endswith("bwd") and at == 3:
            continue  # the gradient that comes in may be overwritten by the one that goes out
        with pytest.raises(ValueError, match="overlap"):
            _qk(entry, **{out[0]: _view(at, 32, 8)})
    shifted = _view(1, 32, 8)
    shifted.data += 16
    with pytest.raises(ValueError, match="overlap"):
        _qk(entry, **{out[0]: shifted})
    if entry.endswith("bwd"):
        for more in (dict(d_q_weight=1 * M), dict(d_k_weight=9 * M + 8), dict(d_q_weight=12 * M), dict(d_q_weight=None)):
            with pytest.raises(ValueError, match="overlap|null"):
                _qk(entry, **more)
        from tt_rsl_rl_amd import _lib as L

        with pytest.raises(ValueError, match="null arguments"):
            L.call(entry, None, 13 * M, 1 << 23, None)


def _decay(entry="ppo_decay_attention_fwd", space=1 << 23, **more):
    from tt_rsl_rl_amd import _lib as L

    d = dict(q=_view(1, 32, 8), k=_view(2, 16, 8), v=_view(3, 24, 12), out=_view(4, 48, 12), d_q=_view(5, 32, 8), d_k=_view(6, 16, 8), d_v=_view(7, 24, 12),
             log_decay=8 * M, cu_seqlens=9 * M, initial_state=10 * M, final_state=11 * M, d_final_state=12 * M, d_initial_state=13 * M, tokens=6, sequences=2,
             scale=1.0, q_heads=4, kv_heads=2, key_dim=8, value_dim=12)
    L.call(entry, ctypes.byref(L.DecayAttentionArgs(**{**d, **more})), 15 * M, space, None)


@pytest.mark.parametrize("entry", ["ppo_decay_attention_fwd", "ppo_decay_attention_bwd"])
def test_decay_attention_refusals(entry):
    for more, what in [(dict(tokens=-1), "tokens"), (dict(tokens=1 << 31), "tokens"), (dict(sequences=0), "sequences"), (dict(q_heads=3), "q_heads"),
                       (dict(kv_heads=0), "kv_heads"), (dict(key_dim=0), "key_dim"), (dict(key_dim=129), "key_dim"), (dict(value_dim=129), "value_dim"),
                       (dict(type=5), "type"), (dict(cu_type=2), "cu_type"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
                       (dict(cu_seqlens=None), "without cu_seqlens"), (dict(log_decay=None), "null"), (dict(k=_view(None, 16, 8)), "null"),
                       (dict(cu_seqlens=9 * M + 2), "aligned"), (dict(initial_state=10 * M + 2), "aligned")]:
        with pytest.raises(ValueError, match=what):
            _decay(entry, **more)
    with pytest.raises(ValueError, match="workspace"):
        _decay(entry, space=16)
    outs = ("out",) if entry.endswith("fwd") else ("d_q", "d_k", "d_v")
    for name in outs:
        for at in (1, 2, 3, 8, 9, 10) + (() if entry.endswith("fwd") else (4, 12)):
            with pytest.raises(ValueError, match="overlap"):
                _decay(entry, **{name: _view(at, 48, 12)})
        with pytest.raises(ValueError, match="rows of"):
            _decay(entry, **{name: _view(14, 6, 3)})
        with pytest.raises(ValueError, match="apart"):
            _decay(entry, **{name: _view(14, 1 << 31, 12)})
    state = "final_state" if entry.endswith("fwd") else "d_initial_state"
    for at in (1 * M, 9 * M, 8 * M, (10 if entry.endswith("fwd") else 12) * M + 4):
        with pytest.raises(ValueError, match="overlap"):
            _decay(entry, **{state: at})
    if entry.endswith("bwd"):
        with pytest.raises(ValueError, match="overlap"):
            _decay(entry, d_k=_view(5, 32, 8))


def _step(**more):
    from tt_rsl_rl_amd import _lib as L

    d = dict(q=_view(1, 32, 8), k=_view(2, 16, 8), v=_view(3, 24, 12), out=_view(4, 48, 12), log_decay=5 * M, states=6 * M, slots=7 * M, fresh=8 * M, rows=3,
             num_slots=4, scale=1.0, q_heads=4, kv_heads=2, key_dim=8, value_dim=12)
    L.call("ppo_decay_attention_step", ctypes.byref(L.DecayStepArgs(**{**d, **more})), None)


def test_decay_step_refusals():
    for more, what in [(dict(rows=-1), "rows"), (dict(rows=1 << 24), "rows"), (dict(num_slots=-1), "num_slots"), (dict(q_heads=5), "q_heads"),
                       (dict(key_dim=200), "key_dim"), (dict(type=4), "type"), (dict(slot_type=3), "slot_type"), (dict(scale=math.nan), "scale"),
                       (dict(slots=None, rows=5), "rows for"), (dict(states=None), "null"), (dict(log_decay=None), "null"), (dict(states=6 * M + 2), "aligned"),
                       (dict(out=_view(6, 48, 12)), "overlap"), (dict(out=_view(1, 48, 12)), "overlap"), (dict(states=3 * M), "overlap"),
                       (dict(states=7 * M), "overlap"), (dict(out=_view(8, 48, 12)), "overlap"), (dict(out=_view(4, 48, 6)), "rows of")]:
        with pytest.raises(ValueError, match=what):
            _step(**more)


def _linear(entry="ppo_linear_cross_entropy", space=1 << 30, **more):
    from tt_rsl_rl_amd import _lib as L

    d = dict(hidden=1 * M, ld_hidden=8, weight=2 * M, ld_weight=8, tokens=3 * M, mask=4 * M, d_hidden=5 * M, ld_d_hidden=8, d_weight=6 * M, ld_d_weight=8, logp=7 * M,
             entropy=8 * M, stats=9 * M, rows=5, vocab=20, dim=8, temperature=1.0)
    L.call(entry, ctypes.byref(L.LinearLossArgs(**{**d, **more})), 16 * M, space, None)


def test_linear_loss_refusals():
    for more, what in [(dict(rows=-1), "rows"), (dict(rows=1 << 22), "rows"), (dict(vocab=0), "vocab"), (dict(dim=0), "dim"), (dict(type=3), "type"),
                       (dict(token_type=2), "token_type"), (dict(temperature=0.0), "temperature"), (dict(temperature=math.nan), "temperature"),
                       (dict(ld_hidden=7), "leading"), (dict(ld_weight=7), "leading"), (dict(ld_d_weight=7), "leading"), (dict(ld_weight=1 << 22), "ld_weight"),
                       (dict(weight=None), "null"), (dict(hidden=None), "null"), (dict(tokens=None), "null"), (dict(stats=None), "null"),
                       (dict(denom=-1.0), "denom"), (dict(hidden=1 * M + 2), "aligned"), (dict(d_hidden=1 * M), "overlap"), (dict(d_weight=2 * M + 4), "overlap"),
                       (dict(logp=3 * M), "overlap"), (dict(stats=7 * M), "overlap"), (dict(entropy=5 * M), "overlap"), (dict(d_hidden=6 * M + 32), "overlap")]:
        with pytest.raises(ValueError, match=what):
            _linear(**more)
    for entry in ("ppo_linear_cross_entropy", "ppo_linear_log_probs"):
        with pytest.raises(ValueError, match="workspace"):
            _linear(entry, space=64)
    with pytest.raises(ValueError, match="overlap"):
        _linear("ppo_linear_log_probs", logp=1 * M)


def test_tensors_are_checked():
    from tt_rsl_rl_amd import ops
    from tt_rsl_rl_amd.tokens import DecayMixer

    q, k, w, p, f = torch.zeros(3, 2, 4), torch.zeros(3, 1, 4), torch.ones(4), torch.zeros(3, dtype=torch.int64), torch.ones(2, dtype=torch.float64)
    v, ld, s, x = torch.zeros(3, 1, 6), torch.zeros(1), torch.zeros(1, 1, 4, 6), torch.zeros(3, 4)
    calls = (lambda: ops.qk_norm_rotary_fwd(q, k, w, w, p, f, q, k), lambda: ops.qk_norm_rotary_bwd(q, k, q, k, w, w, p, f, q, k, w, w),
             lambda: ops.decay_attention_fwd(q, k, v, ld, torch.zeros(3, 2, 6)), lambda: ops.decay_attention_bwd(torch.zeros(3, 2, 6), q, k, v, ld, q, k, v),
             lambda: ops.decay_attention_step(q, k, v, ld, s, torch.zeros(3, 2, 6)), lambda: ops.linear_log_probs(x, x, p, torch.zeros(3)),
             lambda: ops.linear_cross_entropy(x, x, p, x, x, torch.zeros(4)))
    for call in calls:
        with pytest.raises(ValueError, match="GPU"):
            call()
    for bad in (0, 3, -2):
        with pytest.raises(ValueError, match="rotary_frequencies"):
            ops.rotary_frequencies(bad)
    assert torch.allclose(ops.rotary_frequencies(4, 100.0), torch.tensor([1.0, 0.1], dtype=torch.float64))
    with pytest.raises(ValueError, match="kv_heads"):
        DecayMixer(8, 3, 2)


def test_shapes_and_types_are_checked(monkeypatch):
    """What is wrong is said before the library is called (the check of the device is taken out: there is none here)."""
    from tt_rsl_rl_amd import _lib as L
    from tt_rsl_rl_amd import ops

    called = []
    monkeypatch.setattr(ops, "_current_gpu", lambda *a: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda d: 0)
    monkeypatch.setattr(L, "call", lambda *a: called.append(a[0]))
    z = torch.zeros
    q, k, w, p, f = z(3, 2, 4), z(3, 1, 4), torch.ones(4), z(3, dtype=torch.int64), torch.ones(2, dtype=torch.float64)
    fwd = lambda **m: ops.qk_norm_rotary_fwd(**{**dict(q=q, k=k, q_weight=w, k_weight=w, positions=p, freqs=f, q_out=z(3, 2, 4), k_out=z(3, 1, 4)), **m})  # noqa: E731
    fwd()
    for more in (dict(q=z(3, 8)), dict(k=z(2, 1, 4)), dict(k=z(3, 1, 6)), dict(q=q.double()), dict(q_weight=z(5)), dict(k_weight=w.bfloat16()),
                 dict(q_weight=w.half(), k_weight=w.half()), dict(k_weight=z(1, 4)), dict(positions=p.float()), dict(positions=p[:2]), dict(freqs=f.float()),
                 dict(q_out=z(3, 2, 4).half()), dict(k_out=z(3, 2, 4)), dict(q_out=z(3, 4, 2).transpose(1, 2)), dict(k=k.half())):
        with pytest.raises(ValueError, match="qk_norm_rotary_fwd"):
            fwd(**more)
    v, ld, out, s = z(3, 1, 6), z(1), z(3, 2, 6), z(2, 1, 4, 6)
    cu = torch.tensor([0, 1, 3])
    mix = lambda **m: ops.decay_attention_fwd(**{**dict(q=q, k=k, v=v, log_decay=ld, out=out, cu_seqlens=cu, initial_state=s, final_state=s.clone()), **m})  # noqa: E731
    mix()
    for more in (dict(k=z(3, 2, 5)), dict(v=z(2, 1, 6)), dict(q=z(3, 3, 4), k=z(3, 2, 4), v=z(3, 2, 6)), dict(v=v.half()), dict(log_decay=ld.double()),
                 dict(log_decay=z(2)), dict(out=z(3, 2, 4)), dict(cu_seqlens=cu.float()), dict(cu_seqlens=cu[:1]), dict(initial_state=s[:1]),
                 dict(final_state=s.half())):
        with pytest.raises(ValueError, match="decay_attention_fwd"):
            mix(**more)
    step = lambda **m: ops.decay_attention_step(**{**dict(q=q, k=k, v=v, log_decay=ld, state=s, out=out, slots=z(3, dtype=torch.int32), fresh=z(3, dtype=torch.bool)), **m})  # noqa: E731
    step()
    for more in (dict(state=s[0]), dict(state=s.half()), dict(state=z(2, 1, 6, 4)), dict(slots=z(2, dtype=torch.int32)), dict(slots=z(3)), dict(fresh=z(3)),
                 dict(fresh=z(2, dtype=torch.bool))):
        with pytest.raises(ValueError, match="decay_attention_step"):
            step(**more)
    x, y = z(3, 4), z(7, 4)
    loss = lambda **m: ops.linear_cross_entropy(**{**dict(hidden=x, weight=y, tokens=p, d_hidden=z(3, 4), d_weight=z(7, 4), stats=z(4)), **m})  # noqa: E731
    loss()
    for more in (dict(weight=z(7, 5)), dict(weight=y.half()), dict(tokens=p[:2]), dict(tokens=p.float()), dict(mask=z(3)), dict(mask=z(2, dtype=torch.bool)),
                 dict(d_hidden=z(3, 4).half()), dict(d_weight=z(4, 7)), dict(stats=z(8)), dict(logp=z(2)), dict(denom=0.0)):
        with pytest.raises(ValueError, match="linear_cross_entropy"):
            loss(**more)
    assert called == ["ppo_qk_rotary_fwd", "ppo_decay_attention_fwd", "ppo_decay_attention_step", "ppo_linear_cross_entropy"]


def test_launches_hold_fewer_than_2_to_the_32_threads():
    """Sizes whose launches would hold more are refused, or cut: a linear loss's pieces, which the workspace shows, shrink as its rows grow."""
    from tt_rsl_rl_amd import _lib as L

    for entry in ("ppo_qk_rotary_fwd", "ppo_qk_rotary_bwd"):
        with pytest.raises(ValueError, match="tokens"):
            _qk(entry, tokens=(1 << 28) - 16)
    rows, vocab, dim = (1 << 22) - 1, 1 << 29, 63  # 2^14 tiles of rows, so that 2^8 tiles of columns are 2^22 blocks
    args = ctypes.byref(L.LinearLossArgs(hidden=M, ld_hidden=dim, weight=2 * M, ld_weight=dim, rows=rows, vocab=vocab, dim=dim, temperature=1.0, type=1))
    sums, hidden = 3 * (vocab >> 8) * (rows + 1) * 4, (rows + 1) * 64 * 2
    assert L.load().ppo_linear_loss_workspace_bytes(args, 0) <= sums + hidden + 40 * (rows + 1) + (1 << 16) * 64 * 2 + 8192
