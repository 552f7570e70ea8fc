"""tokens.AdamW as an optimiser of torch's, without a GPU: what its groups, copies and checkpoints keep.  ``ops.adamw_step`` is
replaced by a recorder."""

from __future__ import annotations

import copy
import pickle

import pytest
import torch

from tt_rsl_rl_amd import ops, tokens


@pytest.fixture
def calls(monkeypatch):
    seen = []

    def record(params, grads, exp_avg, exp_avg_sq, **options):
        seen.append(dict(options, params=params, grads=grads, exp_avg=exp_avg, exp_avg_sq=exp_avg_sq))

    monkeypatch.setattr(ops, "adamw_step", record)
    return seen


def _params(*sizes, dtype=torch.float32):
    out = [torch.nn.Parameter(torch.zeros(n, dtype=dtype)) for n in sizes]
    for p in out:
        p.grad = torch.ones_like(p)
    return out


def test_groups_carry_the_options(calls):
    a, b = _params(3, 4)
    own = dict(betas=(0.5, 0.6), eps=1e-3)
    opt = tokens.AdamW([dict(params=[a], lr=0.1, **own), dict(params=[b], weight_decay=0.3, **own)], lr=0.2)
    opt.step()
    assert (calls[0]["beta1"], calls[0]["beta2"], calls[0]["eps"]) == (0.5, 0.6, 1e-3)
    assert calls[0]["lr"] == [0.1, 0.2] and calls[0]["weight_decay"] == [1e-2, 0.3]
    assert (opt.betas, opt.eps) == ((0.5, 0.6), 1e-3)
    other = tokens.AdamW([a], betas=(0.8, 0.7), eps=1e-5)
    other.step()
    assert (calls[1]["beta1"], calls[1]["beta2"], calls[1]["eps"]) == (0.8, 0.7, 1e-5)


def test_groups_that_do_not_fit_together_are_refused(calls):
    a, b = _params(3, 4)
    for group in (dict(betas=(0.5, 0.999)), dict(eps=1e-3), dict(lr=-1.0), dict(weight_decay=-1.0), dict(betas=(1.0, 0.9)), dict(max_grad_norm=1.0),
                  dict(state_bits=8), dict(masters=False), dict(amsgrad=True), dict(maximize=True)):
        with pytest.raises(ValueError, match="AdamW"):
            tokens.AdamW([dict(params=[a]), dict(params=[b], **group)])
    opt = tokens.AdamW([a], max_grad_norm=1.0)
    with pytest.raises(ValueError, match="betas"):
        opt.add_param_group(dict(params=[b], betas=(0.1, 0.2)))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[b], name="second", max_grad_norm=1.0, amsgrad=False))
    opt.param_groups[1]["eps"] = 1e-3
    with pytest.raises(ValueError, match="same in all groups"):
        opt.step()
    assert not calls


def test_a_checkpoint_keeps_betas_and_eps(calls):
    (a,) = _params(3)
    opt = tokens.AdamW([a], betas=(0.5, 0.6), eps=1e-3)
    opt.step()
    other = tokens.AdamW([a])
    other.load_state_dict(opt.state_dict())
    assert (other.betas, other.eps) == ((0.5, 0.6), 1e-3)
    old = opt.state_dict()  # as it was while they were not the groups'
    old["param_groups"] = [{k: v for k, v in g.items() if k not in ("betas", "eps")} for g in old["param_groups"]]
    third = tokens.AdamW([a], betas=(0.7, 0.8), eps=1e-4)
    third.load_state_dict(old)
    third.step()
    assert (calls[-1]["beta1"], calls[-1]["beta2"], calls[-1]["eps"]) == (0.7, 0.8, 1e-4) and calls[-1]["step"] == [2]


def test_schedulers_that_cycle_the_momentum(calls):
    a, b = _params(3, 4)
    opt = tokens.AdamW([dict(params=[a]), dict(params=[b], weight_decay=0.0)], lr=1e-3)
    schedule = torch.optim.lr_scheduler.OneCycleLR(opt, max_lr=1e-2, total_steps=6)
    for _ in range(5):
        opt.step()
        schedule.step()
    assert len({c["beta1"] for c in calls}) > 2 and {c["beta2"] for c in calls} == {0.999}
    assert [c["lr"][0] for c in calls] == [c["lr"][1] for c in calls]


@pytest.mark.parametrize("how", ["copy", "pickle"])
def test_copies_step(calls, how):
    (a,) = _params(3)
    opt = tokens.AdamW([a], lr=0.1, betas=(0.5, 0.6), eps=1e-3, max_grad_norm=0.7, state_bits=8, masters=False)
    opt.step()
    other = copy.deepcopy(opt) if how == "copy" else pickle.loads(pickle.dumps(opt))
    p = other.param_groups[0]["params"][0]
    p.grad = torch.ones_like(p)
    other.step()
    for key in ("beta1", "beta2", "eps", "max_grad_norm", "lr"):
        assert calls[0][key] == calls[1][key]
    assert calls[1]["step"] == [2] and calls[1]["scales"] is not None and calls[1]["ws"] is not calls[0]["ws"]
    assert other.masters is False and calls[1]["params"][0].data_ptr() == p.data_ptr() != a.data_ptr()
    assert opt.state[a]["step"] == 1


def test_a_checkpoint_of_other_masters(calls):
    """Into masters=True a missing master is the parameter's; into masters=False none is stepped."""
    (a,) = _params(3, dtype=torch.bfloat16)
    with torch.no_grad():
        a.copy_(torch.tensor([1.0, -2.0, 3.0]))
    without, with_ = tokens.AdamW([a], masters=False), tokens.AdamW([a], masters=True)
    without.step()
    with_.step()
    assert calls[0]["masters"] is None and calls[1]["masters"][0].dtype == torch.float32
    with_.load_state_dict(without.state_dict())
    with_.step()
    assert torch.equal(calls[2]["masters"][0], a.detach().float()) and calls[2]["step"] == [2]
    without.load_state_dict(with_.state_dict())
    without.step()
    assert calls[3]["masters"] is None and calls[3]["step"] == [3] and "master" not in without.state[a]


def test_a_checkpoint_of_torch_s_own(calls):
    (a,) = _params(3)
    theirs = torch.optim.AdamW([a], lr=0.1, betas=(0.5, 0.6), amsgrad=False)
    theirs.step()
    opt = tokens.AdamW([a])
    opt.load_state_dict(theirs.state_dict())
    opt.step()
    assert calls[0]["step"] == [2] and opt.state[a]["step"] == 2 and isinstance(opt.state[a]["step"], int)
    assert torch.equal(calls[0]["exp_avg"][0], theirs.state[a]["exp_avg"]) and (opt.betas, calls[0]["lr"]) == ((0.5, 0.6), [0.1])
    theirs = torch.optim.AdamW([a], amsgrad=True)
    theirs.step()
    before = opt.state_dict()["param_groups"]
    with pytest.raises(ValueError, match="amsgrad"):
        opt.load_state_dict(theirs.state_dict())
    assert opt.state_dict()["param_groups"] == before
