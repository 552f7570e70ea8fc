"""What a policy that acts in tokens is built from, beside torch's own layers: an embedding whose gradient is summed by sorted
tokens, and AdamW over many tensors with fp32 masters and, if wanted, 8-bit states.  The loss is ``ops.token_ppo_loss``, which
writes the logits' gradient itself: ``logits.backward(d_logits)`` goes on from there (examples/token_policy.py).

Everything runs in the HIP kernels of ``libppo_hip.so`` on the tensors' GPU; there is no CPU path.
"""

from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import ops


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens: torch.Tensor, table: torch.Tensor, scale: float) -> torch.Tensor:
        out = table.new_empty(tokens.numel(), table.shape[1])
        ops.embedding_fwd(tokens, table, out, scale)
        ctx.save_for_backward(tokens)
        ctx.shape, ctx.scale = table.shape, scale
        return out.view(*tokens.shape, table.shape[1])

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out: torch.Tensor):
        (tokens,) = ctx.saved_tensors
        d_table = d_out.new_empty(ctx.shape)
        ops.embedding_bwd(tokens, d_out.reshape(-1, ctx.shape[1]).contiguous(), d_table, ctx.scale)
        return None, d_table, None


class TokenEmbedding(nn.Module):
    """``scale * weight[tokens]`` for int64 or int32 tokens of any shape; a token outside [0, vocab) (padding) gives zeros and
    no gradient.  The weight is normal of deviation 1 / scale, so that what comes out has deviation 1."""

    def __init__(self, vocab: int, dim: int, scale: float = 1.0, device=None, dtype=None) -> None:
        super().__init__()
        if scale == 0.0:
            raise ValueError("TokenEmbedding: scale must not be 0")
        self.scale = float(scale)
        self.weight = nn.Parameter(torch.empty(vocab, dim, device=device, dtype=dtype))
        nn.init.normal_(self.weight, std=1.0 / abs(self.scale))

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return _Lookup.apply(tokens.contiguous(), self.weight, self.scale)


class AdamW(torch.optim.Optimizer):
    """AdamW on ``ops.adamw_step``: one call for all parameters, their gradients clipped by their common norm first
    (max_grad_norm; ``norm`` holds the last norm and clip coefficient on the GPU).  Parameters are float32 or bfloat16; the
    latter get a float32 master unless ``masters`` is False.  state_bits: 32, or 8 for both moments in 8 bits, rounded by
    chance that the step's number decides, so that the same steps give the same bits.  Groups may have their own lr and
    weight_decay; their betas and eps are one value for all of them (a scheduler may change it between steps).  Parameters
    without a gradient are left alone."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, max_grad_norm: float | None = None, state_bits: int = 32, masters: bool = True) -> None:
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits={state_bits} (8 or 32)")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError(f"AdamW: max_grad_norm={max_grad_norm}")
        self.max_grad_norm, self.state_bits, self.masters = max_grad_norm, state_bits, masters
        self.norm: torch.Tensor | None = None
        self._ws = ops.Workspace()
        defaults = dict(lr=lr, betas=(float(betas[0]), float(betas[1])), eps=float(eps), weight_decay=weight_decay)
        self._check_group(defaults)
        super().__init__(params, defaults)

    def _check_group(self, group: dict) -> None:
        lr, betas, eps, weight_decay = (group[k] for k in ("lr", "betas", "eps", "weight_decay"))
        if lr < 0.0 or not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0 or eps < 0.0 or weight_decay < 0.0:
            raise ValueError(f"AdamW: lr={lr} betas={betas} eps={eps} weight_decay={weight_decay}")
        for key in ("max_grad_norm", "state_bits", "masters"):
            if key in group and group[key] != getattr(self, key):
                raise ValueError(f"AdamW: {key} is the optimiser's, not a group's")
        for key in ("amsgrad", "maximize"):
            if group.get(key):
                raise ValueError(f"AdamW: no {key}")

    def _common(self) -> tuple[tuple[float, float], float]:
        """betas and eps, which all groups share."""
        first = self.param_groups[0]
        betas, eps = tuple(first["betas"]), first["eps"]
        for group in self.param_groups[1:]:
            if tuple(group["betas"]) != betas or group["eps"] != eps:
                raise ValueError(f"AdamW: betas and eps must be the same in all groups, got {betas}, {eps} and {group['betas']}, {group['eps']}")
        return betas, eps

    betas = property(lambda self: self._common()[0])
    eps = property(lambda self: self._common()[1])

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        try:
            self._check_group(self.param_groups[-1])
            self._common()
        except ValueError:
            self.param_groups.pop()
            raise

    def __getstate__(self) -> dict:
        """Copies and pickles: torch's part and the options beside it; scratch memory and the last norm stay behind."""
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm, "state_bits": self.state_bits, "masters": self.masters}

    def __setstate__(self, state: dict) -> None:  # (load_state_dict() comes here too, with a state of two entries)
        super().__setstate__(state)
        if "_ws" not in self.__dict__:
            self.norm, self._ws = None, ops.Workspace()
        for group in self.param_groups:  # (of a state_dict() from before they were the groups')
            for key in ("betas", "eps"):
                group.setdefault(key, self.defaults[key])

    def _init_state(self, p: torch.Tensor, state: dict) -> None:
        state["step"] = 0
        if self.state_bits == 8:
            blocks = -(-p.numel() // L.ADAMW_BLOCK)
            state["exp_avg"] = torch.zeros(p.numel(), dtype=torch.int8, device=p.device)
            state["exp_avg_sq"] = torch.zeros(p.numel(), dtype=torch.uint8, device=p.device)
            state["exp_avg_scale"] = torch.zeros(blocks, device=p.device)
            state["exp_avg_sq_scale"] = torch.zeros(blocks, device=p.device)
        else:
            state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
            state["exp_avg_sq"] = torch.zeros_like(state["exp_avg"])
        if self.masters and p.dtype == torch.bfloat16:
            state["master"] = p.detach().to(torch.float32)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        (beta1, beta2), eps = self._common()
        params, states, lr, decay = [], [], [], []
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    self._init_state(p, state)
                params.append(p.detach())
                states.append(state)
                lr.append(group["lr"])
                decay.append(group["weight_decay"])
        if not params:
            return loss
        grads = [p.grad.detach().contiguous() for group in self.param_groups for p in group["params"] if p.grad is not None]
        if self.norm is None:
            self.norm = torch.zeros(2, device=params[0].device)
        column = lambda key: [s.get(key) for s in states]  # noqa: E731
        masters = column("master")
        ops.adamw_step(params, grads, column("exp_avg"), column("exp_avg_sq"), step=[s["step"] + 1 for s in states], lr=lr,
                       beta1=beta1, beta2=beta2, eps=eps, weight_decay=decay, max_grad_norm=self.max_grad_norm,
                       masters=masters if any(m is not None for m in masters) else None,
                       scales=(column("exp_avg_scale"), column("exp_avg_sq_scale")) if self.state_bits == 8 else None,
                       norm_out=self.norm if self.max_grad_norm is not None else None, ws=self._ws, dither=self.state_bits == 8)
        for s in states:  # (after the call: a refused one leaves the counts as they are)
            s["step"] += 1
        return loss

    def load_state_dict(self, state_dict: dict) -> None:
        """Takes a state_dict() of an optimiser of the same state_bits; the states keep their types (torch's own would be
        cast to the parameters').  Masters go by this optimiser's ``masters``: one that the state_dict() lacks is the
        parameter as it is now, one that is not wanted is left out."""
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i in saved:
            state = state_dict["state"].get(i)
            if state and (state["exp_avg"].dtype == torch.int8) != (self.state_bits == 8):
                raise ValueError(f"AdamW: states of another width than state_bits={self.state_bits}")
        for group in state_dict["param_groups"]:
            self._check_group({**self.defaults, **group})
        super().load_state_dict(state_dict)
        for i, p in zip(saved, (p for group in self.param_groups for p in group["params"]), strict=True):
            if not state_dict["state"].get(i):
                continue
            state = self.state[p]
            for key, value in state_dict["state"][i].items():
                if isinstance(value, torch.Tensor):
                    state[key] = value.to(p.device, copy=True)
            state["step"] = int(state["step"])  # (torch.optim.AdamW's is a tensor)
            if not self.masters or p.dtype != torch.bfloat16:
                state.pop("master", None)
            elif "master" not in state:
                state["master"] = p.detach().to(torch.float32)
