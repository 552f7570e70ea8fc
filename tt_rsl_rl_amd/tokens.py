"""What a policy that acts in tokens is built from, beside torch's own layers: an embedding whose gradient is summed by sorted
tokens, a layer that mixes a sequence's tokens (normed and turned queries and keys, linear attention whose past fades), the cross
entropy of a head without its logits, and AdamW over many tensors with fp32 masters and, if wanted, 8-bit states.  The policy's loss
is ``ops.token_ppo_loss``, which writes the logits' gradient itself: ``logits.backward(d_logits)`` goes on from there
(examples/token_policy.py; examples/sequence_policy.py is taught by demonstrations first).

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


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A gradient as the operators take it: of unit stride in its last dimension (one that is a broadcast scalar is not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


class _QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, freqs, eps: float, interleaved: bool):
        out = q.new_empty(q.shape), k.new_empty(k.shape)
        ops.qk_norm_rotary_fwd(q, k, q_weight, k_weight, positions, freqs, *out, eps=eps, interleaved=interleaved)
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, freqs)
        ctx.options = eps, interleaved
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_q_out, d_k_out):
        q, k, q_weight, k_weight, positions, freqs = ctx.saved_tensors
        eps, interleaved = ctx.options
        grads = q.new_empty(q.shape), k.new_empty(k.shape), torch.empty_like(q_weight), torch.empty_like(k_weight)
        ops.qk_norm_rotary_bwd(_rows(d_q_out), _rows(d_k_out), q, k, q_weight, k_weight, positions, freqs, *grads, eps=eps, interleaved=interleaved)
        return *grads, None, None, None, None


class QkNormRotary(nn.Module):
    """``ops.qk_norm_rotary_fwd`` with its gradient and weights: queries [tokens, heads, dim] and keys [tokens, kv_heads, dim] of each head
    over their root mean square, times a weight of dim elements, turned by their token's position.  rotary: how many of a head's elements
    are turned (all)."""

    def __init__(self, dim: int, rotary: int | None = None, base: float = 10000.0, eps: float = 1e-6, interleaved: bool = False, device=None,
                 dtype=None) -> None:
        super().__init__()
        self.rotary, self.base, self.eps, self.interleaved = dim if rotary is None else rotary, base, eps, interleaved
        self.q_weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        self.k_weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        # not a buffer: angles stay float64 whatever the module is cast to
        self._freqs = ops.rotary_frequencies(self.rotary, base, device=self.q_weight.device)

    def forward(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        if self._freqs.device != q.device:
            self._freqs = ops.rotary_frequencies(self.rotary, self.base, device=q.device)
        return _QkNormRotary.apply(q, k, self.q_weight, self.k_weight, positions, self._freqs, self.eps, self.interleaved)


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, scale: float, cu_seqlens, initial_state, want_state: bool):
        # (tokens of no sequence are 0: what goes on from here multiplies them by gradients of 0)
        out = (q.new_empty if cu_seqlens is None else q.new_zeros)(*q.shape[:2], v.shape[2])
        sequences = 1 if cu_seqlens is None else cu_seqlens.numel() - 1
        final = q.new_empty(sequences, k.shape[1], k.shape[2], v.shape[2], dtype=torch.float32) if want_state else None
        ops.decay_attention_fwd(q, k, v, log_decay, out, scale=scale, cu_seqlens=cu_seqlens, initial_state=initial_state, final_state=final)
        ctx.save_for_backward(q, k, v, log_decay, cu_seqlens, initial_state)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_final):
        q, k, v, log_decay, cu_seqlens, initial_state = ctx.saved_tensors
        if d_out is None:
            d_out = q.new_zeros(*q.shape[:2], v.shape[2])
        # (tokens of no sequence stay 0; without cu_seqlens there are none)
        grads = tuple((x.new_empty if cu_seqlens is None else x.new_zeros)(x.shape) for x in (q, k, v))
        d_initial = torch.empty_like(initial_state) if initial_state is not None and ctx.needs_input_grad[6] else None
        ops.decay_attention_bwd(_rows(d_out), q, k, v, log_decay, *grads, scale=ctx.scale, cu_seqlens=cu_seqlens, initial_state=initial_state,
                                d_final_state=None if d_final is None else d_final.contiguous(), d_initial_state=d_initial)
        return *grads, None, None, None, d_initial, None


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, scale: float = 1.0,
                    cu_seqlens: torch.Tensor | None = None, initial_state: torch.Tensor | None = None,
                    want_state: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``ops.decay_attention_fwd`` with its gradient: the output, and the state that each sequence ends with (None unless wanted).
    log_decay is a constant; tokens of no sequence (cu_seqlens) get an output of 0 and no gradient."""
    if log_decay.requires_grad:
        raise ValueError("decay_attention: log_decay is a constant, it gets no gradient")
    return _DecayAttention.apply(q, k, v, log_decay, float(scale), cu_seqlens, initial_state, want_state)


class DecayMixer(nn.Module):
    """A layer that mixes the tokens of each sequence: queries, keys and values of one projection, queries and keys normed and turned, linear
    attention whose past fades, head h's by 1 - 2^-reach[h] a token, and a projection back.  Sequences lie one after another
    (cu_seqlens); ``forward`` takes them whole (prompts, training), ``step`` one token of each on the states that ``new_state`` makes
    and ``forward`` returns."""

    def __init__(self, dim: int, heads: int, kv_heads: int | None = None, head_dim: int = 64, rotary: int | None = None, base: float = 10000.0,
                 reach: tuple[float, float] = (3.0, 9.0), device=None, dtype=None) -> None:
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"DecayMixer: heads={heads} kv_heads={kv_heads}")
        self.heads, self.kv_heads, self.head_dim, self.scale = heads, kv_heads, head_dim, head_dim**-0.5
        self.project = nn.Linear(dim, (heads + 2 * kv_heads) * head_dim, bias=False, device=device, dtype=dtype)
        self.turn = QkNormRotary(head_dim, rotary, base, device=device, dtype=dtype)
        self.back = nn.Linear(heads * head_dim, dim, bias=False, device=device, dtype=dtype)
        # not a buffer: it stays float32 whatever the module is cast to
        self._log_decay = torch.log1p(-torch.exp2(-torch.linspace(*reach, kv_heads, dtype=torch.float64))).float().to(self.back.weight.device)

    @property
    def log_decay(self) -> torch.Tensor:
        if self._log_decay.device != self.back.weight.device:
            self._log_decay = self._log_decay.to(self.back.weight.device)
        return self._log_decay

    def new_state(self, sequences: int) -> torch.Tensor:
        return torch.zeros(sequences, self.kv_heads, self.head_dim, self.head_dim, device=self.back.weight.device)

    def _heads(self, x: torch.Tensor, positions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        q, k, v = self.project(x).unflatten(-1, (-1, self.head_dim)).split((self.heads, self.kv_heads, self.kv_heads), dim=1)
        return *self.turn(q, k, positions), v

    def forward(self, x: torch.Tensor, positions: torch.Tensor, cu_seqlens: torch.Tensor | None = None, state: torch.Tensor | None = None,
                want_state: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
        """x [tokens, dim] and its tokens' positions -> ([tokens, dim], states or None)."""
        q, k, v = self._heads(x, positions)
        out, state = decay_attention(q, k, v, self.log_decay, self.scale, cu_seqlens, state, want_state)
        return self.back(out.flatten(1)), state

    @torch.no_grad()
    def step(self, x: torch.Tensor, positions: torch.Tensor, state: torch.Tensor, slots: torch.Tensor | None = None,
             fresh: torch.Tensor | None = None) -> torch.Tensor:
        """One token of each sequence, x [rows, dim], on state[slots] in place (ops.decay_attention_step)."""
        q, k, v = self._heads(x, positions)
        out = q.new_empty(q.shape)
        ops.decay_attention_step(q, k, v, self.log_decay, state, out, scale=self.scale, slots=slots, fresh=fresh)
        return self.back(out.flatten(1))


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, tokens, mask, temperature: float, denom, recorded: bool):
        # (needs_input_grad is a parameter's requires_grad, also where no graph is recorded)
        d_hidden = hidden.new_empty(hidden.shape) if recorded and ctx.needs_input_grad[0] else None
        d_weight = torch.empty_like(weight) if recorded and ctx.needs_input_grad[1] else None
        stats = torch.empty(4, device=hidden.device)
        ops.linear_cross_entropy(hidden, weight, tokens, d_hidden, d_weight, stats, mask=mask, temperature=temperature, denom=denom)
        ctx.save_for_backward(d_hidden, d_weight)
        return stats[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss):
        d_hidden, d_weight = ctx.saved_tensors
        # (in float32, since the loss' factor need not be one of the operands' type: as a vector it makes the product float32, rounded as it is stored, without
        # copies of the gradients between)
        scaled = [None if d is None else torch.mul(d, d_loss.reshape(1), out=torch.empty_like(d)) for d in (d_hidden, d_weight)]
        return *scaled, None, None, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, tokens: torch.Tensor, mask: torch.Tensor | None = None,
                         temperature: float = 1.0, denom: float | None = None) -> torch.Tensor:
    """The mean cross entropy of tokens under softmax(hidden weight^T / temperature), hidden [..., dim], without the logits: a float32 scalar
    whose gradients are made with it (``ops.linear_cross_entropy``; not under ``torch.no_grad()``), rounded to their operands' type before the
    factor that the loss is multiplied by: float16 wants a loss scale as denom = N / scale."""
    hidden = hidden.reshape(-1, hidden.shape[-1])
    mask = None if mask is None else mask.reshape(-1).contiguous()
    return _LinearCrossEntropy.apply(_rows(hidden), weight, tokens.reshape(-1).contiguous(), mask, float(temperature), denom, torch.is_grad_enabled())


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
