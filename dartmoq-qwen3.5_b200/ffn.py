"""Gated feed-forward blocks over the dense operators: y = (silu(x Wg^T) * (x Wu^T)) Wd^T.

Both classes hold ``gate_proj`` / ``up_proj`` / ``down_proj`` as the shared expert of the reference's layers does
(quantization/wxa16/bit_partitioned_moe.py:1101-1106), so a state dict of such a block loads unchanged, and either serves as
``shared_expert`` of the MoE modules.

``GatedFeedForward``       16-bit weights, differentiable when it is called by itself (the MoE modules run without gradients)
``W8A8GatedFeedForward``   8-bit weights and activations (one scale a weight row, one a token), inference only
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import dense
from .linear import W8A8Linear


def _is_silu(act) -> bool:
    """Whether an activation (a name, a function or a module) is SiLU: by what it computes."""
    if isinstance(act, str):
        return act.lower() in ("silu", "swish")
    z = torch.linspace(-8.0, 8.0, 65, device="cpu")
    try:
        with torch.no_grad():
            out = act(z.clone())
    except Exception:
        return False
    return torch.is_tensor(out) and out.shape == z.shape and torch.allclose(out.float().cpu(), nn.functional.silu(z), rtol=1e-4, atol=1e-6)


def require_silu(mlp) -> None:
    """ValueError where a block names another activation."""
    for name in ("act_fn", "activation_fn", "act", "activation", "hidden_act"):
        act = getattr(mlp, name, None)
        if (isinstance(act, str) or callable(act)) and not _is_silu(act):
            raise ValueError(f"the gated feed-forward block computes SiLU, the block's {name} is {act!r}")


def _projections(mlp):
    """The three projections of a block that computes down(silu(gate(x)) * up(x)) with plain linears.  What can be told from the
    block is checked (its activation, hooks and forward methods of the linears); its own ``forward`` is taken to be that."""
    parts = [getattr(mlp, name, None) for name in ("gate_proj", "up_proj", "down_proj")]
    if any(not isinstance(p, nn.Linear) for p in parts):
        raise TypeError("expected a block with gate_proj, up_proj and down_proj of type nn.Linear")
    if any(p.bias is not None for p in parts):
        raise ValueError("the gated feed-forward block has no biases")
    for p in parts:
        if type(p).forward is not nn.Linear.forward or "forward" in vars(p):
            raise ValueError(f"{type(p).__name__} computes more than nn.Linear: only its weight would be taken over")
        if p._forward_hooks or p._forward_pre_hooks or p._backward_hooks or p._backward_pre_hooks:
            raise ValueError("hooks of the projections would no longer run: remove them first")
    require_silu(mlp)
    return parts


class GatedFeedForward(nn.Module):
    """The block in bf16 or fp16; trains like the three ``nn.Linear`` it holds.  It reads their weights: hooks that are put on
    the linears later do not run.  As ``shared_expert`` of a MoE module it is served only: those compute without gradients, so
    it is trained by itself (against the outputs of the dense model, say) before or between."""

    def __init__(self, hidden_size: int, intermediate_size: int, dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        kw = dict(bias=False, dtype=dtype, device=device)
        self.hidden_size, self.intermediate_size = hidden_size, intermediate_size
        self.gate_proj = nn.Linear(hidden_size, intermediate_size, **kw)
        self.up_proj = nn.Linear(hidden_size, intermediate_size, **kw)
        self.down_proj = nn.Linear(intermediate_size, hidden_size, **kw)

    @classmethod
    def from_mlp(cls, mlp: nn.Module) -> "GatedFeedForward":
        """Take over the projections of a block with the same names (the parameters are shared, not copied)."""
        gate, up, down = _projections(mlp)
        block = cls(gate.in_features, gate.out_features, dtype=gate.weight.dtype, device="meta")
        block.gate_proj, block.up_proj, block.down_proj = gate, up, down
        return block

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return dense.gated_feed_forward(x, self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight)

    def extra_repr(self) -> str:
        return f"hidden_size={self.hidden_size}, intermediate_size={self.intermediate_size}"


class W8A8GatedFeedForward(nn.Module):
    """The block with 8-bit operands: the tokens are quantised in front of either half."""

    def __init__(self, gate_proj: W8A8Linear, up_proj: W8A8Linear, down_proj: W8A8Linear):
        super().__init__()
        if any(p.bias is not None for p in (gate_proj, up_proj, down_proj)):
            raise ValueError("the gated feed-forward block has no biases")
        if ((gate_proj.in_features, gate_proj.out_features) != (up_proj.in_features, up_proj.out_features)
                or down_proj.in_features != gate_proj.out_features):
            raise ValueError("gate_proj and up_proj must have one shape and down_proj must take their outputs")
        self.gate_proj, self.up_proj, self.down_proj = gate_proj, up_proj, down_proj

    @classmethod
    @torch.no_grad()
    def from_mlp(cls, mlp: nn.Module) -> "W8A8GatedFeedForward":
        """Quantise the 16-bit projections of a block with the same names."""
        return cls(*(W8A8Linear.from_linear(p) for p in _projections(mlp)))

    @torch.no_grad()
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        h = dense.int8_gated_linear(x, self.gate_proj.weight, self.gate_proj.weight_scale, self.up_proj.weight,
                                    self.up_proj.weight_scale)
        return self.down_proj(h)
