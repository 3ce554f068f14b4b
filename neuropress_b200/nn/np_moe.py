"""NPMoE: a mixture-of-experts block over packed 4-bit experts, two kernels for up to 32 tokens.

    y[t] = sum over the top_k experts e of  w_e * down_e(silu(gate_e(x[t])) * up_e(x[t]))

with ``w`` the softmax of the router's logits, renormalised over the chosen experts or not.  A model
keeps its experts as separate linears; lowered one by one (:class:`NPLinear`) a decode step launches
three kernels per chosen expert and needs the choice on the host.  :meth:`NPMoE.from_experts` stacks
their packed weights -- same bytes, same layout, expert after expert -- and ``forward`` runs the router
as it is and then ``kernels.q_moe``: no host synchronisation, so it can be captured in a CUDA graph.
More than 32 tokens run 32 at a time, each 32 reading their experts again: prompts of many hundreds of
tokens are faster through the lowered experts (64 experts, 8 to a token, 4096 x 1376, 2048 tokens: 12 ms
here, 5.1 ms there).  Casting the module casts the router only.  The stacked weights are copies, and the
block is not taken apart again by ``unlower_model``: keep the lowered experts where that is wanted.  No
reference counterpart.
"""

from __future__ import annotations

from collections.abc import Iterable

import torch
from torch import nn

from .. import _cabi
from .np_linear import NPLinear

__all__ = ["NPMoE"]

_NAMES = (("gate_proj", "up_proj", "down_proj"), ("w1", "w3", "w2"))


def _linears_of(expert) -> tuple[NPLinear, NPLinear, NPLinear]:
    """The gate / up / down linears of one expert: a module with one of the usual attribute names, or a
    tuple of the three."""
    if isinstance(expert, (tuple, list)) and len(expert) == 3:
        found = tuple(expert)
    else:
        found = next((tuple(getattr(expert, n) for n in names) for names in _NAMES
                      if all(hasattr(expert, n) for n in names)), ())
    if len(found) != 3 or not all(isinstance(m, NPLinear) for m in found):
        raise ValueError("an expert must hold three NPLinear modules named gate_proj / up_proj / down_proj or "
                         "w1 / w3 / w2, or be a (gate, up, down) tuple of them.")
    return found


class NPMoE(nn.Module):
    """``gate``, ``up`` and ``down`` are ``(codes, scale, zero_point or None)`` as :func:`kernels.q_moe` takes
    them; ``router`` maps ``[T, H]`` to the logits ``[T, E]``."""

    def __init__(self, router: nn.Module, gate: tuple, up: tuple, down: tuple, top_k: int, group_size: int,
                 renormalize: bool = True) -> None:
        super().__init__()
        e, i, half_h = gate[0].shape
        if tuple(up[0].shape) != (e, i, half_h) or tuple(down[0].shape) != (e, 2 * half_h, i // 2):
            raise ValueError("gate and up must be [E, I, H/2], down [E, H, I/2].")
        if e > _cabi.MOE_MAX_EXPERTS or max(2 * half_h, i) > _cabi.MOE_MAX_WIDTH:
            raise ValueError(f"at most {_cabi.MOE_MAX_EXPERTS} experts, H and I at most {_cabi.MOE_MAX_WIDTH}.")
        if not 1 <= top_k <= min(e, _cabi.MOE_MAX_TOP_K):
            raise ValueError(f"top_k must lie in [1, min(number of experts, {_cabi.MOE_MAX_TOP_K})].")
        if group_size % 32 or (2 * half_h) % group_size or i % group_size:
            raise ValueError("group_size must be a multiple of 32 that divides H and I.")
        if (gate[2] is None) != (up[2] is None):
            raise ValueError("gate and up must both have zero points or both have none.")
        self.router = router
        self.num_experts, self.hidden_size, self.intermediate_size = e, 2 * half_h, i
        self.top_k, self.group_size, self.renormalize = top_k, group_size, renormalize
        for name, (codes, scale, zero_point) in (("gate", gate), ("up", up), ("down", down)):
            self.register_buffer(f"{name}_codes", codes.contiguous())
            self.register_buffer(f"{name}_scale", scale.to(torch.float16).reshape(-1).contiguous())
            self.register_buffer(f"{name}_zero_point", None if zero_point is None
                                 else zero_point.to(torch.float16).reshape(-1).contiguous())

    @classmethod
    def from_experts(cls, router: nn.Module, experts: Iterable, top_k: int, renormalize: bool = True) -> "NPMoE":
        """Stack experts of :class:`NPLinear` modules: 4-bit, no bias, one group size, all of one shape, each of the
        three with zero points in every expert or in none."""
        triples = [_linears_of(x) for x in experts]
        if not triples:
            raise ValueError("at least one expert is needed.")
        stacked = []
        for column in zip(*triples):
            first = column[0]
            for m in column:
                if m.nbits != 4 or m.bias is not None or m.group_size != triples[0][0].group_size:
                    raise ValueError("experts must be 4-bit, without bias, of one group size.")
                if (m.out_features, m.in_features, m.qtype) != (first.out_features, first.in_features, first.qtype):
                    raise ValueError("experts must agree in shape and in having zero points.")
            stacked.append((torch.stack([m.u8_blob for m in column]), torch.stack([m.scale for m in column]),
                            None if first.zero_point is None else torch.stack([m.zero_point for m in column])))
        return cls(router, *stacked, top_k, triples[0][0].group_size, renormalize)

    def _apply(self, fn, recurse: bool = True):
        """A cast of the module (``.to(torch.bfloat16)`` for the router, say) leaves the scales and zero points fp16: they
        are part of the packed format.  They move with the device."""
        packed = {n: b for n, b in self._buffers.items() if b is not None and b.dtype == torch.float16}
        super()._apply(fn, recurse)
        for name, before in packed.items():
            after = self._buffers[name]
            if after.dtype != torch.float16:
                self._buffers[name] = before.to(after.device)
        return self

    def _weight(self, name: str) -> tuple:
        return getattr(self, f"{name}_codes"), getattr(self, f"{name}_scale"), getattr(self, f"{name}_zero_point")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        from .. import kernels

        *leading, h = x.shape
        x2 = x.reshape(-1, h).contiguous()
        logits = self.router(x2)
        y = kernels.q_moe(x2, logits.contiguous(), self._weight("gate"), self._weight("up"), self._weight("down"),
                          self.top_k, self.group_size, renormalize=self.renormalize)
        return y.reshape(*leading, h)

    def extra_repr(self) -> str:
        return (f"experts={self.num_experts}, top_k={self.top_k}, H={self.hidden_size}, I={self.intermediate_size}, "
                f"group_size={self.group_size}, renormalize={self.renormalize}")
