"""``Linear`` and experts with 4-bit weights and group scales: the layers of a model that ternary weights lose too much of.

Beside ``Linear`` (whose reference is t81/nn/linear.py:18-125); the reference has neither.  The weights are buffers in the products'
order and frozen; gradients reach the activations and the bias of ``Q4Linear``.
"""

from __future__ import annotations

from typing import Callable, Optional

import torch
from torch import nn

from .. import _capi
from .. import torch as t81_torch


class _Q4Module(nn.Module):
    """Holds Q4Tensors as pairs of buffers (``<name>_codes``, ``<name>_scales``).  The buffers' lengths tell rows and columns only up to whole
    tiles, so the state dict has the weights' shapes beside them (``_extra_state``, int64)."""

    _version = 2  # 1: without the shapes

    # the float weight is gone: what saves models asks for this
    _t81_float_released = True

    def __init__(self, group: int) -> None:
        super().__init__()
        if group not in (32, 64, 128):
            raise ValueError(f"groups of 32, 64 or 128 columns, not {group}")
        self.group = group
        self._q4_shapes: dict = {}
        self.__dict__["_q4"] = {}

    def _hold(self, name: str, q: "Optional[t81_torch.Q4Tensor]", shape, device=None) -> None:
        shape = tuple(int(n) for n in shape)
        if any(n < 1 for n in shape):
            raise ValueError(f"a 4-bit weight cannot be {shape}")
        matrices = shape[0] if len(shape) == 3 else 1
        codes = torch.empty(matrices * _capi.lib.t81b200_q4_bytes(*shape[-2:]), dtype=torch.uint8, device=device) if q is None else q.codes
        scales = torch.empty(matrices * _capi.lib.t81b200_q4_scales(*shape[-2:], self.group), dtype=torch.bfloat16, device=device) if q is None else q.scales
        self.register_buffer(name + "_codes", codes)
        self.register_buffer(name + "_scales", scales)
        self._q4_shapes[name] = shape

    def _held(self, name: str) -> "t81_torch.Q4Tensor":
        """The buffers as a Q4Tensor, made again when they were replaced (moved to another device)."""
        buffers = self._buffers
        codes, scales = buffers[name + "_codes"], buffers[name + "_scales"]
        q = self._q4.get(name)
        if q is None or q.codes is not codes or q.scales is not scales:
            q = self._q4[name] = t81_torch.Q4Tensor(codes, scales, self._q4_shapes[name], self.group)
        return q

    def _apply(self, fn, recurse: bool = True):
        # a change of the model's type does not concern the scales: they are part of the format
        before = {name: b for name, b in self._buffers.items() if name.endswith("_scales")}
        super()._apply(fn, recurse)
        for name, b in before.items():
            now = self._buffers[name]
            if now.dtype != torch.bfloat16:
                self._buffers[name] = b.to(now.device)
        return self

    def get_extra_state(self) -> torch.Tensor:
        return torch.tensor([n for shape in self._q4_shapes.values() for n in shape], dtype=torch.int64)

    def set_extra_state(self, state: torch.Tensor) -> None:
        pass  # looked at before anything is loaded

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs) -> None:
        key = prefix + "_extra_state"
        held = state_dict.get(key)
        if held is not None and held.tolist() != self.get_extra_state().tolist():
            error_msgs.append(f"size mismatch for {prefix}{'/'.join(self._q4_shapes)}: the state holds 4-bit weights of other sizes, {held.tolist()}, "
                              f"than this module's, {self.get_extra_state().tolist()}.")
            return
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        if held is None and local_metadata.get("version", 1) < 2 and key in missing_keys:
            missing_keys.remove(key)

    def __getstate__(self):
        return {**self.__dict__, "_q4": {}}  # native calls do not travel


def _check_experts(n: int) -> None:
    if n > _capi.MOST_EXPERTS:
        raise ValueError(f"{n} experts: a mixture in 4 bits has at most {_capi.MOST_EXPERTS}")


class Q4Linear(_Q4Module):
    """``nn.Linear`` with a 4-bit weight: ``x @ W.T + bias`` for 1 to any number of tokens, float32, bfloat16 or float16."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, group: int = 128, device: Optional[torch.device] = None,
                 dtype: Optional[torch.dtype] = None) -> None:
        """An empty layer, for ``load_state_dict``; ``dtype`` is the bias's."""
        super().__init__(group)
        self.in_features, self.out_features = in_features, out_features
        self._hold("weight", None, (out_features, in_features), device)
        self.bias = nn.Parameter(torch.zeros(out_features, dtype=dtype, device=device)) if bias else None

    @classmethod
    def from_quantized(cls, q: "t81_torch.Q4Tensor", bias: Optional[torch.Tensor] = None) -> "Q4Linear":
        if len(q.shape) != 2:
            raise ValueError("Q4Linear takes one matrix")
        if bias is not None and bias.shape != q.shape[:1]:
            raise ValueError("the bias does not match the weight's rows")
        layer = cls.__new__(cls)
        _Q4Module.__init__(layer, q.group)
        layer.out_features, layer.in_features = q.shape
        layer._hold("weight", q, q.shape)
        layer.bias = bias if bias is None or isinstance(bias, nn.Parameter) else nn.Parameter(bias)
        return layer

    @classmethod
    def from_linear(cls, linear: nn.Linear, group: int = 128) -> "Q4Linear":
        """Quantise a float layer's weight; the bias is taken over."""
        layer = cls.from_quantized(t81_torch.Q4Tensor.from_float(linear.weight, group=group), linear.bias)
        return layer.train(linear.training)

    @property
    def weight(self) -> "t81_torch.Q4Tensor":
        return self._held("weight")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        q = self._held("weight")
        product = q._native_product()
        bias = self._parameters["bias"] if "bias" in self._parameters else self.bias
        y = product(x, bias)  # None: a call that needs a conversion, a copy or an autograd node
        if y is not None:
            return y
        if x.shape[-1] != self.in_features:
            raise ValueError("rhs dimension does not match the weight's width")
        return q.matmul_input(x.reshape(-1, self.in_features), bias=bias).reshape(*x.shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, group={self.group}"


class Q4Experts(_Q4Module):
    """The experts of a mixture, each a gated MLP ``down(act(gate(x)) * up(x))``, with 4-bit weights: called with the tokens, the
    ids of the experts that the router chose for each and the router's weights.  For inference: no gradient is recorded."""

    def __init__(self, n_experts: int, hidden: int, ffn: int, act_fn: Callable[[torch.Tensor], torch.Tensor] = nn.functional.silu, group: int = 128,
                 device: Optional[torch.device] = None) -> None:
        """Empty experts, for ``load_state_dict``."""
        super().__init__(group)
        _check_experts(n_experts)
        self.n_experts, self.hidden, self.ffn, self.act_fn = n_experts, hidden, ffn, act_fn
        self._hold("gate_up", None, (n_experts, 2 * ffn, hidden), device)
        self._hold("down", None, (n_experts, hidden, ffn), device)

    @classmethod
    def from_float(cls, gate_up_proj: torch.Tensor, down_proj: torch.Tensor, act_fn: Callable[[torch.Tensor], torch.Tensor] = nn.functional.silu,
                   group: int = 128) -> "Q4Experts":
        """``gate_up_proj`` (experts, 2 ffn, hidden): the gate's rows, then the up projection's; ``down_proj`` (experts, hidden, ffn)."""
        if gate_up_proj.ndim != 3 or down_proj.ndim != 3 or gate_up_proj.shape != (down_proj.shape[0], 2 * down_proj.shape[2], down_proj.shape[1]):
            raise ValueError(f"experts must be (experts, 2 ffn, hidden) and (experts, hidden, ffn), not {tuple(gate_up_proj.shape)} and {tuple(down_proj.shape)}")
        _check_experts(down_proj.shape[0])
        layer = cls.__new__(cls)
        _Q4Module.__init__(layer, group)
        layer.n_experts, layer.hidden, layer.ffn = down_proj.shape
        layer.act_fn = act_fn
        layer._hold("gate_up", t81_torch.Q4Tensor.from_float(gate_up_proj, group=group), gate_up_proj.shape)
        layer._hold("down", t81_torch.Q4Tensor.from_float(down_proj, group=group), down_proj.shape)
        return layer

    @property
    def gate_up(self) -> "t81_torch.Q4Tensor":
        return self._held("gate_up")

    @property
    def down(self) -> "t81_torch.Q4Tensor":
        return self._held("down")

    def forward(self, hidden_states: torch.Tensor, top_k_index: torch.Tensor, top_k_weights: torch.Tensor) -> torch.Tensor:
        """``hidden_states`` (..., hidden); ``top_k_index`` and ``top_k_weights`` (tokens, slots).  Ids outside the experts take no part."""
        if hidden_states.shape[-1] != self.hidden:
            raise ValueError("hidden_states do not match the experts' width")
        x = hidden_states.reshape(-1, self.hidden)
        routing = t81_torch.route(top_k_index, self.n_experts)
        rows = self.gate_up.matmul_sorted(routing.gather(x), routing.offsets)
        rows = self.act_fn(rows[:, :self.ffn]) * rows[:, self.ffn:]
        return routing.combine(self.down.matmul_sorted(rows, routing.offsets), top_k_weights).reshape(hidden_states.shape)

    def extra_repr(self) -> str:
        return f"n_experts={self.n_experts}, hidden={self.hidden}, ffn={self.ffn}, group={self.group}"
