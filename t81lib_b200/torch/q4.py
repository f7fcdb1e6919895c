"""4-bit weights with group scales, and the routing of a mixture of experts.

For the layers that ternary weights lose too much of: language-model heads, first and last layers, experts.  ``Q4Tensor`` stands
beside ``TernaryTensor`` (quantise on the device, multiply from the packed form); ``route`` sorts the (token, slot) pairs that a
router chose by expert, so that ``Q4Tensor.matmul_sorted`` reads each expert's weights once.  The reference has neither.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _capi, ops


class Q4Tensor:
    """A (rows, cols) matrix, or an (experts, rows, cols) stack, of 4-bit codes with a scale per row and ``group`` columns."""

    __slots__ = ("codes", "scales", "shape", "group", "_product", "__weakref__")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, group: int) -> None:
        shape = torch.Size(shape)
        if len(shape) not in (2, 3):
            raise ValueError("a Q4Tensor is a 2D matrix or a 3D stack of them")
        if group not in (32, 64, 128):
            raise ValueError(f"groups of 32, 64 or 128 columns, not {group}")
        matrices, tiles = (shape[0] if len(shape) == 3 else 1), (shape[-2] + 15) // 16
        if codes.dtype != torch.uint8 or codes.numel() != matrices * tiles * ((shape[-1] + 63) // 64) * 512 or scales.dtype != torch.bfloat16 \
                or scales.numel() != matrices * tiles * ((shape[-1] + group - 1) // group + 1) * 16 or scales.device != codes.device:
            raise ValueError(f"codes and scales do not hold a {tuple(shape)} weight with groups of {group}")
        self.codes, self.scales, self.shape, self.group = codes, scales, shape, group

    def __setattr__(self, name: str, value) -> None:
        object.__setattr__(self, name, value)
        if name != "_product":
            object.__setattr__(self, "_product", None)  # the native call; it holds what it was made of

    def __reduce__(self):
        return type(self), (self.codes, self.scales, tuple(self.shape), self.group)  # native calls do not travel

    @classmethod
    def from_float(cls, source: torch.Tensor, group: int = 128) -> "Q4Tensor":
        """Quantise on the device; CPU inputs are moved to the current CUDA device."""
        from . import _to_device_float
        w = _to_device_float(source)
        codes, scales = ops.quantize_q4(w, group)
        return cls(codes, scales, w.shape, group)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def __repr__(self) -> str:
        return f"Q4Tensor(shape={tuple(self.shape)}, group={self.group})"

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The weights that the codes stand for; exact in float32 and bfloat16."""
        matrices = self.shape[0] if len(self.shape) == 3 else 1
        values = ops.dequantize_q4(self.codes, self.scales, self.shape[-2], self.shape[-1], self.group, matrices, dtype)
        return values if len(self.shape) == 3 else values[0]

    def group_scales(self) -> torch.Tensor:
        """bfloat16 (..., rows, groups)."""
        matrices = self.shape[0] if len(self.shape) == 3 else 1
        s = _capi.native.q4_group_scales(self.scales, matrices, self.shape[-2], self.shape[-1], self.group)
        return s if len(self.shape) == 3 else s[0]

    def _native_product(self):
        if self._product is None and len(self.shape) == 2 and self.shape.numel() > 0:
            self._product = _capi.native.Q4Product(self.codes, self.scales, self.shape[0], self.shape[1], self.group)
        return self._product

    def matmul_input(self, input: torch.Tensor, bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """``input @ W.T (+ bias)`` for activations (tokens, cols) -> (tokens, rows)."""
        if len(self.shape) != 2:
            raise ValueError("matmul_input takes one matrix; a stack of experts' goes with matmul_sorted")
        if input.ndim != 2:
            raise ValueError("Q4Tensor products expect 2D activations")
        if input.shape[1] != self.shape[1]:
            raise ValueError("rhs dimension does not match the weight's width")
        _check_type(input)
        if torch.is_grad_enabled() and (input.requires_grad or (bias is not None and bias.requires_grad)):
            return _Q4LinearFunction.apply(self, input, bias, out_dtype)
        product = self._native_product()
        y = product(input, bias, out_dtype) if product is not None else None
        if y is not None:
            return y
        ops.refuse_tangents(input, bias)
        return _multiply(self, input, bias, out_dtype)

    def matmul_sorted(self, rows: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None,
                      out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """Rows sorted by expert (``Routing.gather``) times the matrix of the expert each belongs to; rows ahead of ``offsets[0]`` and from
        ``offsets[-1]`` on come out as 0.  ``bias``: (experts, rows of a matrix).  For inference: no gradient is recorded."""
        if len(self.shape) != 3:
            raise ValueError("matmul_sorted takes an (experts, rows, cols) stack")
        if rows.ndim != 2 or rows.shape[1] != self.shape[2]:
            raise ValueError("rows do not match the weights' width")
        _check_type(rows)
        if offsets.numel() != self.shape[0] + 1:
            raise ValueError("offsets must have one entry more than there are experts")
        if torch.is_grad_enabled() and (rows.requires_grad or (bias is not None and bias.requires_grad)):
            raise NotImplementedError("experts in 4 bits record no gradients: call them under torch.no_grad()")
        ops.refuse_tangents(rows, bias)
        rows, bias = _operand(rows, self.device), _bias(bias, self.device)
        return ops.experts_q4(self.codes, self.scales, self.shape[1], rows, self.shape[2], self.group, offsets, bias, out_dtype)


def _check_type(x: torch.Tensor) -> None:
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"x must be float32, bfloat16 or float16, got {x.dtype}")


def _operand(x: torch.Tensor, device: torch.device) -> torch.Tensor:
    """Activations as the kernels take them: on the weight's device, unit column stride."""
    x = x.detach().as_subclass(torch.Tensor).to(device).resolve_neg()
    return x if x.numel() == 0 or ((x.shape[1] == 1 or x.stride(1) == 1) and (x.shape[0] == 1 or x.stride(0) >= x.shape[1])) else x.contiguous()


def _bias(bias: Optional[torch.Tensor], device: torch.device) -> Optional[torch.Tensor]:
    return None if bias is None else bias.detach().to(device=device, dtype=torch.float32).contiguous()


def _multiply(q: Q4Tensor, x: torch.Tensor, bias, out_dtype) -> torch.Tensor:
    y = ops.linear_q4(q.codes, q.scales, q.shape[0], _operand(x, q.device), q.shape[1], q.group, _bias(bias, q.device), out_dtype)
    return y if x.device == y.device else y.to(x.device)


class _Q4LinearFunction(torch.autograd.Function):
    """matmul_input under autograd: gradients of the activations and the bias; the weight is frozen."""

    @staticmethod
    def forward(ctx, q: Q4Tensor, x: torch.Tensor, bias, out_dtype):
        ctx.q, ctx.x_device, ctx.x_dtype, ctx.bias = q, x.device, x.dtype, None if bias is None else (bias.dtype, bias.device)
        return _multiply(q, x, bias, out_dtype)

    @staticmethod
    def backward(ctx, grad_output: torch.Tensor):
        # the dense form, as TernaryTensor has it
        g = grad_output.to(device=ctx.q.device, dtype=torch.float32)
        grad_x = g.matmul(ctx.q.dequantize()).to(device=ctx.x_device, dtype=ctx.x_dtype) if ctx.needs_input_grad[1] else None
        grad_bias = g.sum(dim=0).to(dtype=ctx.bias[0], device=ctx.bias[1]) if ctx.bias and ctx.needs_input_grad[2] else None
        return None, grad_x, grad_bias, None


class Routing:
    """(token, slot) pairs sorted by expert (``route``): ``order``, ``position`` and ``offsets`` as ``ops.sort_by_expert`` gives them."""

    __slots__ = ("order", "position", "offsets")

    def __init__(self, order: torch.Tensor, position: torch.Tensor, offsets: torch.Tensor) -> None:
        self.order, self.position, self.offsets = order, position, offsets

    def gather(self, x: torch.Tensor) -> torch.Tensor:
        """Each token's row of ``x`` (tokens, width) at the positions of its slots: (tokens * slots, width), sorted by expert; rows from
        ``offsets[-1]`` on are 0.  Differentiable: a token's gradient is the sum over its slots, in float32, in slot order."""
        return ops.gather_rows(x, self.position, self.offsets)

    def combine(self, rows: torch.Tensor, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The experts' results back: (tokens, width), the sum over a token's slots of weight (tokens, slots; 1 without) times row, in
        float32, in slot order, rounded once.  Slots that go to no expert take no part.  Differentiable in both."""
        return ops.combine_rows(rows, weights, self.position, self.offsets)


def route(experts: torch.Tensor, n_experts: int) -> Routing:
    """Sort the pairs of a router's choice, (tokens, slots) int64 or int32 expert ids, by expert (at most 1024).  Pairs of one expert
    keep their order; ids outside 0 .. n_experts - 1 (padding, beyond a capacity) go to no expert."""
    return Routing(*ops.sort_by_expert(experts, n_experts))
