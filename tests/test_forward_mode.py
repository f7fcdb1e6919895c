"""Ternary products under torch.autograd.forward_ad: a tangent is refused, not dropped."""

import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_ternary_products_refuse_tangents(lib_built, grad):
    import torch.autograd.forward_ad as fwd
    from t81lib_b200 import torch as t81_torch
    from t81lib_b200.nn import Linear
    torch.manual_seed(0)
    dev = torch.device("cuda", 0)
    weight = t81_torch.TernaryTensor.from_float(torch.randn(48, 96, device=dev), rule="absmean")
    layer = Linear(96, 48, bias=False, device=dev, rule="absmean").eval()
    x, bias = torch.randn(4, 96, device=dev), torch.randn(48, device=dev)
    want, want_layer = weight.matmul_input(x, bias), layer(x)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        dual, dual_bias = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(bias, torch.ones_like(bias))
        for call in (lambda: layer(dual), lambda: layer(dual.view(2, 2, 96)), lambda: layer(dual.half()), lambda: weight.matmul_input(dual),
                     lambda: weight.matmul_input(dual.t().contiguous().t()), lambda: weight.matmul_input(x, dual_bias), lambda: weight.matmul_input(x.half(), dual_bias),
                     lambda: weight.matmul_input(dual.cpu()), lambda: torch.matmul(weight, fwd.make_dual(x.t().contiguous(), x.t().contiguous()))):
            with pytest.raises((NotImplementedError, RuntimeError), match="forward|jvp"):
                call()
        assert torch.equal(weight.matmul_input(x, bias), want) and torch.equal(layer(x), want_layer)
