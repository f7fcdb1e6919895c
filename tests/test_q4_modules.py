"""4-bit layers as a model has them: Q4Linear, Q4Experts, conversion, and the whole block run together."""

import copy

import pytest
import torch
from torch import nn

import _q4_reference as ref


class Experts(nn.Module):
    """Stacked experts as model code holds them."""

    def __init__(self, experts=6, hidden=96, ffn=40):
        super().__init__()
        self.gate_up_proj = nn.Parameter(torch.randn(experts, 2 * ffn, hidden) * 0.1)
        self.down_proj = nn.Parameter(torch.randn(experts, hidden, ffn) * 0.1)
        self.act_fn = nn.SiLU()

    def forward(self, hidden_states, top_k_index, top_k_weights):
        raise NotImplementedError


class Mixture(nn.Module):
    def __init__(self, experts=6, hidden=96):
        super().__init__()
        self.router = nn.Linear(hidden, experts, bias=False)
        self.experts = Experts(experts, hidden)

    def forward(self, x):
        values, ids = torch.topk(self.router(x).float(), 2, dim=-1)
        return x + self.experts(x, ids, torch.softmax(values, -1))


class Model(nn.Module):
    def __init__(self):
        super().__init__()
        self.layers = nn.ModuleList([Mixture(), Mixture()])
        self.proj = nn.Linear(96, 96)
        self.lm_head = nn.Linear(96, 200, bias=False)

    def forward(self, x):
        for layer in self.layers:
            x = layer(x)
        return self.lm_head(self.proj(x))


def test_convert_refusals_leave_the_model_alone(lib_built, tmp_path):
    from t81lib_b200 import convert
    model = Model()
    with pytest.raises(ValueError, match="CUDA device"):
        convert.convert_module(model, four_bit=["lm_head"])
    with pytest.raises(ValueError, match="no nn.Linear and no stacked experts are named 'head'"):
        convert.convert_module(model, four_bit=["head"])
    with pytest.raises(TypeError, match="sequence"):
        convert.convert_module(model, four_bit="lm_head")
    with pytest.raises(ValueError, match="groups of"):
        convert.convert_module(model, q4_group=100)
    assert type(model.lm_head) is nn.Linear and isinstance(model.layers[0].experts, Experts)
    model._t81_four_bit, model._t81_q4_group = ["lm_head"], 64
    convert.save_pretrained_t81(model, tmp_path, call_save_pretrained=False)
    assert convert.read_metadata(tmp_path)["four_bit"] == ["lm_head"] and convert.read_metadata(tmp_path)["q4_group"] == 64
    with pytest.raises(ValueError, match="CUDA device"):
        convert.from_pretrained_t81(None, tmp_path, loader=lambda path: Model())


@pytest.fixture(scope="module")
def dev(lib_built):
    from t81lib_b200 import _capi
    assert _capi.device_available(), _capi.last_error()
    yield torch.device("cuda", 0)
    assert _capi.kernel_status(reset=True) == 0  # no bounded wait of a kernel ran out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_linear_layer(dev, dtype):
    from t81lib_b200.nn import Q4Linear
    torch.manual_seed(0)
    source = nn.Linear(200, 120, device=dev, dtype=dtype)
    layer = Q4Linear.from_linear(source, group=64)
    assert layer.bias is source.bias and layer.weight.shape == (120, 200) and "group=64" in repr(layer)
    values = ref.quantize(source.weight.detach(), 64)[2]
    for shape in ((200,), (3, 200), (2, 5, 200), (2, 2, 3, 200), (0, 200)):
        x = torch.randn(shape, device=dev).to(dtype)
        with torch.no_grad():
            y = layer(x)
        want, magnitude = ref.product(x.reshape(-1, 200), values, source.bias)
        assert y.shape == (*shape[:-1], 120) and y.dtype == dtype
        magnitude = magnitude + source.bias.double().abs()
        assert bool(((y.reshape(-1, 120).double() - want).abs() <= ref.tolerance(magnitude, want, 200, dtype)).all())
        recorded = layer(x.requires_grad_(True))  # under autograd: the same values
        assert torch.equal(recorded, y) and recorded.requires_grad
    with pytest.raises(ValueError):
        layer(torch.zeros(3, 199, device=dev, dtype=dtype))
    again = Q4Linear(200, 120, group=64, device=dev, dtype=dtype)
    again.load_state_dict(layer.state_dict())
    x = torch.randn(4, 200, device=dev).to(dtype)
    with torch.no_grad():
        assert torch.equal(again(x), layer(x))
        assert torch.equal(copy.deepcopy(layer)(x), layer(x))
        # new weights of the same layer, in place: nothing kept answers for them
        again.weight_codes.copy_(Q4Linear.from_linear(nn.Linear(200, 120, device=dev, dtype=dtype), group=64).weight_codes)
        assert not torch.equal(again(x), layer(x))
        moved = copy.deepcopy(layer).cpu().to(dev)
        assert torch.equal(moved(x), layer(x))
        assert torch.equal(layer(x.cpu()), layer(x).cpu())


def _experts_in_64_bits(x, ids, weights, gate_up, down):
    y = torch.zeros_like(x)
    for t in range(x.shape[0]):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            if 0 <= e < gate_up.shape[0]:
                gate, up = (gate_up[e] @ x[t]).chunk(2)
                y[t] += weights[t, j] * (down[e] @ (nn.functional.silu(gate) * up))
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 5, 60])
def test_experts_block(dev, tokens):
    """float32: sort, gather, two products, activation and combination against 64 bits."""
    from t81lib_b200.nn import Q4Experts
    torch.manual_seed(tokens)
    source = Experts().to(dev)
    block = Q4Experts.from_float(source.gate_up_proj, source.down_proj, source.act_fn, group=32)
    x, weights = torch.randn(tokens, 96, device=dev), torch.rand(tokens, 2, device=dev)
    ids = torch.randint(-1, 6, (tokens, 2), device=dev)
    with torch.no_grad():
        y = block(x, ids, weights)
        y3 = block(x.view(1, tokens, 96), ids, weights)
    want = _experts_in_64_bits(x.double(), ids, weights.double(), ref.quantize(source.gate_up_proj.detach(), 32)[2], ref.quantize(source.down_proj.detach(), 32)[2])
    # a product's result is off by at most some 30 steps of 2^-23 of its magnitudes (96 and 40 terms), which are a few times the results;
    # two products and the activation between them: far below 1e-4 of the largest
    assert float((y.double() - want).abs().max()) <= 1e-4 * float(want.abs().max())
    assert torch.equal(y3[0], y)
    again = Q4Experts(6, 96, 40, group=32, device=dev)
    again.load_state_dict(block.state_dict())
    with torch.no_grad():
        assert torch.equal(again(x, ids, weights), y)
    with pytest.raises(NotImplementedError, match="no_grad"):
        block(x.requires_grad_(True), ids, weights)


@pytest.mark.gpu
def test_converted_model_runs_and_decodes_from_a_graph(dev, tmp_path):
    from t81lib_b200 import convert
    from t81lib_b200.nn import Linear, Q4Experts, Q4Linear
    torch.manual_seed(1)
    model = Model().to(dev).eval()
    head, gate_up = model.lm_head.weight.detach().clone(), model.layers[1].experts.gate_up_proj.detach().clone()
    stats = convert.convert_module(model, rule="absmean", verbose=False, four_bit=["lm_head", "layers.*.experts"], q4_group=32)
    assert stats.four_bit == 3 and stats.replaced == 3 and stats.four_bit_bytes > 0
    assert isinstance(model.lm_head, Q4Linear) and all(isinstance(m.experts, Q4Experts) and isinstance(m.router, Linear) for m in model.layers)
    assert torch.equal(model.lm_head.weight.dequantize().double(), ref.quantize(head, 32)[2])
    assert torch.equal(model.layers[1].experts.gate_up.dequantize().double(), ref.quantize(gate_up, 32)[2])
    with pytest.raises(RuntimeError, match="released"):
        convert.save_pretrained_t81(model, tmp_path, save_fn=lambda m, d: None)
    again = convert.convert_module(model, rule="absmean", verbose=False)  # 4-bit modules stay
    assert again.replaced == 0 and isinstance(model.lm_head, Q4Linear)
    x = torch.randn(7, 96, device=dev)
    with torch.no_grad():
        want = model(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            model(x)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = model(x)
        graph.replay()
        assert torch.equal(y, want)
        x.normal_()
        graph.replay()
        assert torch.equal(y, model(x))


@pytest.mark.gpu
def test_a_module_of_two_names_is_replaced_under_both(dev):
    from t81lib_b200 import convert
    from t81lib_b200.nn import Q4Linear
    for pattern in ("first", "second"):
        model = nn.Module()
        model.first = model.second = nn.Linear(64, 48).to(dev)
        stats = convert.convert_module(model, verbose=False, four_bit=[pattern])
        assert isinstance(model.first, Q4Linear) and model.second is model.first and stats.four_bit == 1 and stats.replaced == 0


@pytest.mark.gpu
def test_pickled_layers(dev):
    import pickle
    from t81lib_b200.nn import Q4Linear
    layer = Q4Linear.from_linear(nn.Linear(64, 48).to(dev)).eval()
    x = torch.randn(3, 64, device=dev)
    with torch.no_grad():
        y = layer(x)
        held = layer.weight
        assert torch.equal(pickle.loads(pickle.dumps(layer))(x), y) and layer.weight is held
