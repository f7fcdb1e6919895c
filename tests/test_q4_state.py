"""What 4-bit layers and tensors keep of themselves: state dicts, copies, the names a model was converted by."""

import copy
import io
import pickle
from collections import OrderedDict

import pytest
import torch
from torch import nn


def _filled(module, seed):
    """Codes and scales that tell modules apart."""
    gen = torch.Generator().manual_seed(seed)
    for b in module.buffers():
        b.copy_(torch.randint(0, 255, b.shape, generator=gen).to(b.dtype))
    return module


def test_state_of_another_size_is_refused(lib_built):
    """Rows and columns that round up to the same tiles: the buffers are as long, the weights are not the same."""
    from t81lib_b200.nn import Q4Experts, Q4Linear
    pairs = [(lambda: Q4Linear(4096, 300, bias=False), lambda: Q4Linear(4090, 295, bias=False)), (lambda: Q4Linear(64, 48), lambda: Q4Linear(50, 48)),
             (lambda: Q4Experts(3, 100, 40, group=32), lambda: Q4Experts(3, 100, 39, group=32)), (lambda: Q4Experts(3, 96, 40), lambda: Q4Experts(3, 90, 40))]
    for one, other in pairs:
        target, source = _filled(one(), 1), _filled(other(), 2)
        assert [b.shape for b in target.buffers()] == [b.shape for b in source.buffers()]
        before = {k: v.clone() for k, v in target.state_dict().items()}
        for strict in (True, False):
            for assign in (True, False):
                with pytest.raises(RuntimeError, match="size mismatch"):
                    target.load_state_dict(source.state_dict(), strict=strict, assign=assign)
                with pytest.raises(RuntimeError, match="size mismatch"):
                    nn.Sequential(target).load_state_dict(nn.Sequential(source).state_dict(), strict=strict, assign=assign)
        assert all(torch.equal(v, before[k]) for k, v in target.state_dict().items())  # nothing was loaded


def test_state_comes_back(lib_built):
    from t81lib_b200.nn import Q4Experts, Q4Linear
    for make in (lambda: nn.Sequential(Q4Linear(100, 40, group=32), Q4Linear(40, 7, bias=False)), lambda: Q4Experts(3, 100, 40, group=32)):
        source = _filled(make(), 3)
        file = io.BytesIO()
        torch.save(source.state_dict(), file)
        file.seek(0)
        state = torch.load(file, weights_only=True)
        assert all(isinstance(v, torch.Tensor) for v in state.values())  # formats that hold tensors alone take it
        target = _filled(make(), 4)
        assert str(target.load_state_dict(state)) == "<All keys matched successfully>"
        for target_of in (lambda s: s, lambda s: dict(s), lambda s: OrderedDict((k, v) for k, v in s.items())):
            target = _filled(make(), 4)
            target.load_state_dict(target_of(state))
            assert all(torch.equal(a, b) for a, b in zip(target.buffers(), source.buffers()))
        # states without the shapes, as they were once
        bare = OrderedDict((k, v) for k, v in state.items() if not k.endswith("_extra_state"))
        target = _filled(make(), 4)
        target.load_state_dict(bare)
        assert all(torch.equal(a, b) for a, b in zip(target.buffers(), source.buffers()))
        # of this version they belong to it
        bare._metadata = state._metadata
        with pytest.raises(RuntimeError, match="_extra_state"):
            make().load_state_dict(bare)


class Model(nn.Module):
    def __init__(self):
        super().__init__()
        self.first, self.second, self.third, self.last = (nn.Linear(96, 96) for _ in range(4))


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [(64, 64), (128, 32), (32, 32, 128)])
def test_converted_in_several_calls(lib_built, tmp_path, groups):
    """Names of every call are kept: a model loaded by them has the 4-bit weights of all."""
    from t81lib_b200 import convert
    from t81lib_b200.nn import Linear, Q4Linear
    names = ["first", "thi*", "second"][:len(groups)]
    torch.manual_seed(0)
    floats = Model().state_dict()
    model = Model().cuda()
    model.load_state_dict(floats)
    for name, group in zip(names, groups):
        convert.convert_module(model, rule="absmean", verbose=False, four_bit=[name], q4_group=group)
    convert.save_pretrained_t81(model, tmp_path, call_save_pretrained=False)

    def loader(path):
        again = Model()
        again.load_state_dict(floats)
        return again.cuda()

    again = convert.from_pretrained_t81(None, tmp_path, loader=loader)
    x = torch.randn(3, 96, device="cuda")
    for leaf in ("first", "second", "third", "last"):
        one, other = getattr(model, leaf).eval(), getattr(again, leaf).eval()
        assert type(one) is type(other) and isinstance(one, Linear if leaf == "last" or (leaf == "second" and len(groups) == 2) else Q4Linear)
        assert not isinstance(one, Q4Linear) or one.group == other.group
        with torch.no_grad():
            assert torch.equal(one(x), other(x))
    # and saved once more the names are the same
    convert.save_pretrained_t81(again, tmp_path / "again", call_save_pretrained=False)
    assert convert.read_metadata(tmp_path / "again") == convert.read_metadata(tmp_path)


def test_copies_of_a_tensor(lib_built):
    from t81lib_b200.torch import Q4Tensor
    codes, scales = torch.randint(0, 255, (512,)).to(torch.uint8), torch.rand(32).to(torch.bfloat16)
    q = Q4Tensor(codes, scales, (16, 64), 64)
    for again in (copy.deepcopy(q), pickle.loads(pickle.dumps(q)), copy.copy(q)):
        assert again.shape == q.shape and isinstance(again.shape, torch.Size) and again.group == 64
        assert torch.equal(again.codes, codes) and torch.equal(again.scales, scales)
    assert copy.copy(q).codes is codes and copy.deepcopy(q).codes is not codes


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [2, 40])
def test_copies_and_new_weights_after_a_product(lib_built, tokens):
    from t81lib_b200.torch import Q4Tensor
    torch.manual_seed(tokens)
    q, other = (Q4Tensor.from_float(torch.randn(48, 96, device="cuda"), group=32) for _ in range(2))
    x = torch.randn(tokens, 96, device="cuda")
    y, want = q.matmul_input(x), other.matmul_input(x)
    assert torch.equal(copy.deepcopy(q).matmul_input(x), y) and torch.equal(pickle.loads(pickle.dumps(q)).matmul_input(x), y)
    file = io.BytesIO()
    torch.save({"head": q}, file)
    file.seek(0)
    assert torch.equal(torch.load(file, weights_only=False)["head"].matmul_input(x), y)
    q.codes, q.scales = other.codes, other.scales  # what was multiplied by is not kept
    assert torch.equal(q.matmul_input(x), want) and torch.equal(q.dequantize(), other.dequantize())
    q.codes = other.codes[:-1]
    with pytest.raises(ValueError, match="do not hold"):
        q.matmul_input(x)


class Experts(nn.Module):
    def __init__(self, experts):
        super().__init__()
        self.gate_up_proj, self.down_proj = nn.Parameter(torch.zeros(experts, 4, 3)), nn.Parameter(torch.zeros(experts, 3, 2))
        self.act_fn = nn.SiLU()


def test_more_experts_than_the_routing_takes(lib_built):
    """Refused before a float weight is given up for experts that no call could run."""
    from t81lib_b200 import convert
    from t81lib_b200.nn import Q4Experts
    assert Q4Experts(1024, 3, 2).n_experts == 1024
    with pytest.raises(ValueError, match="at most 1024"):
        Q4Experts(1025, 3, 2)
    many = Experts(1025)
    with pytest.raises(ValueError, match="at most 1024"):
        Q4Experts.from_float(many.gate_up_proj, many.down_proj)
    model = nn.Module()
    model.first, model.second = nn.Linear(4, 4), many
    with pytest.raises(ValueError, match="second has 1025 experts"):
        convert.convert_module(model, four_bit=["second"])
    assert model.second is many and type(model.first) is nn.Linear
