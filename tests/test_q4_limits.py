"""4-bit weights where types end: scales of one row far apart, activations beside the largest numbers."""

import pytest
import torch

import _q4_reference as ref


@pytest.fixture(scope="module")
def dev(lib_built):
    from t81lib_b200 import _capi
    assert _capi.device_available(), _capi.last_error()
    yield torch.device("cuda", 0)
    assert _capi.kernel_status(reset=True) == 0  # no bounded wait of a kernel ran out


def _check(y, x, values, bias=None):
    want, magnitude = ref.product(x, values, bias)
    if bias is not None:
        magnitude = magnitude + bias.double().abs()
    off = (y.double() - want).abs()
    assert y.shape == want.shape and bool((off <= ref.tolerance(magnitude, want, x.shape[1], y.dtype)).all()), float((off / magnitude).nan_to_num().max())


def _far_apart(gen, dev, rows, cols, group, plain):
    """Weights of which every row but each `plain`-th has groups 2^-16 to 2^-60 below its largest, and activations that are 0 beside the large groups."""
    w = torch.randn(rows, cols, generator=gen, device=dev)
    factor = torch.ones(rows, (cols + group - 1) // group, device=dev)
    for i, e in enumerate((-16, -20, -21, -25, -29, -30, -31, -35, -41, -60)):
        if i + 1 < factor.shape[1]:
            factor[:, i + 1] = 2.0 ** e
    factor[::plain] = 1.0
    factor[1::plain, 0] = 0.0                     # rows without the large group: the next one is the largest
    return w * factor.repeat_interleave(group, 1)[:, :cols]


def _quiet(x, group):
    """Activations that meet one small group each, by their row."""
    groups = (x.shape[1] + group - 1) // group
    at = torch.arange(x.shape[0], device=x.device) % groups
    return x * (torch.arange(x.shape[1], device=x.device) // group == at[:, None])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,group,plain", [(2048, 4096, 64, 3), (2000, 4090, 128, 50), (520, 8192, 32, 2), (5000, 1032, 64, 40), (37, 14336, 128, 5)])
def test_scales_of_a_row_far_apart(dev, rows, cols, group, plain):
    """float16 holds 40 binades and a row's scales span more: the result does not depend on how many rows of x there are."""
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(rows)
    q = t81_torch.Q4Tensor.from_float(_far_apart(gen, dev, rows, cols, group, plain), group=group)
    values = q.dequantize().double()
    bias = torch.randn(rows, generator=gen, device=dev) * 2.0 ** -40
    for tokens in (3, 130, 1200):
        x = torch.randn(tokens, cols, generator=gen, device=dev).half()
        for each, b in ((x, None), (_quiet(x, group), None), (_quiet(x, group), bias)):
            _check(q.matmul_input(each, b, out_dtype=torch.float32), each, values, b)
        y = q.matmul_input(_quiet(x, group))
        assert y.dtype == torch.float16
        _check(y, _quiet(x, group), values)


@pytest.mark.gpu
def test_infinite_activations_beside_small_scales(dev):
    """An infinity beside a weight that float16 would hold as 0 is an infinity of the product's sign."""
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(4)
    w = torch.randint(1, 8, (1024, 4096), generator=gen, device=dev).float()
    w[:, ::64] = -8.0
    w[:, 64:128] *= 2.0 ** -50
    q = t81_torch.Q4Tensor.from_float(w, group=64)
    for tokens in (2, 200):
        x = torch.randn(tokens, 4096, generator=gen, device=dev).half()
        x[0, 64], x[1, 70] = float("inf"), float("-inf")
        y = q.matmul_input(x, out_dtype=torch.float32)
        assert bool((y[:2] == -float("inf")).all()) and bool(torch.isfinite(y[2:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("counts,behind", [([300, 0, 40, 257, 1], 7), ([700] * 9, 0)])
def test_experts_with_scales_far_apart(dev, counts, behind):
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(len(counts))
    rows, cols, group = 1500, 1024, 64
    w = torch.stack([_far_apart(gen, dev, rows, cols, group, 2 + 20 * e) for e in range(len(counts))])
    w[0] = torch.randn(rows, cols, generator=gen, device=dev)  # an expert without such rows
    q = t81_torch.Q4Tensor.from_float(w, group=group)
    offsets = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    total = sum(counts)
    x = _quiet(torch.randn(total + behind, cols, generator=gen, device=dev).half(), group)
    bias = torch.randn(len(counts), rows, generator=gen, device=dev) * 2.0 ** -30
    y = q.matmul_sorted(x, offsets, bias, out_dtype=torch.float32)
    values, at = q.dequantize().double(), offsets.tolist()
    assert not y[total:].any()
    for e in range(len(counts)):
        _check(y[at[e]:at[e + 1]], x[at[e]:at[e + 1]], values[e], bias[e])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("offsets,total", [([4, 5, 5, 9], 10), ([300, 500, 700, 1100], 1200), ([7, 7, 7, 7], 7), ([2500, 2500, 2500, 2500], 2500), ([3, 900, 1000, 1500], 1500)])
def test_rows_ahead_of_the_first_expert(dev, offsets, total, dtype):
    """Slices of a sorted batch: rows that belong to an expert that is not there come out as 0, like the ones behind the last."""
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(total)
    for rows, cols in ((70, 200), (1000, 1024), (1001, 256)):
        q = t81_torch.Q4Tensor.from_float(torch.randn(3, rows, cols, generator=gen, device=dev) * 0.02, group=64)
        x = torch.randn(total, cols, generator=gen, device=dev).to(dtype)
        x[:offsets[0]], x[offsets[-1]:] = float("nan"), float("nan")
        torch.full((total, rows), float("nan"), device=dev, dtype=dtype)  # what the result's memory may hold
        y = q.matmul_sorted(x, torch.tensor(offsets, dtype=torch.int32, device=dev))
        assert not y[:offsets[0]].any() and not y[offsets[-1]:].any()
        values = q.dequantize().double()
        for e in range(3):
            lo, hi = offsets[e], offsets[e + 1]
            _check(y[lo:hi], x[lo:hi], values[e])


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(dev, grad):
    """A tangent of the activations or the bias is not dropped without a word, whatever path a call takes."""
    import torch.autograd.forward_ad as fwd
    from t81lib_b200 import torch as t81_torch
    from t81lib_b200.nn import Q4Experts, Q4Linear
    layer = Q4Linear.from_linear(torch.nn.Linear(64, 48, bias=False, device=dev), group=32)
    stack = t81_torch.Q4Tensor.from_float(torch.randn(2, 48, 64, device=dev), group=32)
    block = Q4Experts.from_float(torch.randn(2, 64, 48, device=dev), torch.randn(2, 48, 32, device=dev), group=32)
    offsets = torch.tensor([0, 1, 4], dtype=torch.int32, device=dev)
    x, bias = torch.randn(4, 64, device=dev), torch.randn(48, device=dev)
    ids, weights = torch.zeros(4, 1, dtype=torch.int64, device=dev), torch.ones(4, 1, device=dev)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        dual, dual_bias = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(bias, torch.ones_like(bias))
        assert layer(x).shape == (4, 48) and layer.weight.matmul_input(x, bias).shape == (4, 48)
        for call in (lambda: layer(dual), lambda: layer(dual.half()), lambda: layer.weight.matmul_input(dual), lambda: layer.weight.matmul_input(dual.t().contiguous().t()),
                     lambda: layer.weight.matmul_input(x, dual_bias), lambda: layer.weight.matmul_input(dual.cpu()),
                     lambda: stack.matmul_sorted(dual, offsets), lambda: stack.matmul_sorted(x, offsets, dual_bias.expand(2, 48)),
                     lambda: layer(dual.requires_grad_(True) if grad else dual)):
            with pytest.raises(NotImplementedError, match="forward|jvp"):
                call()
        with pytest.raises(RuntimeError, match="jvp"):
            block(fwd.make_dual(torch.randn(4, 48, device=dev), torch.ones(4, 48, device=dev)), ids, weights)
        with pytest.raises(RuntimeError, match="jvp"):
            t81_torch.route(ids, 2).combine(x, fwd.make_dual(weights, torch.ones_like(weights)))
        assert layer(x).shape == (4, 48)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("largest", [2.0 ** 119, 3.3e38])
def test_the_largest_activations(dev, dtype, largest):
    """Activations beside the end of their type: results that are numbers come out as those, however many rows there are."""
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(7)
    for rows, cols, group in ((300, 512, 128), (2048, 4096, 32), (100, 1032, 64)):
        q = t81_torch.Q4Tensor.from_float(torch.randn(rows, cols, generator=gen, device=dev) * 2.0 ** -20, group=group)
        values = q.dequantize().double()
        for tokens in (1, 8, 12, 200):
            x = (torch.rand(tokens, cols, generator=gen, device=dev) * 2 - 1).to(dtype) * largest
            x[0] = largest
            x[tokens // 2] = -largest
            assert bool(torch.isfinite(x).all())
            y = q.matmul_input(x)
            assert bool(torch.isfinite(y).all())
            _check(y, x, values)
            stack = t81_torch.Q4Tensor(q.codes, q.scales, (1, rows, cols), group)
            _check(stack.matmul_sorted(x, torch.tensor([0, tokens], dtype=torch.int32, device=dev)), x, values)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_results_near_the_smallest_numbers(dev, dtype):
    """The smallest scales there are and small activations: off by at most 2^-135, the last place of float32 brought up by the sums' 2^10, 16 times."""
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(8)
    q = t81_torch.Q4Tensor.from_float(torch.randn(300, 512, generator=gen, device=dev) * 2.0 ** -96, group=64)
    values = q.dequantize().double()
    for tokens in (3, 12, 200):
        for factor in (1.0, 2.0 ** -16, 2.0 ** -24):
            x = torch.randn(tokens, 512, generator=gen, device=dev).to(dtype) * factor
            want, magnitude = ref.product(x, values)
            off = (q.matmul_input(x, out_dtype=torch.float32).double() - want).abs()
            assert bool((off <= ref.tolerance(magnitude, want, 512, torch.float32) + 2.0 ** -135).all()), float(off.max())
