"""float32 activations beside 4-bit weights: all 24 bits in every kernel, and sums that long rows do not wear away."""

import pytest
import torch


@pytest.fixture(scope="module")
def dev(lib_built):
    from t81lib_b200 import _capi
    assert _capi.device_available(), _capi.last_error()
    yield torch.device("cuda", 0)
    assert _capi.kernel_status(reset=True) == 0  # no bounded wait of a kernel ran out


def _powers(gen, dev, *shape):
    """Weights that are powers of two, which 4 bits hold as they are in groups of 32 and more."""
    w = 2.0 ** torch.randint(0, 3, shape, generator=gen, device=dev).float()
    w *= torch.randint(0, 2, shape, generator=gen, device=dev).float() * 2 - 1
    w[..., ::32] = -8.0
    return w * 2.0 ** (torch.arange(shape[-2], device=dev) % 5 - 2.0)[:, None]


def _one_each(gen, dev, tokens, cols):
    """One number of 24 bits a row, the last bit among them, at a column of its own; and where."""
    value = (torch.randint(1 << 22, 1 << 23, (tokens,), generator=gen, device=dev) * 2 + 1).float() * 2.0 ** -20
    at = (torch.arange(tokens, device=dev) * 37 + 11) % cols
    x = torch.zeros(tokens, cols, device=dev)
    x[torch.arange(tokens, device=dev), at] = value
    # Two bf16 numbers do not hold it, so a product that dropped the third would be off: what the first leaves is an odd number of up to 2^15 units,
    # and the second holds it only below 2^8, one in 128.
    first = value.bfloat16().float()
    assert bool((first + (value - first).bfloat16().float() != value).any())
    return x, value, at


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,tokens", [(300, 700, 1), (300, 700, 8), (1999, 3001, 77), (2048, 4096, 256), (600, 6144, 500), (9000, 2048, 300), (5000, 14336, 90), (20000, 520, 33)])
def test_every_bit_arrives(dev, rows, cols, tokens):
    """A number times a power of two is a number of float32: equal, bit for bit."""
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(rows + tokens)
    w = _powers(gen, dev, rows, cols)
    q = t81_torch.Q4Tensor.from_float(w, group=(32, 64, 128)[tokens % 3])
    assert torch.equal(q.dequantize(), w)
    x, value, at = _one_each(gen, dev, tokens, cols)
    assert torch.equal(q.matmul_input(x), value[:, None] * w.t()[at])


@pytest.mark.gpu
@pytest.mark.parametrize("experts,rows,cols,each", [(5, 300, 700, 2), (16, 2048, 1024, 60), (3, 1000, 4096, 300), (40, 520, 320, 129)])
def test_every_bit_arrives_of_experts(dev, experts, rows, cols, each):
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(experts)
    w = _powers(gen, dev, experts, rows, cols)
    q = t81_torch.Q4Tensor.from_float(w, group=64)
    counts = (torch.arange(experts, device=dev) * 7) % (2 * each) + 1
    offsets = torch.cat([torch.zeros(1, dtype=torch.int32, device=dev), counts.cumsum(0).int()])
    total = int(offsets[-1])
    x, value, at = _one_each(gen, dev, total, cols)
    of = torch.repeat_interleave(torch.arange(experts, device=dev), counts)
    y = q.matmul_sorted(x, offsets)
    for e in range(experts):
        mine = of == e
        assert torch.equal(y[mine], value[mine][:, None] * w[e].t()[at[mine]])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,tokens", [(10240, 6144, 256), (2048, 6144, 200), (8192, 14336, 256), (1024, 14336, 256), (700, 14336, 3), (600, 30720, 100)])
def test_sums_of_long_rows_do_not_wear_away(dev, rows, cols, tokens):
    """The tensor core cuts an accumulator off at every 16 columns, always towards 0: 5.6e-7 of the result's norm after 2048 columns, 1.4e-6 after
    4096, 7e-6 after 14336 in one.  Accumulators per 2048 columns are each off by their own 5.6e-7 at most, and so is their sum, with a
    rounding of 2^-24 per accumulator; 1e-6 lies between that and one accumulator's figure for any of these widths.  The streaming kernel rounds
    group by group and stays far below."""
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(cols + rows)
    q = t81_torch.Q4Tensor.from_float(torch.randn(rows, cols, generator=gen, device=dev) * 0.02, group=128)
    x = torch.randn(tokens, cols, generator=gen, device=dev)
    want = x.double() @ q.dequantize().double().t()
    y = q.matmul_input(x).double()
    assert float((y - want).norm() / want.norm()) < 1e-6
    # experts' sums are made the same way
    stack = t81_torch.Q4Tensor(q.codes, q.scales, (1, rows, cols), 128)
    y = stack.matmul_sorted(x, torch.tensor([0, tokens], dtype=torch.int32, device=dev)).double()
    assert float((y - want).norm() / want.norm()) < 1e-6
