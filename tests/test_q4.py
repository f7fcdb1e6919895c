"""4-bit weights with group scales: the quantiser and its layout against their definition, exactly; products against 64 bits."""

import ctypes

import pytest
import torch

import _q4_reference as ref


@pytest.fixture(scope="module")
def dev(lib_built):
    from t81lib_b200 import _capi
    assert _capi.device_available(), _capi.last_error()
    yield torch.device("cuda", 0)
    assert _capi.kernel_status(reset=True) == 0  # no bounded wait of a kernel ran out


# ---- on the CPU ----


def test_refusals_need_no_device(lib_built):
    from t81lib_b200 import _capi, ops
    from t81lib_b200 import torch as t81_torch
    from t81lib_b200.nn import Q4Experts, Q4Linear
    lib = _capi.lib
    assert lib.t81b200_q4_bytes(17, 65) == 2 * 2 * 512 and lib.t81b200_q4_bytes(-1, 4) == -1
    assert lib.t81b200_q4_scales(17, 65, 32) == 2 * 4 * 16 and lib.t81b200_q4_scales(17, 65, 33) == -1
    buf = ctypes.create_string_buffer(64)
    assert lib.t81b200_quantize_q4(buf, 0, 1, 4, 8, 4, 0, 32, buf, buf, None) == _capi.EINVAL      # ld below cols
    assert lib.t81b200_quantize_q4(buf, 0, 1, 4, 8, 8, 0, 48, buf, buf, None) == _capi.EINVAL      # group
    assert lib.t81b200_dequantize_q4(buf, buf, 1, -4, 8, 32, buf, 0, None) == _capi.EINVAL
    assert lib.t81b200_linear_q4(buf, buf, None, buf, 4, buf, 1, 4, 1, 4, 1, 8, 32, None, 0, None) == _capi.EINVAL   # ldb below K
    assert lib.t81b200_linear_q4(buf, buf, None, buf, 4, buf, 3, 8, 1, 4, 1, 8, 32, None, 0, None) == _capi.EINVAL   # type of B
    assert lib.t81b200_experts_q4(buf, buf, None, buf, 4, buf, 1, 8, 1, 4, 1, 8, 32, None, 2, None, 0, None) == _capi.EINVAL  # no offsets
    assert "offsets" in _capi.last_error()
    for w in (torch.zeros(4, 8), torch.zeros(8)):
        with pytest.raises(ValueError):
            ops.quantize_q4(w, 32)
    with pytest.raises(ValueError, match="groups of 32, 64 or 128"):
        Q4Linear(64, 64, group=16)
    with pytest.raises(ValueError, match="cannot be"):
        Q4Linear(0, 64)
    with pytest.raises(ValueError, match="do not hold"):
        t81_torch.Q4Tensor(torch.zeros(512, dtype=torch.uint8), torch.zeros(16, dtype=torch.bfloat16), (17, 64), 64)
    with pytest.raises(ValueError, match="experts must be"):
        Q4Experts.from_float(torch.zeros(2, 8, 4), torch.zeros(2, 4, 3))
    q = t81_torch.Q4Tensor(torch.zeros(512, dtype=torch.uint8), torch.zeros(32, dtype=torch.bfloat16), (16, 64), 64)
    with pytest.raises(ValueError, match="2D activations"):
        q.matmul_input(torch.zeros(64))
    with pytest.raises(ValueError, match="width"):
        q.matmul_input(torch.zeros(2, 63))
    for bad in (torch.float64, torch.int32):
        with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
            q.matmul_input(torch.zeros(2, 64, dtype=bad))
    with pytest.raises(ValueError, match="stack"):
        q.matmul_sorted(torch.zeros(2, 64), torch.zeros(2, dtype=torch.int32))


def test_scales_survive_a_change_of_type(lib_built):
    from t81lib_b200.nn import Q4Linear
    layer = Q4Linear(100, 40, group=32)
    layer.weight_scales.fill_(2.0 ** -60)  # fp16 would lose it
    layer.half()
    assert layer.weight_scales.dtype == torch.bfloat16 and float(layer.weight_scales[0]) == 2.0 ** -60 and layer.bias.dtype == torch.float16
    assert layer.weight.codes is layer.weight_codes
    layer.load_state_dict(Q4Linear(100, 40, group=32).state_dict())


# ---- quantise ----


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (16, 64), (17, 65), (37, 129), (100, 200), (64, 1000), (5, 31), (33, 96)])
def test_quantise_is_the_definition(dev, rows, cols, dtype, group):
    from t81lib_b200 import ops
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator().manual_seed(rows * 7 + cols)
    w = (torch.randn(rows, cols, generator=gen) * 0.02).to(dtype)
    codes, scales, values = ref.quantize(w, group)
    q = t81_torch.Q4Tensor.from_float(w.to(dev), group=group)
    want_words, want_scales = ref.pack(codes, scales, group)
    assert torch.equal(q.codes.cpu().view(torch.int32).long() & 0xFFFFFFFF, want_words)
    assert torch.equal(q.scales.cpu(), want_scales)
    assert torch.equal(q.group_scales().cpu().double(), scales)
    for out in (torch.float32, torch.bfloat16):
        assert torch.equal(q.dequantize(out).cpu().double(), values)  # exact in both
    assert torch.equal(q.dequantize(torch.float16).cpu(), values.to(torch.float16))
    assert torch.equal(ops.dequantize_q4(q.codes, q.scales, rows, cols, group)[0].cpu().double(), values)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantise_at_its_borders(dev, group):
    """Weights halfway between two codes, equal magnitudes of both signs, zeros, what is no number, the largest and the smallest."""
    from t81lib_b200 import torch as t81_torch
    w = torch.zeros(40, 300)
    halves = torch.arange(-17, 18) / 2.0
    for r in range(8):
        w[r, :35] = halves * 2.0 ** (r - 4)
        w[r, 40 + r] = -8.0 * 2.0 ** (r - 4)
    w[8, 3], w[8, 90], w[9, 3], w[9, 90] = 4.0, -4.0, -4.0, 4.0                  # the first of equals gives the sign, in every group size
    w[10, 0], w[10, 1] = 4.0, -4.0
    w[11, 5], w[11, 6] = float("nan"), 1.0
    w[12, 5], w[12, 6] = float("inf"), 1.0
    w[13, 5], w[13, 6] = -float("inf"), float("nan")
    w[14, :] = 2.0 ** -101
    w[15, :] = 2.0 ** -100
    w[16, :] = 3.3e38
    w[17, :20] = torch.nextafter(torch.tensor(2.5), torch.tensor(3.0))          # one place beside a border
    w[17, 20:24] = torch.nextafter(torch.tensor(2.5), torch.tensor(2.0))
    w[17, 24] = -8.0
    w[18, :30] = torch.linspace(-1.0, 1.0, 30) * 1.07
    w[19, 299] = 1e-3                                                            # the last, shorter group
    w[20:] = torch.randn(20, 300, generator=torch.Generator().manual_seed(1))
    codes, scales, values = ref.quantize(w, group)
    q = t81_torch.Q4Tensor.from_float(w.to(dev), group=group)
    assert torch.equal(q.group_scales().cpu().double(), scales)
    assert torch.equal(q.dequantize().cpu().double(), values)
    assert torch.equal(q.codes.cpu().view(torch.int32).long() & 0xFFFFFFFF, ref.pack(codes, scales, group)[0])


@pytest.mark.gpu
def test_quantise_strided_and_stacked(dev):
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator().manual_seed(5)
    wide = torch.randn(3, 40, 210, generator=gen)
    for w in (wide[:, :, 5:180], wide[:, 1:38], wide.transpose(1, 2), wide[1], wide[0, :, 3:7], wide[::2], wide[:, :, :1]):
        for dtype in (torch.float32, torch.bfloat16):
            source = w.to(dtype)
            on = torch.empty(0)
            if w.stride(-1) == 1:  # the same view on the device
                base = wide.to(dev).to(dtype)
                on = base.as_strided(w.shape, w.stride(), w.storage_offset())
            else:
                on = wide.to(dev).to(dtype).transpose(1, 2)
            q = t81_torch.Q4Tensor.from_float(on, group=64)
            assert q.shape == w.shape
            _, scales, values = ref.quantize(source, 64)
            assert torch.equal(q.dequantize().cpu().double(), values) and torch.equal(q.group_scales().cpu().double(), scales)


@pytest.mark.gpu
def test_quantise_nothing(dev):
    from t81lib_b200 import torch as t81_torch
    for shape in ((0, 40), (40, 0), (0, 4, 4), (2, 0, 4)):
        q = t81_torch.Q4Tensor.from_float(torch.zeros(shape, device=dev), group=32)
        assert q.dequantize().shape == shape and q.codes.numel() == 0


# ---- products ----


def _case(gen, dev, rows, cols, tokens, dtype, group, bias):
    from t81lib_b200 import torch as t81_torch
    w = torch.randn(rows, cols, generator=gen, device=dev) * 0.02
    q = t81_torch.Q4Tensor.from_float(w, group=group)
    x = torch.randn(tokens, cols, generator=gen, device=dev).to(dtype)
    b = torch.randn(rows, generator=gen, device=dev) * 0.1 if bias else None
    return q, x, b


def _check(y, x, q, b):
    want, magnitude = ref.product(x, q.dequantize().double(), b)
    if b is not None:
        magnitude = magnitude + b.double().abs()
    off = (y.double() - want).abs()
    assert y.shape == want.shape and bool((off <= ref.tolerance(magnitude, want, x.shape[1], y.dtype)).all()), float(off.max())


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (16, 64), (33, 130), (100, 1000), (300, 4096), (257, 2049), (1024, 520), (48, 14336)])
def test_product(dev, rows, cols, dtype, group):
    gen = torch.Generator(device="cuda").manual_seed(rows + cols)
    for tokens in (1, 2, 7, 8, 9, 16, 17, 33, 64, 130):
        q, x, b = _case(gen, dev, rows, cols, tokens, dtype, group, tokens % 2 == 1)
        _check(q.matmul_input(x, b), x, q, b)
        _check(q.matmul_input(x, b, out_dtype=torch.float32), x, q, b)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,tokens", [(512, 512, 300), (1000, 777, 515), (256, 4096, 1024), (2050, 256, 257), (128, 64, 2048), (4096, 128, 129)])
def test_product_of_many_rows(dev, rows, cols, tokens):
    gen = torch.Generator(device="cuda").manual_seed(rows + tokens)
    for i, dtype in enumerate((torch.bfloat16, torch.float16, torch.float32)):
        q, x, b = _case(gen, dev, rows, cols, tokens, dtype, (32, 64, 128)[i], i == 0)
        _check(q.matmul_input(x, b), x, q, b)
        _check(q.matmul_input(x, None, out_dtype=torch.float32), x, q, None)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,tokens", [(300, 2048, 300), (256, 2049, 70), (300, 6144, 200), (513, 8200, 129), (100, 14336, 150), (64, 31000, 40), (40, 40000, 65), (20000, 128, 33)])
def test_float32_sums_of_long_rows(dev, rows, cols, tokens):
    """Many float32 rows: accumulators per 2048 columns keep the error below what 2048 columns' worth of cut-off steps and a few roundings make."""
    gen = torch.Generator(device="cuda").manual_seed(cols)
    q, x, b = _case(gen, dev, rows, cols, tokens, torch.float32, 64, True)
    want, magnitude = ref.product(x, q.dequantize().double(), b)
    y = q.matmul_input(x, b)
    _check(y, x, q, b)
    # 128 steps of at most 2^-23 of the sum so far, which is at most some three times the root of the terms' squares, twenty more roundings; the
    # accumulators' errors are independent of one another
    rms = (x.double() ** 2 @ (q.dequantize().double() ** 2).t()).sqrt()
    assert bool(((y.double() - want).abs() <= (128 * 3 + 20 * 5) * 2.0 ** -23 * rms + 2.0 ** -23 * b.double().abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,tokens", [(512, 512, 300), (1000, 4100, 70), (33, 130, 9), (300, 6144, 200)])
def test_float32_rows_with_16_bit_results(dev, rows, cols, tokens):
    gen = torch.Generator(device="cuda").manual_seed(rows + tokens)
    for out_dtype in (torch.bfloat16, torch.float16):
        q, x, b = _case(gen, dev, rows, cols, tokens, torch.float32, 64, True)
        y = q.matmul_input(x, b, out_dtype=out_dtype)
        assert y.dtype == out_dtype
        _check(y, x, q, b)
        assert torch.equal(y, q.matmul_input(x, b).to(out_dtype))  # the same sums, rounded once


@pytest.mark.gpu
def test_more_elements_than_31_bits_count(dev):
    """Weights, results and activations of more than 2^31 elements each, at their far ends."""
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(3)
    rows, cols = 66001, 32800
    w = torch.empty(rows, cols, dtype=torch.bfloat16, device=dev).normal_(generator=gen)
    q = t81_torch.Q4Tensor.from_float(w, group=64)
    last = t81_torch.Q4Tensor.from_float(w[-17:].contiguous(), group=64)  # 66001 = 16 * 4125 + 1: row tiles begin alike
    del w
    for tokens in (3, 40):
        x = torch.randn(tokens, cols, generator=gen, device=dev).to(torch.bfloat16)
        y = q.matmul_input(x, out_dtype=torch.float32)
        _check(y[:, -17:], x, last, None)
    del q, y
    q = t81_torch.Q4Tensor.from_float(torch.randn(1003, 64, generator=gen, device=dev), group=64)
    x = torch.randn(2150000, 64, generator=gen, device=dev).to(torch.bfloat16)
    y = q.matmul_input(x)
    _check(y[-300:], x[-300:], q, None)
    _check(y[1000000:1000300], x[1000000:1000300], q, None)
    del y
    wide = torch.zeros(33, 1 << 26, dtype=torch.bfloat16, device=dev)  # rows 2^26 elements apart
    wide[:, :64] = x[:33]
    for few in (5, 33):
        _check(q.matmul_input(wide[-few:, :64]), x[33 - few:33], q, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens", [1, 8, 20, 200])
def test_whole_numbers_come_back_whole(dev, dtype, tokens):
    """Codes and activations that are whole numbers, scales powers of two: every sum is exact in float32, whatever its order."""
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    for rows, cols, group in ((70, 300, 32), (512, 1024, 64), (200, 4096, 128), (129, 2056, 64)):
        w = torch.randint(-7, 8, (rows, cols), generator=gen, device=dev).float()
        w[:, ::32] = -8.0  # every group's scale is 1
        q = t81_torch.Q4Tensor.from_float(w, group=group)
        assert torch.equal(q.dequantize(), w)
        x = torch.randint(-4, 5, (tokens, cols), generator=gen, device=dev).to(dtype)
        assert torch.equal(q.matmul_input(x, out_dtype=torch.float32).double(), x.double() @ w.double().t())


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 40, 300])
def test_strided_and_unaligned_activations(dev, tokens):
    from t81lib_b200 import ops
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        for cols in (256, 250, 321):
            q, _, b = _case(gen, dev, 200, cols, 1, dtype, 64, True)
            wide = torch.full((tokens, cols + 24), float("nan"), device=dev, dtype=dtype)
            for skip in (0, 1, 3, 8):
                x = wide[:, skip:skip + cols]
                wide.fill_(float("nan"))
                x.copy_(torch.randn(tokens, cols, generator=gen, device=dev))
                _check(q.matmul_input(x, b), x, q, b)  # nothing beside the rows is used
            x = torch.randn(cols, tokens, generator=gen, device=dev).to(dtype).t()  # columns apart
            _check(q.matmul_input(x, b), x, q, b)
            x = torch._neg_view(torch.randn(tokens, cols, generator=gen, device=dev).to(dtype))
            _check(q.matmul_input(x, b), x, q, b)
            assert torch.equal(ops.linear_q4(q.codes, q.scales, 200, x, cols, 64), ops.linear_q4(q.codes, q.scales, 200, x.resolve_neg(), cols, 64))
            x = torch.randn(1, cols, generator=gen, device=dev).to(dtype).expand(tokens, cols)  # one row, many times
            _check(q.matmul_input(x, b), x, q, b)
            assert ops.linear_q4(q.codes, q.scales, 200, x.contiguous(), cols, 64).shape == (tokens, 200)


@pytest.mark.gpu
def test_tiny_and_huge_weights_in_every_type(dev):
    """Scales far outside fp16: the products keep them, whatever the activations' type."""
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(3)
    for factor in (2.0 ** -40, 2.0 ** -18, 1.0, 2.0 ** 20):
        w = torch.randn(256, 512, generator=gen, device=dev) * factor
        w[::2] *= 2.0 ** -12
        q = t81_torch.Q4Tensor.from_float(w, group=64)
        for dtype in (torch.bfloat16, torch.float16, torch.float32):
            for tokens in (2, 40, 256):
                x = torch.randn(tokens, 512, generator=gen, device=dev).to(dtype)
                _check(q.matmul_input(x, out_dtype=torch.float32), x, q, None)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 20, 200])
def test_infinities_and_nan_stay_in_their_rows(dev, tokens):
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        q, x, _ = _case(gen, dev, 100, 200, tokens, dtype, 32, False)
        clean = q.matmul_input(x)
        x[0, 7], x[tokens // 2, 199] = float("inf"), float("nan")
        y = q.matmul_input(x)
        hit = sorted({0, tokens // 2})
        assert not torch.isfinite(y[hit]).any()
        rest = [t for t in range(tokens) if t not in hit]
        assert torch.equal(y[rest], clean[rest])


@pytest.mark.gpu
def test_empty_products(dev):
    from t81lib_b200 import ops
    from t81lib_b200 import torch as t81_torch
    q = t81_torch.Q4Tensor.from_float(torch.randn(40, 64, device=dev), group=32)
    assert q.matmul_input(torch.zeros(0, 64, device=dev)).shape == (0, 40)
    none = t81_torch.Q4Tensor.from_float(torch.zeros(40, 0, device=dev), group=32)
    bias = torch.arange(40.0, device=dev)
    assert torch.equal(none.matmul_input(torch.zeros(3, 0, device=dev), bias), bias.expand(3, 40))
    assert ops.linear_q4(none.codes, none.scales, 40, torch.zeros(3, 0, device=dev), 0, 32).abs().sum() == 0


@pytest.mark.gpu
def test_gradients(dev):
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, x, b = _case(gen, dev, 60, 100, 5, torch.float32, 32, True)
    x.requires_grad_(True), b.requires_grad_(True)
    g = torch.randn(5, 60, generator=gen, device=dev)
    gx, gb = torch.autograd.grad(q.matmul_input(x, b), [x, b], g)
    # sums of 60 and 5 float32 products: at most that many roundings of the magnitudes
    assert bool(((gx.double() - g.double() @ q.dequantize().double()).abs() <= 62 * 2.0 ** -24 * (g.double().abs() @ q.dequantize().double().abs())).all())
    assert bool(((gb.double() - g.double().sum(0)).abs() <= 6 * 2.0 ** -24 * g.double().abs().sum(0)).all())


# ---- experts ----


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("counts,behind", [([3], 0), ([0, 0, 5], 2), ([1, 0, 9, 16, 0, 17, 1], 3), ([0, 0], 4), ([40, 0, 300, 7], 0), ([129, 64, 1, 255], 10), ([1] * 70, 1)])
def test_experts(dev, counts, behind, dtype):
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(len(counts) + behind)
    offsets = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    n = sum(counts) + behind
    for out_f, in_f, group, bias in ((48, 200, 32, True), (130, 256, 128, False), (300, 1000, 64, True)):
        w = torch.randn(len(counts), out_f, in_f, generator=gen, device=dev) * 0.02
        q = t81_torch.Q4Tensor.from_float(w, group=group)
        x = torch.randn(n, in_f, generator=gen, device=dev).to(dtype)
        x[sum(counts):] = float("nan")  # rows of no expert are not read into any result
        b = torch.randn(len(counts), out_f, generator=gen, device=dev) if bias else None
        y = q.matmul_sorted(x, offsets, b)
        values = q.dequantize()
        for e in range(len(counts)):
            lo, hi = int(offsets[e]), int(offsets[e + 1])
            one = t81_torch.Q4Tensor.from_float(w[e], group=group)
            assert torch.equal(one.dequantize(), values[e])
            if hi > lo:
                _check(y[lo:hi], x[lo:hi], one, None if b is None else b[e])
        assert y.shape == (n, out_f) and not y[sum(counts):].any()


@pytest.mark.gpu
@pytest.mark.parametrize("experts,most,rows,cols", [(100, 600, 300, 512), (33, 2000, 520, 256), (1024, 90, 264, 192), (7, 3000, 2000, 320), (64, 40, 1400, 1024)])
def test_experts_of_many_sizes(dev, experts, most, rows, cols):
    """Tiles of every width, in more rounds than one, experts without rows among them."""
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(experts)
    counts = (torch.rand(experts, generator=gen, device=dev) * most).int()
    counts[torch.rand(experts, generator=gen, device=dev) < 0.2] = 0
    counts[experts // 2] = most
    offsets = torch.cat([torch.zeros(1, dtype=torch.int32, device=dev), counts.cumsum(0).int()])
    total = int(offsets[-1])
    q = t81_torch.Q4Tensor.from_float(torch.randn(experts, rows, cols, generator=gen, device=dev) * 0.02, group=64)
    bias = torch.randn(experts, rows, generator=gen, device=dev) * 0.1
    values = q.dequantize().double()
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = torch.randn(total + 5, cols, generator=gen, device=dev).to(dtype)
        y = q.matmul_sorted(x, offsets, bias)
        assert bool((y[total:] == 0).all())
        at = offsets.tolist()
        for e in range(experts):
            lo, hi = at[e], at[e + 1]
            want, magnitude = ref.product(x[lo:hi], values[e], bias[e])
            off = (y[lo:hi].double() - want).abs()
            assert bool((off <= ref.tolerance(magnitude + bias[e].double().abs(), want, cols, dtype)).all()), e


@pytest.mark.gpu
def test_experts_refusals_and_bad_offsets(dev):
    from t81lib_b200 import torch as t81_torch
    q = t81_torch.Q4Tensor.from_float(torch.randn(3, 32, 64, device=dev), group=32)
    x = torch.randn(10, 64, device=dev)
    with pytest.raises(ValueError, match="one entry more"):
        q.matmul_sorted(x, torch.zeros(3, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError, match="int32"):
        q.matmul_sorted(x, torch.zeros(4, dtype=torch.int64, device=dev))
    with pytest.raises(ValueError, match="width"):
        q.matmul_sorted(x[:, :60], torch.zeros(4, dtype=torch.int32, device=dev))
    with pytest.raises(NotImplementedError, match="no_grad"):
        q.matmul_sorted(x.requires_grad_(True), torch.zeros(4, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError, match="one matrix"):
        q.matmul_input(x.detach())


@pytest.mark.gpu
def test_products_on_other_streams_and_captured(dev):
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(9)
    q, x, b = _case(gen, dev, 512, 777, 40, torch.bfloat16, 64, True)  # rows that are staged: a workspace per call
    small = x[:3].clone()
    want, want_small = q.matmul_input(x, b), q.matmul_input(small, b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for s in streams * 4:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            results.append(q.matmul_input(x, b))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results)
    graphs = []
    with torch.cuda.stream(streams[0]):
        for source in (x, small):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=streams[0]):
                graphs.append((g, q.matmul_input(source, b)))
    torch.cuda.synchronize()
    for (g, _), s in zip(graphs, streams):  # both at once
        with torch.cuda.stream(s):
            for _ in range(3):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want_small)
    x.normal_(generator=gen)
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1], q.matmul_input(x, b))
