"""(token, slot) pairs sorted by expert and back: whole numbers exactly, rows and gradients against 64 bits and against differences."""

import os
import subprocess
import sys

import pytest
import torch

import _q4_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(lib_built):
    from t81lib_b200 import _capi
    assert _capi.device_available(), _capi.last_error()
    yield torch.device("cuda", 0)
    assert _capi.kernel_status(reset=True) == 0  # no bounded wait of a kernel ran out


@pytest.mark.parametrize("tokens,top,experts", [(1, 1, 1), (1, 6, 64), (16, 6, 64), (33, 1, 3), (100, 8, 8), (512, 2, 60), (513, 2, 1024), (1500, 4, 100), (3000, 7, 33), (40, 3, 1024)])
@pytest.mark.parametrize("id_type", [torch.int64, torch.int32])
def test_sort(dev, tokens, top, experts, id_type):
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator().manual_seed(tokens + experts)
    for kind in range(4):
        ids = torch.randint(0, experts, (tokens, top), generator=gen)
        if kind == 1:
            ids = torch.randint(-2, experts + 3, (tokens, top), generator=gen)  # some of no expert
        elif kind == 2:
            ids.fill_(experts - 1)
        elif kind == 3:
            ids.fill_(-1)
        r = t81_torch.route(ids.to(id_type).to(dev), experts)
        for got, want in zip((r.order, r.position, r.offsets), ref.route(ids, experts)):
            assert got.dtype == torch.int32 and torch.equal(got.cpu(), want), kind


def test_sort_of_many_pairs(dev):
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(0)
    for n, experts in ((400_000, 64), (1_000_003, 7)):
        ids = torch.randint(-1, experts, (n, 1), generator=gen, device=dev)
        r = t81_torch.route(ids, experts)
        key, order = torch.sort(torch.where(ids.flatten() < 0, experts, ids.flatten()), stable=True)
        kept = int((key < experts).sum())
        assert torch.equal(r.order[:kept].long(), order[:kept]) and bool((r.order[kept:] == -1).all())
        assert torch.equal(r.offsets.long(), torch.searchsorted(key, torch.arange(experts + 1, device=dev)))
        assert torch.equal(r.position.flatten()[order[:kept]].long(), torch.arange(kept, device=dev))


def test_no_tokens(dev):
    from t81lib_b200 import torch as t81_torch
    r = t81_torch.route(torch.zeros(0, 4, dtype=torch.int64, device=dev), 5)
    assert r.order.numel() == 0 and r.offsets.tolist() == [0] * 6
    x = torch.zeros(0, 8, device=dev, requires_grad=True)
    rows = r.gather(x)
    y = r.combine(rows, torch.zeros(0, 4, device=dev))
    assert rows.shape == (0, 8) and y.shape == (0, 8)
    y.sum().backward()
    assert x.grad.shape == (0, 8)


def _routing(dev, tokens, top, experts, seed, dropped=True):
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(-1 if dropped else 0, experts, (tokens, top), generator=gen, device=dev)
    if dropped:
        ids[tokens // 2] = -1  # a token of padding
    return gen, t81_torch.route(ids, experts)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("w_dtype", [torch.float32, torch.bfloat16, None])
@pytest.mark.parametrize("tokens,top,experts,width", [(1, 1, 1, 1), (7, 3, 4, 8), (33, 2, 8, 1537), (64, 8, 16, 2048), (5, 1, 9, 4100), (20, 6, 64, 36), (300, 4, 32, 515)])
def test_gather_combine_and_gradients(dev, tokens, top, experts, width, dtype, w_dtype):
    gen, r = _routing(dev, tokens, top, experts, tokens + width)
    n, kept = tokens * top, int(r.offsets[-1])
    new = lambda *s: torch.randn(*s, generator=gen, device=dev).to(dtype)  # noqa: E731
    x, out, g_rows, g_y = new(tokens, width).requires_grad_(True), new(n, width).requires_grad_(True), new(n, width), new(tokens, width)
    w = None if w_dtype is None else torch.rand(tokens, top, generator=gen, device=dev).to(w_dtype).requires_grad_(True)
    with torch.no_grad():
        out[kept:] = float("nan")      # rows of no expert, their gradients and the weights of such slots are not read
        g_rows[kept:] = float("nan")
        if w is not None:
            w[r.position < 0] = float("nan")
    rows, y = r.gather(x), r.combine(out, w)
    grads = torch.autograd.grad([rows, y], [x, out] + ([] if w is None else [w]), [g_rows, g_y])
    kept_slots, at = r.position >= 0, r.position.clamp(min=0).long()
    token = r.order[:kept].long() // top
    assert torch.equal(rows[:kept], x[token]) and not rows[kept:].any()
    W = torch.ones(tokens, top, device=dev, dtype=torch.float64) if w is None else w.detach().double()
    W = torch.where(kept_slots, W, 0.0)
    slots = torch.where(kept_slots[..., None], out.detach().double()[at], 0.0)
    half = torch.finfo(dtype).eps / 2

    def close(got, want, magnitude, terms, step):
        # a rounding per term and product in float32, then one to the result's type
        assert bool(((got.double() - want).abs() <= (terms + 1) * 2.0 ** -24 * magnitude + step * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -24 * torch.finfo(got.dtype).smallest_normal * 2.0 ** 14).all())
    close(y, (slots * W[..., None]).sum(1), (slots.abs() * W[..., None]).sum(1), top, half)
    shares = torch.where(kept_slots[..., None], g_rows.double()[at], 0.0)
    close(grads[0], shares.sum(1), shares.abs().sum(1), top, half)
    want = torch.zeros(n, width, device=dev, dtype=torch.float64)
    want[:kept] = g_y.double()[token] * W.flatten()[r.order[:kept].long()][:, None]
    close(grads[1], want, want.abs(), 1, half)
    assert not grads[1][kept:].any()
    if w is not None:
        terms = slots * g_y.double()[:, None]
        close(grads[2], terms.sum(-1), terms.abs().sum(-1), width, torch.finfo(w_dtype).eps / 2)
        assert grads[2].dtype == w_dtype and not grads[2][~kept_slots].any()


def test_gradients_against_differences(dev):
    """float32 throughout: both maps are linear, so a difference is their gradient up to its rounding."""
    gen, r = _routing(dev, 6, 3, 4, 1)
    x, w = torch.randn(6, 12, generator=gen, device=dev, requires_grad=True), torch.rand(6, 3, generator=gen, device=dev, requires_grad=True)
    g = torch.randn(6, 12, generator=gen, device=dev)
    f = lambda x, w: (r.combine(r.gather(x) * 2.0, w).double() * g.double()).sum()  # noqa: E731
    gx, gw = torch.autograd.grad(f(x, w), [x, w])
    for _ in range(4):
        dx, dw = torch.randn(6, 12, generator=gen, device=dev), torch.randn(6, 3, generator=gen, device=dev)
        with torch.no_grad():
            # differences of step 1/2 in one argument at a time: no curvature, values below 100 in float32 sums of 3 terms
            assert abs(float(f(x + 0.5 * dx, w) - f(x - 0.5 * dx, w) - (gx.double() * dx.double()).sum())) < 72 * 100 * 2.0 ** -23
            assert abs(float(f(x, w + 0.5 * dw) - f(x, w - 0.5 * dw) - (gw.double() * dw.double()).sum())) < 72 * 100 * 2.0 ** -23


def test_second_gradients(dev):
    gen, r = _routing(dev, 5, 2, 3, 2)
    x = torch.randn(5, 4, generator=gen, device=dev, requires_grad=True)
    w = torch.rand(5, 2, generator=gen, device=dev, requires_grad=True)
    kept, at = r.position >= 0, r.position.clamp(min=0).long()

    def plain(x, w):
        rows = torch.zeros(10, 4, device=dev).index_put((r.position[kept].long(),), x[:, None].expand(5, 2, 4)[kept])
        return (torch.where(kept[..., None], torch.tanh(rows)[at], 0.0) * w[..., None]).sum(1)
    results = []
    for f in (lambda x, w: r.combine(torch.tanh(r.gather(x)), w), plain):
        gx, gw = torch.autograd.grad((f(x, w) ** 2).sum(), [x, w], create_graph=True)
        results.append(torch.autograd.grad((gx ** 2).sum() + (gw ** 3).sum(), [x, w]))
    for a, b in zip(*results):  # the same sums of a few float32 terms in another order
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5 * float(b.abs().max()))


def test_strided_rows_and_broadcast_gradients(dev):
    gen, r = _routing(dev, 9, 2, 4, 3)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(9, 100, generator=gen, device=dev).to(dtype)
        for x in (wide[:, 1:70], wide[:, 8:72], wide[:, ::2], wide[:1].expand(9, 100), wide.t().contiguous().t()):
            x = x.detach().requires_grad_(True)
            rows = r.gather(x)
            kept = int(r.offsets[-1])
            assert torch.equal(rows[:kept], x[r.order[:kept].long() // 2])
            y = r.combine(rows)
            (g,) = torch.autograd.grad(y.sum(), [x])  # a gradient of one value, broadcast
            slots = (r.position >= 0).sum(1, keepdim=True)
            assert torch.equal(g, slots.to(dtype).expand(x.shape))


def test_refusals(dev):
    from t81lib_b200 import _capi
    from t81lib_b200 import torch as t81_torch
    ids = torch.zeros(4, 2, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError, match="int64 or int32"):
        t81_torch.route(ids.float(), 3)
    with pytest.raises(ValueError, match="tokens, slots"):
        t81_torch.route(ids.flatten(), 3)
    with pytest.raises(ValueError, match="CUDA"):
        t81_torch.route(ids.cpu(), 3)
    with pytest.raises(ValueError, match="positive"):
        t81_torch.route(ids, 0)
    with pytest.raises(_capi.LimitError, match="1024 experts"):
        t81_torch.route(ids, 1025)
    r = t81_torch.route(ids, 3)
    for bad in (torch.zeros(3, 8, device=dev), torch.zeros(4, 8, device=dev, dtype=torch.float64), torch.zeros(4, device=dev), torch.zeros(4, 8)):
        with pytest.raises(ValueError):
            r.gather(bad)
    rows = torch.zeros(8, 8, device=dev)
    for bad in (torch.zeros(4, 3, device=dev), torch.zeros(4, 2), torch.zeros(4, 2, device=dev, dtype=torch.float64)):
        with pytest.raises(ValueError, match="weights"):
            r.combine(rows, bad)
    with pytest.raises(ValueError, match="one row per"):
        r.combine(rows[:7], torch.zeros(4, 2, device=dev))


def test_captured_step(dev):
    """Forward and backward inside a graph, with eager results of the same leaves alive that were made on its stream, replayed on new inputs."""
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(4)
    ids = torch.randint(-1, 8, (50, 2), generator=gen, device=dev)
    x = torch.randn(50, 64, generator=gen, device=dev, requires_grad=True)
    w = torch.rand(50, 2, generator=gen, device=dev, requires_grad=True)
    g = torch.randn(50, 64, generator=gen, device=dev)

    def step():
        r = t81_torch.route(ids, 8)
        y = r.combine(r.gather(x), w)
        return [y, *torch.autograd.grad(y, [x, w], g)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        alive = step()[0]
        with torch.cuda.graph(graph, stream=side):
            captured = step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad():
        ids.copy_(torch.randint(-1, 8, (50, 2), generator=gen, device=dev))
        x.normal_(generator=gen)
    graph.replay()
    torch.cuda.synchronize()
    del alive
    for a, b in zip(captured, step()):
        assert torch.equal(a, b)


_CHILD = """
import torch
from t81lib_b200 import torch as t81_torch
x = torch.randn(50, 64, device="cuda", requires_grad=True)
r = t81_torch.route(torch.randint(0, 8, (50, 2), device="cuda"), 8)
alive = r.combine(r.gather(x))
torch.cuda.synchronize()
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        torch.autograd.grad(r.combine(r.gather(x)).sum(), x)
except RuntimeError as e:
    print("refused", type(e).__name__)
else:
    print("captured")
"""


def test_capture_beside_an_eager_graph_of_the_default_stream(lib_built):
    """The leaf's gradient node belongs to the default stream there, which torch's engine then joins to the capture: CUDA refuses that, whatever
    the operations between are.  It must be an exception, not the end of the process."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", _CHILD], capture_output=True, text=True, timeout=300, cwd=root)
    assert res.returncode == 0 and ("refused" in res.stdout or "captured" in res.stdout), res.stdout + res.stderr


def test_saved_tensors_that_come_back_otherwise_and_batched_gradients(dev):
    gen, r = _routing(dev, 12, 3, 4, 5)
    x = torch.randn(12, 8, generator=gen, device=dev, requires_grad=True)
    w = torch.rand(12, 3, generator=gen, device=dev, requires_grad=True)
    v = torch.randn(4, 12, 8, generator=gen, device=dev)
    y = r.combine(r.gather(x), w)
    want = [torch.autograd.grad(y, [x, w], v[i], retain_graph=True) for i in range(4)]
    for got, one in zip(torch.autograd.grad(y, [x, w], v, retain_graph=True, is_grads_batched=True), zip(*want)):
        assert torch.allclose(got, torch.stack(one), rtol=1e-5, atol=1e-5)  # sums of at most 8 float32 terms in another order
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.t().contiguous() if t.ndim == 2 else t, lambda t: t.t() if t.ndim == 2 else t):
        y = r.combine(r.gather(x), w)
    for got, one in zip(torch.autograd.grad(y, [x, w], v[0]), want[0]):
        assert torch.equal(got, one)
    with torch.autograd.graph.save_on_cpu():
        y = r.combine(r.gather(x), w)
    for got, one in zip(torch.autograd.grad(y, [x, w], v[0]), want[0]):
        assert torch.equal(got, one)
    for wrong in (lambda t: t.cpu(), lambda t: t.double() if t.is_floating_point() else t.long(), lambda t: t[:-1]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, wrong):
            y = r.combine(r.gather(x), w)
        with pytest.raises(ValueError):
            torch.autograd.grad(y, [x, w], v[0])


def test_more_elements_than_31_bits_count(dev):
    from t81lib_b200 import torch as t81_torch
    gen = torch.Generator(device="cuda").manual_seed(5)
    tokens, top, width = 70000, 4, 8192  # 2.3e9 elements in the sorted rows
    ids = torch.randint(0, 9, (tokens, top), generator=gen, device=dev)  # expert 8 takes no part
    routing = t81_torch.route(ids, 8)
    x = torch.randn(tokens, width, generator=gen, device=dev).to(torch.bfloat16)
    rows = routing.gather(x)
    kept = int(routing.offsets[-1])
    some = torch.arange(kept - 100, kept, device=dev)
    assert torch.equal(rows[kept - 100:kept], x[routing.order[some].long() // top]) and bool((rows[-100:] == 0).all())
    weights = torch.rand(tokens, top, generator=gen, device=dev)
    at = torch.arange(tokens - 64, tokens, device=dev)
    share = torch.where(routing.position[at] >= 0, weights[at], torch.zeros_like(weights[at])).double().sum(1, keepdim=True)
    y = routing.combine(rows, weights)
    want = share * x[at].double()  # four roundings of fp32 and one of bf16
    assert bool(((y[at].double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -20)).all())
    rows.requires_grad_(True)
    weights.requires_grad_(True)
    g = torch.randn(tokens, width, generator=gen, device=dev).to(torch.bfloat16)
    grad_rows, grad_weights = torch.autograd.grad(routing.combine(rows, weights), (rows, weights), g)
    pair = routing.order[some].long()
    want = weights.detach().flatten()[pair].double().unsqueeze(1) * g[pair // top].double()
    assert bool(((grad_rows[kept - 100:kept].double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -20)).all()) and bool((grad_rows[-100:] == 0).all())
    dots = (g[at].double() * x[at].double()).sum(1, keepdim=True) * (routing.position[at] >= 0)
    magnitude = (g[at].double() * x[at].double()).abs().sum(1, keepdim=True)
    assert bool(((grad_weights[at].double() - dots).abs() <= magnitude * (width / 32 + 6) * 2.0 ** -24).all())
