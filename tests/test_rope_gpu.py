"""cmpext3.ops.rope on a B200 against its 64-bit definition: types, pair layouts, sections, position types and
shapes, far positions, odd sizes and strides, the gradient, and use in graphs and on other streams."""
from __future__ import annotations

import pytest
import torch

import cmpext3
from cmpext3 import _native as N
from tests import serving_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def _freqs(pairs):
    return (10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float()


def _check(x, positions, freqs, sections=None, interleaved=False, dev=torch.device("cuda", 0), what="rope"):
    y = cmpext3.ops.rope(x if x.is_cuda else x.to(dev), positions.to(dev), freqs.to(dev), sections, interleaved)
    torch.cuda.synchronize()
    want, bound = O.rope(x.cpu(), positions.cpu(), freqs, sections, interleaved)
    O.assert_within(y, want, bound, what)
    assert y.dtype == x.dtype
    return y


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape,pairs", [
    ((1, 1, 1, 2), 1), ((2, 3, 5, 64), 32), ((1, 10, 77, 64), 32), ((2, 8, 33, 40), 20), ((1, 4, 9, 40), 10),
    ((1, 5, 17, 128), 64), ((3, 2, 7, 96), 16), ((1, 2, 300, 256), 128), ((1, 33, 4, 80), 40), ((2, 2, 3, 7), 3),
    ((1, 2, 5, 255), 1), ((2, 40, 1000, 128), 64)])
def test_matches_the_definition(cuda_device, dtype, interleaved, shape, pairs):
    g = torch.Generator().manual_seed(sum(shape) + pairs)
    x = torch.randn(shape, generator=g).to(dtype)
    positions = torch.randint(0, 5000, (shape[0], shape[2]), generator=g, dtype=torch.int32)
    _check(x, positions, _freqs(pairs), None, interleaved)
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("sections", [(32,), (10, 22), (8, 12, 12), (8, 8, 8, 8), (0, 32, 0), (31, 0, 1)])
def test_sections(cuda_device, dtype, sections):
    g = torch.Generator().manual_seed(len(sections))
    x = torch.randn(2, 3, 50, 72, generator=g).to(dtype)
    positions = torch.randint(-40, 4000, (len(sections), 2, 50), generator=g, dtype=torch.int32)
    for interleaved in (False, True):
        _check(x, positions, _freqs(32), sections, interleaved)
    _check(x, positions[:, 0], _freqs(32), sections)       # [axes, tokens]
    _check(x, positions[:, :1], _freqs(32), sections)      # one batch row for all


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_position_types_and_layouts(cuda_device, kind):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 2, 40, 64, generator=g)
    base = torch.randint(-3000, 3000, (3, 40), generator=g)
    positions = base.to(kind) / 4 if kind == torch.float32 else base.to(kind)
    for p in (positions, positions[0], positions[:1], positions.t().contiguous().t()):
        _check(x, p, _freqs(32))
    wide = torch.zeros(3, 80, dtype=kind)
    wide[:, ::2] = positions
    _check(x.to(cuda_device), wide.to(cuda_device)[:, ::2], _freqs(32))


def test_far_positions_keep_their_precision(cuda_device):
    x = torch.randn(1, 2, 6, 64, generator=torch.Generator().manual_seed(4))
    positions = torch.tensor([0, 1, 10 ** 6, 2 ** 31 - 1, 123456789, -(2 ** 31)], dtype=torch.int32)
    _check(x, positions, _freqs(32))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_strided_views(cuda_device, dtype):
    g = torch.Generator().manual_seed(5)
    positions = torch.randint(0, 900, (2, 30), generator=g, dtype=torch.int32)
    base = torch.randn(2, 30, 6, 64, generator=g).to(dtype).to(cuda_device)
    y = _check(base.transpose(1, 2), positions, _freqs(32))           # [B, L, H, D] memory
    assert y.stride() == base.transpose(1, 2).stride()
    fused = torch.randn(2, 30, 3 * 6 * 64 + 3, generator=g).to(dtype).to(cuda_device)
    odd = fused[..., 1:1 + 6 * 64].unflatten(-1, (6, 64)).transpose(1, 2)   # rows on odd boundaries
    _check(odd, positions, _freqs(32))
    _check(base.transpose(2, 3).contiguous().transpose(2, 3).transpose(1, 2), positions, _freqs(32))  # head_dim strided
    _check(base[:, :, :1].expand(2, 30, 6, 64).transpose(1, 2), positions, _freqs(32))                # one head for all


def test_empty_input(cuda_device):
    p = torch.zeros(0, dtype=torch.int32, device=cuda_device)
    y = cmpext3.ops.rope(torch.empty(2, 3, 0, 64, device=cuda_device), p, _freqs(32).to(cuda_device))
    assert y.shape == (2, 3, 0, 64)
    p = torch.zeros(5, dtype=torch.int32, device=cuda_device)
    assert cmpext3.ops.rope(torch.empty(0, 3, 5, 64, device=cuda_device), p, _freqs(32).to(cuda_device)).shape == (0, 3, 5, 64)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_is_the_rotation_back(cuda_device, dtype, interleaved):
    g = torch.Generator().manual_seed(6)
    x, gy = torch.randn(2, 3, 21, 40, generator=g).to(dtype), torch.randn(2, 3, 21, 40, generator=g).to(dtype)
    positions = torch.randint(0, 300, (2, 2, 21), generator=g, dtype=torch.int64)
    leaf = x.to(cuda_device).requires_grad_()
    y = cmpext3.ops.rope(leaf, positions.to(cuda_device), _freqs(16).to(cuda_device), (6, 10), interleaved)
    (grad,) = torch.autograd.grad(y, leaf, gy.to(cuda_device))
    want, bound = O.rope(gy, positions, _freqs(16), (6, 10), interleaved, sign=-1.0)
    O.assert_within(grad, want, bound, "gradient")


def test_gradient_against_differences(cuda_device):
    # the operator is linear: <gy, R(x + h) - R(x - h)> / 2 = <gx, h> up to fp32 sums
    g = torch.Generator().manual_seed(7)
    x, h, gy = (torch.randn(1, 2, 9, 24, generator=g).to(cuda_device) for _ in range(3))
    positions = torch.arange(9, device=cuda_device)
    freqs = _freqs(8).to(cuda_device)
    leaf = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(cmpext3.ops.rope(leaf, positions, freqs), leaf, gy)
    up, down = (cmpext3.ops.rope(x + s * h, positions, freqs).double() for s in (1, -1))
    left, right = (gy.double() * (up - down) / 2).sum(), (gx.double() * h.double()).sum()
    # each of 432 products is off by a few 2^-24 of at most |gy| (|x| + |h|)
    size = (gy.abs().double() * (x.abs() + h.abs() + 1)).sum()
    assert (left - right).abs() <= 8 * 2.0 ** -22 * size


def test_broadcast_gradient_and_second_gradient(cuda_device):
    g = torch.Generator().manual_seed(8)
    x = torch.randn(1, 2, 9, 24, generator=g).to(cuda_device).requires_grad_()
    positions, freqs = torch.arange(9, device=cuda_device), _freqs(12).to(cuda_device)
    y = cmpext3.ops.rope(x.expand(3, 2, 9, 24), positions, freqs)
    (gx,) = torch.autograd.grad(y.sum(), x)                       # an expanded gradient, summed over the batch
    want, bound = O.rope(torch.ones(1, 2, 9, 24), positions.cpu(), freqs.cpu(), sign=-1.0)
    O.assert_within(gx, 3 * want, 3 * bound + 3 * 2.0 ** -23 * want.abs(), "broadcast gradient")
    gy = torch.randn(1, 2, 9, 24, generator=g).to(cuda_device).requires_grad_()
    (gx,) = torch.autograd.grad(cmpext3.ops.rope(x, positions, freqs), x, gy, create_graph=True)
    (ggy,) = torch.autograd.grad(gx, gy, x.detach())              # d<gx, x>/d gy = R x
    want, bound = O.rope(x.detach().cpu(), positions.cpu(), freqs.cpu())
    O.assert_within(ggy, want, bound, "second gradient")


def test_positions_changed_before_the_backward_pass_are_reported(cuda_device):
    x = torch.randn(1, 1, 4, 8, device=cuda_device, requires_grad=True)
    positions, freqs = torch.arange(4, device=cuda_device), _freqs(4).to(cuda_device)
    y = cmpext3.ops.rope(x, positions, freqs)
    positions.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_in_a_graph_with_its_gradient(cuda_device):
    g = torch.Generator().manual_seed(9)
    x = torch.randn(2, 4, 64, 64, generator=g).to(torch.bfloat16).to(cuda_device)
    gy = torch.randn(2, 4, 64, 64, generator=g).to(torch.bfloat16).to(cuda_device)
    positions, freqs = torch.arange(64, dtype=torch.int32, device=cuda_device), _freqs(32).to(cuda_device)

    def step():
        leaf = x.detach().requires_grad_()
        y = cmpext3.ops.rope(leaf, positions, freqs)
        return y.detach(), torch.autograd.grad(y, leaf, gy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for shift in (0, 1000):
        positions.copy_(torch.arange(64, dtype=torch.int32) + shift)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_on_another_stream(cuda_device):
    x = torch.randn(1, 2, 100, 64, generator=torch.Generator().manual_seed(10))
    positions, freqs = torch.arange(100), _freqs(32)
    xd, pd, fd = x.to(cuda_device), positions.to(cuda_device), freqs.to(cuda_device)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = cmpext3.ops.rope(xd, pd, fd)
    s.synchronize()
    O.assert_within(y, *O.rope(x, positions, freqs), "side stream")


def test_a_capture_of_a_leaf_with_an_eager_graph_is_refused(cuda_device):
    x = torch.randn(1, 1, 8, 16, device=cuda_device, requires_grad=True)
    positions, freqs = torch.arange(8, device=cuda_device), _freqs(8).to(cuda_device)
    eager = cmpext3.ops.rope(x, positions, freqs)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph of this leaf"):
        with torch.cuda.graph(graph):
            cmpext3.ops.rope(x, positions, freqs)
    del eager
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):      # a warm-up, whose graph stays alive
        warm = cmpext3.ops.rope(x, positions, freqs)
        torch.autograd.grad(warm.sum(), x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cmpext3.ops.rope(x, positions, freqs)
        (grad,) = torch.autograd.grad(y.sum(), x)
    graph.replay()
    torch.cuda.synchronize()
    O.assert_within(grad, *O.rope(torch.ones(1, 1, 8, 16), positions.cpu(), freqs.cpu(), sign=-1.0), "captured gradient")
