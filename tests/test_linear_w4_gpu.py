"""cmpext3.ops.linear_w4 on a B200 against its 64-bit definition: types, groups, token counts, odd rows,
zero points, layouts, special values, graphs."""
from __future__ import annotations

import pytest
import torch

import cmpext3
from cmpext3 import _native as N
from tests import serving_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def _make(dtype, m, n, k, group, zeros, bias, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g).to(dtype)
    w = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    s = (torch.rand(n, k // group, generator=g) * 0.02 - 0.005).to(dtype)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    b = torch.randn(n, generator=g).to(dtype) if bias else None
    return x, w, s, z, b


def _check(args, dev, what):
    y = cmpext3.ops.linear_w4(*(None if t is None else t.to(dev) for t in args))
    torch.cuda.synchronize()
    O.assert_within(y, *O.linear_w4(*args), what)
    return y


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("zeros,bias", [(False, False), (True, True)])
@pytest.mark.parametrize("m,n,k,group", [
    (1, 1, 32, 32), (1, 16, 64, 64), (1, 17, 96, 32), (1, 512, 4096, 128), (2, 33, 160, 32), (3, 100, 192, 96),
    (4, 1000, 640, 64), (5, 7, 8192, 128), (7, 129, 1024, 256), (8, 64, 512, 512), (9, 40, 256, 64), (16, 130, 2560, 128),
    (17, 24, 384, 128), (33, 65, 96, 96), (70, 31, 128, 64), (1, 1, 16384, 64), (2, 4096, 64, 32), (1, 300, 1056, 1056)])
def test_matches_the_definition(cuda_device, dtype, zeros, bias, m, n, k, group):
    _check(_make(dtype, m, n, k, group, zeros, bias, m + n + k), cuda_device, f"{m}x{n}x{k} group {group}")
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_every_token_count(cuda_device, dtype):
    for m in range(1, 35):
        _check(_make(dtype, m, 48, 256, 64, True, False, m), cuda_device, f"{m} tokens")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_every_code_and_zero_point(cuda_device, dtype):
    # one weight a row: row 16 z + c has code c against zero point z at k = 5, and zero elsewhere
    k = 32
    codes = torch.arange(16).repeat(16)
    zeros = torch.arange(16).repeat_interleave(16)
    grid = zeros[:, None].repeat(1, k)
    grid[:, 5] = codes
    w = (grid[:, 0::2] | (grid[:, 1::2] << 4)).to(torch.uint8)
    x = torch.full((1, k), 3.0, dtype=dtype)
    y = cmpext3.ops.linear_w4(x.to(cuda_device), w.to(cuda_device), torch.ones(256, 1, dtype=dtype, device=cuda_device),
                              zeros[:, None].to(torch.uint8).to(cuda_device))
    assert torch.equal(y[0].cpu().double(), 3.0 * (codes - zeros).double())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_where_each_weight_goes(cuda_device, dtype):
    # x is one at a single k: the output is that column of W
    k, n = 256, 40
    g = torch.Generator().manual_seed(1)
    w = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    codes = torch.stack((w & 15, w >> 4), -1).reshape(n, k)
    y = cmpext3.ops.linear_w4(torch.eye(k, dtype=dtype, device=cuda_device), w.to(cuda_device),
                              torch.ones(n, k // 32, dtype=dtype, device=cuda_device))
    assert torch.equal(y.cpu().double(), codes.t().double() - 8)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layouts(cuda_device, dtype):
    x, w, s, z, b = _make(dtype, 6, 50, 256, 64, True, True, 2)
    want = cmpext3.ops.linear_w4(*(t.to(cuda_device) for t in (x, w, s, z, b)))
    wide = torch.zeros(6, 300, dtype=dtype, device=cuda_device)
    wide[:, 3:259] = x
    wd = torch.zeros(50, 150, dtype=torch.uint8, device=cuda_device)
    wd[:, 5:133] = w
    sd = s.t().contiguous().to(cuda_device).t()
    zd = torch.zeros(50, 9, dtype=torch.uint8, device=cuda_device)
    zd[:, 1:5] = z
    bd = torch.zeros(100, dtype=dtype, device=cuda_device)
    bd[::2] = b
    assert torch.equal(cmpext3.ops.linear_w4(wide[:, 3:259], wd[:, 5:133], sd, zd[:, 1:5], bd[::2]), want)
    three = cmpext3.ops.linear_w4(x.view(2, 3, 256).to(cuda_device), *(t.to(cuda_device) for t in (w, s, z, b)))
    assert three.shape == (2, 3, 50) and torch.equal(three.view(6, 50), want)
    one = cmpext3.ops.linear_w4(x[0].to(cuda_device), *(t.to(cuda_device) for t in (w, s, z, b)))
    assert one.shape == (50,)
    assert cmpext3.ops.linear_w4(x[:0].to(cuda_device), *(t.to(cuda_device) for t in (w, s, z, b))).shape == (0, 50)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_a_token_does_not_depend_on_its_neighbours(cuda_device, dtype):
    x, w, s, z, b = (t.to(cuda_device) for t in _make(dtype, 8, 70, 512, 128, True, True, 3))
    x[3, 100], x[5, 7] = float("nan"), float("inf")
    y = cmpext3.ops.linear_w4(x, w, s, z, b)
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[5]).any()
    keep = [0, 1, 2, 4, 6, 7]
    assert torch.isfinite(y[keep]).all()
    x[3, 100], x[5, 7] = 0.0, 0.0
    assert torch.equal(cmpext3.ops.linear_w4(x, w, s, z, b)[keep], y[keep])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_large_and_small_values(cuda_device, dtype):
    x, w, s, z, _ = _make(dtype, 2, 64, 256, 64, True, False, 4)
    top = torch.finfo(dtype).max / 2048 if dtype == torch.float16 else 1e30
    _check(((x.float() * (top / 4)).to(dtype), w, (s.float() * 0.05).to(dtype), z, None), cuda_device, "large")
    low = 1e-4 if dtype == torch.float16 else 1e-30
    _check(((x.float() * low).to(dtype), w, s, z, None), cuda_device, "small")


def test_in_a_graph(cuda_device):
    x, w, s, z, b = (t.to(cuda_device) for t in _make(torch.bfloat16, 4, 300, 1024, 128, True, True, 5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cmpext3.ops.linear_w4(x, w, s, z, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cmpext3.ops.linear_w4(x, w, s, z, b)
    for _ in range(3):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, cmpext3.ops.linear_w4(x, w, s, z, b))
