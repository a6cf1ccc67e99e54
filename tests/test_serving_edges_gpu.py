"""Calls of the serving operators at the edges of what they take (needs a B200; marked gpu): special values, views with
odd strides, far positions, kept signatures that meet other pointers."""
from __future__ import annotations

import pytest
import torch

import cmpext3
from cmpext3 import _native as N
from tests.test_paged_attention_gpu import DTYPES, IDS

pytestmark = pytest.mark.gpu

SCHEDULES = [(40, "one CTA"), (3000, "cluster"), (9500, "equal shares")]


def _cache(n, heads_kv, dim, dtype, dev, page=16):
    """Caches of one sequence of n tokens (zeros) whose pages lie in order, its page table and its length."""
    pages = -(-n // page)
    k, v = (torch.zeros(pages, heads_kv, page, dim, dtype=dtype, device=dev) for _ in range(2))
    return (k, v, torch.arange(pages, dtype=torch.int32, device=dev)[None], torch.tensor([n], dtype=torch.int32, device=dev))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,schedule", SCHEDULES)
@pytest.mark.parametrize("gap", [20, 40, 80])
def test_an_infinite_value_stays_infinite_under_a_small_weight(cuda_device, dtype, n, schedule, gap):
    # one key's score is `gap` above all the others', whose weights, exp(-gap), are above 2^-126 of the largest
    k, v, table, length = _cache(n, 1, 64, dtype, cuda_device)
    q = torch.zeros(1, 2, 1, 64, dtype=dtype, device=cuda_device)
    q[..., 0] = 8.0
    v.fill_(1.0)
    for top, at in ((0, n - 1), (n - 1, 0), (n // 2, n // 2 + 1)):
        k.zero_()
        k[top // 16, 0, top % 16, 0] = gap
        v[at // 16, 0, at % 16, 3], v[at // 16, 0, at % 16, 6] = float("inf"), -float("inf")
        assert schedule in N.paged_attention_plan(q, k, v, table, length)
        out = cmpext3.ops.paged_attention(q, k, v, table, length)[0, :, 0].cpu()
        v[at // 16, 0, at % 16] = 1.0
        assert (out[:, 3] == float("inf")).all() and (out[:, 6] == -float("inf")).all()
        rest = out[:, [d for d in range(64) if d not in (3, 6)]].double()
        # values that are all 1: the weights' parts add up to the sum, but for the least parts of fp16's tiny weights
        # (2^-37 of the largest each, below 2^-23 for 9500 keys), two roundings of 2^-24 a tile or part (700) and one
        assert (rest - 1).abs().max() <= torch.finfo(dtype).eps / 2 + 1400 * 2.0 ** -24


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_an_infinite_value_without_weight_has_no_product(cuda_device, dtype):
    # a score of -inf: 0 * inf, in the definition too
    k, v, table, length = _cache(40, 1, 64, dtype, cuda_device)
    q = torch.ones(1, 2, 1, 64, dtype=dtype, device=cuda_device)
    k[0, 0, 7, 5], v[0, 0, 7, 3] = -float("inf"), float("inf")
    out = cmpext3.ops.paged_attention(q, k, v, table, length)[0, :, 0]
    assert torch.isnan(out[:, 3]).all() and (out[:, :3] == 0).all() and (out[:, 4:] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_queries_with_odd_strides_along_dimensions_of_one(cuda_device, dtype):
    g = torch.Generator().manual_seed(30)
    k, v, table, length = _cache(300, 2, 64, dtype, cuda_device)
    for c in (k, v):
        c.copy_(torch.randn(c.shape, generator=g))
    wide = torch.randn(4, 515, generator=g).to(dtype).to(cuda_device)
    row = wide[:, :512].unflatten(1, (8, 64)).unsqueeze(2)[0:1]      # [1, 8, 1, 64], batch stride 515
    want = cmpext3.ops.paged_attention(row.clone(memory_format=torch.contiguous_format).view(1, 8, 1, 64), k, v, table, length)
    for _ in range(2):                                               # the second call has a kept signature
        assert torch.equal(cmpext3.ops.paged_attention(row, k, v, table, length), want)
    turned = cmpext3.ops.kv_append(k[:1, :, :1].clone(), v[:1, :, :1].clone(), k, v, table, length, query=row)
    assert torch.equal(turned, row)
    assert cmpext3.ops.paged_attention(turned, k, v, table, length).shape == row.shape
    one = torch.randn(3 * 64 + 515, generator=g).to(dtype).to(cuda_device).as_strided((3, 1, 1, 64), (64, 515, 64, 1))
    table, length = table.expand(3, -1), torch.tensor([300, 17, 0], dtype=torch.int32, device=cuda_device)
    want = cmpext3.ops.paged_attention(one.reshape(3, 64).clone().view(3, 1, 1, 64), k[:, :1], v[:, :1], table, length)
    assert torch.equal(cmpext3.ops.paged_attention(one, k[:, :1], v[:, :1], table, length), want)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_caches_and_rows_with_odd_strides_along_dimensions_of_one(cuda_device, dtype):
    g = torch.Generator().manual_seed(31)
    i32 = dict(dtype=torch.int32, device=cuda_device)
    freqs = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().to(cuda_device)
    for shape, at, tokens in (((1, 2, 16, 64), 0, 3), ((4, 1, 16, 64), 1, 20), ((4, 2, 1, 64), 2, 3)):
        pages, heads, page, dim = shape
        k, v = (torch.randn(shape, generator=g).to(dtype).to(cuda_device) for _ in range(2))
        stride = list(k.stride())
        stride[at] = 12345
        table = torch.arange(pages, **i32)[None]
        length = torch.tensor([tokens], **i32)
        new, query = (torch.randn(1, h, 1, dim, generator=g).to(dtype).to(cuda_device) for h in (heads, 2 * heads))
        seen = []
        for odd in (False, True):
            kc, vc = k.clone(), v.clone()
            if odd:
                kc, vc = (c.as_strided(shape, stride) for c in (kc, vc))
            turned = cmpext3.ops.kv_append(new, new, kc, vc, table, length, query=query, freqs=freqs)
            seen.append((kc, vc, turned, cmpext3.ops.paged_attention(turned, kc, vc, table, length)))
        assert all(torch.equal(a, b) for a, b in zip(*seen))
    x = torch.randn(1, 3, 5, 64, generator=g).to(dtype).to(cuda_device)
    y = cmpext3.ops.rope(x, torch.arange(5, device=cuda_device), freqs)
    odd = x.as_strided(x.shape, (12345, *x.stride()[1:]))
    assert torch.equal(cmpext3.ops.rope(odd, torch.arange(5, device=cuda_device), freqs), y)


def test_dual_tensors_are_refused_with_a_kept_signature_too(cuda_device):
    from torch.autograd import forward_ad as fa
    x = torch.randn(1, 2, 3, 16, device=cuda_device)
    positions, freqs = torch.arange(3, device=cuda_device), torch.ones(8, device=cuda_device)
    want = cmpext3.ops.rope(x, positions, freqs)
    with fa.dual_level():
        assert torch.equal(cmpext3.ops.rope(x, positions, freqs), want)    # a level without duals changes nothing
        dual = fa.make_dual(x, x.clone())
        with pytest.raises(RuntimeError, match="forward-mode"):
            cmpext3.ops.rope(dual, positions, freqs)
        with pytest.raises(RuntimeError, match="forward-mode"):
            cmpext3.ops.rope(fa.make_dual(x.clone().requires_grad_(), x.clone()), positions, freqs)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_angles_are_exact_to_fp32(cuda_device, kind, interleaved):
    # angles up to 2^50 radians, reduced here in 80 decimal digits
    import math
    from decimal import Decimal, localcontext
    places = [2 ** 28 + 32, 2 ** 31 - 128, -(2 ** 31)]
    if kind != torch.int32:
        places += [2 ** 40 + 2 ** 17, 2 ** 49 - 2 ** 25, -(2 ** 49) - 2 ** 30]
    if kind == torch.int64:
        places += [2 ** 31 - 1, 2 ** 40 + 3, 2 ** 49 - 1, 10 ** 14 + 7]
    positions, freqs = torch.tensor(places).to(kind), torch.tensor([1.0, 0.3, 1e-3, 1.7])
    assert [int(p) for p in positions.tolist()] == places
    x = torch.randn(1, 2, len(places), 10, generator=torch.Generator().manual_seed(32))
    y = cmpext3.ops.rope(x.to(cuda_device), positions.to(cuda_device), freqs.to(cuda_device), interleaved=interleaved).cpu().double()
    with localcontext() as ctx:
        ctx.prec = 80
        turn = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")
        rest = torch.tensor([[float(Decimal(p) * Decimal(f) % turn) for f in freqs.tolist()] for p in places], dtype=torch.float64)
    cos, sin = torch.cos(rest), torch.sin(rest)
    re, im = (slice(0, 8, 2), slice(1, 8, 2)) if interleaved else (slice(0, 4), slice(4, 8))
    u, w = x[..., re].double(), x[..., im].double()
    # cos and sin are off by at most 2^-23 (half a step of the fp32 remainder, and their polynomials' own), the two products
    # and the sum by 2^-24 each of at most |u| + |w|, the result by its rounding
    bound = (u.abs() + w.abs()) * 2.0 ** -21
    for got, want in ((y[..., re], u * cos - w * sin), (y[..., im], u * sin + w * cos)):
        assert ((got - want).abs() - bound).max() <= 0, (got - want).abs().amax((0, 1, 3))
    assert torch.equal(y[..., 8:], x[..., 8:].double()) and math.isfinite(y.sum())


# ---- a kept signature meets other pointers -----------------------------------------------------

def _shifted(t):
    """Copies of t, contiguous: at a new allocation's begin, and one element behind it."""
    return [torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)[at:at + t.numel()].view(t.shape).copy_(t) for at in (0, 1)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_a_kept_signature_with_misaligned_tensors(cuda_device, dtype):
    g = torch.Generator().manual_seed(33)
    dev, ops = cuda_device, cmpext3.ops

    def randn(*shape):
        return torch.randn(shape, generator=g).to(dtype).to(dev)

    def both(call, *tensors):
        """call(*tensors), aligned, a second time with its kept signature, then with each tensor misaligned in turn."""
        pairs = [_shifted(t) for t in tensors]
        first = [p[0] for p in pairs]
        want = call(*first)
        assert torch.equal(call(*first), want)
        for i, (_, off) in enumerate(pairs):
            assert off.data_ptr() % 16 and off.stride() == first[i].stride()
            assert torch.equal(call(*first[:i], off, *first[i + 1:]), want), i
        assert torch.equal(call(*first), want)
    freqs = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().to(dev)
    both(ops.rope, randn(2, 3, 5, 64), torch.arange(5, device=dev), freqs)
    k, v, table, length = _cache(300, 2, 64, dtype, dev)
    k.copy_(randn(*k.shape)), v.copy_(randn(*v.shape))
    both(lambda q, t, n: ops.paged_attention(q, k, v, t, n), randn(1, 8, 1, 64), table, length)

    def append(key, value, t, n, new, query, f):
        kc, vc = k.clone(), v.clone()
        out = ops.kv_append(key, value, kc, vc, t, n, new, query, freqs=f)
        return torch.cat((kc.flatten(), vc.flatten(), out.flatten()))
    both(append, randn(1, 2, 3, 64), randn(1, 2, 3, 64), table, length, torch.tensor([2], dtype=torch.int32, device=dev),
         randn(1, 4, 3, 64), freqs)
    w = torch.randint(0, 256, (40, 128), generator=g, dtype=torch.uint8).to(dev)
    zeros = torch.randint(0, 16, (40, 4), generator=g, dtype=torch.uint8).to(dev)
    both(ops.linear_w4, randn(3, 256), w, randn(40, 4), zeros, randn(40))
    # a cache off its 16-byte boundaries has no other way: refused, kept signature or not
    off = _shifted(k)[1]
    for _ in range(2):
        with pytest.raises(N.CmpxError, match="aligned"):
            ops.paged_attention(randn(1, 8, 1, 64), off, v, table, length)
        with pytest.raises(N.CmpxError, match="aligned"):
            ops.kv_append(randn(1, 2, 3, 64), randn(1, 2, 3, 64), off, v, table, length)
    assert N.device_status() == 0


def test_more_signatures_than_are_kept(cuda_device, monkeypatch):
    from cmpext3 import _serving as S
    monkeypatch.setattr(S, "_SIGNATURES", {})
    monkeypatch.setattr(S, "_SIGNATURES_MOST", 5)
    freqs = torch.ones(8, device=cuda_device)
    xs = [torch.randn(1, 2, n, 16, device=cuda_device) for n in range(1, 14)]
    want = [cmpext3.ops.rope(x, torch.arange(x.shape[2], device=cuda_device), freqs) for x in xs]
    assert 1 <= len(S._SIGNATURES) <= 5
    for _ in range(2):
        for x, y in zip(xs, want):
            assert torch.equal(cmpext3.ops.rope(x, torch.arange(x.shape[2], device=cuda_device), freqs), y)
            assert len(S._SIGNATURES) <= 5


# ---- linear_w4: all three parts of fp32 activations ----------------------------------------------

@pytest.mark.parametrize("m", [1, 8, 9, 16])
@pytest.mark.parametrize("k,group", [(64, 64), (96, 32), (160, 32), (256, 128), (4096, 32), (4096, 64), (4096, 128), (16384, 128)])
def test_low_parts_of_full_precision_activations(cuda_device, m, k, group):
    # x = 1 + a 2^-12 + b 2^-22, a < 16, b < 4: a value in each part of 8 bits.  Weights are +1 for k % 8 < 4 and -1 else, so that the
    # ones cancel in every product of 16 k; what is left are multiples of 2^-22, below 2 in all partial sums: exact in fp32
    g = torch.Generator().manual_seed(m + k + group)
    a, b = torch.randint(0, 16, (m, k), generator=g), torch.randint(0, 4, (m, k), generator=g)
    x = (1 + a * 2.0 ** -12 + b * 2.0 ** -22).float()
    assert torch.equal(x.double(), 1 + a * 2.0 ** -12 + b * 2.0 ** -22)
    sign = torch.where(torch.arange(k) % 8 < 4, 1, -1)
    codes = (8 + sign).to(torch.uint8).expand(24, k)
    w = codes[:, 0::2] | (codes[:, 1::2] << 4)
    want = (x.double() * sign).sum(1)
    assert want.abs().max() < 2
    y = cmpext3.ops.linear_w4(x.to(cuda_device), w.to(cuda_device), torch.ones(24, k // group, device=cuda_device))
    assert torch.equal(y.cpu().double(), want[:, None].expand(m, 24))


@pytest.mark.parametrize("m,k,group", [(1, 384, 128), (1, 4096, 128), (8, 4096, 128), (16, 4096, 128), (8, 4096, 64), (3, 2560, 32)])
def test_full_precision_sums_are_fp32_sums(cuda_device, m, k, group):
    from tests import serving_oracle as O
    from tests.test_linear_w4_gpu import _make
    x, w, s, z, _ = args = _make(torch.float32, m, 1001, k, group, True, False, k + group)
    y = cmpext3.ops.linear_w4(*(None if t is None else t.to(cuda_device) for t in args)).cpu().double()
    want = O.linear_w4(*args)[0]
    codes = torch.stack((w & 15, w >> 4), -1).reshape(1001, -1, group).double()
    weights = ((codes - z.double()[..., None]) * s.double()[..., None]).reshape(1001, k)
    root = ((x.double() ** 2) @ (weights ** 2).t()).sqrt()          # of an output's squared products: about its size
    # For every 32 k two sums are cut off at 2^-23 of a partial sum about as large as the root of its products' squares, with
    # the sign of that sum, 2 * 2^-23 of the whole's; up to 24 fp32 sums of 2^-24 (8 words a warp, 16 warps), and a rounding
    off = ((2 * 2.0 ** -23) ** 2 + 24 * (2.0 ** -24) ** 2) ** 0.5 + 2.0 ** -24
    assert (y - want).norm() <= off * root.norm()
