"""cmpext3.ops.paged_attention on a B200 under close bounds: that every key counts once in every schedule, and that fp32 products on
the tensor cores keep the low parts of all four operands (that the bounds see such mistakes: test_serving_bounds_host.py)."""
from __future__ import annotations

import pytest
import torch

import cmpext3
from cmpext3 import _native as N
from tests import serving_bounds as B
from tests import serving_oracle as O
from tests.test_kv_append_gpu import _table
from tests.test_paged_attention_gpu import DTYPES, IDS, Case

pytestmark = pytest.mark.gpu

HEADS = [(1, 1, 128), (8, 4, 64), (8, 1, 40), (8, 1, 96), (16, 2, 128), (7, 1, 160), (8, 1, 192), (4, 1, 256), (33, 1, 128)]
LENGTHS = [([40, 1, 17], "one CTA"), ([500], "cluster"), ([130, 129, 128] * 30, "one CTA"), ([513, 0, 1], "cluster"), ([3000], "cluster"), ([9500], "equal shares"),
           ([9000, 3, 0, 1200], "equal shares")]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("H,Hkv,D", HEADS)
@pytest.mark.parametrize("lengths,schedule", LENGTHS)
@pytest.mark.parametrize("page", [16, 24])
def test_every_key_counts_once(cuda_device, dtype, H, Hkv, D, lengths, schedule, page):
    # equal scores, one key's value in each column, until every key has been in one
    table, pool = _table(lengths, page, torch.Generator().manual_seed(len(lengths)))
    table = table.to(cuda_device)
    shape = (pool, Hkv, page, D)
    q = torch.zeros(len(lengths), H, 1, D, dtype=dtype, device=cuda_device)
    k = torch.randn(shape, generator=torch.Generator(cuda_device).manual_seed(1), device=cuda_device).to(dtype)
    now = torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    assert schedule in N.paged_attention_plan(q, k, k, table, now)
    worst = torch.zeros((), dtype=torch.float64, device=cuda_device)
    for start in range(0, max(lengths), Hkv * D):
        v, want = B.marked(lengths, table, shape, start, dtype, cuda_device)
        out = cmpext3.ops.paged_attention(q, k, v, table, now)[:, :, 0].double()
        want = want.repeat_interleave(H // Hkv, 1)
        worst = torch.maximum(worst, ((out - want).abs() - B.marked_bound(want, dtype)).max())
    assert worst <= 0
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_every_key_of_a_long_context_counts_once(cuda_device, dtype):
    n, page, D = 70001, 64, 128
    table, pool = _table([n], page, torch.Generator().manual_seed(2))
    table, now = table.to(cuda_device), torch.tensor([n], dtype=torch.int32, device=cuda_device)
    q = torch.zeros(1, 1, 1, D, dtype=dtype, device=cuda_device)
    k = torch.ones(pool, 1, page, D, dtype=dtype, device=cuda_device)
    worst = torch.zeros((), dtype=torch.float64, device=cuda_device)
    for start in range(0, n, D):
        v, want = B.marked([n], table, k.shape, start, dtype, cuda_device)
        out = cmpext3.ops.paged_attention(q, k, v, table, now)[:, :, 0].double()
        worst = torch.maximum(worst, ((out - want).abs() - B.marked_bound(want, dtype)).max())
    assert worst <= 0


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("H,Hkv,D", HEADS)
@pytest.mark.parametrize("lengths", [[300, 1, 30], [4096] * 3, [9500], [20000, 3, 0, 1200], [600] * 100])
def test_random_inputs_within_close_bounds(cuda_device, dtype, H, Hkv, D, lengths):
    c = Case(dtype, H, Hkv, D, 24, lengths, seed=H + D + len(lengths))
    out = cmpext3.ops.paged_attention(*c.args)[:, :, 0]
    torch.cuda.synchronize()
    for b, n in list(enumerate(lengths))[:7]:
        want, bound = B.attention(c.q[b, :, 0], c.k[b], c.v[b], D ** -0.5) if n else (torch.zeros(H, D, dtype=torch.float64),) * 2
        O.assert_within(out[b], want, bound, f"sequence {b} of length {n}")
    assert N.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_a_long_context_within_close_bounds(cuda_device, dtype):
    c = Case(dtype, 1, 1, 128, 64, [70001], seed=3)
    out = cmpext3.ops.paged_attention(*c.args)[0, :, 0]
    O.assert_within(out, *B.attention(c.q[0, :, 0], c.k[0], c.v[0], 128 ** -0.5), "70001 keys")


@pytest.mark.parametrize("part", ["queries", "keys", "weights", "values"])
@pytest.mark.parametrize("n", [40, 3000, 9500])
@pytest.mark.parametrize("heads,D", [(8, 40), (5, 64), (8, 64), (2, 80), (4, 96), (8, 96), (8, 128), (6, 160), (8, 160), (8, 192),
                                     (1, 64), (4, 128), (8, 256)])
def test_low_parts_in_full_precision(cuda_device, part, n, heads, D):
    g = torch.Generator().manual_seed(n + D)
    page, pages = 16, -(-n // 16)
    cases = [B.low_parts(part, heads, n, D, g) for _ in range(2)]                          # a key head each
    kc, vc = torch.zeros(pages, 2, page, D), torch.zeros(pages, 2, page, D)
    for h, (_, k, v, _) in enumerate(cases):
        for cache, rows in ((kc, k), (vc, v)):
            for p in range(pages):
                cache[p, h, :min(page, n - p * page)] = rows[p * page:(p + 1) * page]
    q = torch.cat([c[0] for c in cases])[None, :, None]
    table = torch.arange(pages, dtype=torch.int32)[None]
    dev = [t.to(cuda_device) for t in (q, kc, vc, table, torch.tensor([n], dtype=torch.int32))]
    out = cmpext3.ops.paged_attention(*dev, 1.0)[0, :, 0]
    for h, c in enumerate(cases):
        want, bound = B.low_parts_want(part, *c, tensor_cores=D <= 192 and (heads > 4 or heads > 1 and 64 < D <= 96))
        O.assert_within(out[h * heads:(h + 1) * heads], want, bound, f"key head {h}")


@pytest.mark.parametrize("D", [40, 64, 80, 96, 128, 160, 192, 256])
def test_one_key_gives_its_value_in_full_precision(cuda_device, D):
    # a weight of one: a value's leading 11 bits are rounded, and of the rest, at most 2^-11 of it, 11 bits are left: within
    # 2^-23 of the value; one key in each of 50 sequences, in pages of one
    g = torch.Generator().manual_seed(D)
    k, v = (torch.randn(50, 2, 1, D, generator=g).to(cuda_device) for _ in range(2))
    q = torch.randn(50, 16, 1, D, generator=g).to(cuda_device)
    table = torch.arange(50, dtype=torch.int32, device=cuda_device)[:, None]
    out = cmpext3.ops.paged_attention(q, k, v, table, torch.ones(50, dtype=torch.int32, device=cuda_device))
    want = v.double().repeat_interleave(8, 1)
    assert ((out.double() - want).abs() <= 2.0 ** -23 * want.abs()).all()


@pytest.mark.parametrize("D", [40, 64, 96, 128, 160, 192])
def test_the_largest_values_stay_finite_in_full_precision(cuda_device, D):
    # rounded to 11 bits they would be infinite; the second of two keys has a weight of exp(-30) and a small value
    top = torch.finfo(torch.float32).max
    k, v = (torch.zeros(1, 1, 16, D, device=cuda_device) for _ in range(2))
    k[0, 0, 0, 0], v[0, 0, 0], v[0, 0, 1] = 30.0, top, 1.0
    v[0, 0, 0, 1::2] = -top
    q = torch.zeros(1, 8, 1, D, device=cuda_device)
    q[..., 0] = 1.0
    table = torch.zeros(1, 1, dtype=torch.int32, device=cuda_device)
    for n in (1, 2):
        out = cmpext3.ops.paged_attention(q, k, v, table, torch.tensor([n], dtype=torch.int32, device=cuda_device), 1.0)[0, :, 0]
        want = v[0, 0, 0].double() / (1 + (n - 1) * torch.exp(torch.tensor(-30.0, dtype=torch.float64)).item())
        # two parts cut off: 3 * 2^-23, and the sums and the quotient 2^-22
        assert torch.isfinite(out).all() and ((out.double() - want).abs() <= 5 * 2.0 ** -23 * want.abs()).all()
