"""cmpext3.ops.paged_attention on a B200 against its 64-bit definition: lengths from none to long,
head groups, head sizes, pages that end inside a tile, cache layouts, what lies behind the last token,
bad pages, graphs, streams, and the split schedule."""
from __future__ import annotations

import math

import pytest
import torch

import cmpext3
from cmpext3 import _native as N
from tests import serving_oracle as O
from tests.test_kv_append_gpu import _table

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


class Case:
    def __init__(self, dtype, H, Hkv, D, page, lengths, seed=0, dev="cuda", tokens_first=False, sharp=1.0, fill=0.0):
        g = torch.Generator().manual_seed(seed)
        self.lengths = lengths
        self.q = (sharp * torch.randn(len(lengths), H, 1, D, generator=g)).to(dtype)
        self.table, pool = _table(lengths, page, g)
        self.k = [torch.randn(Hkv, n, D, generator=g).to(dtype) for n in lengths]
        self.v = [torch.randn(Hkv, n, D, generator=g).to(dtype) for n in lengths]
        # what no sequence has written holds `fill`
        self.kc, self.vc = (torch.full((pool, Hkv, page, D), fill, dtype=dtype) for _ in range(2))
        for b, n in enumerate(lengths):
            for p in range(-(-n // page)):
                m = min(page, n - p * page)
                at = int(self.table[b, p])
                self.kc[at, :, :m] = self.k[b][:, p * page:p * page + m]
                self.vc[at, :, :m] = self.v[b][:, p * page:p * page + m]
        self.args = [self.q.to(dev), self.kc.to(dev), self.vc.to(dev), self.table.to(dev),
                     torch.tensor(lengths, dtype=torch.int32, device=dev)]
        if tokens_first:
            for i in (1, 2):
                self.args[i] = self.args[i].transpose(1, 2).contiguous().transpose(1, 2)

    def check(self, scale=None, what="paged attention"):
        out = cmpext3.ops.paged_attention(*self.args, scale)
        torch.cuda.synchronize()
        s = 1 / math.sqrt(self.q.shape[3]) if scale is None else scale
        for b in range(len(self.lengths)):
            want, bound = O.attention(self.q[b, :, 0], self.k[b], self.v[b], s)
            O.assert_within(out[b, :, 0], want, bound, f"{what}, sequence {b} of length {self.lengths[b]}")
        assert out.shape == self.q.shape and out.dtype == self.q.dtype
        assert N.device_status() == 0
        return out


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("H,Hkv,D", [(1, 1, 8), (8, 8, 40), (8, 2, 64), (32, 8, 128), (5, 1, 96), (12, 2, 80),
                                     (16, 1, 160), (40, 2, 192), (8, 2, 256), (33, 1, 128), (7, 7, 128)])
def test_head_layouts(cuda_device, dtype, H, Hkv, D):
    Case(dtype, H, Hkv, D, 16, [1, 77, 300], seed=H + D).check()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("page", [1, 5, 16, 24, 64, 100, 256])
def test_pages_end_anywhere(cuda_device, dtype, page):
    Case(dtype, 4, 2, 64, page, [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 500], seed=page).check()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_every_short_length(cuda_device, dtype):
    Case(dtype, 4, 4, 32, 8, list(range(0, 140)), seed=2).check()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("lengths,schedule", [
    ([20000], "equal shares"), ([9000, 3, 0, 1200], "equal shares"), ([0, 0, 0, 9000], "equal shares"),
    ([600] * 300, "equal shares"), ([1, 0, 1300, 17] * 40, "equal shares"),
    ([0, 0, 0], "one CTA"), ([1] * 700, "one CTA"), ([130, 129, 128] * 30, "one CTA"), ([500] * 200, "one CTA"),
    ([4096] * 3, "cluster"), ([513], "cluster"), ([8192], "cluster"), ([600, 0, 1, 599], "cluster"), ([2000, 15] * 4, "cluster")])
def test_every_schedule(cuda_device, dtype, lengths, schedule):
    c = Case(dtype, 8, 2, 64, 16, lengths, seed=len(lengths))
    assert schedule in N.paged_attention_plan(*c.args)
    c.check()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("H,Hkv,D", [(1, 1, 8), (8, 8, 40), (32, 8, 128), (5, 1, 96), (12, 2, 80), (16, 1, 160), (40, 2, 192),
                                     (8, 2, 256), (33, 1, 128)])
@pytest.mark.parametrize("lengths", [[3000, 1], [9500]])
def test_head_layouts_of_long_caches(cuda_device, dtype, H, Hkv, D, lengths):
    Case(dtype, H, Hkv, D, 16, lengths, seed=H + D + 1).check()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("D", [64, 256])
def test_many_rows_beside_a_long_one(cuda_device, dtype, D):
    # more rows than SMs, one of them in many parts; then more sequences than a block has threads
    Case(dtype, 8, 2, D, 16, [9000] + [20] * 30, seed=17).check()
    Case(dtype, 2, 2, D, 16, [1500] + [7, 0, 300] * 60, seed=18).check()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_one_head_over_a_long_context(cuda_device, dtype):
    Case(dtype, 1, 1, 128, 64, [70001], seed=3).check()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_cache_layouts(cuda_device, dtype):
    Case(dtype, 8, 2, 64, 16, [100, 40], seed=4, tokens_first=True).check()
    c = Case(dtype, 8, 2, 64, 16, [100, 40], seed=4)
    both = torch.stack([c.args[1], c.args[2]], 1)          # keys and values of a page side by side
    c.args[1], c.args[2] = both[:, 0], both[:, 1]
    c.check()
    wide = torch.zeros(2, 8, 1, 71, dtype=dtype, device=cuda_device)
    wide[..., 3:67] = c.args[0]
    c.args[0] = wide[..., 3:67]                            # a query on odd boundaries
    c.check()
    c.args[0] = c.q.to(cuda_device).transpose(1, 3).contiguous().transpose(1, 3)
    c.check()
    pad = torch.full((2, 20), -5, dtype=torch.int32, device=cuda_device)
    pad[:, :c.table.shape[1]] = c.args[3]
    c.args[3] = pad                                        # a wider table, its free entries anything
    c.check()
    c.args[3] = pad[:, :c.table.shape[1]]                  # and a view of it
    c.check()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf")])
def test_what_lies_behind_the_last_token_does_not_count(cuda_device, dtype, fill):
    Case(dtype, 8, 2, 64, 24, [1, 23, 24, 25, 100, 1000, 0], seed=5, fill=fill).check()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("scale", [1.0, -0.5, 0.0, 1e-3])
def test_scales(cuda_device, dtype, scale):
    Case(dtype, 4, 2, 64, 16, [300, 5], seed=6).check(scale)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_sharp_scores(cuda_device, dtype):
    # scores of some hundreds: one key has nearly all the weight, wherever it lies
    Case(dtype, 8, 2, 64, 16, [1, 50, 700, 3000], seed=7, sharp=30.0).check()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n", [40, 3000, 9000])
def test_infinite_values_and_scores(cuda_device, dtype, n):
    c = Case(dtype, 4, 2, 64, 16, [n], seed=16)
    page, row = int(c.table[0, (n - 1) // 16]), (n - 1) % 16
    c.args[2][page, 0, row, 5] = float("inf")             # a value: its column is infinite, the others stay
    out = cmpext3.ops.paged_attention(*c.args)[0, :, 0]
    assert (out[:2, 5] == float("inf")).all()
    rest = torch.cat((out[:2, :5], out[:2, 6:]), 1)
    assert torch.isfinite(rest).all() and torch.isfinite(out[2:]).all()
    c.args[2][page, 0, row, 5] = 0.0
    c.args[0][0, :, 0, 3] = 2.0
    c.args[1][page, 1, row, 3] = -float("inf")            # a score of -inf: the key does not count
    c.q[0, :, 0, 3] = 2.0
    out = cmpext3.ops.paged_attention(*c.args)[0, 2:, 0]
    torch.cuda.synchronize()
    want, bound = O.attention(c.q[0, 2:, 0], c.k[0][1:, :n - 1], c.v[0][1:, :n - 1], 1 / 8)
    O.assert_within(out, want, bound, "a key with a score of -inf")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("lengths", [[40, 0], [3000, 0], [9000, 0], [9000, 0] + [20] * 300])
def test_scores_that_are_all_minus_infinity_have_no_softmax(cuda_device, dtype, lengths):
    c = Case(dtype, 4, 2, 64, 16, lengths, seed=19)
    c.args[0][..., 3] = 2.0
    c.args[1][:, 1, :, 3] = -float("inf")
    out = cmpext3.ops.paged_attention(*c.args)
    some = [b for b, n in enumerate(lengths) if n]
    assert torch.isnan(out[some][:, 2:]).all() and torch.isfinite(out[some][:, :2]).all() and (out[1] == 0).all()


@pytest.mark.parametrize("D", [40, 64, 96, 128, 160, 192, 256])
@pytest.mark.parametrize("n", [40, 3000, 9000])
def test_infinite_values_and_scores_with_many_heads_in_full_precision(cuda_device, D, n):
    c = Case(torch.float32, 16, 2, D, 16, [n, 30], seed=20)
    page, row = int(c.table[0, (n - 1) // 16]), (n - 1) % 16
    c.args[2][page, 0, row, 5] = -float("inf")
    c.args[0][0, :, 0, 3] = 2.0
    c.args[1][page, 1, row, 3] = -float("inf")
    c.q[0, :, 0, 3] = 2.0
    out = cmpext3.ops.paged_attention(*c.args)[:, :, 0]
    torch.cuda.synchronize()
    assert (out[0, :8, 5] == -float("inf")).all()
    want, bound = O.attention(c.q[0, :8, 0], c.k[0][:1], c.v[0][:1], D ** -0.5)
    want[:, 5], bound[:, 5] = 0, 1                                            # (seen above)
    out[0, :8, 5] = 0
    O.assert_within(out[0, :8], want, bound, "the other columns")
    want, bound = O.attention(c.q[0, 8:, 0], c.k[0][1:, :n - 1], c.v[0][1:, :n - 1], D ** -0.5)
    O.assert_within(out[0, 8:], want, bound, "a key with a score of -inf")
    want, bound = O.attention(c.q[1, :, 0], c.k[1], c.v[1], D ** -0.5)
    O.assert_within(out[1], want, bound, "the other sequence")
    c.args[1][page, 0, row, 0] = float("nan")
    out = cmpext3.ops.paged_attention(*c.args)[:, :, 0]
    assert torch.isnan(out[0, :8]).all() and torch.isfinite(out[0, 8:]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("H,Hkv,D", [(8, 1, 40), (5, 1, 64), (16, 2, 64), (12, 2, 96), (24, 3, 128), (6, 1, 160), (14, 2, 192)])
@pytest.mark.parametrize("lengths", [list(range(0, 70)), [600] * 300, [9500, 3, 0], [4096] * 3])
def test_many_heads_in_full_precision(cuda_device, H, Hkv, D, lengths):
    Case(torch.float32, H, Hkv, D, 24, lengths, seed=H + D, fill=float("nan")).check()


def test_nan_and_infinite_keys_spread_to_their_sequence_alone(cuda_device):
    c = Case(torch.bfloat16, 4, 2, 64, 16, [40, 700, 30], seed=8)
    c.args[1][int(c.table[1, 20]), 0, 3] = float("nan")
    out = cmpext3.ops.paged_attention(*c.args)
    assert torch.isnan(out[1, :2]).all() and torch.isfinite(out[1, 2:]).all()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[2]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_bad_pages_and_lengths_make_their_sequence_nan(cuda_device, dtype):
    c = Case(dtype, 8, 2, 64, 16, [40, 900, 30, 50, 20], seed=9)
    good = c.check()
    c.args[3][1, 30] = c.kc.shape[0]          # behind the cache
    c.args[3][2, 0] = -1
    c.args[4][3] = c.table.shape[1] * 16 + 1  # longer than the table
    c.args[4][4] = -4                         # shorter than empty
    out = cmpext3.ops.paged_attention(*c.args)
    assert N.device_status() == N.DEVFLAG_BAD_PAGE
    assert torch.equal(out[0], good[0])
    assert torch.isnan(out[1:4]).all() and (out[4] == 0).all()
    assert N.device_status() == 0


def test_empty_calls(cuda_device):
    i32 = dict(dtype=torch.int32, device=cuda_device)
    cache = torch.zeros(2, 2, 8, 64, device=cuda_device)
    q = torch.empty(0, 4, 1, 64, device=cuda_device)
    assert cmpext3.ops.paged_attention(q, cache, cache, torch.zeros(0, 3, **i32), torch.zeros(0, **i32)).shape == q.shape
    q = torch.ones(3, 4, 1, 64, device=cuda_device)
    for pages, width in ((2, 0), (0, 4)):
        out = cmpext3.ops.paged_attention(q, cache[:pages], cache[:pages], torch.zeros(3, width, **i32), torch.zeros(3, **i32))
        assert (out == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_the_same_call_gives_the_same_bits(cuda_device, dtype):
    c = Case(dtype, 8, 2, 64, 16, [5000, 3, 900], seed=10)
    first = cmpext3.ops.paged_attention(*c.args)
    for _ in range(5):
        assert torch.equal(cmpext3.ops.paged_attention(*c.args), first)


@pytest.mark.parametrize("longest", [100, 3000, 12000])   # a CTA, a cluster, shares and a join
def test_two_graphs_at_once_and_other_lengths(cuda_device, longest):
    c = Case(torch.bfloat16, 8, 2, 128, 16, [longest, 50, 1], seed=11)
    d = Case(torch.bfloat16, 8, 2, 128, 16, [longest - 7, longest // 2], seed=12)
    graphs = []
    for case in (c, d):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            cmpext3.ops.paged_attention(*case.args)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = cmpext3.ops.paged_attention(*case.args)
        graphs.append((graph, out, case))
    streams = [torch.cuda.Stream() for _ in graphs]
    for lengths in ([longest, 50, 1], [17, 0, 1], [longest - 1, 20, 0]):
        c.args[4].copy_(torch.tensor(lengths, dtype=torch.int32))
        torch.cuda.synchronize()
        for (graph, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(10):
                    graph.replay()
        torch.cuda.synchronize()
        for _, out, case in graphs:
            assert torch.equal(out, cmpext3.ops.paged_attention(*case.args))


@pytest.mark.parametrize("longest", [6000, 15000])
def test_two_streams_at_once(cuda_device, longest):
    cases = [Case(torch.float16, 8, 2, 64, 16, [longest, 30], seed=s) for s in (13, 14)]
    want = [cmpext3.ops.paged_attention(*c.args) for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cmpext3.ops.paged_attention(*cases[i].args))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_offsets_beyond_32_bits(cuda_device):
    # a cache of 2^32 and more elements, of which the sequence uses the last pages
    pages = 2 ** 32 // (1 * 64 * 128) + 4
    kc, vc = (torch.empty(pages, 1, 64, 128, dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    g = torch.Generator().manual_seed(15)
    c = Case(torch.bfloat16, 4, 1, 128, 64, [200], seed=15)
    last = torch.arange(pages - 4, pages, dtype=torch.int32)
    for i in range(4):
        kc[pages - 4 + i], vc[pages - 4 + i] = (t[int(c.table[0, i])].to(cuda_device) for t in (c.kc, c.vc))
    c.args[1], c.args[2], c.args[3] = kc, vc, last[None].to(cuda_device)
    c.check()
    k, v = (torch.randn(1, 1, 2, 128, generator=g).to(torch.bfloat16).to(cuda_device) for _ in range(2))
    cmpext3.ops.kv_append(k, v, kc, vc, c.args[3], torch.tensor([202], dtype=torch.int32, device=cuda_device))
    assert torch.equal(kc[pages - 1, 0, 8:10], k[0, 0]) and torch.equal(vc[pages - 1, 0, 8:10], v[0, 0])
