"""cmpext3.ops.kv_append on a B200 against its 64-bit definition: which slots are written (and that no
other is), padding rows, pages that end anywhere, cache layouts, the rotation on the way, bad pages."""
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


def _table(total, page, gen, spare=3):
    """A page table for sequences of these lengths, its pages in random order, and the pool's size."""
    counts = [-(-n // page) for n in total]
    pool = sum(counts) + spare
    order = torch.randperm(pool, generator=gen).to(torch.int32)
    table = torch.full((len(total), max(1, max(counts))), -7, dtype=torch.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    return table, pool


class Case:
    def __init__(self, dtype, B, H, Hkv, D, page, L, past, new=None, seed=0, tokens_first=False):
        g = torch.Generator().manual_seed(seed)
        self.new = [L] * B if new is None else new
        self.total = [p + n for p, n in zip(past, self.new)]
        self.table, pool = _table(self.total, page, g)
        self.k, self.v = (torch.randn(B, Hkv, L, D, generator=g).to(dtype) for _ in range(2))
        self.q = torch.randn(B, H, L, D, generator=g).to(dtype) if H else None
        self.kc, self.vc = (torch.randn(pool, Hkv, page, D, generator=g).to(dtype) for _ in range(2))
        self.ragged, self.page, self.tokens_first = new is not None, page, tokens_first

    def run(self, dev, **rot):
        kc, vc = self.kc.to(dev), self.vc.to(dev)
        if self.tokens_first:  # [pages, page_size, heads_kv, head_dim] memory
            kc, vc = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (kc, vc))
        lengths = torch.tensor(self.total, dtype=torch.int32, device=dev)
        new = torch.tensor(self.new, dtype=torch.int32, device=dev) if self.ragged else None
        rot = {n: t.to(dev) if isinstance(t, torch.Tensor) else t for n, t in rot.items()}
        q = cmpext3.ops.kv_append(self.k.to(dev), self.v.to(dev), kc, vc, self.table.to(dev), lengths, new,
                                  None if self.q is None else self.q.to(dev), **rot)
        torch.cuda.synchronize()
        return q, kc.cpu(), vc.cpu()

    def check(self, dev, **rot):
        q, kc, vc = self.run(dev, **rot)
        B, _, L, _ = self.k.shape
        place = torch.tensor([[t - n + i for i in range(L)] for t, n in zip(self.total, self.new)])
        positions = rot.get("positions", None)
        how = (rot.get("freqs"), rot.get("sections"), rot.get("interleaved", False))

        def turned(x):
            if how[0] is None:
                return x.double(), torch.zeros_like(x, dtype=torch.float64)
            return O.rope(x, place if positions is None else positions, *how)
        kt, kb = turned(self.k)
        want_k, want_v, bound = self.kc.double(), self.vc.double(), torch.zeros_like(self.kc, dtype=torch.float64)
        for b in range(B):
            for i in range(self.new[b]):
                t = int(place[b, i])
                p, r = int(self.table[b, t // self.page]), t % self.page
                want_k[p, :, r], bound[p, :, r] = kt[b, :, i], kb[b, :, i]
                want_v[p, :, r] = self.v[b, :, i].double()
        O.assert_within(kc, want_k, bound, "k_cache")
        assert torch.equal(vc.double(), want_v), "v_cache"
        if self.q is None:
            assert q is None
        else:
            want, b = turned(self.q)
            for i in range(B):  # padding rows come back as they were
                want[i, :, self.new[i]:], b[i, :, self.new[i]:] = self.q[i, :, self.new[i]:].double(), 0
            O.assert_within(q, want, b, "query")
        assert N.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,H,Hkv,D,page,L,past,new", [
    (1, 1, 1, 8, 1, 1, [0], None),                       # the first token, pages of one row
    (3, 8, 2, 64, 16, 1, [15, 16, 17], None),            # a step at a page's end, beginning and second row
    (5, 32, 8, 128, 64, 1, [0, 1, 63, 64, 1000], None),
    (2, 0, 4, 40, 24, 7, [20, 3], None),                 # no query; across a page's end
    (4, 5, 5, 96, 10, 33, [0, 9, 10, 11], [33, 0, 1, 20]),
    (2, 20, 4, 256, 7, 5, [13, 2], [0, 0]),              # nothing new at all
    (1, 128, 16, 80, 100, 130, [70], [129]),
])
def test_matches_the_definition(cuda_device, dtype, interleaved, B, H, Hkv, D, page, L, past, new):
    c = Case(dtype, B, H, Hkv, D, page, L, past, new, seed=B + D)
    c.check(cuda_device, freqs=_freqs(D // 2), interleaved=interleaved)
    c.check(cuda_device, freqs=_freqs(max(1, D // 8)), interleaved=interleaved)   # a part of the head
    c.check(cuda_device)                                                          # no rotation


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_given_positions_and_sections(cuda_device, dtype):
    c = Case(dtype, 3, 6, 2, 64, 16, 12, [5, 0, 30], [12, 4, 0], seed=5, tokens_first=True)
    g = torch.Generator().manual_seed(1)
    c.check(cuda_device, freqs=_freqs(32), positions=torch.randint(0, 99, (3, 12), generator=g, dtype=torch.int32))
    c.check(cuda_device, freqs=_freqs(32), positions=torch.randint(0, 99, (3, 3, 12), generator=g), sections=(12, 10, 10))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_strided_inputs(cuda_device, dtype):
    c = Case(dtype, 2, 4, 2, 64, 16, 9, [3, 14], seed=6)
    for name in ("k", "v", "q"):   # rows of a fused projection, on odd boundaries
        t = getattr(c, name)
        wide = torch.zeros(2, 9, t.shape[1] * 64 + 5, dtype=dtype)
        view = wide[..., 3:3 + t.shape[1] * 64].unflatten(-1, (t.shape[1], 64)).transpose(1, 2)
        view.copy_(t)
        setattr(c, name, view)
    c.check(cuda_device, freqs=_freqs(32))
    c.k, c.v = c.k[:, :1].expand(2, 2, 9, 64), c.v[:, :, :1].expand(2, 2, 9, 64)
    c.check(cuda_device, freqs=_freqs(32))


def test_a_slice_of_a_larger_cache(cuda_device):
    # keys and values of all layers in one tensor: [pages, 2, heads_kv, page, dim]
    g = torch.Generator().manual_seed(7)
    both = torch.randn(6, 2, 2, 16, 64, generator=g).to(cuda_device)
    before = both.clone()
    k, v = (torch.randn(1, 2, 3, 64, generator=g).to(cuda_device) for _ in range(2))
    table = torch.tensor([[4, 2]], dtype=torch.int32, device=cuda_device)
    lengths = torch.tensor([18], dtype=torch.int32, device=cuda_device)
    cmpext3.ops.kv_append(k, v, both[:, 0], both[:, 1], table, lengths)
    for i, (p, r) in enumerate([(4, 15), (2, 0), (2, 1)]):
        before[p, 0, :, r], before[p, 1, :, r] = k[0, :, i], v[0, :, i]
    assert torch.equal(both, before)


def test_tokens_outside_the_cache_are_reported_and_not_stored(cuda_device):
    # sequences: a negative place, behind the table, a page number too large, a negative one, a good one
    dev = cuda_device
    kc, vc = torch.zeros(4, 1, 8, 16, device=dev), torch.zeros(4, 1, 8, 16, device=dev)
    k = v = torch.ones(5, 1, 2, 16, device=dev)
    table = torch.tensor([[0, 0], [0, 0], [0, 4], [0, -1], [1, 2]], dtype=torch.int32, device=dev)
    lengths = torch.tensor([0, 18, 10, 10, 9], dtype=torch.int32, device=dev)
    q = cmpext3.ops.kv_append(k, v, kc, vc, table, lengths, query=k, freqs=_freqs(8).to(dev))
    assert N.device_status() == N.DEVFLAG_BAD_PAGE
    assert torch.isfinite(q).all()
    stored = {(int(p), int(r)) for p, _, r, _ in (vc != 0).nonzero()}
    assert stored == {(1, 7), (2, 0)}
    assert N.device_status() == 0


def test_new_lengths_outside_the_rows_are_clipped(cuda_device):
    dev = cuda_device
    kc, vc = torch.zeros(3, 1, 8, 16, device=dev), torch.zeros(3, 1, 8, 16, device=dev)
    k = torch.ones(2, 1, 2, 16, device=dev)
    table = torch.tensor([[0], [2]], dtype=torch.int32, device=dev)
    new = torch.tensor([9, -3], dtype=torch.int32, device=dev)
    cmpext3.ops.kv_append(k, k, kc, vc, table, torch.tensor([5, 5], dtype=torch.int32, device=dev), new)
    assert {(int(p), int(r)) for p, _, r, _ in (vc != 0).nonzero()} == {(0, 3), (0, 4)}
    assert N.device_status() == 0


def test_empty_calls(cuda_device):
    dev = cuda_device
    kc, vc = torch.ones(3, 2, 8, 16, device=dev), torch.ones(3, 2, 8, 16, device=dev)
    none = torch.empty(0, 2, 1, 16, device=dev)
    i32 = dict(dtype=torch.int32, device=dev)
    assert cmpext3.ops.kv_append(none, none, kc, vc, torch.zeros(0, 1, **i32), torch.zeros(0, **i32)) is None
    none = torch.empty(2, 2, 0, 16, device=dev)
    q = cmpext3.ops.kv_append(none, none, kc, vc, torch.zeros(2, 1, **i32), torch.zeros(2, **i32), query=none)
    assert q.shape == (2, 2, 0, 16) and (kc == 1).all()


def test_the_caches_count_as_changed_in_place(cuda_device):
    dev = cuda_device
    kc, vc = torch.ones(3, 2, 8, 16, device=dev), torch.ones(3, 2, 8, 16, device=dev)
    k = torch.zeros(1, 2, 1, 16, device=dev)
    i32 = dict(dtype=torch.int32, device=dev)
    versions = kc._version, vc._version
    cmpext3.ops.kv_append(k, k, kc, vc, torch.zeros(1, 1, **i32), torch.ones(1, **i32))
    assert (kc._version, vc._version) == (versions[0] + 1, versions[1] + 1)
    with torch.inference_mode():
        kc, vc = torch.ones(3, 2, 8, 16, device=dev), torch.ones(3, 2, 8, 16, device=dev)
        cmpext3.ops.kv_append(k, k, kc, vc, torch.zeros(1, 1, **i32), torch.ones(1, **i32))
