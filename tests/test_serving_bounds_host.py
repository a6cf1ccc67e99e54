"""That the close bounds of the attention tests see the mistakes they are for, played in the definition on the CPU."""
from __future__ import annotations

import pytest
import torch

from tests import serving_bounds as B


def _random(n, d, dtype, heads=1, seed=0):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(s, generator=g).to(dtype) for s in ((heads, d), (1, n, d), (1, n, d)))


def _attend(q, k, v, scale, keep=None, tf32=(), rounded=True):
    """The definition over the keys `keep`, with the operands named in tf32 as one part of 11 bits."""
    if keep is not None:
        k, v = k[:, keep], v[:, keep]
    q, k, v = (B.one_part(t, rounded).double() if w in tf32 else t.double() for t, w in ((q, "queries"), (k[0], "keys"), (v[0], "values")))
    p = torch.softmax(q @ k.t() * scale, -1)
    if "weights" in tf32:
        top = p.amax(-1, keepdim=True)                      # the kernels' weights are at most 1
        p = B.one_part(p / top, rounded).double() * top
    return p @ v


def _seen(got, want, bound):
    return ((got - want).abs() > bound).any().item()


@pytest.mark.parametrize("n,d", [(70001, 128), (20000, 64), (9500, 40), (3000, 192)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_lost_keys_are_seen(n, d, dtype):
    q, k, v = _random(n, d, dtype, seed=n)
    scale = d ** -0.5
    want, bound = B.attention(q, k, v, scale)
    every = torch.arange(n)
    assert not _seen(_attend(q, k, v, scale).to(dtype).double(), want, bound)
    for lost in (slice(n // 2, n // 2 + 16), slice(n - 16, n), slice(0, 16)):         # a tile
        keep = torch.ones(n, dtype=torch.bool)
        keep[lost] = False
        assert _seen(_attend(q, k, v, scale, every[keep]).to(dtype).double(), want, bound), lost
    twice = torch.cat((every, every[100:116]))                                         # a tile twice
    assert _seen(_attend(q, k, v, scale, twice).to(dtype).double(), want, bound)
    if dtype == torch.float32:
        assert _seen(_attend(q, k, v, scale, every[every != n // 3]), want, bound)      # a key


@pytest.mark.parametrize("n,d", [(300, 40), (300, 192), (4096, 128), (9500, 160), (20000, 64)])
@pytest.mark.parametrize("part", ["queries", "keys", "weights", "values"])
def test_operands_of_one_part_are_seen_in_full_precision(n, d, part):
    q, k, v = _random(n, d, torch.float32, heads=8, seed=d)
    want, bound = B.attention(q, k, v, d ** -0.5)
    assert not _seen(_attend(q, k, v, d ** -0.5).float().double(), want, bound)
    for rounded in (False, True):
        assert _seen(_attend(q, k, v, d ** -0.5, tf32=(part,), rounded=rounded), want, bound)


@pytest.mark.parametrize("n", [40, 3000, 9500])
@pytest.mark.parametrize("d", [40, 64, 80, 96, 128, 160, 192])
@pytest.mark.parametrize("part", ["queries", "keys", "weights", "values"])
def test_low_parts_hang_on_their_part(n, d, part):
    q, k, v, scale = B.low_parts(part, 8, n, d, torch.Generator().manual_seed(n + d))
    want, bound = B.low_parts_want(part, q, k, v, scale)
    assert not _seen(_attend(q, k[None], v[None], scale).float().double(), want, bound)
    off = (_attend(q, k[None], v[None], scale, tf32=(part,)) - want).abs()
    assert (off.amax(-1) > 20 * bound.amax(-1)).all()        # every head's result is far off without it
    assert (off.amax(-1) > 4 * B.low_parts_want(part, q, k, v, scale, tensor_cores=False)[1].amax(-1)).all()
    for other in {"queries", "keys", "weights", "values"} - {part}:   # (and those of the others are not asked for)
        if other in ("queries", "keys") or part in ("weights", "values") and other != "weights":
            assert not _seen(_attend(q, k[None], v[None], scale, tf32=(other,)), want, bound)


def test_marked_columns_see_every_key():
    lengths, page, heads, dim = [70, 0, 33], 8, 2, 16
    counts = [-(-n // page) for n in lengths]
    table, at = torch.full((3, max(counts)), -1, dtype=torch.int32), 0
    for b, c in enumerate(counts):
        table[b, :c] = torch.arange(at, at + c)
        at += c
    seen = [set() for _ in lengths]
    for start in range(0, max(lengths), heads * dim):
        v, want = B.marked(lengths, table, (at, heads, page, dim), start, torch.float32, "cpu")
        for b, n in enumerate(lengths):
            t = torch.arange(n)
            rows = v[table[b].long()[t // page], :, t % page]                           # [n, heads, dim]
            if n:
                assert torch.equal(rows.double().mean(0), want[b])
                less = rows[torch.arange(n) != start % n].double().mean(0)               # one key lost
                assert ((less - want[b]).abs() > B.marked_bound(want[b], torch.bfloat16)).any() or start >= n
            seen[b] |= {int(i) for i in rows.flatten(1).any(1).nonzero()}
    assert [len(s) for s in seen] == lengths
