"""The serving operators without a GPU: what the binding and the C ABI refuse, the descriptors' layout, and
the arithmetic of the paged attention's schedule, restated."""
from __future__ import annotations

import ctypes
import random
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import cmpext3
from cmpext3 import _native as N
from cmpext3 import _serving as S

HEADER_DIR = Path(__file__).resolve().parents[1] / "include"


@pytest.fixture
def cpu(monkeypatch):
    """Lets CPU tensors through the device check, so that the checks behind it can be tested; no call is launched."""
    monkeypatch.setattr(S, "_rows", lambda name, t: t.device)
    monkeypatch.setattr(S, "_run", lambda *a: pytest.fail("the call was not refused"))


def refused(match, fn, *args, error=RuntimeError, **kwargs):
    with pytest.raises(error, match=match):
        fn(*args, **kwargs)


# ---- descriptors ------------------------------------------------------------------------------

def test_descriptors_have_the_header_layout(tmp_path):
    structs = {"cmpx_rotation": S.Rotation, "cmpx_rope_desc": S.RopeDesc, "cmpx_paged_cache": S.PagedCache,
               "cmpx_kv_append_desc": S.KvAppendDesc, "cmpx_paged_attn_desc": S.PagedAttnDesc,
               "cmpx_linear_w4_desc": S.LinearW4Desc}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "cmpx_b200.h"', "int main(void) {"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} %zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {field}));' for field, _ in cls._fields_]
        lines.append('printf("\\n");')
    source = tmp_path / "layout.c"
    source.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", str(HEADER_DIR), str(source), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout
    for line in out.splitlines():
        name, size, *offsets = line.split()
        cls = structs[name]
        assert int(size) == ctypes.sizeof(cls), name
        assert [int(o) for o in offsets] == [getattr(cls, f).offset for f, _ in cls._fields_], name


def test_ops_offer_the_serving_operators():
    for name in ("rope", "kv_append", "paged_attention", "linear_w4"):
        assert callable(getattr(cmpext3.ops, name)) and callable(getattr(cmpext3.ops, name + "_plan"))
        assert name in N.__all__


# ---- refusals of the binding ------------------------------------------------------------------

def test_cpu_tensors_are_refused():
    x = torch.randn(1, 2, 3, 8)
    i = torch.zeros(1, dtype=torch.int32)
    refused("CUDA", cmpext3.ops.rope, x, torch.arange(3), torch.ones(4))
    refused("CUDA", cmpext3.ops.kv_append, x, x, x, x, i[None], i)
    refused("CUDA", cmpext3.ops.paged_attention, x, x, x, i[None], i)
    refused("CUDA", cmpext3.ops.linear_w4, torch.randn(2, 64), torch.zeros(3, 32, dtype=torch.uint8), torch.ones(3, 1))


def test_rope_refusals(cpu):
    x, p, f = torch.randn(2, 3, 5, 8), torch.arange(5), torch.ones(4)
    ops = cmpext3.ops
    refused("freqs must be a Tensor", ops.rope, x, p, [1.0], error=TypeError)
    refused("positions must be a Tensor", ops.rope, x, None, f, error=TypeError)
    refused("positions must be a Tensor", ops.rope, x, 3, f, error=TypeError)
    refused("int32, int64 or float32", ops.rope, x, p.half(), f)
    refused("freqs must be torch.float32", ops.rope, x, p, f.double())
    refused("freqs must be 1D", ops.rope, x, p, f[None])
    refused("1 to head_dim // 2", ops.rope, x, p, torch.ones(5))
    refused("1 to head_dim // 2", ops.rope, x, p, torch.ones(0))
    refused("positions .* must be", ops.rope, x, torch.arange(4), f)
    refused("positions .* must be", ops.rope, x, torch.zeros(3, 5), f)
    refused("positions .* must be", ops.rope, x, torch.zeros(2, 2, 5), f)
    refused("must begin with the 2 axes", ops.rope, x, torch.zeros(3, 5), f, (2, 2))
    refused("must begin with the 2 axes", ops.rope, x, torch.tensor(0), f, (2, 2))
    refused("add up to 4", ops.rope, x, torch.zeros(2, 5), f, (2, 1))
    refused("add up to 4", ops.rope, x, torch.zeros(2, 5), f, (5, -1))
    refused("sections must be 1 to 4", ops.rope, x, torch.zeros(5, 5), f, (1, 1, 1, 1, 0))
    refused("sections must be 1 to 4", ops.rope, x, torch.zeros(0, 5), f, ())
    refused("whole numbers", ops.rope, x, torch.zeros(2, 5), f, (2.0, 2.0), error=TypeError)
    refused("whole numbers", ops.rope, x, torch.zeros(2, 5), f, (torch.tensor(2), 2), error=TypeError)
    refused("no gradient", ops.rope, x, p, f.clone().requires_grad_())
    refused("no gradient", ops.rope, x, p.float().requires_grad_(), f)


def _cache_args(B=2, Hkv=2, D=16, page=4, pages=3, width=2, dtype=torch.float32):
    cache = [torch.zeros(pages, Hkv, page, D, dtype=dtype) for _ in range(2)]
    return cache + [torch.zeros(B, width, dtype=torch.int32), torch.ones(B, dtype=torch.int32)]


def _cache_refusals(call):
    """call(k_cache, v_cache, page_table, lengths) with one argument wrong at a time."""
    kc, vc, table, lengths = _cache_args()
    refused("k_cache must be torch.float32", call, kc.half(), vc, table, lengths)
    refused("v_cache must be 4D", call, kc, vc[0], table, lengths)
    refused("does not match k_cache", call, kc, vc[:, :, :2], table, lengths)
    refused("none of the last three 0", call, kc[:, :, :0], vc[:, :, :0], table, lengths)
    refused("contiguous along head_dim", call, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, table, lengths)
    refused("page_table must be torch.int32", call, kc, vc, table.long(), lengths)
    refused("lengths must be torch.int32", call, kc, vc, table, lengths.long())
    refused("page_table must be 2D", call, kc, vc, table[0], lengths)
    refused("must have batch 2 rows", call, kc, vc, table[:1], lengths)
    refused("must have batch 2 rows", call, kc, vc, table, lengths[:1])
    refused("must be contiguous", call, kc, vc, torch.zeros(2, 2, dtype=torch.int32).t(), lengths)
    refused("must be contiguous", call, kc, vc, table, torch.zeros(4, dtype=torch.int32)[::2])
    refused("lengths must be a Tensor", call, kc, vc, table, [1, 1], error=TypeError)


def test_a_leaf_with_an_eager_graph_is_refused_in_a_capture(monkeypatch):
    # the note on the leaf's autograd node, with the streams played on the CPU
    stream = [0]
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: stream[0], raising=False)
    x = torch.randn(3, requires_grad=True)
    S._check_leaf(x)
    eager = x * 2
    S._note_leaf(eager, x.device)
    with pytest.raises(RuntimeError, match="eager graph of this leaf"):
        S._check_leaf(x)
    del eager                          # the node goes with the last graph that uses it
    S._check_leaf(x)
    stream[0] = 5                      # a warm-up on a side stream may stay alive
    eager = x * 2
    S._note_leaf(eager, x.device)
    S._check_leaf(x)


def test_kv_append_refusals(cpu):
    ops = cmpext3.ops
    k, q, f = torch.randn(2, 2, 3, 16), torch.randn(2, 4, 3, 16), torch.ones(8)
    args = _cache_args()
    _cache_refusals(lambda *c: ops.kv_append(k, k, *c))
    refused("value .* does not match key", ops.kv_append, k, k[:, :, :2], *args)
    refused("value must be torch.float32", ops.kv_append, k, k.half(), *args)
    refused("does not hold key", ops.kv_append, k[..., :8], k[..., :8], *args)
    refused("does not hold key", ops.kv_append, k[:, :1], k[:, :1], *args)
    refused("query .* does not match key", ops.kv_append, k, k, *args, query=q[:, :, :2])
    refused("query must be torch.float32", ops.kv_append, k, k, *args, query=q.half())
    refused("new_lengths must be torch.int32", ops.kv_append, k, k, *args, torch.ones(2))
    refused("new_lengths must be 2", ops.kv_append, k, k, *args, torch.ones(3, dtype=torch.int32))
    refused("need freqs", ops.kv_append, k, k, *args, positions=torch.arange(3))
    refused("need freqs", ops.kv_append, k, k, *args, sections=(8,))
    refused("need positions", ops.kv_append, k, k, *args, freqs=f, sections=(8,))
    refused("no gradient", ops.kv_append, k.clone().requires_grad_(), k, *args)
    one = torch.zeros(1, 2, 4, 16)
    refused("expanded", ops.kv_append, k, k, one.expand(3, 2, 4, 16), args[1], *args[2:])


def test_paged_attention_refusals(cpu):
    ops = cmpext3.ops
    q, args = torch.randn(2, 4, 1, 16), _cache_args()
    _cache_refusals(lambda *c: ops.paged_attention(q, *c))
    refused("one token per sequence", ops.paged_attention, torch.randn(2, 4, 2, 16), *args)
    refused("does not match query", ops.paged_attention, q[..., :8], *args)
    refused("does not match query", ops.paged_attention, torch.randn(2, 3, 1, 16), *args)
    refused("scale must be finite", ops.paged_attention, q, *args, float("inf"))
    refused("no gradient", ops.paged_attention, q.clone().requires_grad_(), *args)


def test_linear_w4_refusals(monkeypatch):
    monkeypatch.setattr(S, "_run", lambda *a: pytest.fail("the call was not refused"))
    ops = cmpext3.ops

    class Cuda(torch.Tensor):   # a CPU tensor that passes the device check
        is_cuda = True
    x, w, s = torch.randn(3, 64).as_subclass(Cuda), torch.zeros(5, 32, dtype=torch.uint8), torch.ones(5, 2)
    refused("input must be a Tensor", ops.linear_w4, [1.0], w, s, error=TypeError)
    refused("weight must be torch.uint8", ops.linear_w4, x, w.int(), s)
    refused("weight must be 2D", ops.linear_w4, x, w[0], s)
    refused("scales must be torch.float32", ops.linear_w4, x, w, s.half())
    refused("does not match weight", ops.linear_w4, x[:, :32], w, s)
    refused("scales .* must be", ops.linear_w4, x, w, s[:4])
    refused("scales .* must be", ops.linear_w4, x, w, torch.ones(5, 4))      # groups of 16
    refused("scales .* must be", ops.linear_w4, x, w, torch.ones(5, 3))
    refused("scales .* must be", ops.linear_w4, x, w, torch.ones(5, 0))
    refused("zeros must be torch.uint8", ops.linear_w4, x, w, s, s)
    refused("zeros .* does not match", ops.linear_w4, x, w, s, torch.zeros(5, 1, dtype=torch.uint8))
    refused("bias must have 5", ops.linear_w4, x, w, s, None, torch.ones(4))
    refused("bias must be torch.float32", ops.linear_w4, x, w, s, None, torch.ones(5).half())
    refused("no gradient", ops.linear_w4, x, w, s.clone().requires_grad_())


# ---- refusals of the C ABI --------------------------------------------------------------------

PTR = 0x10000


def _status(fn, desc):
    buf = ctypes.create_string_buffer(128)
    return fn(ctypes.byref(desc), buf, 128), buf.value.decode()


def _rotation(pairs=32, axes=1, kind=1, ends=None):
    ends = ends or (pairs, 0, 0, 0)
    return S.Rotation(PTR, PTR, S._I64x3(0, 0, 1), kind, pairs, axes, 0, S._I32x4(*ends))


def _rope(dtype=2, D=64, ptr=PTR, stride=64, **rot):
    return S.RopeDesc(ptr, PTR, _rotation(**rot), 2, 3, 5, D, S._I64x3(15 * stride, 5 * stride, stride),
                      S._I64x3(15 * D, 5 * D, D), dtype, 0)


def test_rope_plans_and_statuses():
    f = N.lib.cmpx_rope_plan
    assert _status(f, _rope()) == (N.OK, "rope<16-byte vectors>")
    assert _status(f, _rope(stride=66)) == (N.OK, "rope<4-byte vectors>")
    assert _status(f, _rope(stride=65)) == (N.OK, "rope<single values>")
    assert _status(f, _rope(ptr=PTR + 2)) == (N.OK, "rope<single values>")
    assert _status(f, _rope(pairs=10)) == (N.OK, "rope<4-byte vectors>")
    assert _status(f, _rope(dtype=7))[0] == N.ERR_UNSUPPORTED_DTYPE
    assert _status(f, _rope(D=512, stride=512))[0] == N.ERR_UNSUPPORTED_SHAPE
    for bad in (dict(pairs=33), dict(pairs=-1), dict(axes=0), dict(axes=5), dict(kind=0), dict(kind=4),
                dict(axes=2, ends=(20, 30, 0, 0)), dict(axes=2, ends=(40, 32, 0, 0))):
        assert _status(f, _rope(**bad))[0] == N.ERR_INVALID_ARGUMENT, bad
    assert N.lib.cmpx_rope(None, None) == N.ERR_INVALID_ARGUMENT
    d = _rope()
    d.len = 0
    assert N.lib.cmpx_rope(ctypes.byref(d), None) == N.OK      # nothing to do


def _cache(D=64, page=16, pages=100, Hkv=2, width=8, ptr=PTR):
    st = S._I64x3(Hkv * page * D, page * D, D)
    return S.PagedCache(ptr, PTR, PTR, PTR, pages, page, Hkv, D, st, st, width, width)


def _attn(dtype=2, H=8, B=3, scale=0.1, **cache):
    c = _cache(**cache)
    st = S._I64x2(H * c.head_dim, c.head_dim)
    return S.PagedAttnDesc(PTR, PTR, None, c, 0, B, H, st, st, scale, dtype, 0)


def test_paged_attention_plans_and_statuses():
    f = N.lib.cmpx_paged_attn_plan
    assert _status(f, _attn()) == (N.OK, "paged_attn<one CTA per item>")
    assert _status(f, _attn(width=200)) == (N.OK, "paged_attn<cluster per item>")
    assert _status(f, _attn(width=1000)) == (N.OK, "paged_attn<equal shares, join>")
    assert _status(f, _attn(width=200, B=300)) == (N.OK, "paged_attn<equal shares, join>")
    assert _status(f, _attn(dtype=3))[0] == N.ERR_UNSUPPORTED_DTYPE
    for bad in (dict(H=7), dict(scale=float("nan")), dict(page=0), dict(Hkv=0, H=0), dict(pages=-1), dict(ptr=None)):
        assert _status(f, _attn(**bad))[0] == N.ERR_INVALID_ARGUMENT, bad
    for bad in (dict(D=264), dict(D=4), dict(D=12), dict(width=2 ** 28)):
        assert _status(f, _attn(**bad))[0] == N.ERR_UNSUPPORTED_SHAPE, bad
    assert _status(f, _attn(dtype=0, D=4))[0] == N.OK
    assert _status(f, _attn(ptr=PTR + 8))[0] == N.ERR_MISALIGNED
    d = _attn()
    d.q = PTR + 2
    assert _status(f, d)[0] == N.ERR_MISALIGNED
    assert N.lib.cmpx_paged_attn(None, None) == N.ERR_INVALID_ARGUMENT
    assert N.lib.cmpx_paged_attn_workspace_size(None) == 0
    assert N.lib.cmpx_paged_attn_workspace_size(ctypes.byref(_attn())) == 0
    assert N.lib.cmpx_paged_attn_workspace_size(ctypes.byref(_attn(width=1000))) > 0


def _append(dtype=2, H=4, **cache):
    c = _cache(**cache)
    st = S._I64x3(c.heads_kv * 5 * c.head_dim, 5 * c.head_dim, c.head_dim)
    return S.KvAppendDesc(PTR, PTR, PTR if H else None, PTR if H else None, None, c, _rotation(kind=0), 2, H, 5,
                          st, st, st, st, dtype, 0)


def test_kv_append_plans_and_statuses():
    f = N.lib.cmpx_kv_append_plan
    assert _status(f, _append()) == (N.OK, "kv_append<16-byte vectors>")
    assert _status(f, _append(H=0)) == (N.OK, "kv_append<16-byte vectors>")
    d = _append()
    d.k_in_stride[2] = 65
    assert _status(f, d) == (N.OK, "kv_append<single values>")
    assert _status(f, _append(ptr=PTR + 2))[0] == N.ERR_MISALIGNED
    assert _status(f, _append(dtype=9))[0] == N.ERR_UNSUPPORTED_DTYPE
    assert _status(f, _append(D=60))[0] == N.ERR_INVALID_ARGUMENT          # 32 pairs do not fit
    d = _append()
    d.q = None
    assert _status(f, d)[0] == N.ERR_INVALID_ARGUMENT
    assert N.lib.cmpx_kv_append(None, None) == N.ERR_INVALID_ARGUMENT


def _linear(m=2, n=10, k=256, group=64, dtype=2, xs=None, ws=None, ptr=PTR):
    return S.LinearW4Desc(ptr, PTR, PTR, None, None, PTR, m, n, k, group, xs or k, n, ws or k // 2, k // group, 0, dtype, 0)


def test_linear_w4_plans_and_statuses():
    f = N.lib.cmpx_linear_w4_plan
    assert _status(f, _linear())[0] == N.OK
    for bad in (dict(k=0), dict(group=0), dict(group=96)):
        assert _status(f, _linear(**bad) if bad != dict(group=0) else S.LinearW4Desc(
            PTR, PTR, PTR, None, None, PTR, 2, 10, 256, 0, 256, 10, 128, 4, 0, 2, 0))[0] == N.ERR_INVALID_ARGUMENT, bad
    assert _status(f, _linear(group=16))[0] == N.ERR_UNSUPPORTED_SHAPE
    assert _status(f, _linear(ws=(1 << 27) + 16))[0] == N.ERR_UNSUPPORTED_SHAPE
    assert _status(f, _linear(n=1 << 30, k=1 << 20))[0] == N.ERR_UNSUPPORTED_SHAPE
    assert _status(f, _linear(dtype=4))[0] == N.ERR_UNSUPPORTED_DTYPE
    assert _status(f, _linear(xs=257))[0] == N.ERR_MISALIGNED
    assert _status(f, _linear(ws=130))[0] == N.ERR_MISALIGNED
    assert _status(f, _linear(ptr=PTR + 4))[0] == N.ERR_MISALIGNED
    assert N.lib.cmpx_linear_w4(None, None) == N.ERR_INVALID_ARGUMENT


def test_the_new_device_flag_is_the_header_s():
    text = (HEADER_DIR / "cmpx_b200.h").read_text()
    assert f"#define CMPX_DEVFLAG_BAD_PAGE {N.DEVFLAG_BAD_PAGE}u" in text


# ---- the schedule of the paged attention ------------------------------------------------------

TILE, COST, LEAST = 16, 3, 6


def _stretches(lengths, items, workers):
    """What every warp does, as the kernels find it: (sequence, item, tile0, tile1, slot or None)."""
    tiles = [max(1, -(-n // TILE)) for n in lengths]
    total = sum((t + COST) * items for t in tiles)
    share = max(LEAST, -(-total // workers))
    out = []
    for w in range(workers):
        cur, end = w * share, min(total, (w + 1) * share)
        before, b = 0, 0
        while cur < end:
            units = tiles[b] + COST
            while cur >= before + units * items:
                before += units * items
                b += 1
                units = tiles[b] + COST
            item, unit0 = divmod(cur - before, units)
            unit1 = min(units, unit0 + end - cur)
            cur += unit1 - unit0
            tile0, tile1 = max(unit0 - COST, 0), unit1 - COST
            if tile1 <= tile0:
                continue
            whole = tile0 == 0 and tile1 == tiles[b]
            out.append((b, item, tile0, tile1, None if whole else 2 * w + (tile0 == 0)))
    return tiles, total, share, out


def test_every_tile_is_done_once_and_the_join_finds_every_part():
    rng = random.Random(0)
    for _ in range(400):
        lengths = [rng.choice([0, 1, 15, 16, 17, rng.randrange(1, 3000)]) for _ in range(rng.randrange(1, 12))]
        items, workers = rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 7, 64, 1184])
        tiles, total, share, stretches = _stretches(lengths, items, workers)
        done, slots = {}, set()
        for b, item, t0, t1, slot in stretches:
            done.setdefault((b, item), []).append((t0, t1, slot))
            assert slot is None or slot not in slots
            slots.add(slot) if slot is not None else None
        first = 0
        for b, t in enumerate(tiles):
            for item in range(items):
                parts = sorted(done[b, item])
                assert parts[0][0] == 0 and parts[-1][1] == t
                assert all(x[1] == y[0] for x, y in zip(parts, parts[1:]))
                begin = first + item * (t + COST) + COST       # as the join kernel finds the slots
                c0, c1 = begin // share, (begin + t - 1) // share
                want = [None] if c0 == c1 else [2 * c + (c == c0) for c in range(c0, c1 + 1)]
                assert [p[2] for p in parts] == want
            first += items * (t + COST)


def test_divisions_by_the_page_size_are_exact():
    rng = random.Random(1)
    for d in list(range(1, 400)) + [2 ** i + j for i in range(9, 31) for j in (-1, 0, 1)] + [2 ** 31 - 1]:
        log2 = (d - 1).bit_length()
        p = 31 + log2
        m = -(-2 ** p // d)
        assert m < 2 ** 32
        for t in [0, 1, d - 1, d, 2 * d - 1, 2 ** 31 - 1] + [rng.randrange(2 ** 31) for _ in range(20)]:
            if t < 2 ** 31:
                assert (t * m) >> p == t // d


def test_traced_ranges_wrap_the_serving_operators():
    code = ("import sys; sys.path[:0] = ['torch-cmp-patch_b200', '.']\n"
            "from cmpext3 import _native as N\n"
            "assert all(hasattr(f, '__wrapped__') for f in (N.rope, N.kv_append, N.paged_attention, N.linear_w4))\n"
            "print('ok')\n")
    import os
    env = dict(os.environ, CMPEXT3_NVTX="1", CMPEXT3_AUTOPATCH="0")
    out = subprocess.run([sys.executable, "-c", code], cwd=HEADER_DIR.parent, env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stderr[-2000:]
