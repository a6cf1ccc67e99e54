"""Calls of the serving operators at the edges of what they take, without a GPU: views with odd strides, arguments that
look like kept ones, derivatives that the kernels do not carry."""
from __future__ import annotations

import pytest
import torch

import cmpext3
from cmpext3 import _native as N
from cmpext3 import _serving as S
from tests.test_serving_host import _cache_args, cpu, refused  # noqa: F401


# ---- strides of dimensions of size one ---------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_a_query_s_stride_along_a_dimension_of_one_does_not_count(cpu, dtype):
    kc, vc, table, lengths = _cache_args(B=4, D=64, dtype=dtype)
    rows = torch.zeros(4, 515, dtype=dtype)[:, :512].unflatten(1, (8, 64)).unsqueeze(2)   # as a projection leaves them
    one = rows[0:1]                                                  # contiguous for torch, with a stride of 515
    assert one.is_contiguous() and one.stride(0) == 515
    assert "paged_attn" in N.paged_attention_plan(one, kc, vc, table[:1], lengths[:1])
    assert S._paged_attn_desc(one, kc, vc, table[:1], lengths[:1], None)[2] is one               # and it is not copied
    heads = torch.zeros(3, 1, 1, 515, dtype=dtype)[..., :64].as_strided((3, 1, 1, 64), (64, 515, 64, 1))
    assert "paged_attn" in N.paged_attention_plan(heads, kc[:, :1], vc[:, :1], table[:3], lengths[:3])
    desc, out, used = S._paged_attn_desc(rows, kc, vc, table, lengths, None)                # rows on odd boundaries are copied
    assert used is not rows and desc.q_stride[0] * rows.element_size() % 16 == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_strides_along_dimensions_of_one_do_not_narrow_the_vectors_or_refuse_a_cache(cpu, dtype):
    def odd(shape, at):
        """Zeros of this shape, whose dimension `at`, of one, has an odd stride."""
        t = torch.zeros(shape, dtype=dtype)
        stride = list(t.stride())
        stride[at] = 12345
        return t.as_strided(shape, stride)
    positions, freqs = torch.arange(5), torch.ones(32)
    for shape, at, p in (((1, 3, 5, 64), 0, positions), ((2, 1, 5, 64), 1, positions), ((2, 3, 1, 64), 2, positions[:1])):
        assert N.rope_plan(odd(shape, at), p, freqs) == "rope<16-byte vectors>"
    i32 = dict(dtype=torch.int32)
    for shape, at in (((1, 2, 16, 64), 0), ((4, 1, 16, 64), 1), ((4, 2, 1, 64), 2)):
        heads = shape[1]
        cache, table, lengths = odd(shape, at), torch.zeros(1, 2, **i32), torch.ones(1, **i32)
        row = odd((1, heads, 1, 64), 0)
        assert N.kv_append_plan(row, row, cache, cache, table, lengths, query=row, freqs=freqs) == "kv_append<16-byte vectors>"
        assert "paged_attn" in N.paged_attention_plan(row, cache, cache, table, lengths)
    wide = torch.zeros(3, 2, 4, 67, dtype=dtype)[..., :64]            # rows that are apart by 67 do count
    assert N.rope_plan(wide, torch.arange(4), freqs) == "rope<single values>"
    with pytest.raises(N.CmpxError):
        N.paged_attention_plan(torch.zeros(1, 2, 1, 64, dtype=dtype), wide, wide, torch.zeros(1, 2, **i32), torch.ones(1, **i32))


def test_a_single_row_of_4_bit_weights_may_have_any_stride():
    from tests.test_serving_host import _linear, _status
    assert _status(N.lib.cmpx_linear_w4_plan, _linear(n=1, ws=(1 << 27) + 3))[0] == N.OK
    assert _status(N.lib.cmpx_linear_w4_plan, _linear(m=1, xs=257))[0] == N.OK
    assert _status(N.lib.cmpx_linear_w4_plan, _linear(n=2, ws=(1 << 27) + 16))[0] == N.ERR_UNSUPPORTED_SHAPE


# ---- derivatives -------------------------------------------------------------------------------

def test_dual_tensors_are_refused(cpu):
    # their tangents would be lost: in each differentiable argument, with autograd on and off
    from torch.autograd import forward_ad as fa
    ops = cmpext3.ops
    x, p, f = torch.randn(2, 2, 3, 16), torch.arange(3.0), torch.ones(8)
    k, v, table, lengths = _cache_args()
    one = torch.randn(2, 4, 1, 16)
    w, act, scale, bias = torch.zeros(5, 32, dtype=torch.uint8), torch.randn(3, 64), torch.ones(5, 2), torch.ones(5)
    calls = [(ops.rope, (x, p, f), (0, 1, 2)),
             (lambda *a: ops.kv_append(*a[:6], query=a[6], positions=a[7], freqs=a[8]),
              (x, x.clone(), k, v, table, lengths, x.clone(), p, f), (0, 1, 2, 3, 6, 7, 8)),
             (ops.paged_attention, (one, k, v, table, lengths), (0, 1, 2)),
             (lambda *a: ops.linear_w4(*a[:3], None, a[3]), (act, w, scale, bias), (0, 2, 3))]
    with fa.dual_level():
        for call, args, wheres in calls:
            for i in wheres:
                dual = list(args)
                dual[i] = fa.make_dual(args[i].clone(), torch.ones_like(args[i]))
                refused("no forward-mode derivative", call, *dual)
                with torch.no_grad():
                    refused("no forward-mode derivative", call, *dual)
                dual[i] = dual[i].detach()
                with pytest.raises(BaseException) as e:   # detached it goes on to the device check or the launch
                    call(*dual)
                assert "forward-mode" not in str(e.value)


def test_a_gradient_with_a_tangent_is_refused_in_the_backward_pass(cpu, monkeypatch):
    from torch.autograd import forward_ad as fa
    monkeypatch.setattr(S, "_run", lambda *a: None)
    monkeypatch.setattr(S, "_note_leaf", lambda *a: None)
    x, p, f = torch.randn(1, 2, 3, 16, requires_grad=True), torch.arange(3), torch.ones(8)
    y = cmpext3.ops.rope(x, p, f)
    with fa.dual_level():
        grad = fa.make_dual(torch.ones_like(y), torch.ones_like(y))
        refused("no forward-mode derivative", torch.autograd.grad, y, x, grad)


# ---- kept signatures ---------------------------------------------------------------------------

def test_sections_that_equal_kept_ones_are_refused_all_the_same(cpu, monkeypatch):
    class Kept(dict):
        def get(self, key, default=None):
            return (b"", b"", 0) if key[0] == "kv_append" else (b"", 0)
    monkeypatch.setattr(S, "_SIGNATURES", Kept())
    monkeypatch.setattr(S, "_direct", lambda *a: N.OK)
    x, f = torch.randn(2, 2, 3, 16), torch.ones(8)
    positions, cache = torch.zeros(2, 3), _cache_args()
    cmpext3.ops.rope(x, positions, f, (4, 4))
    for sections in ((4.0, 4.0), [4, 4.0], (True, 7), (torch.tensor(4), 4)):
        refused("whole numbers", cmpext3.ops.rope, x, positions, f, sections, error=TypeError)
        refused("whole numbers", cmpext3.ops.kv_append, x, x, *cache, positions=positions, freqs=f, sections=sections,
                error=TypeError)


# ---- the scale ---------------------------------------------------------------------------------

def test_a_scale_that_is_infinite_in_fp32_is_refused(cpu):
    from tests.test_serving_host import _attn, _status
    q, args = torch.randn(2, 4, 1, 16), _cache_args()
    for scale in (1e300, -1e39, 3e38, float("nan"), float("-inf")):
        refused("scale must be finite", cmpext3.ops.paged_attention, q, *args, scale)
        assert _status(N.lib.cmpx_paged_attn_plan, _attn(scale=scale))[0] == N.ERR_INVALID_ARGUMENT
    for scale in (2.3e38, -1e30, 0.0):
        assert "paged_attn" in N.paged_attention_plan(q, *args, scale)
