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
