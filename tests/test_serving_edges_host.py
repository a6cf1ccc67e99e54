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
