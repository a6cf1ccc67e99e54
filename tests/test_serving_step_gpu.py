"""The serving operators together, as a transformer layer's step uses them (needs a B200; marked gpu): 4-bit
projections, the rotated append, one-token attention over the paged cache, the 4-bit output projection -- eagerly
and replayed from one captured graph whose lengths move on -- and a prompt through rope and SDPA against
the same prompt through the cache."""
from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import cmpext3
from cmpext3 import _native as N
from tests import serving_oracle as O

pytestmark = pytest.mark.gpu

H, HKV, D, PAGE, MODEL = 8, 2, 64, 16, 512
QKV = (H + 2 * HKV) * D


def _w4(n, k, group, dtype, gen):
    w = torch.randint(0, 256, (n, k // 2), generator=gen, dtype=torch.uint8)
    s = (torch.rand(n, k // group, generator=gen) * 0.01 + 0.002).to(dtype)
    z = torch.randint(6, 10, (n, k // group), generator=gen, dtype=torch.uint8)
    return w, s, z


class Layer:
    def __init__(self, dtype, batch, room, dev, seed):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.dev = dtype, dev
        self.qkv, self.out = _w4(QKV, MODEL, 128, dtype, g), _w4(MODEL, H * D, 64, dtype, g)
        width = -(-room // PAGE)
        pages = batch * width + 2
        self.table = torch.randperm(pages, generator=g)[:batch * width].reshape(batch, width).to(torch.int32)
        self.freqs = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float()
        self.k, self.v = (torch.zeros(pages, HKV, PAGE, D, dtype=dtype, device=dev) for _ in range(2))
        self.on = [tuple(t.to(dev) for t in w) for w in (self.qkv, self.out)] + [self.table.to(dev), self.freqs.to(dev)]

    def project(self, x):
        """x [batch, tokens, MODEL] -> query, key, value [batch, heads, tokens, D] views of one tensor."""
        qkv = cmpext3.ops.linear_w4(x, *self.on[0]).unflatten(-1, (H + 2 * HKV, D)).transpose(1, 2)
        return qkv[:, :H], qkv[:, H:H + HKV], qkv[:, H + HKV:]

    def step(self, x, lengths):
        """x [batch, 1, MODEL]; everything that the step computed."""
        q, k, v = self.project(x)
        turned = cmpext3.ops.kv_append(k, v, self.k, self.v, self.on[2], lengths, query=q, freqs=self.on[3])
        a = cmpext3.ops.paged_attention(turned, self.k, self.v, self.on[2], lengths)
        y = cmpext3.ops.linear_w4(a.transpose(1, 2).flatten(2), *self.on[1])
        return q, k, v, turned, a, y

    def kept(self, b, n):
        """Keys and values [HKV, n, D] that the cache holds for sequence b."""
        at = torch.arange(n)
        pages = self.table[b].long()[at // PAGE]
        return tuple(c.cpu()[pages, :, at % PAGE].transpose(0, 1) for c in (self.k, self.v))

    def check(self, x, lengths, results):
        q, k, v, turned, a, y = (t.cpu() for t in results)
        want, bound = O.linear_w4(x.reshape(-1, MODEL).cpu(), *self.qkv)
        got = torch.cat((q, k, v), 1).transpose(1, 2).flatten(2)[:, 0]
        O.assert_within(got, want, bound, "projection")
        place = torch.tensor(lengths)[:, None] - 1
        O.assert_within(turned, *O.rope(q, place, self.freqs), "turned query")
        kt, kb = O.rope(k, place, self.freqs)
        for b, n in enumerate(lengths):
            ck, cv = self.kept(b, n)
            O.assert_within(ck[:, -1], kt[b, :, 0], kb[b, :, 0], "stored key")
            assert torch.equal(cv[:, -1], v[b, :, 0])
            O.assert_within(a[b, :, 0], *O.attention(turned[b, :, 0], ck, cv, D ** -0.5), "attention")
        O.assert_within(y[:, 0], *O.linear_w4(a.transpose(1, 2).flatten(2)[:, 0], *self.out), "output projection")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
def test_decoding_steps_eager_and_from_a_graph(cuda_device, dtype):
    g = torch.Generator().manual_seed(1)
    layer = Layer(dtype, 3, 200, cuda_device, seed=2)
    lengths = [1, 16, 100]            # a first token, a page's end, the middle
    now = torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    x = torch.randn(3, 1, MODEL, generator=g).to(dtype).to(cuda_device)
    for c in (layer.k, layer.v):
        c.normal_()
    layer.check(x, lengths, layer.step(x, now))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step(x, now)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        now.add_(1)
        results = layer.step(x, now)
    for step in range(4):
        x.copy_(torch.randn(3, 1, MODEL, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        layer.check(x, [n + 1 + step for n in lengths], results)
    assert N.device_status() == 0


def test_a_prompt_through_the_cache_matches_rope_and_sdpa(cuda_device, patched):
    # the prompt's last token by one-token attention over the cache, and by rope + causal SDPA over the prompt
    n, dtype = 150, torch.bfloat16
    layer = Layer(dtype, 2, n, cuda_device, seed=3)
    x = torch.randn(2, n, MODEL, generator=torch.Generator().manual_seed(4)).to(dtype).to(cuda_device)
    with torch.no_grad():
        q, k, v = layer.project(x)
        positions = torch.arange(n, device=cuda_device)
        qr, kr = (cmpext3.ops.rope(t, positions, layer.on[3]) for t in (q, k))
        dense = F.scaled_dot_product_attention(qr, kr, v, is_causal=True, enable_gqa=True)
        now = torch.full((2,), n, dtype=torch.int32, device=cuda_device)
        turned = cmpext3.ops.kv_append(k, v, layer.k, layer.v, layer.on[2], now, query=q, freqs=layer.on[3])
        assert torch.equal(turned, qr)
        for b in range(2):
            ck, cv = layer.kept(b, n)
            assert torch.equal(ck, kr[b].cpu()) and torch.equal(cv, v[b].cpu())
        last = cmpext3.ops.paged_attention(turned[:, :, -1:], layer.k, layer.v, layer.on[2], now)
    for b in range(2):
        want, bound = O.attention(qr[b, :, -1].cpu(), kr[b].cpu(), v[b].cpu(), D ** -0.5)
        O.assert_within(last[b, :, 0], want, bound, "paged")
        # the SDPA kernel rounds its weights, which add up to 1, to bf16 before the second product
        O.assert_within(dense[b, :, -1], want, bound + 2.0 ** -8 * v[b].cpu().double().abs().amax(), "dense")
