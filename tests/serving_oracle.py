"""64-bit definitions of the serving operators on CPU tensors, and the error their kernels may have.

Bounds are sums of: the one rounding to the output type (eps / 2 of the value, half the smallest step
below the normal range), and the fp32 arithmetic before it (each addition or product is off by at most
2^-24 of its result, a tensor-core addition by 2^-23)."""
from __future__ import annotations

import math

import torch

TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}


def rounding(value: torch.Tensor, dtype) -> torch.Tensor:
    return value.abs() * (torch.finfo(dtype).eps / 2) + TINY[dtype]


def assert_within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    g = got.detach().cpu().double()
    assert g.shape == want.shape, (what, g.shape, want.shape)
    assert torch.isfinite(g).all(), f"{what}: not finite"
    off = (g - want).abs() - bound
    worst = off.max().item() if off.numel() else 0.0
    at = int(off.argmax()) if off.numel() else 0
    assert worst <= 0, (f"{what}: value {at} is {(g - want).abs().flatten()[at].item():.3e} off, "
                        f"{bound.expand_as(want).flatten()[at].item():.3e} allowed")


def rope(x, positions, freqs, sections=None, interleaved=False, sign=1.0):
    """(turned, bound): x [B, H, L, D] CPU; positions as cmpext3.ops.rope takes them."""
    b, _, n, _ = x.shape
    pairs = freqs.numel()
    pos = positions.double()
    if sections is None:
        angle = pos.expand(b, n)[..., None] * freqs.double()
    else:
        pos = pos[:, None, :].expand(len(sections), b, n) if pos.dim() == 2 else pos.expand(len(sections), b, n)
        axis = [a for a, c in enumerate(sections) for _ in range(c)]
        angle = torch.stack([pos[a] * freqs[j].double() for j, a in enumerate(axis)], -1)
    cos, sin = torch.cos(angle)[:, None], sign * torch.sin(angle)[:, None]
    out = x.double().clone()
    size, far = torch.zeros_like(out), torch.zeros_like(out)
    re, im = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    u, w = x[..., re].double(), x[..., im].double()
    out[..., re], out[..., im] = u * cos - w * sin, u * sin + w * cos
    size[..., re] = size[..., im] = u.abs() + w.abs()
    far[..., re] = far[..., im] = angle.abs()[:, None].expand_as(u)
    # cos and sin are off by at most 2^-23 (half a step of the fp32 remainder, and their
    # polynomials' own), the two products and the sum by 2^-24 each of at most |u| + |w|; an angle of a
    # radians carries four roundings of 2^-53 a between the kernel and this definition
    return out, rounding(out, x.dtype) + size * (2.0 ** -21 + far * 2.0 ** -51)


def attention(q, k, v, scale):
    """(out, bound) of one sequence: q [H, D], k and v [Hkv, n, D]."""
    h, d = q.shape
    group = h // k.shape[0]
    out, bound = torch.zeros(h, d, dtype=torch.float64), torch.zeros(h, d, dtype=torch.float64)
    if k.shape[1]:
        kk, vv = (t.double().repeat_interleave(group, 0) for t in (k, v))
        qq = q.double()[:, None]
        s = (qq @ kk.transpose(1, 2)) * scale
        size = (qq.abs() @ kk.abs().transpose(1, 2)).amax(-1, keepdim=True) * abs(scale)
        p = torch.softmax(s, -1)
        out = (p @ vv)[:, 0]
        # a score is a sum of d products and two more factors (2^-23 each of the sum of sizes); a
        # weight takes twice that (its own score and the maximum's), the exponential's 2^-21 and, for
        # 16-bit types, 2^-16 for two 16-bit parts; the sums over the keys carry at most n + 64 additions, in
        # chains of which no term passes more than 1/8 (eight warps or more)
        weight = 2 * (d + 4) * 2.0 ** -23 * size + 2.0 ** -21 + (2.0 ** -16 if q.dtype != torch.float32 else 0.0)
        adds = (k.shape[1] / 8 + 64) * 2.0 ** -23
        bound = ((2 * weight + 2 * adds) * (p @ vv.abs()))[:, 0]
    return out, bound + rounding(out, q.dtype)


def linear_w4(x, weight, scales, zeros=None, bias=None):
    """(y, bound): CPU tensors as cmpext3.ops.linear_w4 takes them, x [M, K]."""
    n, k = weight.shape[0], 2 * weight.shape[1]
    group = k // scales.shape[1]
    codes = torch.stack((weight & 15, weight >> 4), -1).reshape(n, -1, group).double()
    z = 8.0 if zeros is None else zeros.double()[..., None]
    w = ((codes - z) * scales.double()[..., None]).reshape(n, k)
    y, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    # a term passes at most group additions in its group, one product with the scale, one addition a
    # group, and 16 more between lanes, warps and the bias
    return y, rounding(y, x.dtype) + (group + k // group + 20) * 2.0 ** -23 * size
