"""Close bounds for one-token attention, for random inputs with symmetric signs, and inputs whose result hangs on one key or on
the low parts of values.

The worst case of a sum grows with its length, the sum of values with random signs with its square root only: over
70000 keys a bound of the first kind lets pass what a lost tile would change.  Here errors that each meet a
value of random sign are added up as such: the sum of terms e_i with independent signs is beyond 8 sqrt(sum e_i^2)
with a probability below 2 exp(-32) (Hoeffding)."""
from __future__ import annotations

import torch

from tests import serving_oracle as O

TILES = 32     # tiles that a warp goes through, at most, in the tests that use this
CHAIN = 8 * TILES + 64 + 64   # additions of 2^-23 that a value passes: in a warp (an fp32 tile of 16 keys in
                              # one lane group is 16 of 2^-24), over the parts of an item, between lanes and warps


def attention(q, k, v, scale):
    """(out, bound) of one sequence: q [H, D], k and v [Hkv, n, D], v with independent symmetric signs."""
    h, d = q.shape
    group = h // k.shape[0]
    kk, vv = (t.double().repeat_interleave(group, 0) for t in (k, v))
    qq = q.double()[:, None]
    s = (qq @ kk.transpose(1, 2)) * scale                                            # [H, 1, n]
    p = torch.softmax(s, -1)
    out = (p @ vv)[:, 0]
    # A score's products are off by 1.25 * 2^-20 each at most (two tf32 parts a value, rounded or cut: the product of the rests,
    # 2^-21, and what two rests lose, 2 * 1.5 * 2^-22; less in the other kernels), with the signs of q and k; its 24
    # additions at most (chains of 16 products, of 8 per lane) by 2^-23 of a partial sum, on average of the size below, the
    # maximum's subtraction and the scale's product by 2^-23 of the score.
    size = ((qq ** 2) @ (kk ** 2).transpose(1, 2)).sqrt() * abs(scale) + s.abs()
    # the exponential and the weights' parts
    part = {torch.float32: 2.0 ** -20, torch.float16: 2.0 ** -20, torch.bfloat16: 2.0 ** -16}[q.dtype]
    each = p * (4.25 * 2.0 ** -20 * size + part)
    root = ((p ** 2) @ (vv ** 2)).sqrt()[:, 0]                                          # what out's size is about
    bound = 8 * ((each ** 2) @ (vv ** 2)).sqrt()[:, 0]
    # sums over the keys: partial sums are below 6 times their root mean square; the sum of weights and the quotient
    bound += CHAIN * 2.0 ** -23 * (6 * root + out.abs()) + part * out.abs()
    return out, bound + O.rounding(out, q.dtype)


# ---- one key a column ---------------------------------------------------------------------------

HEIGHT = 2.0 ** 15


def marked(lengths, table, shape, start, dtype, dev):
    """A cache of values [pages, heads, page, dim] that is zero but for HEIGHT at key start + c of each sequence in column c =
    head * dim + d, and the attention with equal weights over it, [batch, heads, dim] in 64 bits."""
    pages, heads, page, dim = shape
    v = torch.zeros(shape, dtype=dtype, device=dev)
    want = torch.zeros(len(lengths), heads * dim, dtype=torch.float64, device=dev)
    for b, n in enumerate(lengths):
        t = torch.arange(start, max(start, min(n, start + heads * dim)), device=dev)
        if not t.numel():
            continue
        c = t - start
        v[table[b].long()[t // page], c // dim, t % page, c % dim] = HEIGHT
        want[b, c] = HEIGHT / n
    return v, want.view(len(lengths), heads, dim)


def marked_bound(want, dtype):
    # equal weights are exact powers of two, their sum and the one value in a column exact; the least
    # parts of fp16 weights are 2^-38 of them; then a quotient, a product or two and the rounding
    return want.abs() * 2.0 ** -21 + torch.where(want == 0, 0.0, O.rounding(want, dtype))


# ---- low parts ----------------------------------------------------------------------------------

def low_parts(which, heads, n, dim, gen):
    """(q [heads, dim], k, v [n, dim], scale) in fp32 whose attention hangs on bits 12 and 13 behind the leading one of the keys, the
    queries, the weights or the values: 11 leading bits alone (one tf32 part) give something else altogether."""
    q, k = torch.zeros(heads, dim), torch.zeros(n, dim)
    pairs = dim // 2
    step = 2.0 ** (12 - (pairs - 1).bit_length())         # times the pairs' sum of 2^-12: between 1/2 and 1
    v = torch.randint(0, 2, (n, dim), generator=gen) * 2.0 - 1
    if which == "keys":                                   # 1 + m 2^-12 against 1
        m = torch.randint(0, 4, (n, 1), generator=gen)
        q[:, 0::2], q[:, 1::2] = step, -step
        k[:, 0::2], k[:, 1::2] = 1 + m * 2.0 ** -12, 1.0
    elif which == "queries":
        sign = torch.randint(0, 2, (heads, 1), generator=gen) * 2.0 - 1
        q[:, 0::2], q[:, 1::2] = step * (1 + sign * 2.0 ** -12), -step
        k[:] = torch.randint(1, 5, (n, 1), generator=gen).float()
    elif which == "weights":                              # 1 against exp(-2^-13), with values that cancel
        q[:, 0] = 1.0
        k[1::2, 0] = -(2.0 ** -13)
        v[0::2], v[1::2] = 1.0, -1.0
    else:                                                 # equal weights, values 1 + m 2^-12 against -1
        v[0::2], v[1::2] = 1 + torch.randint(0, 4, v[0::2].shape, generator=gen) * 2.0 ** -12, -1.0
    return q, k, v, 1.0


def low_parts_want(which, q, k, v, scale, tensor_cores=True):
    """(out, bound): every product of parts is exact here; left are the exponential (2^-22 a weight, as of its sum) and the
    sums over the keys: of values around 1 with random signs, or, where neighbours cancel, of what is left of them.
    Without tensor cores the queries are multiplied by the scale first, which rounds each by 2^-24 of itself: where "queries"
    1 + 2^-12 and -1 cancel, that stays, and a score is off by up to 2^-24 of its sum of sizes, and its sums by as much again."""
    s = q.double() @ k.double().t() * scale
    p = torch.softmax(s, -1)
    out = p @ v.double()
    if which in ("weights", "values"):
        return out, torch.full_like(out, 2.0 ** -20)
    bound = 2.0 ** -19 + CHAIN * 2.0 ** -23 * (6 * (p ** 2 @ v.double() ** 2).sqrt() + out.abs())
    if which == "queries" and not tensor_cores:
        off = 2 * 2.0 ** -24 * (q.double().abs() @ k.double().abs().t()) * abs(scale)
        bound += 8 * ((p * off) ** 2 @ v.double() ** 2).sqrt()     # (of values with random signs)
    return out, bound


def one_part(x, rounded):
    """x rounded, or cut off, to 11 bits, in fp32."""
    bits = x.float().view(torch.int32) + (0x1000 if rounded else 0)
    return (bits & ~0x1FFF).view(torch.float32)
