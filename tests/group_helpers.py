"""Plain 64-bit forms of the grouped and block-scaled products, and their error bounds.

Bounds. A product of two bf16, fp16 or e4m3 values is exact in float32, so a sum of K of them held in float32 is
off by at most K + 8 roundings (of up to one unit in the last place each, whatever the order and the matrix
instructions' own alignment) of the sum of magnitudes S: (K + 8) 2^-23 S. A block-scaled sum rounds a scale's
product and two more results for each block of 128: 3 ceil(K / 128) more. The result is then rounded once to
its type: half a step, eps / 2 of the value, or half the least subnormal.

The matrix instructions' sum of fp8 products is not quite a float32 one. They add the products of 8 consecutive
reduction steps on a fixed-point grid: with E the largest sum of two factors' exponents among the 8, what a product
has under 2^(E - 13) is cut off (measured: of 448 * 448 - 448 * 448 + t, E = 16, a power of two t is kept down to 2^3
and lost from 2^2 on; of 1 - 1 + t down to 2^-13; steps 8 apart do not touch each other). A product of two e4m3 values
has 8 significant bits, so the largest is whole, and the 7 others lose less than 2^(E - 13) <= 2^-13 of the largest
product's magnitude each: 7 * 2^-13 * (the sum over the groups of 8 of the largest product), `fp8_slack` below.
A subnormal's exponent counts as the least one, -6, whatever its leading zeros (measured: of 2^-9 * 256 - 2^-9 * 256 +
t, E = -6 + 8 = 2, t is kept down to 2^-11 and lost from 2^-12 on; a zero times 448 hides nothing). Its product's lowest
bit is still 2^(E - 6) or more, so whole, but the product itself can be less than 2^E. "The largest product" is
therefore that of the factors' magnitudes with a subnormal's raised to 2^-6: `raised64` gives such operands.
"""

import torch


def random_sizes(t, e, seed, empty=()):
    """Sizes of e groups that add up to t; the groups in `empty` have no rows."""
    g = torch.Generator().manual_seed(seed)
    p = torch.rand(e, generator=g) ** 2 + 0.01
    for i in empty:
        p[i] = 0.0
    if t == 0:
        return [0] * e
    return torch.bincount(torch.multinomial(p, t, replacement=True, generator=g), minlength=e).tolist()


def offsets_of(sizes, first=0, device="cpu"):
    o = [first]
    for s in sizes:
        o.append(o[-1] + s)
    return torch.tensor(o, dtype=torch.int32, device=device)


def tolerance(ref, mag, terms, dtype):
    eps = torch.finfo(dtype).eps / 2
    low = torch.finfo(dtype).smallest_normal * eps
    sums = (terms + 8) * 2.0 ** -23 * mag
    return eps * (ref.abs() + sums) + sums + low


def raised64(q, s, block_rows):
    """The magnitudes of the block-scaled codes q, those of subnormal codes raised to the least normal one's."""
    v = q.double().abs()
    return dequantize64(torch.where(v > 0, v.clamp_min(2.0 ** -6), v), s, block_rows)


def fp8_slack(x, w):
    """7 * 2^-13 * sum over groups of 8 reduction steps of the largest |x w|, for each element of x @ w.T; x and w as
    `raised64` gives them."""
    x, w = (torch.nn.functional.pad(v.abs(), (0, -v.shape[1] % 8)) for v in (x, w))
    total = torch.zeros((x.shape[0], w.shape[0]), dtype=torch.float64, device=x.device)
    for k in range(0, x.shape[1], 8):
        largest = torch.zeros_like(total)
        for i in range(k, k + 8):
            torch.maximum(largest, x[:, i, None] * w[None, :, i], out=largest)
        total += largest
    return 7 * 2.0 ** -13 * total


def grouped_fp8_slack(x, w, offsets):
    s = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.float64, device=x.device)
    o = offsets.tolist()
    for i in range(w.shape[0]):
        s[o[i] : o[i + 1]] = fp8_slack(x[o[i] : o[i + 1]], w[i])
    return s


def check(got, ref, mag, terms, slack=0.0):
    """got (any float type) against ref (float64), element by element; `slack`: error of the sum itself."""
    assert got.shape == ref.shape
    err = (got.double() - ref).abs()
    tol = tolerance(ref, mag, terms, got.dtype) + slack * (1 + torch.finfo(got.dtype).eps / 2)
    bad = ~(err <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off; first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0].item()} for {ref[bad][0].item()} (tolerance {tol[bad][0].item():.3e})")


def forward64(a, bt, offsets):
    """(c, S) of the grouped product, rows without an expert zero."""
    c = torch.zeros((a.shape[0], bt.shape[1]), dtype=torch.float64, device=a.device)
    s = torch.zeros_like(c)
    o = offsets.tolist()
    for i in range(bt.shape[0]):
        r = slice(o[i], o[i + 1])
        c[r] = a[r].double() @ bt[i].double().t()
        s[r] = a[r].double().abs() @ bt[i].double().abs().t()
    return c, s


def dgrad64(dc, bt, offsets):
    c = torch.zeros((dc.shape[0], bt.shape[2]), dtype=torch.float64, device=dc.device)
    s = torch.zeros_like(c)
    o = offsets.tolist()
    for i in range(bt.shape[0]):
        r = slice(o[i], o[i + 1])
        c[r] = dc[r].double() @ bt[i].double()
        s[r] = dc[r].double().abs() @ bt[i].double().abs()
    return c, s


def wgrad64(dc, a, offsets):
    o = offsets.tolist()
    e = len(o) - 1
    c = torch.zeros((e, dc.shape[1], a.shape[1]), dtype=torch.float64, device=dc.device)
    s = torch.zeros_like(c)
    for i in range(e):
        r = slice(o[i], o[i + 1])
        c[i] = dc[r].double().t() @ a[r].double()
        s[i] = dc[r].double().abs().t() @ a[r].double().abs()
    return c, s


def dequantize64(q, s, block_rows):
    s = s.float().double().repeat_interleave(128, dim=-1)[..., : q.shape[-1]]
    if block_rows > 1:
        s = s.repeat_interleave(128, dim=-2)[..., : q.shape[-2], :]
    return q.double() * s


def quantize64(x, block_rows, e8):
    """(values, scales) of the quantiser's definition, every step exact or in 64 bits."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -cols % 128, 0, -rows % block_rows))
    v = v.view(-1, block_rows, v.shape[1] // 128, 128)
    amax = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(dim=(1, 3))
    amax = amax.clamp_min(448.0 * 2.0 ** -126)
    if e8:
        m, ex = torch.frexp(amax)
        s = power_of_two(ex - 9 + (m > 0.875).int())
        y = v / s[:, None, :, None]
    else:
        s = amax / 448.0
        y = v * 448.0 / amax[:, None, :, None]
    finite = torch.isfinite(y)
    y0 = torch.where(finite, y, torch.zeros_like(y))
    _, ex = torch.frexp(y0)
    step = power_of_two((ex - 1).clamp_min(-6) - 3)
    q = torch.where(finite, torch.round(y0 / step) * step, torch.full_like(y, float("nan")))
    return q.view(-1, q.shape[2] * 128)[:rows, :cols], s


def power_of_two(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)
