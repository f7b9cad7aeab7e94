"""Measured cases of the block-scaled fp8 and the grouped matrix products.

Five operators, each reached the way a program reaches it:

* ``quantize``: a matrix to fp8 e4m3fn with one scale per block of 128 columns, of one row
  (activations) or of 128 rows (weights); scales in float32 or as powers of two (e8m0);
* ``fp8``: the product of two such matrices;
* ``grouped_fp8``: the same, rows sorted by expert, one weight matrix for each expert;
* ``grouped``: the product of bf16 / fp16 rows sorted by expert with their experts' weights;
* ``train``: that product with its gradients for the rows and for the weights.

The product's shape is ``c[m, n] = sum_k a[m, k] bt[n, k]``, both operands K-major.
"""

import math

import torch

own = False

BLOCK = 128            # columns (and, for weights, rows) that share a scale
E4M3_MAX = 448.0
LEAST_SCALE = 2.0 ** -126

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a decode step's activations, one token: the launch is all there is
        dict(name="quantize token", op="quantize", rows=1, cols=4096, block_rows=1, dtype="bf16", scale="fp32"),
        # a prefill batch's activations at the validator's square size
        dict(name="quantize batch", op="quantize", rows=16384, cols=8192, block_rows=1, dtype="bf16", scale="e8m0"),
        # a weight matrix loaded in float32, neither side a whole number of blocks
        dict(name="quantize weight", op="quantize", rows=12200, cols=8256, block_rows=128, dtype="fp32", scale="fp32"),
        # one decode step of a few sequences: the weights' bytes count
        dict(name="fp8 decode", op="fp8", m=16, n=8192, k=8192, scale="fp32"),
        # the validator's headline size
        dict(name="fp8 square", op="fp8", m=8192, n=8192, k=8192, scale="fp32"),
        # ragged rows, a last tile of every kind, powers of two as scales
        dict(name="fp8 odd", op="fp8", m=4001, n=5136, k=4176, scale="e8m0"),
        # a decode step over many experts, most of which get a row or none
        dict(name="grouped fp8 decode", op="grouped_fp8", t=64, e=64, n=4096, k=2048, tail=0, scale="fp32"),
        # a prefill batch over experts with a padded tail
        dict(name="grouped fp8 batch", op="grouped_fp8", t=16384, e=32, n=4096, k=4096, tail=1024, scale="fp32"),
        # single tokens through bf16 experts
        dict(name="grouped decode", op="grouped", t=8, e=16, n=4096, k=4096, tail=0, dtype="bf16"),
        # a prefill batch through a few large experts
        dict(name="grouped batch", op="grouped", t=16384, e=8, n=8192, k=4096, tail=0, dtype="bf16"),
        # a training step's product and its two gradients, many experts, odd sizes
        dict(name="train small", op="train", t=2083, e=32, n=1032, k=2056, tail=35, dtype="fp16"),
        # a training step's product and its two gradients
        dict(name="train batch", op="train", t=16384, e=16, n=4096, k=4096, tail=0, dtype="bf16"),
    ]


def _log_int(rng, lo, hi, multiple=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return max(lo, min(hi, int(v) // multiple * multiple))


def draw(rng):
    """A case of the listed ones' ranges: one token to 16384 rows, widths to 8192, aligned or odd."""
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["quantize", "fp8", "grouped_fp8", "grouped", "train"])
        odd = rng.random() < 0.25
        width = lambda lo, hi, mul: _log_int(rng, lo, hi, 1 if odd else mul)  # noqa: E731
        if op == "quantize":
            case = dict(op=op, rows=_log_int(rng, 1, 16384), cols=width(128, 8192, 16), block_rows=rng.choice([1, 128]),
                        dtype=rng.choice(["bf16", "fp16", "fp32"]), scale=rng.choice(["fp32", "e8m0"]))
        elif op == "fp8":
            case = dict(op=op, m=_log_int(rng, 1, 8192), n=width(256, 8192, 16), k=width(256, 8192, 16),
                        scale=rng.choice(["fp32", "e8m0"]))
        else:
            t = _log_int(rng, 1 if op != "train" else 256, 16384)
            case = dict(op=op, t=t, e=_log_int(rng, 4, 64), n=width(512, 4096, 16), k=width(512, 4096, 16),
                        tail=rng.choice([0, t // 16]))
            if op == "grouped_fp8":
                case["scale"] = rng.choice(["fp32", "e8m0"])
            else:
                case["dtype"] = rng.choice(["bf16", "fp16"])
        if _cost(case) <= most:
            return case


def _cost(case):
    w = work(case)
    return w["flops"] + 200.0 * w["bytes"]


def work(case):
    op = case["op"]
    if op == "quantize":
        r, c = case["rows"], case["cols"]
        size = 4 if case["dtype"] == "fp32" else 2
        blocks = -(-r // case["block_rows"]) * -(-c // BLOCK)
        return {"bytes": r * c * (size + 1) + blocks * _scale_size(case), "flops": 3 * r * c}
    if op == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // BLOCK)
        scales = (m + -(-n // BLOCK)) * kb * _scale_size(case)
        return {"bytes": (m + n) * k + scales + 2 * m * n, "flops": 2 * m * n * k}
    t, e, n, k = case["t"], case["e"], case["n"], case["k"]
    rows = t - case["tail"]
    # experts that get at least one row, on average over the inputs
    busy = sum(1.0 - (1.0 - p) ** rows for p in _shares(e))
    if op == "grouped_fp8":
        kb = -(-k // BLOCK)
        scales = (rows + busy * -(-n // BLOCK)) * kb * _scale_size(case)
        return {"bytes": rows * k + busy * n * k + scales + 2 * t * n + 4 * (e + 1), "flops": 2 * rows * n * k}
    if op == "grouped":
        return {"bytes": 2 * (rows * k + busy * n * k + t * n) + 4 * (e + 1), "flops": 2 * rows * n * k}
    # a, bt, dout in; out, da, dbt out (dbt whole: an idle expert's gradient is zeros)
    return {"bytes": 2 * (rows * k + busy * n * k + rows * n + t * n + t * k + e * n * k) + 4 * (e + 1),
            "flops": 6 * rows * n * k}


def _scale_size(case):
    return 4 if case["scale"] == "fp32" else 1


def _shares(e):
    """Experts' shares of the rows, as a router leaves them: uneven, one in eight idle."""
    p = [0.0 if i % 8 == 7 else (i + 1) ** -0.5 for i in range(e)]
    return [x / sum(p) for x in p]


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _device():
    return torch.device("cuda", 0) if torch.cuda.is_available() else torch.device("cpu")


def _activations(rows, cols, g, dtype):
    """Rows of unit size with a few columns twenty times as large, as normed hidden states have them."""
    x = torch.randn((rows, cols), generator=g, device=g.device)
    big = torch.rand((1, cols), generator=g, device=g.device) < 0.01
    return torch.where(big, 20.0 * x, x).to(dtype)


def _weights(shape, g, dtype):
    return (torch.randn(shape, generator=g, device=g.device) * shape[-1] ** -0.5).to(dtype)


def _quantized(x, block_rows, scale):
    """fp8 operand and scales of x [.., rows, cols] in one pass of float32, as a checkpoint holds them."""
    rows, cols = x.shape[-2:]
    pad = torch.nn.functional.pad(x.float(), (0, -cols % BLOCK, 0, -rows % block_rows))
    v = pad.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, block_rows))
    s = v.abs().amax(dim=(-1, -3), keepdim=True).clamp_min(1e-30) / E4M3_MAX
    if scale == "e8m0":
        s = torch.exp2(torch.ceil(torch.log2(s)))
    q = (v / s).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    q = q.flatten(-4, -3).flatten(-2, -1)[..., :rows, :cols].contiguous()
    s = s.squeeze(-1).squeeze(-2).contiguous()
    return q, s.to(torch.float8_e8m0fnu) if scale == "e8m0" else s


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]
    state = dict(case)
    if op == "quantize":
        make = _weights if case["block_rows"] > 1 else lambda s, g, d: _activations(*s, g, d)
        state["x"] = make((case["rows"], case["cols"]), g, _DTYPES[case["dtype"]])
        return state
    if op == "fp8":
        state["a"], state["a_scale"] = _quantized(_activations(case["m"], case["k"], g, torch.bfloat16), 1, case["scale"])
        state["bt"], state["bt_scale"] = _quantized(_weights((case["n"], case["k"]), g, torch.bfloat16), BLOCK, case["scale"])
        return state
    t, e = case["t"], case["e"]
    hg = torch.Generator().manual_seed(seed)
    shares = torch.tensor(_shares(e), dtype=torch.float64)[torch.randperm(e, generator=hg)]
    picks = torch.multinomial(shares, t - case["tail"], replacement=True, generator=hg)
    sizes = torch.bincount(picks, minlength=e)
    state["longest"] = int(sizes.max())          # a program that plans its batch on the host knows it
    state["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)]).to(torch.int32).to(dev)
    dtype = _DTYPES[case.get("dtype", "bf16")]
    a = _activations(t, case["k"], g, dtype)
    bt = _weights((e, case["n"], case["k"]), g, dtype)
    if op == "grouped_fp8":
        state["a"], state["a_scale"] = _quantized(a, 1, case["scale"])
        state["bt"], state["bt_scale"] = _quantized(bt, BLOCK, case["scale"])
        return state
    state["a"], state["bt"] = a, bt
    if op == "train":
        state["a"].requires_grad_(True)
        state["bt"].requires_grad_(True)
        state["dout"] = (torch.randn((t, case["n"]), generator=g, device=dev) * 0.05).to(dtype)
    return state


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "quantize":
        return _plain_quantize(state["x"], state["block_rows"], state["scale"])
    if op == "fp8":
        a = _plain_dequantize(state["a"], state["a_scale"], 1)
        bt = _plain_dequantize(state["bt"], state["bt_scale"], BLOCK)
        return (a @ bt.t()).to(torch.bfloat16)
    if op == "grouped_fp8":
        a = _plain_dequantize(state["a"], state["a_scale"], 1)
        bt = _plain_dequantize(state["bt"], state["bt_scale"], BLOCK)
        return _plain_grouped(a, bt, state["offsets"], state["longest"]).to(torch.bfloat16)
    a, bt = state["a"].detach(), state["bt"].detach()
    out = _plain_grouped(a.float(), bt.float(), state["offsets"], state["longest"]).to(a.dtype)
    if op == "grouped":
        return out
    da, dbt = _plain_grads(state["dout"].float(), a.float(), bt.float(), state["offsets"], state["longest"])
    return out, da.to(a.dtype), dbt.to(a.dtype)


def _run_own(state):
    from gpu_operator_amd.ops import blockscale, grouped

    op = state["op"]
    if op == "quantize":
        scale_dtype = torch.float32 if state["scale"] == "fp32" else torch.float8_e8m0fnu
        q, s = blockscale.quantize_fp8_block(state["x"], state["block_rows"], scale_dtype=scale_dtype)
        return q, s.float()
    if op == "fp8":
        return blockscale.gemm_fp8_block(state["a"], state["a_scale"], state["bt"], state["bt_scale"])
    if op == "grouped_fp8":
        return blockscale.gemm_grouped_fp8_block(state["a"], state["a_scale"], state["bt"], state["bt_scale"],
                                                 state["offsets"])
    if op == "grouped":
        return grouped.gemm_grouped(state["a"], state["bt"], state["offsets"])
    out = grouped.grouped_linear(state["a"], state["bt"], state["offsets"])
    return out.detach(), *torch.autograd.grad(out, (state["a"], state["bt"]), state["dout"])


def _power_of_two(e):
    """2 ** e in float64, by its exponent's bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _to_e4m3(v):
    """v (float64) to the nearest e4m3 value, ties to the even one, without a rounding in between."""
    _, ex = torch.frexp(v)
    step = _power_of_two((ex - 1).clamp_min(-6) - 3)
    return (torch.round(v / step) * step).to(torch.float8_e4m3fn)


def _plain_quantize(x, block_rows, scale):
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -cols % BLOCK, 0, -rows % block_rows))
    v = v.view(-1, block_rows, v.shape[1] // BLOCK, BLOCK)
    amax = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(dim=(1, 3))
    amax = amax.clamp_min(E4M3_MAX * LEAST_SCALE)
    if scale == "e8m0":
        mant, ex = torch.frexp(amax)
        s = _power_of_two(ex - 9 + (mant > 0.875).to(ex.dtype))
        q = _to_e4m3(v / s[:, None, :, None])
    else:
        s = amax / E4M3_MAX
        q = _to_e4m3(v * E4M3_MAX / amax[:, None, :, None])
    return q.view(-1, q.shape[2] * BLOCK)[:rows, :cols].contiguous(), s.float()


def _plain_dequantize(q, s, block_rows):
    rows, cols = q.shape[-2:]
    s = s.float().repeat_interleave(BLOCK, dim=-1)[..., :cols]
    if block_rows > 1:
        s = s.repeat_interleave(block_rows, dim=-2)[..., :rows, :]
    return q.float() * s


def _plain_padded(x, offsets, longest):
    """Rows sorted by expert as one zero-padded matrix for each expert."""
    at = torch.arange(longest, device=x.device)
    there = at < (offsets[1:] - offsets[:-1])[:, None]
    rows = (offsets[:-1, None] + at).clamp_max(x.shape[0] - 1)
    return torch.where(there[..., None], x[rows], x.new_zeros(()))


def _plain_sorted(y, offsets, total):
    """Back from one padded matrix for each expert to rows sorted by expert; other rows are zero."""
    t = torch.arange(total, device=y.device, dtype=offsets.dtype)
    expert = torch.searchsorted(offsets[1:].contiguous(), t, right=True).clamp_max(y.shape[0] - 1)
    pos = (t - offsets[expert]).clamp(0, y.shape[1] - 1)
    owned = (t >= offsets[0]) & (t < offsets[-1])
    return torch.where(owned[:, None], y[expert, pos], y.new_zeros(()))


def _plain_grouped(a, bt, offsets, longest):
    y = torch.bmm(_plain_padded(a, offsets, longest), bt.transpose(1, 2).contiguous())
    return _plain_sorted(y, offsets, a.shape[0])


def _plain_grads(dout, a, bt, offsets, longest):
    d = _plain_padded(dout, offsets, longest)
    da = _plain_sorted(torch.bmm(d, bt), offsets, a.shape[0])
    return da, torch.bmm(d.transpose(1, 2).contiguous(), _plain_padded(a, offsets, longest))


# ------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_quantize(st["x"], case["block_rows"], case["scale"])
    if op == "fp8":
        return _exact_values(st["a"], st["a_scale"], 1) @ _exact_values(st["bt"], st["bt_scale"], BLOCK).t()
    edges = st["offsets"].tolist()
    t, n, k = case["t"], case["n"], case["k"]
    dev = st["a"].device
    out = torch.zeros((t, n), dtype=torch.float64, device=dev)
    da = torch.zeros((t, k), dtype=torch.float64, device=dev)
    dbt = torch.zeros((case["e"], n, k) if op == "train" else (0,), dtype=torch.float64, device=dev)
    for i in range(case["e"]):
        rows = slice(edges[i], edges[i + 1])
        if op == "grouped_fp8":
            x = _exact_values(st["a"][rows], st["a_scale"][rows], 1)
            w = _exact_values(st["bt"][i], st["bt_scale"][i], BLOCK)
        else:
            x, w = st["a"][rows].detach().double(), st["bt"][i].detach().double()
        out[rows] = x @ w.t()
        if op == "train":
            d = st["dout"][rows].double()
            da[rows] = d @ w
            dbt[i] = d.t() @ x
    return (out, da, dbt) if op == "train" else out


def _exact_values(q, s, block_rows):
    row = torch.arange(q.shape[0], device=q.device) // block_rows
    col = torch.arange(q.shape[1], device=q.device) // BLOCK
    return q.to(torch.float64) * s.to(torch.float32).to(torch.float64)[row][:, col]


def _exact_quantize(x, block_rows, scale):
    # every e4m3 value and the borders half way between neighbours; a border belongs to the even neighbour
    codes = torch.arange(0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).to(torch.float64).to(x.device)
    border = (codes[1:] + codes[:-1]) / 2
    v = x.to(torch.float64)
    rb = torch.arange(v.shape[0], device=v.device) // block_rows
    cb = torch.arange(v.shape[1], device=v.device) // BLOCK
    peak = torch.zeros((int(rb[-1]) + 1, v.shape[1]), dtype=torch.float64, device=v.device)
    peak = peak.index_reduce_(0, rb, v.abs(), "amax")
    peak = torch.zeros((peak.shape[0], int(cb[-1]) + 1), dtype=torch.float64, device=v.device).index_reduce_(1, cb, peak, "amax")
    peak = peak.clamp_min(E4M3_MAX * LEAST_SCALE)
    s = peak / E4M3_MAX
    if scale == "e8m0":
        powers = torch.tensor([2.0 ** i for i in range(-126, 128)], dtype=torch.float64, device=v.device)
        s = powers[torch.searchsorted(powers, s)]              # the least that is not under s
        ratio = v / s[rb][:, cb]
    else:
        ratio = E4M3_MAX * v / peak[rb][:, cb]
    size = ratio.abs()
    at = torch.searchsorted(border, size)                     # border[at - 1] < size <= border[at]
    tie = (at < border.numel()) & (border[at.clamp_max(border.numel() - 1)] == size)
    at = at + (tie & (at % 2 == 1))
    return torch.copysign(codes[at], ratio), s
