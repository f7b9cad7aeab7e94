"""The grouped and block-scaled products at the sizes that fill the card: every tile shape, each against 64 bits."""

import pytest
import torch

import group_helpers as H

pytestmark = pytest.mark.gpu

SCALES = [torch.float32, torch.float8_e8m0fnu]


def _rand(dev, seed, dtype, *shape, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)


def _codes(dev, seed, *shape):
    g = torch.Generator(device=dev).manual_seed(seed)
    c = torch.randint(0, 256, shape, generator=g, device=dev, dtype=torch.int16)
    return torch.where((c & 0x7F) == 0x7F, c ^ 1, c).to(torch.uint8).view(torch.float8_e4m3fn)


def _scales(dev, seed, dtype, *shape):
    g = torch.Generator(device=dev).manual_seed(seed)
    s = torch.exp2(torch.randint(-12, 3, shape, generator=g, device=dev).float())
    return s * (1 + torch.rand(shape, generator=g, device=dev)) if dtype == torch.float32 else s.to(dtype)


# sizes, N, K, rows before the first expert, rows behind the last. Over 205 tiles of 256 x 256 and over 128 rows a
# group, so the largest tiles: reductions of one, two, three and many panels, a last panel that is not whole, column
# tails of 1 to 255, last row tiles of 1 to 256 rows, empty experts, more experts than a wave has lanes.
BIG = [
    ([3000, 0, 1, 257, 2500, 255, 1200, 64], 1536, 1024, 0, 0),
    ([2048, 2048, 2100, 2040], 1800, 64, 0, 5),
    ([4000, 129, 0, 0, 4200], 1601, 100, 3, 0),
    ([1500, 1501, 1502, 1503, 1504], 1793, 130, 0, 70),
    ([9000], 1544, 520, 0, 0),
    ([150 + i for i in range(130)], 520, 200, 11, 300),
    ([700, 900, 500], 8200, 72, 40, 1),
    ([6000, 10], 2304, 8, 0, 0),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,n,k,first,tail", BIG)
def test_forward(cuda_device, sizes, n, k, first, tail, dtype):
    from gpu_operator_amd.ops import grouped as G

    t, owned = first + sum(sizes) + tail, slice(first, first + sum(sizes))
    a = _rand(cuda_device, 1, dtype, t, k)
    bt = _rand(cuda_device, 2, dtype, len(sizes), n, k, scale=k ** -0.5)
    off = H.offsets_of(sizes, first, cuda_device)
    a[:first], a[t - tail:] = float("nan"), float("inf")
    got = G.gemm_grouped(a, bt, off)
    ref, mag = H.forward64(a, bt, off)
    H.check(got, ref, mag, k)
    out = torch.full((t, n + 8), 7.0, dtype=dtype, device=cuda_device)
    G.gemm_grouped(a, bt, off, out[:, :n])
    assert torch.equal(out[owned, :n], got[owned])
    out[owned, :n] = 7.0
    assert (out == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,n,k,first,tail", BIG)
def test_dgrad(cuda_device, sizes, n, k, first, tail, dtype):
    """The same sizes with the reduction over K columns of the weights and N outputs."""
    from gpu_operator_amd.ops import grouped as G

    t = first + sum(sizes) + tail
    dc = _rand(cuda_device, 3, dtype, t, k)
    bt = _rand(cuda_device, 4, dtype, len(sizes), k, n, scale=k ** -0.5)
    off = H.offsets_of(sizes, first, cuda_device)
    dc[:first], dc[t - tail:] = float("nan"), float("inf")
    ref, mag = H.dgrad64(dc, bt, off)
    H.check(G.gemm_grouped_dgrad(dc, bt, off), ref, mag, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,n,k,first,tail", [
    ([0, 1, 63, 64, 65, 128, 129, 600, 0, 500], 1500, 1000, 0, 0),
    ([2000, 31, 0], 2304, 2056, 5, 70),
    ([300] * 12, 1030, 1032, 0, 3),
    ([1] + [250] * 8, 1281, 1281, 1, 0),
])
def test_wgrad(cuda_device, sizes, n, k, first, tail, dtype):
    from gpu_operator_amd.ops import grouped as G

    t = first + sum(sizes) + tail
    a, dc = _rand(cuda_device, 5, dtype, t, k), _rand(cuda_device, 6, dtype, t, n)
    off = H.offsets_of(sizes, first, cuda_device)
    for x in (a, dc):
        x[:first], x[t - tail:] = float("nan"), float("inf")
    ref, mag = H.wgrad64(dc, a, off)
    H.check(G.gemm_grouped_wgrad(dc, a, off), ref, mag, max(sizes))


@pytest.mark.parametrize("scale_dtype", SCALES)
@pytest.mark.parametrize("sizes,n,k,first,tail", BIG)
def test_grouped_fp8(cuda_device, sizes, n, k, first, tail, scale_dtype):
    from gpu_operator_amd.ops import blockscale as B

    t, e, kb, nb = first + sum(sizes) + tail, len(sizes), -(-k // 128), -(-n // 128)
    a, bt = _codes(cuda_device, 7, t, k), _codes(cuda_device, 8, e, n, k)
    sa, sb = _scales(cuda_device, 9, scale_dtype, t, kb), _scales(cuda_device, 10, scale_dtype, e, nb, kb)
    off = H.offsets_of(sizes, first, cuda_device)
    for r in (slice(0, first), slice(t - tail, t)):
        a.view(torch.uint8)[r] = 0x7F
    x, w = H.dequantize64(a, sa, 1), H.dequantize64(bt, sb, 128)
    ref, mag = H.forward64(x, w, off)
    slack = H.grouped_fp8_slack(H.raised64(a, sa, 1), H.raised64(bt, sb, 128), off)
    H.check(B.gemm_grouped_fp8_block(a, sa, bt, sb, off), ref, mag, k + 3 * kb, slack)


@pytest.mark.parametrize("scale_dtype", SCALES)
@pytest.mark.parametrize("m,n,k", [(4096, 4096, 128), (4097, 3840, 300), (3500, 4104, 1152), (8000, 1793, 96), (6000, 2304, 272)])
def test_fp8(cuda_device, m, n, k, scale_dtype):
    from gpu_operator_amd.ops import blockscale as B

    kb, nb = -(-k // 128), -(-n // 128)
    a, bt = _codes(cuda_device, 11, m, k), _codes(cuda_device, 12, n, k)
    sa, sb = _scales(cuda_device, 13, scale_dtype, m, kb), _scales(cuda_device, 14, scale_dtype, nb, kb)
    x, w = H.dequantize64(a, sa, 1), H.dequantize64(bt, sb, 128)
    got = B.gemm_fp8_block(a, sa, bt, sb)
    H.check(got, x @ w.t(), x.abs() @ w.abs().t(), k + 3 * kb, H.fp8_slack(H.raised64(a, sa, 1), H.raised64(bt, sb, 128)))
    # scales stored column by column
    cols = [s.view(torch.uint8 if scale_dtype != torch.float32 else scale_dtype).t().contiguous().t().view(scale_dtype) for s in (sa, sb)]
    assert torch.equal(B.gemm_fp8_block(a, cols[0], bt, cols[1]), got)


# cases for each smaller tile shape in each direction, for parts of the largest tiles on an idle card, and for many groups
# of a few rows: (sizes, N, K)
MIDDLE = [([64, 70, 0, 130] * 8, 1992, 256), ([64, 70, 0, 130] * 8, 256, 1992), ([8, 12, 0, 9] * 16, 640, 320),
          ([2, 1, 0, 3], 200, 4104), ([1, 0, 2] * 25, 2056, 136),
          ([1800], 4096, 200), ([900, 850], 200, 4100), ([1500, 1536], 1400, 264),
          ([40, 30, 0, 50] * 8, 2048, 256), ([100] * 16, 2000, 320), ([300, 200, 10, 0], 1000, 1000), ([2000], 264, 520),
          ([20] * 60, 1288, 200), ([500, 490], 1792, 136)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,n,k", MIDDLE)
def test_middle_sizes(cuda_device, sizes, n, k, dtype):
    from gpu_operator_amd.ops import blockscale as B
    from gpu_operator_amd.ops import grouped as G

    t, e = sum(sizes), len(sizes)
    off = H.offsets_of(sizes, 0, cuda_device)
    a, dc = _rand(cuda_device, 15, dtype, t, k), _rand(cuda_device, 16, dtype, t, n)
    bt = _rand(cuda_device, 17, dtype, e, n, k, scale=k ** -0.5)
    for got, (ref, mag), terms in ((G.gemm_grouped(a, bt, off), H.forward64(a, bt, off), k),
                                   (G.gemm_grouped_dgrad(dc, bt, off), H.dgrad64(dc, bt, off), n),
                                   (G.gemm_grouped_wgrad(dc, a, off), H.wgrad64(dc, a, off), max(sizes))):
        H.check(got, ref, mag, terms)
    for scale_dtype in SCALES:
        qa, sa = B.quantize_fp8_block(a, scale_dtype=scale_dtype)
        qb, sb = B.quantize_fp8_block(bt, 128, scale_dtype=scale_dtype)
        x, w = H.dequantize64(qa, sa, 1), H.dequantize64(qb, sb, 128)
        ref, mag = H.forward64(x, w, off)
        slack = H.grouped_fp8_slack(H.raised64(qa, sa, 1), H.raised64(qb, sb, 128), off)
        H.check(B.gemm_grouped_fp8_block(qa, sa, qb, sb, off), ref, mag, k + 3 * -(-k // 128), slack)


def _shifted(x):
    """x at an address and with rows that are not on 16 bytes."""
    flat = torch.empty(1 + x[..., 0].numel() * (x.shape[-1] + 1), dtype=x.dtype, device=x.device)
    v = flat[1:].view(*x.shape[:-1], x.shape[-1] + 1)[..., : x.shape[-1]]
    v.copy_(x)
    return v


def test_unaligned_operands_at_every_size(cuda_device):
    """Operands that have to be laid out first: the aligned ones' bits, for the largest tiles and small ones, in every
    direction; an fp8 product whose N and K are not multiples of 16."""
    from gpu_operator_amd.ops import blockscale as B
    from gpu_operator_amd.ops import grouped as G

    for sizes, n, k in (([3000, 0, 4000, 1], 1801, 515), ([70, 0, 33], 135, 77)):
        t, e = sum(sizes), len(sizes)
        off = H.offsets_of(sizes, 0, cuda_device)
        a, dc = _rand(cuda_device, 18, torch.bfloat16, t, k), _rand(cuda_device, 19, torch.bfloat16, t, n)
        bt = _rand(cuda_device, 20, torch.bfloat16, e, n, k, scale=k ** -0.5)
        for fn, x, y, (ref, mag), terms in ((G.gemm_grouped, a, bt, H.forward64(a, bt, off), k),
                                            (G.gemm_grouped_dgrad, dc, bt, H.dgrad64(dc, bt, off), n),
                                            (G.gemm_grouped_wgrad, dc, a, H.wgrad64(dc, a, off), max(sizes))):
            got = fn(x, y, off)
            H.check(got, ref, mag, terms)
            assert torch.equal(fn(_shifted(x), _shifted(y), off), got)
    a, bt = _codes(cuda_device, 21, 5000, 301), _codes(cuda_device, 22, 3001, 301)
    sa, sb = _scales(cuda_device, 23, torch.float32, 5000, 3), _scales(cuda_device, 24, torch.float32, 24, 3)
    x, w = H.dequantize64(a, sa, 1), H.dequantize64(bt, sb, 128)
    H.check(B.gemm_fp8_block(a, sa, bt, sb), x @ w.t(), x.abs() @ w.abs().t(), 301 + 9, H.fp8_slack(H.raised64(a, sa, 1), H.raised64(bt, sb, 128)))


@pytest.mark.parametrize("sizes,n,k", [([3000, 0, 4000, 1], 1801, 515), ([70, 0, 33], 135, 77), ([2, 0, 1], 135, 77), ([17, 0, 30], 70, 6)])
def test_unaligned_operands_in_a_graph(cuda_device, sizes, n, k):
    """The workspace that unaligned operands are laid out in belongs to the graph: replays over new inputs, with eager
    calls of the same operators between them, give the eager results."""
    from gpu_operator_amd.ops import grouped as G

    t, e = sum(sizes), len(sizes)
    off = H.offsets_of(sizes, 0, cuda_device)
    a, dc = _rand(cuda_device, 25, torch.bfloat16, t, k), _rand(cuda_device, 26, torch.bfloat16, t, n)
    bt = _rand(cuda_device, 27, torch.bfloat16, e, n, k)

    def step():
        return G.gemm_grouped(a, bt, off), G.gemm_grouped_dgrad(dc, bt, off), G.gemm_grouped_wgrad(dc, a, off)

    step()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    for seed in range(3):
        for x in (a, dc, bt):
            x.copy_(_rand(cuda_device, 28 + seed, torch.bfloat16, *x.shape))
        for graph in graphs:
            graph.replay()
        want = step()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_two_streams_at_once(cuda_device):
    """Products of either kind queued on two streams without a wait between them: each stream's own results."""
    from gpu_operator_amd.ops import blockscale as B
    from gpu_operator_amd.ops import grouped as G

    work = []
    for seed in range(2):
        sizes = H.random_sizes(8000, 6, seed=seed + 1)
        off = H.offsets_of(sizes, 0, cuda_device)
        a = _rand(cuda_device, 40 + seed, torch.bfloat16, 8000, 515)          # unaligned: laid out on its own stream
        bt = _rand(cuda_device, 50 + seed, torch.bfloat16, 6, 1544, 515)
        dc = _rand(cuda_device, 60 + seed, torch.bfloat16, 8000, 1544)

        def step(a=a, bt=bt, dc=dc, off=off):
            q, s = B.quantize_fp8_block(a)
            qw, sw = B.quantize_fp8_block(bt, 128)
            return (G.gemm_grouped(a, bt, off), G.gemm_grouped_dgrad(dc, bt, off), G.gemm_grouped_wgrad(dc, a, off),
                    B.gemm_grouped_fp8_block(q, s, qw, sw, off))

        work.append((step, torch.cuda.Stream()))
    want = [step() for step, _ in work]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i, (step, stream) in enumerate(work):
            with torch.cuda.stream(stream):
                got[i].append(step())
    torch.cuda.synchronize()
    for w, rounds in zip(want, got):
        for r in rounds:
            assert all(torch.equal(p, q) for p, q in zip(r, w))


def test_a_gradient_of_the_gradients_is_refused(cuda_device):
    from gpu_operator_amd.ops import grouped as G

    a = _rand(cuda_device, 70, torch.bfloat16, 20, 64).requires_grad_(True)
    bt = _rand(cuda_device, 71, torch.bfloat16, 2, 32, 64).requires_grad_(True)
    dc = _rand(cuda_device, 72, torch.bfloat16, 20, 32).requires_grad_(True)
    off = H.offsets_of([7, 13], 0, cuda_device)
    da, dbt = torch.autograd.grad(G.grouped_linear(a, bt, off), (a, bt), dc, create_graph=True)
    assert torch.equal(da, G.gemm_grouped_dgrad(dc.detach(), bt.detach(), off))
    assert torch.equal(dbt, G.gemm_grouped_wgrad(dc.detach(), a.detach(), off))
    with pytest.raises(RuntimeError, match="twice"):
        da.float().sum().backward()


@pytest.mark.parametrize("scale_dtype", SCALES)
def test_strides_of_single_rows_say_nothing(cuda_device, scale_dtype):
    """A dimension of one may have any stride: the results are those of contiguous operands."""
    from gpu_operator_amd.ops import blockscale as B
    from gpu_operator_amd.ops import grouped as G

    def odd(t, far):
        return t.as_strided(t.shape, [far if n == 1 else st for n, st in zip(t.shape, t.stride())])

    a, bt = _codes(cuda_device, 80, 1, 96), _codes(cuda_device, 81, 1, 48, 96)
    sa, sb = _scales(cuda_device, 82, scale_dtype, 1, 1), _scales(cuda_device, 83, scale_dtype, 1, 1, 1)
    off = torch.tensor([0, 1], dtype=torch.int32, device=cuda_device)
    want = B.gemm_grouped_fp8_block(a, sa, bt, sb, off)
    got = B.gemm_grouped_fp8_block(odd(a, 3), odd(sa, 1 << 40), odd(bt, 7), odd(sb, 1 << 40), off, odd(torch.empty_like(want), 5))
    assert torch.equal(got, want)
    assert torch.equal(B.gemm_fp8_block(odd(a, 3), odd(sa, 1 << 40), bt[0], odd(sb[0], 1 << 40)), want)
    x, w = _rand(cuda_device, 84, torch.bfloat16, 1, 96), _rand(cuda_device, 85, torch.bfloat16, 1, 48, 96)
    dc = _rand(cuda_device, 86, torch.bfloat16, 1, 48)
    assert torch.equal(G.gemm_grouped(odd(x, 3), odd(w, 7), off), G.gemm_grouped(x, w, off))
    assert torch.equal(G.gemm_grouped_dgrad(odd(dc, 1 << 40), odd(w, 7), off), G.gemm_grouped_dgrad(dc, w, off))
    dw = G.gemm_grouped_wgrad(dc, x, off)
    assert torch.equal(G.gemm_grouped_wgrad(odd(dc, 3), odd(x, 1 << 40), off, odd(torch.empty_like(dw), 1 << 40)), dw)


@pytest.mark.parametrize("m", [5, 40, 200, 4000])
def test_power_of_two_scales_at_their_ends(cuda_device, m):
    """The least and the largest scale together, and NaN (code 255), in every kernel: NaN stays in its row or columns."""
    from gpu_operator_amd.ops import blockscale as B

    n, k = 4000 if m == 4000 else 272, 384
    a, bt = _codes(cuda_device, 87, m, k), _codes(cuda_device, 88, n, k)
    sa = torch.full((m, 3), 254, dtype=torch.uint8, device=cuda_device)          # 2^127
    sb = torch.zeros((-(-n // 128), 3), dtype=torch.uint8, device=cuda_device)   # 2^-127
    sa[1], sb[1] = 127 - 60, 127 + 60
    sa[2] = 0                                                                    # rows times 2^-254, and of 2^-67
    e8 = torch.float8_e8m0fnu
    x64 = lambda q, s, rows: H.dequantize64(q, torch.exp2(s.double() - 127), rows)  # noqa: E731
    x, w = x64(a, sa, 1), x64(bt, sb, 128)
    keep = [r for r in range(m) if r != 3]
    sa[3, 2] = 255
    got = B.gemm_fp8_block(a, sa.view(e8), bt, sb.view(e8))
    assert torch.isnan(got[3]).all()
    ref, mag = x @ w.t(), x.abs() @ w.abs().t()
    cols = slice(0, 128)                  # (the others' products of 2^127 and 2^60 leave the type's range)
    slack = H.fp8_slack(H.raised64(a, torch.exp2(sa.double() - 127), 1), H.raised64(bt, torch.exp2(sb.double() - 127), 128))
    H.check(got[keep][:, cols], ref[keep][:, cols], mag[keep][:, cols], k + 9, slack[keep][:, cols])
    sb[0, 0] = 255
    got = B.gemm_fp8_block(a, sa.view(e8), bt, sb.view(e8))
    assert torch.isnan(got[:, :128]).all() and not torch.isnan(got[2, 128:]).any()


@pytest.mark.parametrize("sizes,n,k", [([17, 0, 33, 5], 300, 259), ([16] * 5, 77, 1030), ([3, 40], 33, 7), ([1, 1, 0, 9], 130, 641),
                                       ([20, 20], 64, 15), ([2], 100, 64)])
def test_few_rows_from_any_address(cuda_device, sizes, n, k):
    """Rows that start on each byte of a word (fp8), on 2 and 4 bytes (16 bits), with widths that end inside a piece: the bits
    of aligned copies; nothing behind the operands is read into the results."""
    from gpu_operator_amd.ops import blockscale as B
    from gpu_operator_amd.ops import grouped as G

    t, e, kb = sum(sizes), len(sizes), -(-k // 128)
    off = H.offsets_of(sizes, 0, cuda_device)

    def at(x, lead, pad):
        flat = torch.full((lead + x[..., 0].numel() * (x.shape[-1] + pad) + 64,), 0x7F, dtype=torch.uint8, device=x.device)
        if x.dtype != torch.float8_e4m3fn:
            flat = torch.full((flat.numel(),), float("nan"), dtype=x.dtype, device=x.device)
        v = flat[lead : lead + x[..., 0].numel() * (x.shape[-1] + pad)].view(*x.shape[:-1], -1)[..., : x.shape[-1]]
        v.copy_(x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x)
        return v.view(x.dtype)

    a, bt = _codes(cuda_device, 90, t, k), _codes(cuda_device, 91, e, n, k)
    sa, sb = _scales(cuda_device, 92, torch.float32, t, kb), _scales(cuda_device, 93, torch.float32, e, -(-n // 128), kb)
    x, w = H.dequantize64(a, sa, 1), H.dequantize64(bt, sb, 128)
    ref, mag = H.forward64(x, w, off)
    slack = H.grouped_fp8_slack(H.raised64(a, sa, 1), H.raised64(bt, sb, 128), off)
    for lead, pad in ((0, 0), (1, 0), (2, 1), (3, 2), (0, 3), (5, 7)):
        got = B.gemm_grouped_fp8_block(at(a, lead, pad), sa, at(bt, lead + 1, pad), sb, off)
        H.check(got, ref, mag, k + 3 * kb, slack)
        if len(sizes) == 1:
            assert torch.equal(B.gemm_fp8_block(at(a, lead, pad), sa, at(bt, lead, pad)[0], sb[0]), got)
    for dtype in (torch.bfloat16, torch.float16):
        x, w = _rand(cuda_device, 94, dtype, t, k), _rand(cuda_device, 95, dtype, e, n, k, scale=k ** -0.5)
        ref, mag = H.forward64(x, w, off)
        for lead, pad in ((0, 0), (1, 0), (2, 2), (0, 1), (3, 5)):
            H.check(G.gemm_grouped(at(x, lead, pad), at(w, lead + 1, pad), off), ref, mag, k)
