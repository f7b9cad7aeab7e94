"""The grouped matrix products (bf16, fp16) and their gradients against a 64-bit plain form."""

import pytest
import torch

import group_helpers as H

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]

# sizes of the groups, N, K: single tokens, empty groups, tile edges and their neighbours, odd widths
CASES = [
    ([1], 1, 1), ([1], 16, 8), ([0], 40, 24), ([0, 0, 3], 17, 33), ([1, 0, 2, 1], 64, 128),
    ([1] * 9, 136, 72), ([16, 17, 0, 15], 130, 70), ([33, 0, 63, 64, 65], 256, 64), ([127, 128, 129], 128, 192),
    ([255, 0, 256, 257], 264, 136), ([300], 520, 1032), ([5, 0, 0, 700, 1, 90], 384, 320), ([2, 3] * 40, 96, 200),
    ([640, 1, 1], 1, 640), ([77, 11], 640, 1), ([513, 31], 255, 257), ([1000], 1000, 1000),
]


def _inputs(dev, sizes, n, k, dtype, seed=0, tail=0, first=0):
    t, e = first + sum(sizes) + tail, len(sizes)
    g = torch.Generator(device=dev).manual_seed(seed + 7 * n + k)
    a = torch.randn((t, k), generator=g, device=dev).to(dtype)
    bt = (torch.randn((e, n, k), generator=g, device=dev) / max(1, k) ** 0.5).to(dtype)
    dc = torch.randn((t, n), generator=g, device=dev).to(dtype)
    return a, bt, dc, H.offsets_of(sizes, first, dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,n,k", CASES)
def test_forward(cuda_device, sizes, n, k, dtype):
    from gpu_operator_amd.ops import grouped as G

    a, bt, _, off = _inputs(cuda_device, sizes, n, k, dtype)
    ref, mag = H.forward64(a, bt, off)
    H.check(G.gemm_grouped(a, bt, off), ref, mag, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,n,k", CASES)
def test_dgrad(cuda_device, sizes, n, k, dtype):
    from gpu_operator_amd.ops import grouped as G

    _, bt, dc, off = _inputs(cuda_device, sizes, n, k, dtype)
    ref, mag = H.dgrad64(dc, bt, off)
    H.check(G.gemm_grouped_dgrad(dc, bt, off), ref, mag, n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,n,k", CASES)
def test_wgrad(cuda_device, sizes, n, k, dtype):
    from gpu_operator_amd.ops import grouped as G

    a, _, dc, off = _inputs(cuda_device, sizes, n, k, dtype)
    ref, mag = H.wgrad64(dc, a, off)
    H.check(G.gemm_grouped_wgrad(dc, a, off), ref, mag, max(sizes))


def _spread(x, pad, lead):
    """x with `pad` more elements between its rows, starting `lead` elements into its memory."""
    shape = (*x.shape[:-1], x.shape[-1] + pad)
    flat = torch.full((lead + x[..., 0].numel() * shape[-1],), float("nan"), dtype=x.dtype, device=x.device)
    v = flat[lead:].view(shape)[..., : x.shape[-1]]
    v.copy_(x)
    return v


@pytest.mark.parametrize("pad,lead", [(8, 0), (64, 8), (1, 0), (0, 1), (3, 5), (24, 4)])
def test_strided_operands_and_outputs(cuda_device, pad, lead):
    """Rows apart, not on 16 bytes, NaN between them: the results are those of packed operands, bit for bit, and what
    lies between the output's rows stays."""
    from gpu_operator_amd.ops import grouped as G

    a, bt, dc, off = _inputs(cuda_device, [130, 0, 3, 70], 200, 136, torch.bfloat16)
    sa, sb, sd = (_spread(x, pad, lead) for x in (a, bt, dc))
    for want, fn, ops in ((G.gemm_grouped(a, bt, off), G.gemm_grouped, (sa, sb)),
                          (G.gemm_grouped_dgrad(dc, bt, off), G.gemm_grouped_dgrad, (sd, sb)),
                          (G.gemm_grouped_wgrad(dc, a, off), G.gemm_grouped_wgrad, (sd, sa))):
        assert torch.equal(fn(*ops, off), want)
        out = _spread(torch.zeros_like(want), pad, lead)
        assert fn(*ops, off, out) is out
        assert torch.equal(out, want)
        whole = out.as_strided((out[..., 0].numel(), out.shape[-1] + pad), (out.stride(-2), 1))
        if pad:
            assert torch.isnan(whole[:-1, out.shape[-1]:]).all()


@pytest.mark.parametrize("first,tail", [(0, 5), (3, 0), (7, 200)])
def test_rows_that_no_expert_owns(cuda_device, first, tail):
    """Padding rows full of NaN reach nothing; an output of the caller's keeps its padding rows, a new one has zeros."""
    from gpu_operator_amd.ops import grouped as G

    sizes, n, k = [40, 0, 129], 72, 96
    a, bt, dc, off = _inputs(cuda_device, sizes, n, k, torch.bfloat16, tail=tail, first=first)
    owned = torch.zeros(a.shape[0], dtype=torch.bool, device=cuda_device)
    owned[first : first + sum(sizes)] = True
    a[~owned] = float("nan")
    dc[~owned] = float("inf")
    for fn, x, y, w in ((G.gemm_grouped, a, bt, n), (G.gemm_grouped_dgrad, dc, bt, k)):
        fresh = fn(x, y, off)
        assert torch.isfinite(fresh).all() and (fresh[~owned] == 0).all()
        out = torch.full_like(fresh, 123.0)
        fn(x, y, off, out)
        assert torch.equal(out[owned], fresh[owned]) and (out[~owned] == 123.0).all()
    ref, mag = H.wgrad64(dc, a, off)
    H.check(G.gemm_grouped_wgrad(dc, a, off), ref, mag, max(sizes))


def test_a_nan_stays_with_its_expert(cuda_device):
    """One expert's NaN row, column and weights change only what they multiply, in every direction."""
    from gpu_operator_amd.ops import grouped as G

    sizes = [60, 70, 50]
    a, bt, dc, off = _inputs(cuda_device, sizes, 100, 104, torch.float16)
    want = [G.gemm_grouped(a, bt, off), G.gemm_grouped_dgrad(dc, bt, off), G.gemm_grouped_wgrad(dc, a, off)]
    a[61], dc[62], bt[1, 5, 7] = float("nan"), float("inf"), float("nan")
    got = [G.gemm_grouped(a, bt, off), G.gemm_grouped_dgrad(dc, bt, off), G.gemm_grouped_wgrad(dc, a, off)]
    for g, w in zip(got[:2], want[:2]):
        assert torch.equal(g[:60], w[:60]) and torch.equal(g[130:], w[130:])
    clean = torch.ones(100, dtype=torch.bool, device=cuda_device)
    clean[5] = False
    rows = [r for r in range(60, 130) if r != 61]
    assert torch.equal(got[0][rows][:, clean], want[0][rows][:, clean]) and torch.isnan(got[0][rows][:, 5]).all()
    assert torch.equal(got[2][[0, 2]], want[2][[0, 2]]) and not torch.isfinite(got[2][1]).any()


def test_offsets_are_clamped_to_the_rows(cuda_device):
    from gpu_operator_amd.ops import grouped as G

    a, bt, dc, _ = _inputs(cuda_device, [50, 30], 40, 48, torch.bfloat16)
    wild = torch.tensor([-5, 50, 1 << 30], dtype=torch.int32, device=cuda_device)
    tame = torch.tensor([0, 50, 80], dtype=torch.int32, device=cuda_device)
    assert torch.equal(G.gemm_grouped(a, bt, wild), G.gemm_grouped(a, bt, tame))
    assert torch.equal(G.gemm_grouped_dgrad(dc, bt, wild), G.gemm_grouped_dgrad(dc, bt, tame))
    assert torch.equal(G.gemm_grouped_wgrad(dc, a, wild), G.gemm_grouped_wgrad(dc, a, tame))


@pytest.mark.parametrize("e,t", [(64, 500), (65, 65), (200, 900), (1000, 40)])
def test_many_experts(cuda_device, e, t):
    from gpu_operator_amd.ops import grouped as G

    sizes = H.random_sizes(t, e, seed=e, empty=range(0, e, 7))
    a, bt, dc, off = _inputs(cuda_device, sizes, 48, 64, torch.bfloat16)
    for got, (ref, mag), terms in ((G.gemm_grouped(a, bt, off), H.forward64(a, bt, off), 64),
                                   (G.gemm_grouped_dgrad(dc, bt, off), H.dgrad64(dc, bt, off), 48),
                                   (G.gemm_grouped_wgrad(dc, a, off), H.wgrad64(dc, a, off), max(sizes))):
        H.check(got, ref, mag, terms)


def test_large_operands(cuda_device):
    """Several tiles of every kind and long reductions, against 64 bits."""
    from gpu_operator_amd.ops import grouped as G

    sizes = H.random_sizes(3000, 6, seed=3, empty=(2,))
    a, bt, dc, off = _inputs(cuda_device, sizes, 1536, 2048, torch.bfloat16, tail=70)
    for got, (ref, mag), terms in ((G.gemm_grouped(a, bt, off), H.forward64(a, bt, off), 2048),
                                   (G.gemm_grouped_dgrad(dc, bt, off), H.dgrad64(dc, bt, off), 1536),
                                   (G.gemm_grouped_wgrad(dc, a, off), H.wgrad64(dc, a, off), max(sizes))):
        H.check(got, ref, mag, terms)


def test_offsets_past_32_bits(cuda_device):
    """Rows 8 MiB apart: byte offsets of operands and outputs pass 2^32."""
    from gpu_operator_amd.ops import grouped as G

    t, n, k, ld = 600, 64, 72, 1 << 22
    a, bt, dc, off = _inputs(cuda_device, [100, 450, 50], n, k, torch.bfloat16)
    far = torch.empty(t * ld, dtype=torch.bfloat16, device=cuda_device)
    fa = far.as_strided((t, k), (ld, 1))
    fd = far.as_strided((t, n), (ld, 1), 4096)
    fo = far.as_strided((t, n), (ld, 1), 8192)
    fa.copy_(a)
    fd.copy_(dc)
    assert torch.equal(G.gemm_grouped(fa, bt, off, fo), G.gemm_grouped(a, bt, off))
    assert torch.equal(G.gemm_grouped_dgrad(fd, bt, off), G.gemm_grouped_dgrad(dc, bt, off))
    assert torch.equal(G.gemm_grouped_wgrad(fd, fa, off), G.gemm_grouped_wgrad(dc, a, off))


def test_repeated_calls_give_the_same_bits(cuda_device):
    from gpu_operator_amd.ops import grouped as G

    sizes = H.random_sizes(700, 5, seed=1)
    a, bt, dc, off = _inputs(cuda_device, sizes, 272, 400, torch.float16)
    for fn, ops in ((G.gemm_grouped, (a, bt)), (G.gemm_grouped_dgrad, (dc, bt)), (G.gemm_grouped_wgrad, (dc, a))):
        first = fn(*ops, off)
        assert all(torch.equal(fn(*ops, off), first) for _ in range(4))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,n,k,tail", [([0, 37, 5], 24, 40, 3), ([130, 0, 200], 264, 136, 9)])
def test_autograd(cuda_device, sizes, n, k, tail, dtype):
    """The gradients against the formulas', and against differences of the (linear) product itself."""
    from gpu_operator_amd.ops import grouped as G

    a, bt, dc, off = _inputs(cuda_device, sizes, n, k, dtype, tail=tail)
    a.requires_grad_(True)
    bt.requires_grad_(True)
    out = G.grouped_linear(a, bt, off)
    da, dbt = torch.autograd.grad(out, (a, bt), dc)
    ref, mag = H.dgrad64(dc, bt.detach(), off)
    H.check(da, ref, mag, n)
    ref, mag = H.wgrad64(dc, a.detach(), off)
    H.check(dbt, ref, mag, max(sizes))
    # L(a, bt) = <dc, product> is linear in each argument: L(a + u) - L(a - u) = 2 <da, u>, in 64 bits
    g = torch.Generator(device=cuda_device).manual_seed(5)
    for x, gx, loss in ((a, da, lambda v: (H.forward64(v, bt.detach(), off)[0] * dc.double())[: off[-1]].sum()),
                        (bt, dbt, lambda v: (H.forward64(a.detach(), v, off)[0] * dc.double())[: off[-1]].sum())):
        u = torch.randn(x.shape, generator=g, device=cuda_device, dtype=torch.float64)
        x64 = x.detach().double()
        diff = (loss(x64 + u) - loss(x64 - u)) / 2
        slope = (gx.double() * u).sum()
        # every gradient element is off by at most its own tolerance: random signs, so well inside the plain sum
        bound = ((torch.finfo(dtype).eps / 2 + 2.0 ** -12) * (gx.double() * u).abs()).sum() + 1e-6
        assert abs(float(slope - diff)) <= float(bound)


def test_autograd_needs_only_one_gradient_and_broadcast_gradients(cuda_device):
    from gpu_operator_amd.ops import grouped as G

    a, bt, _, off = _inputs(cuda_device, [20, 0, 50], 40, 56, torch.bfloat16)
    bt.requires_grad_(True)
    G.grouped_linear(a, bt, off).sum().backward()          # the sum's gradient has strides of zero
    ones = torch.ones((70, 40), dtype=torch.bfloat16, device=cuda_device)
    assert torch.equal(bt.grad, G.gemm_grouped_wgrad(ones, a, off))
    a.requires_grad_(True)
    (da,) = torch.autograd.grad(G.grouped_linear(a, bt.detach(), off), a, ones)
    assert torch.equal(da, G.gemm_grouped_dgrad(ones, bt.detach(), off))


def test_no_rows_and_no_reduction(cuda_device):
    from gpu_operator_amd.ops import grouped as G

    dev = cuda_device
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=dev)  # noqa: E731
    off = torch.zeros(4, dtype=torch.int32, device=dev)
    assert G.gemm_grouped(z(0, 16), z(3, 8, 16), off).shape == (0, 8)
    assert G.gemm_grouped_dgrad(z(0, 8), z(3, 8, 16), off).shape == (0, 16)
    w = G.gemm_grouped_wgrad(z(0, 8), z(0, 16), off, torch.full((3, 8, 16), 7.0, dtype=torch.bfloat16, device=dev))
    assert (w == 0).all()
    off = torch.tensor([0, 5, 5, 9], dtype=torch.int32, device=dev)
    assert (G.gemm_grouped(z(9, 0), z(3, 8, 0), off, torch.ones((9, 8), dtype=torch.bfloat16, device=dev)) == 0).all()
    assert (G.gemm_grouped_dgrad(z(9, 0), z(3, 0, 8), off, torch.ones((9, 8), dtype=torch.bfloat16, device=dev)) == 0).all()
    assert G.gemm_grouped(z(9, 4), z(3, 0, 4), off).shape == (9, 0)


def test_side_stream_and_graph(cuda_device):
    """A captured step, replayed over new inputs with eager work between the replays, gives the eager results."""
    from gpu_operator_amd.ops import grouped as G

    a, bt, dc, off = _inputs(cuda_device, [100, 3, 57], 144, 208, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = G.gemm_grouped(a, bt, off)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(warm, G.gemm_grouped(a, bt, off))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = G.gemm_grouped(a, bt, off)
        da = G.gemm_grouped_dgrad(dc, bt, off)
        dbt = G.gemm_grouped_wgrad(dc, a, off)
    for seed, sizes in enumerate(([100, 3, 57], [0, 160, 0], [40, 60, 60], [1, 0, 3])):
        na, nb, nd, no = _inputs(cuda_device, sizes, 144, 208, torch.bfloat16, seed=seed + 1, tail=160 - sum(sizes))
        for x, y in ((a, na), (bt, nb), (dc, nd), (off, no)):
            x.copy_(y)
        graph.replay()
        want = G.gemm_grouped(a, bt, off), G.gemm_grouped_dgrad(dc, bt, off), G.gemm_grouped_wgrad(dc, a, off)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((out, da, dbt), want))


def test_training_step_in_a_graph(cuda_device):
    """Forward and backward captured together, replayed: the eager gradients."""
    from gpu_operator_amd.ops import grouped as G

    a, bt, dc, off = _inputs(cuda_device, [60, 0, 100], 136, 72, torch.bfloat16)
    la, lb = a.clone().requires_grad_(True), bt.clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(G.grouped_linear(la, lb, off), (la, lb), dc)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = G.grouped_linear(la, lb, off)
        da, dbt = torch.autograd.grad(out, (la, lb), dc)
    for seed in range(3):
        g = torch.Generator(device=cuda_device).manual_seed(seed)
        dc.copy_(torch.randn(dc.shape, generator=g, device=cuda_device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(da, G.gemm_grouped_dgrad(dc, bt, off)) and torch.equal(dbt, G.gemm_grouped_wgrad(dc, a, off))
