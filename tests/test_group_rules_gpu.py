"""What the grouped and block-scaled products promise beside their formulas."""

import pytest
import torch

import group_helpers as H

pytestmark = pytest.mark.gpu


def _codes(dev, seed, *shape):
    g = torch.Generator(device=dev).manual_seed(seed)
    c = torch.randint(0, 256, shape, generator=g, device=dev, dtype=torch.int16)
    return torch.where((c & 0x7F) == 0x7F, c ^ 1, c).to(torch.uint8).view(torch.float8_e4m3fn)


def _rand(dev, seed, dtype, *shape, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)


def _instruction_sum(a, bt):
    """a @ bt.T of e4m3 codes with each product cut toward zero at 2^(E - 13), E the largest sum of two factors'
    exponents among its 8 reduction steps (a subnormal's is -6, a zero has none); the sum itself in 64 bits."""
    x, w = (torch.nn.functional.pad(v.double(), (0, -v.shape[1] % 8)) for v in (a, bt))
    ex, ew = (torch.where(v == 0, torch.full_like(v, -100).int(), (torch.frexp(v)[1] - 1).clamp_min(-6)) for v in (x, w))
    out = torch.zeros((x.shape[0], w.shape[0]), dtype=torch.float64, device=x.device)
    for k in range(0, x.shape[1], 8):
        top = torch.full(out.shape, -100, dtype=torch.int32, device=x.device)
        for i in range(k, k + 8):
            torch.maximum(top, ex[:, i, None] + ew[None, :, i], out=top)
        step = H.power_of_two(top - 13)
        for i in range(k, k + 8):
            out += torch.trunc(x[:, i, None] * w[None, :, i] / step) * step
    return out


@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.float8_e8m0fnu])
@pytest.mark.parametrize("m,n,k", [(5, 200, 384), (40, 272, 257), (200, 264, 272), (600, 1024, 128), (4001, 4000, 144)])
def test_fp8_sums_are_cut_as_documented_and_no_further(cuda_device, m, n, k, scale_dtype):
    """In every kernel: against the cut products in 64 bits there is nothing but float32 roundings left, also where the
    largest products cancel. (All scales are one, so a block's weight rounds nothing: k roundings of the sum.)"""
    from gpu_operator_amd.ops import blockscale as B

    a, bt = _codes(cuda_device, m, m, k), _codes(cuda_device, n, n, k)
    a[:, 1:k:8] = (-a[:, 0 : k - 1 : 8].float()).to(a.dtype)             # pairs that cancel where bt's are equal
    bt[: n // 2, 1:k:8] = bt[: n // 2, 0 : k - 1 : 8]
    one = lambda *s: torch.ones(s, device=cuda_device).to(scale_dtype)  # noqa: E731
    got = B.gemm_fp8_block(a, one(m, -(-k // 128)), bt, one(-(-n // 128), -(-k // 128)))
    H.check(got, _instruction_sum(a, bt), a.double().abs() @ bt.double().abs().t(), k)


@pytest.mark.parametrize("m", [3, 40, 200])
def test_a_small_product_beside_ones_that_cancel(cuda_device, m):
    """448 * 448 - 448 * 448 + t: t is kept from 2^(16 - 13) on, lost under it, and untouched 8 steps on."""
    from gpu_operator_amd.ops import blockscale as B

    def product(t, at):
        a, b = torch.zeros((m, 128), device=cuda_device), torch.zeros((16, 128), device=cuda_device)
        a[:, 0], a[:, 1], b[:, :2] = 448.0, -448.0, 448.0
        a[:, at], b[:, at] = t / 2.0, 2.0
        f8 = torch.float8_e4m3fn
        return B.gemm_fp8_block(a.to(f8), torch.ones((m, 1), device=cuda_device), b.to(f8), torch.ones((1, 1), device=cuda_device))

    assert (product(8.0, 2) == 8.0).all() and (product(4.0, 2) == 0.0).all()
    assert (product(2.0 ** -8, 8) == 2.0 ** -8).all()


def _calls(dev, dtype=torch.bfloat16):
    """name, a call with or without `out`, the operands it differentiates, for every entry point that takes an `out`."""
    from gpu_operator_amd.ops import blockscale as B
    from gpu_operator_amd.ops import grouped as G

    off = H.offsets_of([7, 0, 33], 0, dev)
    a, bt, dc = _rand(dev, 1, dtype, 40, 64), _rand(dev, 2, dtype, 3, 48, 64, scale=0.1), _rand(dev, 3, dtype, 40, 48)
    qa, sa = B.quantize_fp8_block(a)
    qb, sb = B.quantize_fp8_block(bt, 128)
    return {
        "gemm_grouped": (lambda out, a, bt: G.gemm_grouped(a, bt, off, out), [a, bt]),
        "gemm_grouped_dgrad": (lambda out, dc, bt: G.gemm_grouped_dgrad(dc, bt, off, out), [dc, bt]),
        "gemm_grouped_wgrad": (lambda out, dc, a: G.gemm_grouped_wgrad(dc, a, off, out), [dc, a]),
        "gemm_fp8_block": (lambda out, a, sa, b, sb: B.gemm_fp8_block(a, sa, b, sb, out), [qa, sa, qb[0], sb[0]]),
        "gemm_grouped_fp8_block": (lambda out, a, sa, b, sb: B.gemm_grouped_fp8_block(a, sa, b, sb, off, out), [qa, sa, qb, sb]),
        "quantize_fp8_block": (lambda out, x: B.quantize_fp8_block(x, out=out)[0], [a]),
    }


NAMES = ["gemm_grouped", "gemm_grouped_dgrad", "gemm_grouped_wgrad", "gemm_fp8_block", "gemm_grouped_fp8_block", "quantize_fp8_block"]


@pytest.mark.parametrize("name", NAMES)
def test_an_output_of_the_callers_counts_as_written(cuda_device, name):
    """Autograd has to know that its memory changed: a tensor saved for a backward pass may not be overwritten unnoticed."""
    call, ops = _calls(cuda_device)[name]
    out = torch.empty_like(call(None, *ops))
    before = out._version
    call(out, *ops)
    assert out._version > before
    with torch.inference_mode():
        call(torch.empty_like(out), *ops)               # (has no version)


def test_a_saved_tensor_is_not_overwritten_unnoticed(cuda_device):
    from gpu_operator_amd.ops import blockscale as B

    call, ops = _calls(cuda_device)["gemm_grouped"]
    out = call(None, *ops)
    w = torch.ones_like(out).requires_grad_(True)
    loss = (out * w).float().sum()                      # saves out
    call(out, *ops)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    x = _rand(cuda_device, 4, torch.bfloat16, 5, 300)
    s = torch.ones((5, 3), device=cuda_device)
    w = torch.ones_like(s).requires_grad_(True)
    loss = (s * w).sum()
    B.quantize_fp8_block(x, scale_out=s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("name", NAMES)
def test_no_gradient_is_lost_in_silence(cuda_device, name):
    """Operands that need a gradient: gemm_grouped has one, the others' results say at their backward that they have none; an
    `out` cannot be recorded and is refused, as torch's own are. Without gradients to record everything is as ever."""
    call, ops = _calls(cuda_device)[name]
    want = call(None, *ops)
    assert not want.requires_grad
    for i in range(len(ops)):
        need = [t.detach().clone().requires_grad_(True) if j == i else t for j, t in enumerate(ops)]
        got = call(None, *need)
        assert got.requires_grad and torch.equal(got.detach().view(torch.uint8), want.view(torch.uint8))
        if name == "gemm_grouped":
            assert torch.autograd.grad(got.float().sum(), need[i])[0].shape == need[i].shape
        else:
            with pytest.raises(RuntimeError, match="no gradient"):
                got.float().sum().backward()
        with pytest.raises(RuntimeError, match="automatic differentiation"):
            call(torch.empty_like(want), *need)
        with torch.no_grad():
            out = torch.empty_like(want)
            call(out, *need)
            assert not call(None, *need).requires_grad
        assert torch.equal(out.view(torch.uint8), want.view(torch.uint8))
    with pytest.raises(RuntimeError, match="automatic differentiation"):
        call(torch.empty_like(want).requires_grad_(True), *ops)


def test_gemm_grouped_gives_grouped_linears_gradients(cuda_device):
    from gpu_operator_amd.ops import grouped as G

    off = H.offsets_of([7, 0, 33], 0, cuda_device)
    a = _rand(cuda_device, 1, torch.bfloat16, 43, 64).requires_grad_(True)
    bt = _rand(cuda_device, 2, torch.bfloat16, 3, 48, 64, scale=0.1).requires_grad_(True)
    dc = _rand(cuda_device, 3, torch.bfloat16, 43, 48)
    one, two = G.gemm_grouped(a, bt, off), G.grouped_linear(a, bt, off)
    assert torch.equal(one, two)
    for x, y in zip(torch.autograd.grad(one, (a, bt), dc), torch.autograd.grad(two, (a, bt), dc)):
        assert torch.equal(x, y)
    ref, mag = H.dgrad64(dc, bt.detach(), off)
    H.check(torch.autograd.grad(G.gemm_grouped(a, bt, off), a, dc)[0], ref, mag, 48)


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(cuda_device, name):
    import torch.autograd.forward_ad as fwd

    call, ops = _calls(cuda_device)[name]
    with fwd.dual_level():
        call(None, *ops)
        if ops[0].dtype != torch.float8_e4m3fn:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(None, fwd.make_dual(ops[0], torch.ones_like(ops[0])), *ops[1:])
        else:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(None, ops[0], fwd.make_dual(ops[1], torch.ones_like(ops[1])), *ops[2:])


def test_quantisers_scale_out_is_an_output_too(cuda_device):
    from gpu_operator_amd.ops import blockscale as B

    x = _rand(cuda_device, 7, torch.bfloat16, 5, 300).requires_grad_(True)
    with pytest.raises(RuntimeError, match="automatic differentiation"):
        B.quantize_fp8_block(x, scale_out=torch.empty((5, 3), device=cuda_device))
    q, s = B.quantize_fp8_block(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        s.sum().backward()
    q, s = B.quantize_fp8_block(x, scale_dtype=torch.float8_e8m0fnu)
    with pytest.raises(RuntimeError, match="no gradient"):
        s.float().sum().backward()


@pytest.mark.parametrize("e,n,k", [(3, 48, 64), (3, 300, 520), (70, 260, 1032), (2, 5, 7)])
def test_weight_gradients_to_interleaved_matrices(cuda_device, e, n, k):
    """Experts' matrices that lie row by row among one another (an output stored [N, E, K], or with columns between):
    they do not overlap, so they are written, and nothing between them."""
    from gpu_operator_amd.ops import grouped as G

    sizes = H.random_sizes(200, e, seed=e, empty=(1,))
    off = H.offsets_of(sizes, 0, cuda_device)
    dc, a = _rand(cuda_device, 5, torch.bfloat16, 200, n), _rand(cuda_device, 6, torch.bfloat16, 200, k)
    want = G.gemm_grouped_wgrad(dc, a, off)
    for pad in (0, 8, 3):
        flat = torch.full((n, e, k + pad), 7.0, dtype=torch.bfloat16, device=cuda_device)
        out = flat[..., :k].transpose(0, 1)
        assert G.gemm_grouped_wgrad(dc, a, off, out) is out
        assert torch.equal(out, want) and (flat[..., k:] == 7.0).all()


def test_matrices_that_overlap_are_refused(cuda_device):
    from gpu_operator_amd.ops import grouped as G

    dc, a = torch.ones((9, 4), dtype=torch.bfloat16, device=cuda_device), torch.ones((9, 16), dtype=torch.bfloat16, device=cuda_device)
    off = H.offsets_of([4, 5], 0, cuda_device)
    flat = torch.zeros(1000, dtype=torch.bfloat16, device=cuda_device)
    for strides in ((8, 16, 1), (16, 24, 1), (63, 16, 1), (0, 16, 1), (24, 32, 1)):
        with pytest.raises(ValueError, match="overlap"):
            G.gemm_grouped_wgrad(dc, a, off, flat.as_strided((2, 4, 16), strides))
    for strides in ((64, 16, 1), (16, 32, 1), (20, 36, 1)):
        out = G.gemm_grouped_wgrad(dc, a, off, flat.as_strided((2, 4, 16), strides))
        assert (out[0] == 4.0).all() and (out[1] == 5.0).all()


def test_outputs_that_share_memory_with_an_operand_are_refused(cuda_device):
    """A workgroup would read what another has written. (Rows side by side in one buffer share none.)"""
    from gpu_operator_amd.ops import blockscale as B
    from gpu_operator_amd.ops import grouped as G

    off = H.offsets_of([16, 24], 0, cuda_device)
    a, bt = _rand(cuda_device, 1, torch.bfloat16, 40, 64), _rand(cuda_device, 2, torch.bfloat16, 2, 64, 64)
    q, s = B.quantize_fp8_block(a)
    qb, sb = B.quantize_fp8_block(bt, 128)
    whole = torch.zeros(40 * 64 * 4, dtype=torch.uint8, device=cuda_device)
    x = whole[: 40 * 64 * 2].view(torch.bfloat16).view(40, 64)
    for call in (lambda: G.gemm_grouped(a, bt, off, a), lambda: G.gemm_grouped(a, bt, off, bt.view(-1, 64)[30:70]),
                 lambda: G.gemm_grouped_dgrad(a, bt, off, a), lambda: G.gemm_grouped_wgrad(a, bt[0, :40], off, bt),
                 lambda: B.gemm_fp8_block(q, s, qb[0], whole[:4].view(torch.float32).view(1, 1), x),
                 lambda: B.gemm_grouped_fp8_block(q, whole[: 40 * 4].view(torch.float32).view(40, 1), qb, sb, off, x),
                 lambda: B.quantize_fp8_block(x, out=whole[64 : 64 + 40 * 64].view(torch.float8_e4m3fn).view(40, 64)),
                 lambda: B.quantize_fp8_block(a, out=whole[: 40 * 64].view(torch.float8_e4m3fn).view(40, 64),
                                              scale_out=whole[: 160].view(torch.float32).view(40, 1))):
        with pytest.raises(ValueError, match="shares memory"):
            call()
    both = torch.zeros((40, 128), dtype=torch.bfloat16, device=cuda_device)
    both[:, :64] = a
    assert torch.equal(G.gemm_grouped(both[:, :64], bt, off, both[:, 64:]), G.gemm_grouped(a, bt, off))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("e,n,k", [(70, 512, 1024), (130, 504, 1016), (200, 250, 1021)])
def test_weight_gradients_of_more_experts_than_lanes(cuda_device, e, n, k, dtype):
    """The largest tiles with more than 64 experts, whose order is then the experts' own: experts without rows among them, rows
    that no expert owns around them."""
    from gpu_operator_amd.ops import grouped as G

    sizes = H.random_sizes(3000, e, seed=e, empty=range(3, e, 9))
    a, dc = _rand(cuda_device, 8, dtype, 3020, k), _rand(cuda_device, 9, dtype, 3020, n)
    off = H.offsets_of(sizes, 5, cuda_device)
    for x in (a, dc):
        x[:5], x[3005:] = float("nan"), float("inf")
    ref, mag = H.wgrad64(dc, a, off)
    H.check(G.gemm_grouped_wgrad(dc, a, off), ref, mag, max(sizes))


def test_grouped_linear_has_no_forward_mode(cuda_device):
    import torch.autograd.forward_ad as fwd

    from gpu_operator_amd.ops import grouped as G

    off = H.offsets_of([7, 0, 33], 0, cuda_device)
    a, bt = _rand(cuda_device, 1, torch.bfloat16, 40, 64), _rand(cuda_device, 2, torch.bfloat16, 3, 48, 64)
    with fwd.dual_level():
        for need in (False, True):
            with pytest.raises(RuntimeError):
                G.grouped_linear(fwd.make_dual(a, torch.ones_like(a)), bt.clone().requires_grad_(need), off)
