"""What the grouped and block-scaled products refuse, checked without a GPU: the operands are fake GPU tensors, so a
call that got past the checks would fail on the missing library or memory instead."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from gpu_operator_amd.ops import blockscale as B
from gpu_operator_amd.ops import grouped as G


@pytest.fixture
def fake():
    with FakeTensorMode(allow_non_fake_inputs=False):
        yield


def _t(*shape, dtype=torch.bfloat16, device="cuda"):
    return torch.empty(shape, dtype=dtype, device=device)


def _off(n, dtype=torch.int32, device="cuda"):
    return torch.empty(n, dtype=dtype, device=device)


def test_grouped_refusals(fake):
    a, bt, off = _t(10, 32), _t(3, 16, 32), _off(4)
    for exc, args in [
        (TypeError, (_t(10, 32, dtype=torch.float32), bt, off)),               # type
        (TypeError, (a, _t(3, 16, 32, dtype=torch.float16), off)),             # two types
        (ValueError, (_t(10, 32, device="cpu"), bt, off)),                     # not on the GPU
        (ValueError, (a, _t(3, 16, 32, device="cpu"), off)),
        (ValueError, (_t(32), bt, off)),                                       # dimensions
        (ValueError, (a, _t(16, 32), off)),
        (ValueError, (a, _t(3, 16, 40), off)),                                 # K differs
        (ValueError, (a, _t(0, 16, 32), _off(1))),                             # no experts
        (ValueError, (_t(32, 10).t(), bt, off)),                               # last dimension strided
        (TypeError, (a, bt, _off(4, torch.int64))),                            # offsets
        (TypeError, (a, bt, [0, 1, 2, 3])),
        (ValueError, (a, bt, _off(3))),
        (ValueError, (a, bt, _off(8)[::2])),
        (ValueError, (a, bt, _off(4, device="cpu"))),
        (TypeError, (a, bt, off, _t(10, 16, dtype=torch.float32))),            # out
        (ValueError, (a, bt, off, _t(10, 17))),
        (ValueError, (a, bt, off, _t(1, 16).expand(10, 16))),                  # rows overlap
        (TypeError, ("a", bt, off)),
    ]:
        with pytest.raises(exc):
            G.gemm_grouped(*args)


def test_gradient_refusals(fake):
    dc, a, bt, off = _t(10, 16), _t(10, 32), _t(3, 16, 32), _off(4)
    for exc, fn, args in [
        (ValueError, G.gemm_grouped_dgrad, (_t(10, 17), bt, off)),
        (TypeError, G.gemm_grouped_dgrad, (dc.to(torch.float16), bt, off)),
        (ValueError, G.gemm_grouped_dgrad, (dc, bt, off, _t(10, 31))),
        (ValueError, G.gemm_grouped_wgrad, (dc, _t(9, 32), off)),
        (TypeError, G.gemm_grouped_wgrad, (dc, a.to(torch.float16), off)),
        (ValueError, G.gemm_grouped_wgrad, (dc, a, None)),
        (ValueError, G.gemm_grouped_wgrad, (dc, a, _off(1))),
        (ValueError, G.gemm_grouped_wgrad, (dc, a, off, _t(3, 16, 33))),
        (ValueError, G.gemm_grouped_wgrad, (dc, a, off, _t(1, 16, 32).expand(3, 16, 32))),
    ]:
        with pytest.raises(exc):
            fn(*args)


def test_quantize_refusals(fake):
    x = _t(10, 300)
    for exc, args, kw in [
        (TypeError, (_t(10, 300, dtype=torch.float64),), {}),
        (TypeError, (_t(10, 300, dtype=torch.float8_e4m3fn),), {}),
        (ValueError, (_t(300),), {}),
        (ValueError, (None,), {}),
        (ValueError, (_t(10, 300, device="cpu"),), {}),
        (ValueError, (x, 64), {}),
        (TypeError, (x, 1), dict(scale_dtype=torch.float16)),
        (ValueError, (_t(300, 10).t(),), {}),
        (TypeError, (x,), dict(out=_t(10, 300))),
        (ValueError, (x,), dict(out=_t(10, 301, dtype=torch.float8_e4m3fn))),
        (ValueError, (x,), dict(scale_out=_t(10, 2, dtype=torch.float32))),
        (TypeError, (x,), dict(scale_out=_t(10, 3, dtype=torch.float32), scale_dtype=torch.float8_e8m0fnu)),
        (ValueError, (x,), dict(out=_t(10, 600, dtype=torch.float8_e4m3fn)[:, :300])),
    ]:
        with pytest.raises(exc):
            B.quantize_fp8_block(*args, **kw)


def test_block_product_refusals(fake):
    f8, f32 = torch.float8_e4m3fn, torch.float32
    a, sa, bt, sb = _t(10, 300, dtype=f8), _t(10, 3, dtype=f32), _t(200, 300, dtype=f8), _t(2, 3, dtype=f32)
    for exc, args in [
        (TypeError, (_t(10, 300), sa, bt, sb)),
        (ValueError, (a, sa, _t(200, 301, dtype=f8), sb)),
        (ValueError, (a, _t(10, 2, dtype=f32), bt, sb)),
        (ValueError, (a, sa, bt, _t(3, 2, dtype=f32))),
        (TypeError, (a, sa, bt, _t(2, 3, dtype=torch.float8_e8m0fnu))),
        (TypeError, (a, sa.to(torch.bfloat16), bt, sb)),
        (TypeError, (a, None, bt, sb)),
        (ValueError, (a, _t(10, 3, dtype=f32, device="cpu"), bt, sb)),
        (TypeError, (a, sa, bt, sb, _t(10, 200, dtype=f32))),
        (ValueError, (a, sa, bt, sb, _t(10, 201))),
    ]:
        with pytest.raises(exc):
            B.gemm_fp8_block(*args)
    wt, ws, off = _t(4, 200, 300, dtype=f8), _t(4, 2, 3, dtype=f32), _off(5)
    for exc, args in [
        (TypeError, (a, sa, wt, ws, None)),
        (ValueError, (a, sa, bt, sb, off)),
        (ValueError, (a, sa, wt, sb, off)),
        (ValueError, (a, sa, wt, ws, _off(4))),
        (TypeError, (a, sa, wt, ws, _off(5, torch.int64))),
    ]:
        with pytest.raises(exc):
            B.gemm_grouped_fp8_block(*args)


def test_workspace_of_unaligned_operands():
    """Bytes of the copies: rows of whole lines, of what does not lie on 16 bytes alone; refusals of sizes and kinds."""
    from gpu_operator_amd.ops import _lib

    if not _lib.group_lib_path().exists():
        pytest.skip("the library is not built")
    lib = _lib.load_group()

    def need(mode, rows, cols, red, experts, lda, ldb, b_expert, dtype=0, scale=0, a=1 << 20, b=1 << 21, rows_apart=0):
        return lib.amdgo_group_workspace(_lib.pack_group(a, b, 1 << 22, 0, 0, 1 << 23, lda, ldb, cols, b_expert, 0, rows_apart, 0, 0, 0, 0,
                                                         rows, cols, red, experts, mode, dtype, scale, 0, 0))

    assert need(0, 10, 20, 64, 3, 64, 64, 20 * 64) == 0
    assert need(0, 10, 20, 64, 3, 65, 64, 20 * 64) == 10 * 128                      # a's rows alone
    assert need(0, 10, 20, 64, 3, 64, 64, 20 * 64, b=(1 << 21) + 2) == 3 * 20 * 128
    assert need(0, 10, 20, 65, 3, 72, 72, 20 * 72) == (10 + 3 * 20) * 256           # the reduction's end: both
    assert need(1, 10, 64, 20, 3, 24, 64, 20 * 64) == 10 * 128 + 3 * 24 * 128       # zero rows behind each of bt's
    assert need(2, 33, 64, 500, 3, 33, 64, 0) == 500 * 128
    assert need(0, 10, 20, 130, 3, 130, 130, 20 * 130, dtype=2, scale=1) == (10 + 3 * 20) * 256
    assert need(0, 10, 20, 64, 0, 64, 64, 0) < 0 and need(3, 10, 20, 64, 3, 64, 64, 0) < 0
    assert need(0, 10, 20, 64, 3, 64, 64, 0, dtype=2) < 0 and need(0, 10, 20, 64, 3, 64, 64, 0, scale=1) < 0
    assert need(0, -1, 20, 64, 3, 64, 64, 0) < 0
    assert need(0, 10, 20, 64, 3, 65, 64, 20 * 64, rows_apart=1 << 30, dtype=2, scale=1) < 0   # scales' rows too far apart
    assert need(0, 10, 2 ** 31 - 1, 64, 1, 64, 64, 0) < 0                           # indices past 32 bits
    assert need(0, 10, 20, 2 ** 31 - 1, 3, 2 ** 31 - 1, 2 ** 31 - 1, 0) < 0         # rows too long for a copy
    assert need(0, 2 ** 31 - 1, 2 ** 31 - 1, 63, 2 ** 20, 63, 63, 63) < 0           # too many of them
