"""Block-scaled fp8 matrix products and their quantiser (native/hip/gemm_group.hip, quant_block.hip).

An operand is OCP e4m3fn with one scale for each block of 128 columns: of one row (activations, scales
``[rows, ceil(cols / 128)]``) or of 128 rows (weights, scales ``[ceil(rows / 128), ceil(cols / 128)]``). What it
stands for is ``q * scale``. Scales are float32, or powers of two (``torch.float8_e8m0fnu``), which the matrix
instructions apply themselves.

* :func:`quantize_fp8_block`       a bf16 / fp16 / fp32 matrix to such an operand;
* :func:`gemm_fp8_block`           ``a @ bt.T`` of activations and weights, bf16 out;
* :func:`gemm_grouped_fp8_block`   the same for rows sorted by expert (see :mod:`.grouped`).

Sums are fp32. With float32 scales each block's sum is formed first and then weighted with the product of its
two scales (a float32: scales whose product leaves float32's range are not supported).
"""

from __future__ import annotations

import ctypes

from . import _lib
from .grouped import MODE_FORWARD, _matrix, _offsets, _on, _row_stride, _shape, _written, launch

BLOCK = 128


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def quantize_fp8_block(x, block_rows: int = 1, *, scale_dtype=None, out=None, scale_out=None):
    """``(q, scale)`` of ``x`` ([rows, cols] or [batch, rows, cols]; bf16, fp16 or fp32; any row stride).

    ``block_rows``: 1 (activations) or 128 (weights). ``scale_dtype``: ``torch.float32`` (the default) or
    ``torch.float8_e8m0fnu``. The scale is ``amax / 448`` (or the least power of two not under it) over the block's
    finite values, at least 2^-126; ``q`` is the nearest e4m3 value of the exact quotient, ties to even. An infinity
    or NaN becomes NaN. ``out`` and ``scale_out``, where given, are contiguous tensors of the results' shapes.
    """
    import torch

    scale_dtype = scale_dtype or torch.float32
    codes = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
    _shape(isinstance(x, torch.Tensor) and x.dim() in (2, 3), "x must be a tensor of 2 or 3 dimensions")
    _matrix(x, "x", x.dim(), tuple(codes))
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows must be 1 or {BLOCK}, got {block_rows}")
    if scale_dtype not in (torch.float32, torch.float8_e8m0fnu):
        raise TypeError(f"scale_dtype must be torch.float32 or torch.float8_e8m0fnu, got {scale_dtype}")
    batch, (rows, cols) = (x.shape[0] if x.dim() == 3 else 1), x.shape[-2:]
    scale_shape = (*x.shape[:-2], rows if block_rows == 1 else _blocks(rows), _blocks(cols))
    q = _result(out, "out", tuple(x.shape), torch.float8_e4m3fn, x)
    s = _result(scale_out, "scale_out", scale_shape, scale_dtype, x)
    if x.numel():
        args = _lib.QuantArgs(x=x.data_ptr(), q=q.data_ptr(), s=s.data_ptr(), ld=_row_stride(x),
                              batch_stride=x.stride(0) if x.dim() == 3 else 0, batches=batch, rows=rows, cols=cols,
                              dtype=codes[x.dtype], block_rows=block_rows, e8=int(scale_dtype == torch.float8_e8m0fnu))
        with _on(x.device):
            err = _lib.load_group().amdgo_quantize_fp8_block(ctypes.byref(args),
                                                             torch.cuda.current_stream(x.device).cuda_stream)
        _lib.check(err, "amdgo_quantize_fp8_block")
    return q, s


def _result(out, name, shape, dtype, like):
    import torch

    if out is None:
        return torch.empty(shape, dtype=dtype, device=like.device)
    _matrix(out, name, len(shape), (dtype,), like.device)
    _shape(tuple(out.shape) == shape and out.is_contiguous(), f"{name} must be contiguous {shape}, got {tuple(out.shape)}")
    return out


def _scale(t, name, shape, dtypes, device) -> None:
    import torch

    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, "
                        f"got {getattr(t, 'dtype', type(t).__name__)}")
    _shape(tuple(t.shape) == shape, f"{name} must be {shape}, got {tuple(t.shape)}")
    _shape(t.device == device, f"{name} is on {t.device}, the operands on {device}")


def _product(a, a_scale, bt, bt_scale, offsets, out):
    import torch

    f8 = (torch.float8_e4m3fn,)
    dims = 2 if offsets is None else 3
    _matrix(a, "a", 2, f8)
    _matrix(bt, "bt", dims, f8, a.device)
    m, k = a.shape
    n = bt.shape[-2]
    e = bt.shape[0] if dims == 3 else 1
    _shape(bt.shape[-1] == k, f"a is [{m},{k}], bt is {tuple(bt.shape)}: their last dimensions differ")
    _shape(e >= 1, "bt has no experts")
    _scale(a_scale, "a_scale", (m, _blocks(k)), (torch.float32, torch.float8_e8m0fnu), a.device)
    _scale(bt_scale, "bt_scale", (*bt.shape[:-2], _blocks(n), _blocks(k)), (a_scale.dtype,), a.device)
    if offsets is not None:
        _offsets(offsets, e, a.device)
    rest = 0
    if out is None:
        out, rest = torch.empty((m, n), dtype=torch.bfloat16, device=a.device), int(offsets is not None)
    else:
        _matrix(out, "out", 2, (torch.bfloat16,), a.device)
        _shape(tuple(out.shape) == (m, n), f"out must be [{m},{n}], got {tuple(out.shape)}")
        _written(out, "out")
    if m and n:
        launch(a.device, "amdgo_gemm_group(fp8)", a=a.data_ptr(), b=bt.data_ptr(), c=out.data_ptr(),
               a_scale=a_scale.data_ptr(), b_scale=bt_scale.data_ptr(),
               offsets=None if offsets is None else offsets.data_ptr(), lda=_row_stride(a), ldb=_row_stride(bt),
               ldc=_row_stride(out), b_expert=bt.stride(0) if dims == 3 else 0, as_row=a_scale.stride(0),
               as_k=a_scale.stride(1), bs_expert=bt_scale.stride(0) if dims == 3 else 0, bs_row=bt_scale.stride(-2),
               bs_k=bt_scale.stride(-1), rows=m, cols=n, red=k, experts=e, mode=MODE_FORWARD, dtype=2,
               scale=1 if a_scale.dtype == torch.float32 else 2, zero_rest=rest)
    return out


def gemm_fp8_block(a, a_scale, bt, bt_scale, out=None):
    """``(a * a_scale) @ (bt * bt_scale).T``. ``a``: [M,K] e4m3fn with ``a_scale`` [M, ceil(K/128)], ``bt``: [N,K] with
    ``bt_scale`` [ceil(N/128), ceil(K/128)], both scales of one type and any strides; ``out``: [M,N] bf16."""
    return _product(a, a_scale, bt, bt_scale, None, out)


def gemm_grouped_fp8_block(a, a_scale, bt, bt_scale, offsets, out=None):
    """:func:`gemm_fp8_block` of rows sorted by expert: ``bt`` [E,N,K], ``bt_scale`` [E, ceil(N/128), ceil(K/128)] and
    ``offsets`` int32 [E + 1] as in :func:`gpu_operator_amd.ops.grouped.gemm_grouped`."""
    if offsets is None:
        raise TypeError("offsets must be an int32 tensor")
    return _product(a, a_scale, bt, bt_scale, offsets, out)
