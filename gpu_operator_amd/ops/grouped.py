"""Matrix products of rows sorted by expert: hand-written CDNA4 MFMA kernels (native/hip/gemm_group.hip).

``offsets`` (int32 ``[E + 1]`` on the GPU, non-decreasing) says which rows belong to which expert: expert ``e``
owns the rows ``offsets[e] .. offsets[e + 1]`` and multiplies them with its own weights, any number of them,
none included. The offsets stay on the device: nothing here waits for the GPU. What they hold is clamped to
the rows that exist; offsets that decrease give unspecified rows, never an access outside the operands.

* :func:`gemm_grouped`        ``c[t] = a[t] @ bt[e(t)].T``, bf16 or fp16, fp32 accumulation;
* :func:`gemm_grouped_dgrad`  its gradient for the rows, ``dc[t] @ bt[e(t)]``;
* :func:`gemm_grouped_wgrad`  its gradient for the weights, ``dc_e.T @ a_e`` for each expert;
* :func:`grouped_linear`      the product with both gradients under autograd.

Rows that no expert owns (before ``offsets[0]``, from ``offsets[E]`` on: a batch's padding) are left as they are
in an ``out`` that the caller gives, and are zeros in one that is allocated here. Operands may have any row
stride; only the last dimension has to be contiguous.
"""

from __future__ import annotations

import contextlib
import ctypes

from . import _lib

MODE_FORWARD, MODE_DGRAD, MODE_WGRAD = 0, 1, 2
_INT_MAX = 2 ** 31 - 1


def _matrix(t, name: str, dims: int, dtypes, device=None):
    """A GPU tensor of `dims` dimensions whose last one is contiguous and whose rows do not overlap."""
    import torch

    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other operands on {device}")
    if max(t.shape, default=0) > _INT_MAX:
        raise ValueError(f"{name} has a dimension over 2^31 - 1: {tuple(t.shape)}")
    if t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous, got strides {t.stride()}")
    if any(s < 0 for s in t.stride()):
        raise ValueError(f"{name} has a negative stride")


def _row_stride(t) -> int:
    """Elements between two rows (a single row's own stride says nothing)."""
    return t.stride(-2) if t.shape[-2] > 1 else t.shape[-1]


def _written(t, name: str) -> None:
    """An output's rows (and matrices) may be apart, but not overlap."""
    rows, cols = t.shape[-2:]
    if t.numel() and rows > 1 and t.stride(-2) < cols:
        raise ValueError(f"{name}'s rows overlap: strides {t.stride()}")
    if t.numel() and t.dim() == 3 and t.shape[0] > 1 and t.stride(0) < (rows - 1) * _row_stride(t) + cols:
        raise ValueError(f"{name}'s matrices overlap: strides {t.stride()}")


def _offsets(offsets, experts: int, device) -> None:
    import torch

    if not isinstance(offsets, torch.Tensor) or offsets.dtype != torch.int32:
        raise TypeError("offsets must be an int32 tensor")
    if offsets.dim() != 1 or offsets.shape[0] != experts + 1 or not offsets.is_contiguous():
        raise ValueError(f"offsets must be contiguous [{experts + 1}], got {tuple(offsets.shape)}")
    if offsets.device != device:
        raise ValueError(f"offsets are on {offsets.device}, the operands on {device}")


def _shape(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _on(device):
    """The device that a launch on one of its streams needs current."""
    import torch

    return contextlib.nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def launch(device, what: str, **fields) -> None:
    import torch

    args = _lib.GroupArgs(**fields)
    with _on(device):
        err = _lib.load_group().amdgo_gemm_group(ctypes.byref(args), torch.cuda.current_stream(device).cuda_stream)
    _lib.check(err, what)


def _dtype_code(dtype) -> int:
    import torch

    return 0 if dtype == torch.bfloat16 else 1


def _halves():
    import torch

    return (torch.bfloat16, torch.float16)


def _out(out, shape, like, name="out"):
    """(tensor to write, whether rows that no expert owns have to be cleared)"""
    import torch

    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device), 1
    _matrix(out, name, len(shape), (like.dtype,), like.device)
    _shape(tuple(out.shape) == tuple(shape), f"{name} must be {tuple(shape)}, got {tuple(out.shape)}")
    _written(out, name)
    return out, 0


def gemm_grouped(a, bt, offsets, out=None):
    """``out[t] = a[t] @ bt[e(t)].T``. ``a``: [T,K], ``bt``: [E,N,K], bf16 or fp16; ``out``: [T,N] of their type."""
    _matrix(a, "a", 2, _halves())
    _matrix(bt, "bt", 3, (a.dtype,), a.device)
    t, k = a.shape
    e, n, kb = bt.shape
    _shape(kb == k, f"a is [{t},{k}], bt is [{e},{n},{kb}]: their last dimensions differ")
    _shape(e >= 1, "bt has no experts")
    _offsets(offsets, e, a.device)
    out, rest = _out(out, (t, n), a)
    if t and n:
        launch(a.device, "amdgo_gemm_group", a=a.data_ptr(), b=bt.data_ptr(), c=out.data_ptr(), offsets=offsets.data_ptr(),
               lda=_row_stride(a), ldb=_row_stride(bt), ldc=_row_stride(out), b_expert=bt.stride(0), rows=t, cols=n, red=k,
               experts=e, mode=MODE_FORWARD, dtype=_dtype_code(a.dtype), zero_rest=rest)
    return out


def gemm_grouped_dgrad(dc, bt, offsets, out=None):
    """The product's gradient for its rows: ``out[t] = dc[t] @ bt[e(t)]``. ``dc``: [T,N], ``bt``: [E,N,K]; ``out``: [T,K]."""
    _matrix(dc, "dc", 2, _halves())
    _matrix(bt, "bt", 3, (dc.dtype,), dc.device)
    t, n = dc.shape
    e, nb, k = bt.shape
    _shape(nb == n, f"dc is [{t},{n}], bt is [{e},{nb},{k}]: the middle dimension of bt is not dc's last")
    _shape(e >= 1, "bt has no experts")
    _offsets(offsets, e, dc.device)
    out, rest = _out(out, (t, k), dc)
    if t and k:
        launch(dc.device, "amdgo_gemm_group(dgrad)", a=dc.data_ptr(), b=bt.data_ptr(), c=out.data_ptr(),
               offsets=offsets.data_ptr(), lda=_row_stride(dc), ldb=_row_stride(bt), ldc=_row_stride(out),
               b_expert=bt.stride(0), rows=t, cols=k, red=n, experts=e, mode=MODE_DGRAD, dtype=_dtype_code(dc.dtype),
               zero_rest=rest)
    return out


def gemm_grouped_wgrad(dc, a, offsets, out=None):
    """The product's gradient for its weights: ``out[e] = dc_e.T @ a_e`` over the rows of expert ``e`` (zeros where it
    has none). ``dc``: [T,N], ``a``: [T,K]; ``out``: [E,N,K] of their type, rounded once from the fp32 sum."""
    import torch

    _matrix(dc, "dc", 2, _halves())
    _matrix(a, "a", 2, (dc.dtype,), dc.device)
    t, n = dc.shape
    ta, k = a.shape
    _shape(ta == t, f"dc has {t} rows, a has {ta}")
    _shape(isinstance(offsets, torch.Tensor) and offsets.dim() == 1 and offsets.shape[0] >= 2, "offsets must be [E + 1]")
    e = offsets.shape[0] - 1
    _offsets(offsets, e, dc.device)
    out, _ = _out(out, (e, n, k), dc)
    if n and k:
        launch(dc.device, "amdgo_gemm_group(wgrad)", a=dc.data_ptr(), b=a.data_ptr(), c=out.data_ptr(),
               offsets=offsets.data_ptr(), lda=_row_stride(dc), ldb=_row_stride(a), ldc=_row_stride(out),
               c_expert=out.stride(0), rows=n, cols=k, red=t, experts=e, mode=MODE_WGRAD, dtype=_dtype_code(dc.dtype))
    return out


_FUNCTION = None


def _function():
    """The autograd function, made at its first use (the package imports without torch)."""
    global _FUNCTION
    if _FUNCTION is None:
        import torch

        class GroupedLinear(torch.autograd.Function):
            @staticmethod
            def forward(ctx, a, bt, offsets):
                ctx.save_for_backward(a, bt, offsets)
                return gemm_grouped(a, bt, offsets)

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, dc):
                a, bt, offsets = ctx.saved_tensors
                if dc.dim() == 2 and dc.numel() and (dc.stride(-1) != 1 or _row_stride(dc) < dc.shape[-1]):
                    dc = dc.contiguous()            # a gradient broadcast by a sum has strides of zero
                da = gemm_grouped_dgrad(dc, bt, offsets) if ctx.needs_input_grad[0] else None
                dbt = gemm_grouped_wgrad(dc, a, offsets) if ctx.needs_input_grad[1] else None
                return da, dbt, None

        _FUNCTION = GroupedLinear
    return _FUNCTION


def grouped_linear(a, bt, offsets):
    """:func:`gemm_grouped` under autograd: gradients for ``a`` (zeros in rows that no expert owns) and ``bt``."""
    return _function().apply(a, bt, offsets)
