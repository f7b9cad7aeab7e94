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
in an ``out`` that the caller gives, and are zeros in one that is allocated here. An ``out`` shares no memory with the
operands (rows side by side in one buffer are none).

Autograd records :func:`grouped_linear`, and :func:`gemm_grouped` where an operand needs a gradient. The two gradients
have none themselves: a backward pass that reaches their results raises. A call with an ``out`` cannot be recorded and
is refused where an operand needs a gradient, as are forward-mode gradients. ``torch.func`` transforms end in torch's own
errors, since the kernels take addresses; ``torch.compile`` runs the calls between its graphs.

Operands may have any row stride; only the last dimension has to be contiguous. Operands whose rows do not lie on 16
bytes (or whose reduction does not fill 16-byte pieces) are copied into a workspace of the call first, all experts'
weights with them, to rows of whole 128-byte lines: it is about as large as those operands. Only the forward product of
up to 20 rows an expert reads them in place.
"""

from __future__ import annotations

import struct

from . import _lib

MODE_FORWARD, MODE_DGRAD, MODE_WGRAD = 0, 1, 2

# torch, from the first call on: the package imports without it, and looking it up in every helper took 0.4 us of a call
torch = None
_FORWARD_AD = None
_HALVES = ()


def load_torch():
    """torch, also for this module's helpers. Every entry point calls it before them."""
    global torch, _FORWARD_AD, _HALVES
    if torch is None:
        import torch as module
        import torch.autograd.forward_ad as _FORWARD_AD

        _HALVES = (module.bfloat16, module.float16)
        torch = module
    return torch


def _matrix(t, name: str, dims: int, dtypes, device=None):
    """A GPU tensor of `dims` dimensions whose last one is contiguous; its strides."""
    try:
        strides = t.stride()
        if t.dtype in dtypes and len(strides) == dims and t.is_cuda and (device is None or t.device == device) \
                and (strides[-1] == 1 or t.shape[-1] <= 1 or t.numel() == 0):
            return strides
    except AttributeError:
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}") from None
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if len(strides) != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other operands on {device}")
    raise ValueError(f"{name}'s last dimension must be contiguous, got strides {strides}")


def _row_stride(shape, strides) -> int:
    """Elements between two rows (a single row's own stride says nothing)."""
    return strides[-2] if shape[-2] > 1 else shape[-1]


def _stride(shape, strides, dim: int) -> int:
    """The same of any dimension: 0 where there is no second one."""
    return strides[dim] if shape[dim] > 1 else 0


def _reach(t) -> int:
    """Bytes from t's first to behind its last."""
    last = 1
    for n, s in zip(t.shape, t.stride()):
        last += (n - 1) * s
    return last * t.element_size()


def _rows(t):
    """The addresses of t's rows (of its elements, where those lie apart), sorted, and the bytes of each."""
    size, whole = t.element_size(), t.stride(-1) == 1 or t.shape[-1] == 1
    at = torch.tensor([t.data_ptr()], device="cpu")
    for n, s in list(zip(t.shape, t.stride()))[: -1 if whole else None]:
        at = (at[:, None] + torch.arange(n, device="cpu") * (s * size)).flatten()
    return at.unique(), (t.shape[-1] if whole else 1) * size


def _shares_memory(out, t) -> bool:
    """Whether a byte of `out` is one of t's."""
    load_torch()
    begin, first = out.data_ptr(), t.data_ptr()
    if first >= begin + _reach(out) or begin >= first + _reach(t) or not out.numel() or not t.numel():
        return False
    size, other = out.element_size(), t.element_size()
    if out.dim() == t.dim() == 2 and out.stride(0) > 0 and out.stride(0) * size == t.stride(0) * other and t.stride(1) == 1:
        pitch = out.stride(0) * size                     # rows as far apart: shared, or side by side, in every row alike
        d = (first - begin) % pitch
        if out.shape[1] * size <= d and d + t.shape[1] * other <= pitch:
            return False
    (at, width), (b, wide) = _rows(out), _rows(t)
    i = torch.searchsorted(at, b)                        # at[i - 1] < b <= at[i]
    after, before = at[i.clamp_max(len(at) - 1)], at[(i - 1).clamp_min(0)]
    return bool((((i < len(at)) & (after < b + wide)) | ((i > 0) & (before + width > b))).any())


def _refuse_shared(outs, operands) -> None:
    """Where the library says that the outputs may share memory with the operands, or with each other."""
    for i, out in enumerate(outs):
        for t in (*outs[:i], *operands):
            if t is not None and _shares_memory(out, t):
                raise ValueError("an output shares memory with an operand or with another output")


def _out(out, shape, dtype, device):
    """(tensor to write, its row stride, whether rows that no expert owns have to be cleared). The rows (and matrices)
    of an output may be apart, or lie among one another, but not overlap."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device), shape[-1], 1
    strides = _matrix(out, "out", len(shape), (dtype,), device)
    if out.shape != shape:
        raise ValueError(f"out must be {shape}, got {tuple(out.shape)}")
    ld = _row_stride(shape, strides)
    if out.numel():
        if ld < shape[-1]:
            raise ValueError(f"out's rows overlap: strides {strides}")
        if len(shape) == 3 and shape[0] > 1:
            # the matrices one behind the other, or the rows of one between those of the others
            apart = strides[0] >= (shape[1] - 1) * ld + shape[2]
            among = strides[0] >= shape[2] and (shape[1] == 1 or ld >= (shape[0] - 1) * strides[0] + shape[2])
            if not (apart or among):
                raise ValueError(f"out's matrices overlap: strides {strides}")
    torch._C._increment_version((out,))       # autograd does not see the kernels' writes
    return out, ld, 0


def _offsets(offsets, experts: int, device) -> None:
    if not isinstance(offsets, torch.Tensor) or offsets.dtype != torch.int32:
        raise TypeError("offsets must be an int32 tensor")
    if offsets.dim() != 1 or offsets.shape[0] != experts + 1 or not offsets.is_contiguous():
        raise ValueError(f"offsets must be contiguous [{experts + 1}], got {tuple(offsets.shape)}")
    if offsets.device != device:
        raise ValueError(f"offsets are on {offsets.device}, the operands on {device}")


def needs_gradient(out) -> bool:
    """Whether an output, or None, does (it may be anything yet)."""
    return out is not None and getattr(out, "requires_grad", False)


def recorded(what: str, *outs) -> bool:
    """Whether autograd has to record this call, an operand or output of which needs a gradient. One with an output of the
    caller's (`outs`: those or None) cannot be, and is refused as torch's own are. (launch() refuses forward-mode gradients.)"""
    if not torch.is_grad_enabled():
        return False
    if any(t is not None for t in outs):
        raise RuntimeError(f"{what}: functions with out=... don't support automatic differentiation, but one of the "
                           "arguments requires grad (detach it, or call under torch.no_grad())")
    return True


_NO_GRADIENT = None


def without_gradient(what: str, call, *operands):
    """The results of call() as ones that depend on `operands`: a backward pass that reaches them says that there is no
    gradient, instead of going on without one."""
    global _NO_GRADIENT
    if _NO_GRADIENT is None:
        class NoGradient(torch.autograd.Function):
            @staticmethod
            def forward(ctx, what, call, *operands):
                ctx.set_materialize_grads(False)
                ctx.what = what
                return call()

            @staticmethod
            def backward(ctx, *grads):
                raise RuntimeError(f"{ctx.what} has no gradient: detach its operands, or call it under torch.no_grad()")

        _NO_GRADIENT = NoGradient
    return _NO_GRADIENT.apply(what, call, *operands)


def _shape(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def launch(device, what: str, entry, outs, operands, pack, *fields) -> None:
    """One launch on the device's current stream; `entry`: a function of the library, `pack`: its arguments' packer."""
    try:
        args = pack(*fields)
    except struct.error:
        raise ValueError(f"{what}: a dimension over 2^31 - 1 or a stride over 2^63 - 1") from None
    if _FORWARD_AD._current_level >= 0:
        for t in operands:
            if t is not None and _FORWARD_AD.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what} has no forward-mode gradient")
    # (torch.cuda.current_device() and current_stream() make a call 1.2 us longer)
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        err = entry(args, stream)
    else:                                    # a launch on a device's stream needs that device current
        with torch.cuda.device(index):
            err = entry(args, stream)
    if err:
        if err == _lib.MAY_SHARE:
            _refuse_shared(outs, operands)
            with torch.cuda.device(index):
                err = getattr(_lib.load_group(), entry.__name__ + "_apart")(args, stream)
        if err == _lib.NEEDS_PACKING:
            return _launch_packed(device, what, args, stream)
        _lib.check(err, what)


def _launch_packed(device, what: str, args: bytes, stream: int) -> None:
    """The product on copies, in a workspace of the call, of what the kernels cannot read in place."""
    lib = _lib.load_group()
    need = lib.amdgo_group_workspace(args)
    if need < 0:
        raise ValueError(f"{what}: 256 rows of an operand or of its scales reach over 2 GiB")
    with torch.cuda.device(device):
        space = torch.empty(need, dtype=torch.uint8, device=device)
        err = lib.amdgo_gemm_group_packed(args, space.data_ptr(), stream)
    _lib.check(err, what)


def _dtype_code(dtype) -> int:
    return 0 if dtype == torch.bfloat16 else 1


def gemm_grouped(a, bt, offsets, out=None):
    """``out[t] = a[t] @ bt[e(t)].T``. ``a``: [T,K], ``bt``: [E,N,K], bf16 or fp16; ``out``: [T,N] of their type.
    Where ``a`` or ``bt`` needs a gradient this is :func:`grouped_linear`."""
    load_torch()
    sa = _matrix(a, "a", 2, _HALVES)
    device, dtype = a.device, a.dtype
    sb = _matrix(bt, "bt", 3, (dtype,), device)
    (t, k), (e, n, kb) = a.shape, bt.shape
    if kb != k:
        raise ValueError(f"a is [{t},{k}], bt is [{e},{n},{kb}]: their last dimensions differ")
    if e < 1:
        raise ValueError("bt has no experts")
    _offsets(offsets, e, device)
    if (a.requires_grad or bt.requires_grad or needs_gradient(out)) and recorded("gemm_grouped", out):
        return grouped_linear(a, bt, offsets)
    out, ldc, rest = _out(out, (t, n), dtype, device)
    if t and n:
        launch(device, "amdgo_gemm_group", _lib.load_group().amdgo_gemm_group, (out,), (a, bt, offsets), _lib.pack_group,
               a.data_ptr(), bt.data_ptr(), out.data_ptr(), 0, 0, offsets.data_ptr(),
               _row_stride((t, k), sa), _row_stride((n, k), sb), ldc, _stride((e,), sb, 0), 0, 0, 0, 0, 0, 0,
               t, n, k, e, MODE_FORWARD, _dtype_code(dtype), 0, rest, 0)
    return out


def gemm_grouped_dgrad(dc, bt, offsets, out=None):
    """The product's gradient for its rows: ``out[t] = dc[t] @ bt[e(t)]``. ``dc``: [T,N], ``bt``: [E,N,K]; ``out``: [T,K]."""
    load_torch()
    sd = _matrix(dc, "dc", 2, _HALVES)
    device, dtype = dc.device, dc.dtype
    sb = _matrix(bt, "bt", 3, (dtype,), device)
    (t, n), (e, nb, k) = dc.shape, bt.shape
    if nb != n:
        raise ValueError(f"dc is [{t},{n}], bt is [{e},{nb},{k}]: the middle dimension of bt is not dc's last")
    if e < 1:
        raise ValueError("bt has no experts")
    _offsets(offsets, e, device)
    if (dc.requires_grad or bt.requires_grad or needs_gradient(out)) and recorded("gemm_grouped_dgrad", out):
        return without_gradient("gemm_grouped_dgrad", lambda: gemm_grouped_dgrad(dc, bt, offsets), dc, bt)
    out, ldc, rest = _out(out, (t, k), dtype, device)
    if t and k:
        launch(device, "amdgo_gemm_group(dgrad)", _lib.load_group().amdgo_gemm_group, (out,), (dc, bt, offsets), _lib.pack_group,
               dc.data_ptr(), bt.data_ptr(), out.data_ptr(), 0, 0, offsets.data_ptr(),
               _row_stride((t, n), sd), _row_stride((n, k), sb), ldc, _stride((e,), sb, 0), 0, 0, 0, 0, 0, 0,
               t, k, n, e, MODE_DGRAD, _dtype_code(dtype), 0, rest, 0)
    return out


def gemm_grouped_wgrad(dc, a, offsets, out=None):
    """The product's gradient for its weights: ``out[e] = dc_e.T @ a_e`` over the rows of expert ``e`` (zeros where it
    has none). ``dc``: [T,N], ``a``: [T,K]; ``out``: [E,N,K] of their type, rounded once from the fp32 sum."""
    load_torch()
    sd = _matrix(dc, "dc", 2, _HALVES)
    device, dtype = dc.device, dc.dtype
    sa = _matrix(a, "a", 2, (dtype,), device)
    (t, n), (ta, k) = dc.shape, a.shape
    if ta != t:
        raise ValueError(f"dc has {t} rows, a has {ta}")
    _shape(isinstance(offsets, torch.Tensor) and offsets.dim() == 1 and offsets.shape[0] >= 2, "offsets must be [E + 1]")
    e = offsets.shape[0] - 1
    _offsets(offsets, e, device)
    if (dc.requires_grad or a.requires_grad or needs_gradient(out)) and recorded("gemm_grouped_wgrad", out):
        return without_gradient("gemm_grouped_wgrad", lambda: gemm_grouped_wgrad(dc, a, offsets), dc, a)
    out, ldc, _ = _out(out, (e, n, k), dtype, device)
    if n and k:
        launch(device, "amdgo_gemm_group(wgrad)", _lib.load_group().amdgo_gemm_group, (out,), (dc, a, offsets), _lib.pack_group,
               dc.data_ptr(), a.data_ptr(), out.data_ptr(), 0, 0, offsets.data_ptr(),
               _row_stride((t, n), sd), _row_stride((t, k), sa), ldc, 0, out.stride(0) if e > 1 else 0, 0, 0, 0, 0, 0,
               n, k, t, e, MODE_WGRAD, _dtype_code(dtype), 0, 0, 0)
    return out


_FUNCTION = None


def _function():
    """The autograd function, made at its first use (the package imports without torch)."""
    global _FUNCTION
    load_torch()
    if _FUNCTION is None:
        def gradients(ctx, dc):
            a, bt, offsets = ctx.saved_tensors
            if dc.stride(-1) != 1:
                dc = dc.contiguous()            # a gradient broadcast by a sum has strides of zero
            da = gemm_grouped_dgrad(dc, bt, offsets) if ctx.needs_input_grad[0] else None
            dbt = gemm_grouped_wgrad(dc, a, offsets) if ctx.needs_input_grad[1] else None
            return da, dbt, None

        refusing = torch.autograd.function.once_differentiable(gradients)

        class GroupedLinear(torch.autograd.Function):
            @staticmethod
            def forward(ctx, a, bt, offsets):
                ctx.save_for_backward(a, bt, offsets)
                return gemm_grouped(a, bt, offsets)

            @staticmethod
            def backward(ctx, dc):
                # a gradient of the gradients is refused where one can be asked for (elsewhere that costs a step 18 us)
                return (refusing if torch.is_grad_enabled() else gradients)(ctx, dc)

        _FUNCTION = GroupedLinear
    return _FUNCTION


def grouped_linear(a, bt, offsets):
    """:func:`gemm_grouped` under autograd: gradients for ``a`` (zeros in rows that no expert owns) and ``bt``. A gradient of
    the gradients is refused. A step may be captured into a graph, forward and backward together, once the results of
    earlier calls on the same leaves are gone (torch ends the process where such an eager graph still lives)."""
    return _function().apply(a, bt, offsets)
