"""Which outputs share memory with an operand, checked without a GPU on views of one buffer."""

import itertools

import pytest
import torch

from gpu_operator_amd.ops import grouped as G


def _bytes(t):
    """The addresses of all of t's bytes."""
    at = {t.data_ptr()}
    for n, s in zip(t.shape, t.stride()):
        at = {a + i * s * t.element_size() for a in at for i in range(n)}
    return {a + i for a in at for i in range(t.element_size())} if t.numel() else set()


def test_shared_memory_is_found_exactly():
    """Every pair of views: side by side in the same rows, of other types and pitches, batched, broadcast, single rows, empty."""
    flat = torch.zeros(4096, dtype=torch.uint8)
    half, full = flat.view(torch.bfloat16), flat.view(torch.float32)
    views = [half.as_strided(s, st, at) for s, st, at in [
        ((4, 8), (32, 1), 0), ((4, 8), (32, 1), 8), ((4, 8), (32, 1), 20), ((4, 8), (32, 1), 28), ((4, 8), (32, 1), 7), ((4, 25), (32, 1), 7),
        ((4, 8), (24, 1), 8), ((1, 8), (1, 1), 40), ((1, 8), (7, 1), 48), ((0, 8), (8, 1), 0), ((6, 2), (0, 1), 36), ((4, 8), (32, 1), 1000),
        ((2, 4, 8), (128, 32, 1), 8), ((2, 4, 8), (16, 32, 1), 0), ((2, 4, 8), (8, 40, 1), 4), ((3, 1, 8), (64, 9, 1), 24), ((9, 1), (16, 5), 3),
        ((4, 8), (64, 2), 9)]]
    views += [full.as_strided((4, 2), (16, 1), 4), full.as_strided((4, 3), (1, 5), 6), full.as_strided((5,), (1,), 3)]
    for a, b in itertools.product(views[:-1], views):
        if a.stride(-1) == 1 or a.shape[-1] == 1:
            assert G._shares_memory(a, b) == bool(_bytes(a) & _bytes(b)), (a.shape, a.stride(), b.shape, b.stride())


@pytest.mark.parametrize("e", [1, 3])
def test_rows_side_by_side_do_not_meet(e):
    buf = torch.zeros((50, 96), dtype=torch.bfloat16)
    assert not G._shares_memory(buf[:, :40], buf[:, 40:])
    assert G._shares_memory(buf[:, :41], buf[:, 40:])
    assert not G._shares_memory(buf[: 25], buf[25:].view(e, -1, 32) if e == 3 else buf[25:][None])
    assert G._shares_memory(buf, buf) and not G._shares_memory(buf, torch.zeros_like(buf))


def test_the_library_looks_before_it_launches():
    """Addresses alone: each operand in turn within the output's reach is told to the caller, whatever the mode."""
    from gpu_operator_amd.ops import _lib

    if not _lib.group_lib_path().exists():
        pytest.skip("the library is not built")
    lib, c = _lib.load_group(), 1 << 30

    def group(mode, dtype=0, scale=0, a=1 << 20, b=1 << 21, sa=0, sb=0, off=1 << 23, ldc=64, c_expert=0, lda=64):
        return lib.amdgo_gemm_group(_lib.pack_group(a, b, c, sa, sb, off, lda, 64, ldc, 64 * 64, c_expert, 1, 10, 1, 1, 1,
                                                    10, 64, 64, 3, mode, dtype, scale, 0, 0), None)

    last = c + 10 * 64 * 2
    for mode in (0, 1):
        for at in (c, c - 2, last - 2, c - 10 * 64 * 2 + 2):
            assert group(mode, a=at) == _lib.MAY_SHARE
        for at in (c - 3 * 64 * 64 * 2 + 2, last - 16):
            assert group(mode, b=at) == _lib.MAY_SHARE
        assert group(mode, off=last - 4) == _lib.MAY_SHARE and group(mode, off=c - 12) == _lib.MAY_SHARE
        assert group(mode, a=c + 2 * 64 - 2, ldc=128, lda=128) == _lib.MAY_SHARE       # side by side, but for one element
        assert group(mode, a=c + 2 * 64 + 2, ldc=128, lda=128) == _lib.MAY_SHARE
    assert group(2, a=c + (2 * 640 + 10 * 64) * 2 - 2, c_expert=640) == _lib.MAY_SHARE
    assert group(2, b=c - 64 * 64 * 2 + 2, c_expert=640) == _lib.MAY_SHARE
    for scale, size in ((1, 4), (2, 1)):
        assert group(0, 2, scale, sa=last - size, sb=1 << 24) == _lib.MAY_SHARE
        assert group(0, 2, scale, sa=1 << 24, sb=last - size) == _lib.MAY_SHARE

    def quantize(x=1 << 20, q=1 << 22, s=1 << 24, block_rows=1):
        return lib.amdgo_quantize_fp8_block(_lib.pack_quant(x, q, s, 300, 0, 1, 10, 300, 0, block_rows, 0), None)

    x = 1 << 20
    assert quantize(q=x + 10 * 300 * 2 - 1) == quantize(q=x - 2999) == quantize(s=x + 5996) == quantize(s=x - 116) == _lib.MAY_SHARE
    assert quantize(s=x - 8, block_rows=128) == quantize(s=(1 << 22) + 2996) == _lib.MAY_SHARE
