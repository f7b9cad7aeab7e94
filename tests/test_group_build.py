"""Static audit of the grouped products' and the quantiser's gfx950 code (CPU only: hipcc cross-compiles).

The ping-pong kernel's waits count the memory instructions that a wave has in flight, the stores of its result among them;
a register spilled to memory would be one more that nothing counts."""

import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")


@pytest.fixture(scope="module", params=["gemm_group.hip", "quant_block.hip"])
def kernels(request, tmp_path_factory):
    from gpu_operator_amd import _build

    (target,) = [t for t in _build.TARGETS if t.name == "libamdgo_group.so"]
    flags = [f for f in target.command() if f.startswith(("-O", "-std", "-I", "--offload-arch")) or f in
             ("-Xclang", "-target-feature", "-packed-fp32-ops")]
    out = tmp_path_factory.mktemp("group_asm") / "group.s"
    subprocess.run([HIPCC, *flags, "--cuda-device-only", "-S", os.path.join(ROOT, "native", "hip", request.param), "-o", str(out)],
                   check=True, capture_output=True, timeout=600)
    asm = out.read_text()
    found = {m.group(1): asm[m.start():asm.index(".end_amdhsa_kernel", m.start())]
             for m in re.finditer(r"^(_Z\w*(?:group|quantize|pack)_\w+):", asm, re.M)}
    assert len(found) >= 10
    sizes = re.findall(r"^; ScratchSize: (\d+)", asm, re.M) + re.findall(r"\.vgpr_spill_count:\s+(\d+)", asm)
    return found, sizes


def test_nothing_is_kept_in_memory(kernels):
    found, sizes = kernels
    assert len(sizes) >= 2 * len(found) and set(sizes) == {"0"}
    for name, body in found.items():
        assert "scratch_" not in body, name


def test_no_packed_float32_instructions(kernels):
    for name, body in kernels[0].items():
        assert not re.search(r"\bv_pk_(?:add|mul|fma)_f32\b", body), name


def test_no_atomics(kernels):
    """The same call gives the same bits."""
    for name, body in kernels[0].items():
        assert not re.search(r"\b(?:global|buffer|flat|ds)_(?:atomic|add|cmpst)\w*", body), name
