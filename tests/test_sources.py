"""CPU tier: properties of the CUDA sources that no run can show."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "avelang_b200", "csrc")


def _code(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", text, flags=re.S))


# launched with <<<>>>: they start once everything before them in the stream has ended
ORDERED = ("amax_bf16_kernel", "sf_to_tiled_kernel", "pack_weight_tiles_kernel", "reduce_partials_kernel")


def _without(code, kernel):
    """The source without that kernel's definition."""
    at = re.search(r"__global__[^{;]*\b" + kernel + r"\s*\([^{;]*\{", code)
    if at is None:
        return code
    end, depth = at.end(), 1
    while depth:
        depth += {"{": 1, "}": -1}.get(code[end], 0)
        end += 1
    return code[:at.start()] + code[end:]


def test_ordered_kernels_are_launched_so():
    code = _code("ave_fp4_api.cu") + _code("ave_dense_api.cu")
    for kernel in ORDERED:
        assert re.search(kernel + r"\s*<<<", code), kernel
        assert not re.search(r"cudaLaunchKernelEx\([^;]*\b" + kernel, code), kernel


@pytest.mark.parametrize("name", ["activations.cuh", "gated_backward.cuh", "gemm_dense_sm100.cuh", "gemm_stream_sm100.cuh", "quantize_int8.cuh",
                                  "quantize_fp4.cuh", "gemm_fp4_sm100.cuh", "gemm_fp4_skinny_sm100.cuh"])
def test_no_non_coherent_loads_beside_a_running_predecessor(name):
    """All but the kernels in ORDERED are resident while the previous one in the stream still writes (programmatic stream serialisation), so what they
    read is not read-only for their lifetime: no __ldg, no const __restrict__ parameters, and no intrinsic load that the compiler
    may move above the wait for that kernel."""
    code = _code(name)
    for kernel in ORDERED:
        code = _without(code, kernel)
    found = re.findall(r"__ld(?:g|cs|cg|ca|lu|cv)\s*\(|ld\.global\.nc", code)
    assert not found, found
    for signature in re.findall(r"__global__[^{;]*", code):
        assert "__restrict__" not in signature, signature
