"""CPU tier: properties of the CUDA sources that no run can show."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "avelang_b200", "csrc")


def _code(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", text, flags=re.S))


@pytest.mark.parametrize("name", ["activations.cuh", "gated_backward.cuh", "gemm_dense_sm100.cuh", "gemm_stream_sm100.cuh", "quantize_int8.cuh"])
def test_no_non_coherent_loads_beside_a_running_predecessor(name):
    """These kernels are resident while the previous one in the stream still writes (programmatic stream serialisation), so what they
    read is not read-only for their lifetime: no __ldg, no const __restrict__ parameters, and no intrinsic load that the compiler
    may move above the wait for that kernel."""
    code = _code(name)
    assert not re.findall(r"__ld(?:g|cs|cg|ca|lu|cv)\s*\(|ld\.global\.nc", code)
    for signature in re.findall(r"__global__[^{;]*", code):
        assert "__restrict__" not in signature, signature
