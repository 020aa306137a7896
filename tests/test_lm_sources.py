"""Rules that the language-model kernels keep everywhere, read from their sources:
no run shows a breach reliably."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "voxcpm-inference_b200", "csrc")
KERNELS = ["lm_norm.cuh", "lm_rotary.cuh", "fp8_gemm.cuh", "fp8_gemv.cuh", "paged_attn.cuh", "chunk_attn.cuh"]


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", KERNELS)
def test_operands_are_read_coherently(name):
    """A launch may start while the kernel that writes its operands still runs: they are not constant for its
    lifetime, which is what read-only loads ask for."""
    assert not re.findall(r"__ldg|\.nc\b|__restrict__", source(name))


@pytest.mark.parametrize("name", KERNELS)
def test_waits_that_run_out_are_recorded(name):
    """Every wait is bounded and goes through op_wait, and every kernel that waits records a failure at its end."""
    s = source(name)
    assert not re.findall(r"\bmbar_wait(?:_for)?\s*\(|\bmbar_try_wait\s*\(", s)
    kernels = re.split(r"\b__global__\b", s)[1:]
    for k in kernels:
        assert ("op_wait(" in k) == ("record_abort(" in k)


@pytest.mark.parametrize("name", KERNELS + ["gemm.cuh", "resunit.cuh", "convt_tm.cuh", "encoder.cuh"])
def test_tensor_memory_is_taken_before_dependents_are_released(name):
    """A dependent may take columns before its own wait: it must not find any that this kernel still asks for."""
    for k in re.split(r"\b__global__\b", source(name))[1:]:
        alloc, release = k.find("tmem_alloc("), re.search(r"grid_dep_(?:sync|launch)\(\)", k)
        assert alloc < 0 or release is None or alloc < release.start()
