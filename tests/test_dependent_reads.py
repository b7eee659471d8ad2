"""Kernels that start under their predecessor (programmatic dependent launch) must not promise the compiler that what the predecessor
may still be writing never changes: no const __restrict__ on it, no __ldg. Weights and scales of an int4 product are the
documented exception; they are read before the predecessor ends."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "beantensor_b200", "csrc")
PARAMETERS = {"int4.cu": {"w", "scales"}, "int4_gemv_regs.cu": {"w", "scales"}, "int4_tc.cu": {"scales"}}


def kernels(text):
    """(name, parameter list, body) of every __global__ function."""
    for m in re.finditer(r"__global__\s+void\b", text):
        at = m.end()
        while True:  # attributes such as __launch_bounds__(..) come in front of the name
            n = re.compile(r"\s*(\w+)\s*\(").match(text, at)
            depth, end = 1, n.end()
            while depth:
                depth += {"(": 1, ")": -1}.get(text[end], 0)
                end += 1
            if not n.group(1).startswith("__"):
                break
            at = end
        open_at = text.index("{", end)
        depth, stop = 1, open_at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[stop], 0)
            stop += 1
        yield n.group(1), text[n.end():end - 1], text[open_at:stop]


def dependent_kernels():
    for f in sorted(os.listdir(CSRC)):
        if f.endswith(".cu"):
            with open(os.path.join(CSRC, f)) as src:
                text = src.read()
            for name, params, body in kernels(text):
                if "griddepcontrol.wait" in body:
                    yield f, name, params, body


def test_the_kernels_are_found():
    names = {name for _, name, _, _ in dependent_kernels()}
    assert {"mxfp4_quantize_kernel", "mxfp4_dequant_kernel", "int4_gemv_regs_kernel", "gemm_tc_kernel", "grouped_decode_kernel"} <= names


@pytest.mark.parametrize("f,name,params,body", [pytest.param(*k, id=k[1]) for k in dependent_kernels()])
def test_inputs_of_a_dependent_kernel(f, name, params, body):
    allowed = PARAMETERS.get(f, set())
    promised = {m.group(1) for m in re.finditer(r"const\s+[\w: ]+\*\s*__restrict__\s+(\w+)", params)}
    assert promised <= allowed, (name, promised - allowed)
    for m in re.finditer(r"__ldg\(([^;]*)", body):
        assert allowed and re.match(r"\(?(scales|grow)\b", m.group(1)), (name, m.group(0))


def test_the_bias_of_the_dense_epilogue():
    with open(os.path.join(CSRC, "gemm_epilogue.cuh")) as src:
        assert "__ldg" not in src.read()
