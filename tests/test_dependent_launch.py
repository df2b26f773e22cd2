"""Kernels that may start before the grid ahead of them has ended
(launch_pdl) read no input as read-only data: a non-coherent load promises that
nothing writes its address while the kernel runs, and may be moved in front of
the wait for the grid ahead."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "grpc-unlimited-ocr_b200", "csrc")


def code(path):
    return re.sub(r"//[^\n]*", "", open(path).read())


SOURCES = sorted(os.path.basename(p) for p in glob.glob(os.path.join(CSRC, "*.cu")) if "launch_pdl(" in code(p))


def test_there_are_such_kernels():
    assert {"quantize_tokens.cu", "w8a8_gemm.cu", "w8a8_rows.cu"} <= set(SOURCES)


@pytest.mark.parametrize("name", SOURCES)
def test_inputs_are_read_by_plain_loads(name):
    text = code(os.path.join(CSRC, name))
    assert "__ldg" not in text
    assert not re.search(r"ld\.global[a-z0-9_:.]*\.nc\b", text)
    assert not re.search(r"const\s+\w+\s*\*\s*__restrict__", text)
