"""What the sources of the transformer-block operators promise and no run can show."""
from __future__ import annotations

import os
import re

import pytest

from hexlib_b200 import build

SOURCES = {os.path.basename(p): open(p).read() for p in build._sources()}


def code_of(name):
    """A source without its comments."""
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", SOURCES[name], flags=re.S)


EARLY = [n for n in SOURCES if "ProgrammaticStreamSerialization" in code_of(n)]


def test_some_kernel_starts_early():
    assert EARLY == ["k_gemm_e4m3.cu"]


@pytest.mark.parametrize("name", EARLY)
def test_kernels_that_start_early_use_no_read_only_loads(name):
    # A kernel launched with programmatic serialization is alive while the kernel before
    # still writes its operands; loads through the read-only path are defined only for data
    # that nothing writes during the kernel's whole life.
    code = code_of(name)
    assert not re.search(r"__ldg\s*\(|\.nc\b|ld\.global\.nc|__ldlu|tex1D", code)
    # and the compiler may choose that path by itself for pointers it knows to be alone
    assert "__restrict__" not in code
