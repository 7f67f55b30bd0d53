"""What the transformer-block operators promise and no run on a device can show: sizes and
shared buffers that they refuse, and how their sources read memory."""
from __future__ import annotations

import os
import re

import pytest

from hexlib_b200 import build
from test_block_ops_cpu import BAD, EDGE, EDGE8, OK, P, ROPE, rc, with_

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


BIG = (1 << 30) + 1


@pytest.mark.parametrize("sizes", [dict(T=BIG), dict(T=2 ** 31 - 1), dict(H=BIG), dict(H=2 ** 31 - 1), dict(D=BIG),
                                   dict(D=2 ** 31 - 1), dict(H=2 ** 31 - 1024), dict(D=2 ** 31 - 2, rot=2 ** 31 - 2),
                                   dict(D=30000, rot=24578)])
def test_rope_refuses_more_than_the_largest_sizes(sizes):
    wide = {k: 2 ** 61 for k in ("xs", "ys")}          # rows far enough apart for any of them
    assert rc("rope_pos_fp16", *with_(ROPE, **wide, **sizes)) == BAD
    # with no tokens too
    if "T" not in sizes:
        assert rc("rope_pos_fp16", *with_(ROPE, **wide, **sizes, T=0)) == BAD


def test_rope_takes_no_tokens_of_the_largest_heads():
    most = 1 << 30
    assert rc("rope_pos_fp16", *with_(ROPE, xs=2 ** 60, ys=2 ** 60, H=most, D=most, rot=24576, T=0)) == OK


def test_dequant_refuses_more_than_the_largest_sizes():
    for R, K in ((BIG, 64), (4, BIG), (2 ** 31 - 1, 64), (4, 2 ** 31 - 1)):
        assert rc("dequant_e4m3_fp16", P, P, P, R, K, None) == BAD


# every buffer an address of its own
EDGE_OWN = {**EDGE, **dict(pw=6 * P, pb=7 * P, w=8 * P, b=9 * P)}
EDGE8_OWN = {**EDGE8, **dict(q=10 * P, sc=11 * P, pw=6 * P, pb=7 * P, w=8 * P, b=9 * P)}


@pytest.mark.parametrize("read", ["pw", "pb", "w", "b", "gate"])
def test_edge_refuses_outputs_on_what_every_row_reads(read):
    for out in ("xo", "h"):
        assert rc("norm_gate_residual_fp16", *with_(EDGE_OWN, **{out: EDGE_OWN[read]})) == BAD
    for out in ("xo", "q", "sc"):
        assert rc("norm_gate_residual_e4m3", *with_(EDGE8_OWN, **{out: EDGE8_OWN[read]})) == BAD
