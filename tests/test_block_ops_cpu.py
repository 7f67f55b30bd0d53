"""The transformer-block operators without a device: what each entry refuses, and the
rotary table against frequencies formed in 60 decimal digits."""
from __future__ import annotations

import ctypes
import decimal
import math

import pytest

from hexlib_b200 import _lib

OK, BAD = 1, 6
P = 1 << 20          # a well-aligned address; a refused call reads nothing


def rc(name, *args):
    return getattr(_lib.lib(), "hexlib_b200_" + name)(*args)


def table_of(scaling, rot, theta, factor=1.0, length=0.0, low=0.0, high=0.0):
    """(table as Python ints, mscale)."""
    t, m = (ctypes.c_uint64 * (rot // 2))(), ctypes.c_float()
    assert rc("rope_pos_table", scaling, rot, theta, factor, length, low, high, t, ctypes.byref(m)) == OK
    return list(t), m.value


PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def exact_turns(scaling, rot, theta, factor, length, low, high):
    D = decimal.Decimal
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        theta, out = D(theta), []
        if scaling == 2:
            theta = theta * ((D(rot) / (rot - 2)) * D(factor).ln()).exp()
        for j in range(rot // 2):
            f = (-(D(2 * j) / rot) * theta.ln()).exp()
            if scaling == 1:
                f = f / D(factor)
            if scaling in (3, 4):
                if scaling == 3:
                    at = lambda n: float(rot * (D(length) / (D(n) * 2 * PI)).ln() / (2 * theta.ln()))  # noqa: E731
                    first, last = max(math.floor(at(high)), 0), min(math.ceil(at(low)), rot - 1)
                    last = last if last > first else first + 0.001
                    keep = 1 - min(max((D(j) - first) / (D(last) - D(first)), D(0)), D(1))
                else:
                    keep = min(max((D(length) * f / (2 * PI) - D(low)) / (D(high) - D(low)), D(0)), D(1))
                f = f / D(factor) * (1 - keep) + f * keep
            out.append(f / (2 * PI))
    return out


@pytest.mark.parametrize("rot", [2, 4, 20, 64, 128])
@pytest.mark.parametrize("scaling,theta,args", [(0, 10000.0, (1.0, 0, 0, 0)), (1, 1e6, (4.0, 0, 0, 0)), (1, 10000.0, (0.25, 0, 0, 0)),
                                                (2, 10000.0, (8.0, 0, 0, 0)), (3, 10000.0, (16.0, 4096.0, 1.0, 32.0)),
                                                (4, 500000.0, (8.0, 8192.0, 1.0, 4.0))])
def test_rope_table_matches_exact_frequencies(scaling, rot, theta, args):
    if scaling == 2 and rot == 2:
        assert rc("rope_pos_table", 2, 2, theta, 8.0, 0.0, 0.0, 0.0, (ctypes.c_uint64 * 1)(), ctypes.byref(ctypes.c_float())) == BAD
        return
    table, ms = table_of(scaling, rot, theta, *args)
    for got, want in zip(table, exact_turns(scaling, rot, theta, *args)):
        want = want - int(want)
        # a few roundings of 53 bits on the frequency (the blends subtract numbers of
        # either side of it; pow and log are within an ulp), and the fixed point's own
        off = abs(decimal.Decimal(got) / 2 ** 64 - want)
        assert off <= decimal.Decimal(64) * want * decimal.Decimal(2) ** -53 + decimal.Decimal(2) ** -63
    assert ms == pytest.approx(1 + 0.1 * math.log(args[0]) if scaling == 3 else 1.0, rel=2.0 ** -23)


@pytest.mark.parametrize("args", [(-1, 64, 1e4, 1.0, 0, 0, 0), (5, 64, 1e4, 1.0, 0, 0, 0), (0, 63, 1e4, 1.0, 0, 0, 0),
                                  (0, 0, 1e4, 1.0, 0, 0, 0), (0, 64, 1.0, 1.0, 0, 0, 0), (0, 64, math.nan, 1.0, 0, 0, 0),
                                  (0, 64, math.inf, 1.0, 0, 0, 0), (1, 64, 1e4, 0.0, 0, 0, 0), (1, 64, 1e4, math.nan, 0, 0, 0),
                                  (2, 64, 1e4, -2.0, 0, 0, 0), (2, 64, 1e4, 1e-9, 0, 0, 0), (3, 64, 1e4, 4.0, 0.0, 1.0, 32.0),
                                  (3, 64, 1e4, 4.0, 4096.0, 32.0, 1.0), (4, 64, 1e4, 4.0, 4096.0, 0.0, 4.0),
                                  (4, 64, 1e4, 4.0, math.inf, 1.0, 4.0)])
def test_rope_table_refusals(args):
    t, m = (ctypes.c_uint64 * 64)(), ctypes.c_float()
    assert rc("rope_pos_table", *args, t, ctypes.byref(m)) == BAD
    assert list(t) == [0] * 64
    assert rc("rope_pos_table", 0, 64, 1e4, 1.0, 0.0, 0.0, 0.0, None, ctypes.byref(m)) == BAD


def with_(base, **changes):
    names = list(base)
    assert set(changes) <= set(names)
    return [changes.get(n, base[n]) for n in names]


ROPE = dict(x=P, xs=256, pos=P, axes=1, table=P, axis=None, ms=1.0, y=2 * P, ys=256, T=4, H=4, D=64, rot=64, layout=0, s=None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(y=None), dict(pos=None), dict(table=None), dict(axes=0), dict(axes=5),
                                 dict(xs=255), dict(ys=255), dict(T=-1), dict(H=0), dict(D=0), dict(rot=0), dict(rot=63),
                                 dict(rot=66), dict(layout=2), dict(layout=-1), dict(x=P + 1), dict(y=P + 1), dict(table=P + 4),
                                 dict(pos=P + 2), dict(axis=P + 1), dict(y=P, xs=300)])
def test_rope_refusals(bad):
    assert rc("rope_pos_fp16", *with_(ROPE, **bad)) == BAD


QUANT = dict(x=P, q=P, s=P, R=4, K=100, st=None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(q=None), dict(s=None), dict(R=-1), dict(K=0), dict(K=-5), dict(x=P + 1),
                                 dict(q=P + 8), dict(s=P + 2)])
def test_quantize_refusals(bad):
    assert rc("quantize_e4m3_fp16", *with_(QUANT, **bad)) == BAD
    if "R" not in bad:
        assert rc("quantize_weight_e4m3_fp16", *with_(QUANT, **bad)) == BAD


def test_quantize_weight_refuses_no_columns_and_dequant_its_own():
    assert rc("quantize_weight_e4m3_fp16", P, P, P, 64, 0, None) == BAD
    for bad in ((None, P, P, 4, 64), (P, None, P, 4, 64), (P, P, None, 4, 64), (P, P, P, -1, 64), (P, P, P, 4, 0),
                (P + 1, P, P, 4, 64), (P, P + 1, P, 4, 64), (P, P, P + 1, 4, 64)):
        assert rc("dequant_e4m3_fp16", *bad, None) == BAD
    assert rc("dequant_e4m3_fp16", None, None, None, 0, 64, None) == OK


MM = dict(a=P, as_=P, w=P, ws=P, bias=P, out=P, M=4, K=128, N=64, act=0, s=None)
MMR = dict(a=P, as_=P, w=P, ws=P, bias=P, r=P, out=P, M=4, K=128, N=64, act=0, s=None)


@pytest.mark.parametrize("bad", [dict(a=None), dict(as_=None), dict(w=None), dict(ws=None), dict(out=None), dict(M=-1), dict(K=0),
                                 dict(N=0), dict(act=3), dict(act=-1), dict(a=P + 4), dict(w=P + 8), dict(as_=P + 1), dict(ws=P + 2),
                                 dict(bias=P + 2), dict(out=P + 1)])
def test_product_refusals(bad):
    assert rc("matmul_epilogue_e4m3", *with_(MM, **bad)) == BAD
    assert rc("matmul_epilogue_residual_e4m3", *with_(MMR, **bad)) == BAD


def test_product_refuses_a_missing_or_odd_residual():
    assert rc("matmul_epilogue_residual_e4m3", *with_(MMR, r=None)) == BAD
    assert rc("matmul_epilogue_residual_e4m3", *with_(MMR, r=P + 1)) == BAD


EDGE = dict(x=P, y=2 * P, pw=P, pb=P, gate=3 * P, rows=2, act=1, xs=1.0, ys=1.0, xo=4 * P, w=P, b=P, h=5 * P, R=4, C=64,
            norm=0, eps=1e-6, s=None)
EDGE8 = dict(x=P, y=2 * P, pw=P, pb=P, gate=3 * P, rows=2, act=1, xs=1.0, ys=1.0, xo=4 * P, w=P, b=P, q=5 * P, sc=6 * P, R=4,
             C=64, norm=0, eps=1e-6, s=None)
EDGE_BAD = [dict(x=None), dict(xo=None), dict(R=-1), dict(C=0), dict(norm=2), dict(norm=-1), dict(eps=-1.0), dict(eps=math.nan),
            dict(act=4), dict(act=-1), dict(rows=0), dict(rows=3), dict(rows=-2), dict(gate=None), dict(gate=None, rows=0),
            dict(w=None), dict(w=None, b=None), dict(pw=None), dict(y=None), dict(y=None, pw=None, pb=None, gate=None, rows=0, act=0),
            dict(x=P + 1), dict(y=P + 1), dict(xo=P + 1), dict(gate=P + 1), dict(w=P + 2), dict(b=P + 2), dict(pw=P + 2),
            dict(pb=P + 2), dict(xo=3 * P)]


@pytest.mark.parametrize("bad", EDGE_BAD)
def test_edge_refusals(bad):
    assert rc("norm_gate_residual_fp16", *with_(EDGE, **bad)) == BAD
    assert rc("norm_gate_residual_e4m3", *with_(EDGE8, **bad)) == BAD


@pytest.mark.parametrize("bad", [dict(h=None), dict(h=P + 1), dict(h=4 * P), dict(h=P), dict(h=3 * P)])
def test_edge_refuses_outputs_that_are_missing_or_shared(bad):
    assert rc("norm_gate_residual_fp16", *with_(EDGE, **bad)) == BAD


@pytest.mark.parametrize("bad", [dict(q=None), dict(sc=None), dict(q=None, sc=None), dict(q=5 * P + 8), dict(sc=P + 2),
                                 dict(q=P), dict(q=2 * P), dict(sc=4 * P), dict(sc=3 * P), dict(q=4 * P), dict(sc=5 * P)])
def test_edge_e4m3_refuses_outputs_that_are_missing_or_shared(bad):
    assert rc("norm_gate_residual_e4m3", *with_(EDGE8, **bad)) == BAD


def test_empty_batches_need_nothing():
    assert rc("norm_gate_residual_fp16", *with_(EDGE, R=0)) == OK
    assert rc("matmul_epilogue_e4m3", *with_(MM, M=0)) == OK
    assert rc("quantize_e4m3_fp16", *with_(QUANT, R=0)) == OK
    assert rc("rope_pos_fp16", *with_(ROPE, T=0)) == OK


def test_more_than_the_largest_sizes_are_refused():
    big = (1 << 30) + 1
    for k in ("M", "K", "N"):
        assert rc("matmul_epilogue_e4m3", *with_(MM, **{k: big})) == BAD
    for k in ("R", "K"):
        assert rc("quantize_e4m3_fp16", *with_(QUANT, **{k: big})) == BAD
        assert rc("quantize_weight_e4m3_fp16", *with_(QUANT, **{k: big})) == BAD
    for k in ("R", "C"):
        assert rc("norm_gate_residual_fp16", *with_(EDGE, gate=None, rows=0, act=0, **{k: big})) == BAD
