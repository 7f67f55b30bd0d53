"""The norms of the edge between two blocks where rounding shows: constant and nearly
constant rows, rows far from zero, each width's own layout, with bounds that count the
roundings the kernels make rather than one for every element of the row."""
from __future__ import annotations

import numpy as np
import pytest

import block_ref as B
import gpu_util as U
from test_edge_gpu import run

pytestmark = pytest.mark.gpu

U24 = 2.0 ** -24
# a warp to a row, 128 and 256 threads, each with and without whole vectors, and the
# widths past 8192 whose sums of equal values no longer fit 24 bits
WIDTHS = [1, 96, 256, 768, 1000, 1203, 2048, 3001, 4096, 5000, 8192, 12291, 16384, 20000, 40001]


def steps(C):
    """Additions on the longest path of a row's sum: a row in registers is at most 32
    two-wide steps of a thread, the pair, 5 across a warp and 3 across warps; a wider
    one is C / 256 steps of a thread instead."""
    return 41 if C <= 16384 else -(-C // 256) + 9


def sums_exactly(v):
    """For each row of fp16 values, [R, 1]: whether every partial sum, in any order, is a
    whole number of the row's smallest unit under 2^24 of them, and so exact in fp32."""
    k = np.abs(v * 2.0 ** 24).astype(np.int64)
    bits = np.bitwise_or.reduce(k, axis=1, keepdims=True)
    return k.sum(1, keepdims=True) < 2 ** 24 * np.maximum(bits & -bits, 1)


def norm(v, w, b, layer, eps):
    """(value, bound on the fp32 steps) of a row norm of exact inputs v, for a kernel that
    subtracts a rounded mean m from every element and corrects what is left, d = v - m,
    by the rest of the mean: the division's remainder or, past 8192, the mean of the d.

    u = 2^-24, n = steps + 1 (a division); a sum of terms t is off by at most n u sum|t|,
    or by nothing where it is exact. m is off by gm = n u mean|v|, or by its own
    rounding, 2 u. A deviation is rounded once, u (|D| + gm). m + rest is off by dm:
    the error of the sum and 3 u of the rest; or, taken from the d, by their roundings and
    their own sum, (n + 2) u (mean|D| + gm). The variance is off by (n + 4) u of the mean
    square of the d, mean D^2 + gm^2, and by the error of the square of the rest taken
    off it. The inverse root: half the relative error of its argument (the whole of it is
    taken) and 4 u. Then d inv - shift: the shift's rounding u gm inv and its own u."""
    C = v.shape[1]
    n = steps(C) + 1
    mean, gm, dm = 0.0, 0.0, 0.0
    D = v
    if layer:
        mean = v.mean(1, keepdims=True)
        D = v - mean
        size, exact = np.abs(v).mean(1, keepdims=True), sums_exactly(v)
        gm = np.where(exact, 2, n) * U24 * size
        dm = np.where(exact, 0, n) * U24 * size + 3 * U24 * gm
        if C > 8192:
            dm = (n + 2) * U24 * (np.abs(D).mean(1, keepdims=True) + gm)
    ms = (D * D).mean(1, keepdims=True)
    dv = (n + 4) * U24 * (ms + gm * gm) + 2 * gm * dm + dm * dm
    inv = 1 / np.sqrt(ms + eps)
    rel = dv / (ms + eps) + 4 * U24
    out = D * inv * w
    err = (np.abs(D) * (rel + 3 * U24) + U24 * (np.abs(D) + 2 * gm) + dm) * inv * np.abs(w)
    if b is not None:
        out = out + b
        err = err + 2 * U24 * (np.abs(out) + np.abs(b))
    return out, err


def to_f16(v, err):
    return v, err + (np.abs(v) + err) * B.F16_HALF_STEP + B.F16_TINY


def same_form(form, h):
    q, s = B.quantize(h)
    return np.array_equal(U.host(form[1]), s) and B.same_codes(U.host(form[0]), q)


def weights(rng, C, layer=True):
    return ((1 + 0.2 * rng.standard_normal(C)).astype(np.float32),
            (0.3 * rng.standard_normal(C)).astype(np.float32) if layer else None)


CONSTANTS = np.array([0.1, -3.14, 777, 999, 1000, -2047, 30000, 53248, -65504], np.float16)


@pytest.mark.parametrize("eps", [1e-5, 1e-6, 1e-12])
@pytest.mark.parametrize("C", WIDTHS)
def test_a_constant_row_is_its_shift(C, eps):
    rng = np.random.default_rng(C)
    pre_w, pre_b = weights(rng, C)
    x = np.repeat(CONSTANTS[:, None], C, axis=1)
    c = dict(x=x, y=None, post_w=None, post_b=None, gate=None, pre_w=pre_w, pre_b=pre_b)
    want = np.broadcast_to(pre_b.astype(np.float16), x.shape)
    _, h = run(c, layer=True, eps=eps)
    assert np.array_equal(U.host(h), want)
    _, form = run(c, layer=True, eps=eps, e4m3=True)
    assert same_form(form, want)
    # the norm after a block: the branch is its shift, the stream takes that alone
    post_w, post_b = weights(rng, C)
    s = rng.standard_normal(x.shape).astype(np.float16)
    c = dict(x=s, y=x, post_w=post_w, post_b=post_b, gate=None, pre_w=None, pre_b=None)
    xo, _ = run(c, layer=True, eps=eps)
    assert np.array_equal(U.host(xo), (s.astype(np.float32) + post_b).astype(np.float16))


def far_rows(rng, C):
    """Rows whose mean is far larger than their deviations."""
    x = np.empty((8, C))
    x[0] = 1000
    x[0, C // 2] = 1000.5                               # one element a step away
    x[1] = 30000
    x[1, C // 3] = 29984
    x[2] = 999 + 0.5 * rng.integers(0, 2, C)
    x[3] = -2047 + rng.integers(0, 2, C)
    x[4] = 300 + 2 * rng.standard_normal(C)
    x[5] = 20000 + 16 * rng.integers(-3, 4, C)
    x[6] = 3.14 + 0.002 * rng.integers(0, 2, C)
    x[7] = rng.standard_normal(C)
    return x.astype(np.float16)


@pytest.mark.parametrize("layer", [True, False])
@pytest.mark.parametrize("eps", [1e-5, 1e-6])
@pytest.mark.parametrize("C", WIDTHS[1:])
def test_rows_far_from_zero(C, eps, layer):
    rng = np.random.default_rng(C + 1)
    pre_w, pre_b = weights(rng, C, layer)
    x = far_rows(rng, C)
    eps32 = float(np.float32(eps))
    c = dict(x=x, y=None, post_w=None, post_b=None, gate=None, pre_w=pre_w, pre_b=pre_b)
    _, h = run(c, layer=layer, eps=eps)
    f64 = lambda a: None if a is None else a.astype(np.float64)  # noqa: E731
    ref, bound = to_f16(*norm(f64(x), f64(pre_w), f64(pre_b), layer, eps32))
    B.assert_within(U.host(h), ref, bound, "h")
    _, form = run(c, layer=layer, eps=eps, e4m3=True)
    assert same_form(form, U.host(h))
    # after a block, on a stream of zeros: x' is the normed branch
    c = dict(x=np.zeros_like(x), y=x, post_w=pre_w, post_b=pre_b, gate=None, pre_w=None, pre_b=None)
    xo, _ = run(c, layer=layer, eps=eps)
    B.assert_within(U.host(xo), ref, bound, "x'")
