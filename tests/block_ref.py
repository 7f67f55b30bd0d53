"""Plain 64-bit forms of the transformer-block operators, on numpy arrays, for
their tests: the e4m3 form of a row, the 8-bit product, the edge between two
blocks, rotary positions. Nothing here calls the library."""
from __future__ import annotations

import math

import numpy as np

F16_HALF_STEP = 2.0 ** -11        # of a value, rounding to fp16
F16_TINY = 2.0 ** -25             # half a step of fp16's subnormals


def e4m3_values() -> np.ndarray:
    """The value of each of the 256 codes (sign, 4 exponent bits with bias 7, 3 of
    mantissa; 0x7f and 0xff are NaN)."""
    out = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v = math.nan if c & 0x7F == 0x7F else v
        out[c] = -v if c & 0x80 else v
    return out


VALUES = e4m3_values()


def pitch(K: int) -> int:
    return -(-K // 128) * 128


def groups(K: int) -> int:
    return -(-K // 512)


def quantize(x: np.ndarray):
    """fp16 [R, K] -> (codes [R, Kp], scales [groups, R, 4]) by search: the smallest
    power of two that brings the block within 448, then the nearest code, the even
    one of two equally near."""
    R, K = x.shape
    kp, g = pitch(K), groups(K)
    v = np.zeros((R, kp))
    v[:, :K] = x.astype(np.float64)
    v = v.reshape(R, kp // 128, 128)
    fin = np.where(np.isfinite(v), np.abs(v), 0.0)
    amax = fin.max(axis=2)
    e = np.full(amax.shape, -40)
    for cand in range(-39, 10):
        e = np.where(amax > 448.0 * 2.0 ** (cand - 1), cand, e)
    e = np.where(amax == 0, 0, e)
    s = v * 2.0 ** -e[:, :, None].astype(np.float64)
    pos = VALUES[:127]
    mag = np.abs(np.where(np.isfinite(s), s, 0.0))
    hi = np.clip(np.searchsorted(pos, mag), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = mag - pos[lo], pos[hi] - mag
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.signbit(s), code | 0x80, code)
    code = np.where(np.isfinite(s), code, 0x7F)
    scales = np.full((R, g * 4), 127, np.uint8)
    scales[:, :kp // 128] = e + 127
    return (code.reshape(R, kp).astype(np.uint8),
            np.ascontiguousarray(scales.reshape(R, g, 4).transpose(1, 0, 2)))


def same_codes(a: np.ndarray, b: np.ndarray) -> bool:
    """Equal code for code, any NaN code equal to any other."""
    nan = (a & 0x7F) == 0x7F
    return bool(np.array_equal(nan, (b & 0x7F) == 0x7F) and np.array_equal(a[~nan], b[~nan]))


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """What an e4m3 form stands for, [R, Kp] fp64."""
    R, kp = codes.shape
    s = scales.transpose(1, 0, 2).reshape(R, -1)[:, :kp // 128].astype(np.float64)
    return VALUES[codes] * np.repeat(2.0 ** (s - 127), 128, axis=1)


def gelu(v, act):
    if act == 1:
        return 0.5 * v * (1 + np.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if act == 2:
        return 0.5 * v * (1 + np.vectorize(math.erf, otypes=[float])(v / math.sqrt(2)))
    return v


def product(av, wv, bias, resid, act):
    """(value, bound on the kernel's error) of act(av @ wv.T + bias) + resid. The
    sum is held in fp32 and each of the Kp additions loses at most 2^-23 of the
    magnitudes summed (a truncated step, the tensor core's worst); GELU's slope is
    at most 1.13 and its fp32 evaluation a few 2^-22 of its argument; then one
    rounding to fp16."""
    v, mag = av @ wv.T, np.abs(av) @ np.abs(wv).T
    if bias is not None:
        v, mag = v + bias, mag + np.abs(bias)
    err = mag * (av.shape[1] + 2) * 2.0 ** -23
    if act:
        err = 1.13 * err + np.abs(v) * 2.0 ** -19
    v = gelu(v, act)
    if resid is not None:
        v = v + resid.astype(np.float64)
    return v, err + (np.abs(v) + err) * F16_HALF_STEP + F16_TINY


def norm(v, w, b, layer, eps):
    """(value, bound) of a row norm of exact inputs v, computed in fp32: the mean is
    off by C 2^-24 of the mean magnitude, the mean square by C 2^-24 relative (and
    by twice the mean's error over the deviation), then a few products."""
    C = v.shape[1]
    u = 2.0 ** -24
    mean = v.mean(1, keepdims=True) if layer else 0.0
    dm = (C + 2) * u * np.abs(v).mean(1, keepdims=True) if layer else 0.0
    d = v - mean
    ms = (d * d).mean(1, keepdims=True)
    inv = 1 / np.sqrt(ms + eps)
    dd = dm + u * np.abs(d)
    rel = (C + 8) * u + dm * inv          # of the inverse root: half of the mean square's
    out = d * inv * w
    err = (np.abs(d) * (rel + 4 * u) + dd) * inv * np.abs(w)
    if b is not None:
        out = out + b
        err = err + 2 * u * (np.abs(out) + np.abs(b))
    return out, err


def gate_value(g, act):
    g = g.astype(np.float64)
    sig = 1 / (1 + np.exp(-g))
    return [g, sig, g * sig, np.tanh(g)][act]


def edge_x(x, y, post_w, post_b, gate, act, xs, ys, layer, eps):
    """(x' before rounding, bound after it)."""
    u, err = y.astype(np.float64), 0.0
    if post_w is not None:
        u, err = norm(u, post_w.astype(np.float64), None if post_b is None else post_b.astype(np.float64), layer, eps)
    if gate is not None:
        g = np.repeat(gate_value(gate, act), x.shape[0] // gate.shape[0], axis=0)
        err = err * np.abs(g) + np.abs(u * g) * 2.0 ** -21   # the gate's exponential and division
        u = u * g
    out = xs * x.astype(np.float64) + ys * u
    err = abs(ys) * err + (np.abs(xs * x.astype(np.float64)) + np.abs(ys * u)) * 2.0 ** -22
    return out, err + (np.abs(out) + err) * F16_HALF_STEP + F16_TINY


def edge_h(x_out, pre_w, pre_b, layer, eps):
    """(h, bound) from the stored x'."""
    h, err = norm(x_out.astype(np.float64), pre_w.astype(np.float64), None if pre_b is None else pre_b.astype(np.float64), layer, eps)
    return h, err + (np.abs(h) + err) * F16_HALF_STEP + F16_TINY


def rotary(x, pos, table, axis, mscale, H, D, rot, layout):
    """(y, bound): x [T, >= H D] fp16, pos int [A, T], table Python ints. The phase is
    the exact product modulo 2^64; an fp32 keeps 24 bits of it, which with the sine
    and the products leaves a few 2^-22 of the pair's magnitude."""
    T = x.shape[0]
    v = x[:, :H * D].astype(np.float64).reshape(T, H, D)
    t = np.array([[((int(p) * int(f)) % 2 ** 64) / 2.0 ** 64 for p, f in zip([pos[a][i] for a in axis], table)]
                  for i in range(T)]).reshape(T, 1, rot // 2)
    c, s = mscale * np.cos(2 * np.pi * t), mscale * np.sin(2 * np.pi * t)
    ia = np.arange(rot // 2) * 2 if layout else np.arange(rot // 2)
    ib = ia + 1 if layout else ia + rot // 2
    a, b = v[..., ia], v[..., ib]
    out, err = v.copy(), np.zeros_like(v)
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    err[..., ia] = err[..., ib] = (np.abs(a) + np.abs(b)) * abs(mscale) * 2.0 ** -20
    err[..., :rot] += (np.abs(out[..., :rot]) + err[..., :rot]) * F16_HALF_STEP + F16_TINY
    return out.reshape(T, H * D), err.reshape(T, H * D)


def assert_within(got, ref, bound, what=""):
    got = np.asarray(got, np.float64)
    assert got.shape == ref.shape, f"{what}: shape {got.shape} != {ref.shape}"
    assert np.all(np.isfinite(got)), f"{what}: non-finite values"
    over = np.abs(got - ref) - bound
    if over.size and over.max() > 0:
        i = np.unravel_index(np.argmax(over), over.shape)
        raise AssertionError(f"{what}: {int((over > 0).sum())} of {over.size} outside their bound; worst at {i}: "
                             f"got {got[i]!r}, ref {ref[i]!r}, bound {np.broadcast_to(bound, ref.shape)[i]:.3e}")
