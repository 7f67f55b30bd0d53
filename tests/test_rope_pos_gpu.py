"""Rotary positions against the exact phase: layouts, part of the head, axes, far and
negative positions, packed rows, in place."""
from __future__ import annotations

import math

import numpy as np
import pytest

import block_ref as B
import gpu_util as U
from test_block_ops_cpu import table_of

pytestmark = pytest.mark.gpu


def rotate(x, pos, table, axis, mscale, H, D, rot, layout, y=None, y_stride=None):
    """x a device tensor [T, ld]; pos int32 numpy [A, T]."""
    import torch
    T = x.shape[0]
    t = torch.from_numpy(np.array(table, dtype=np.uint64).view(np.int64)).cuda()
    ax = None if axis is None else U.dev(np.asarray(axis, np.int32))
    ps = U.dev(np.ascontiguousarray(pos, dtype=np.int32))
    y = U.empty((T, H * D), np.float16) if y is None else y
    U.call("hexlib_b200_rope_pos_fp16", U.ptr(x), x.stride(0) if T > 1 else x.shape[1], U.ptr(ps), pos.shape[0], U.ptr(t),
           None if ax is None else U.ptr(ax), mscale, U.ptr(y), y_stride or H * D, T, H, D, rot, layout, U.stream())
    return y


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("T,H,D,rot", [(1, 1, 2, 2), (1, 4, 128, 128), (3, 2, 64, 32), (5, 7, 80, 20), (2, 3, 10, 6),
                                       (9, 1, 256, 256), (33, 12, 64, 64), (8, 20, 128, 32), (17, 5, 96, 96), (4, 2, 33, 2),
                                       (130, 3, 192, 48), (2, 64, 128, 64),
                                       (3, 1, 16, 16), (700, 1, 16, 16), (1300, 2, 32, 16), (900, 1, 8, 8), (2, 1500, 16, 16),
                                       (40, 5, 96, 24), (41, 3, 80, 40), (700, 2, 32, 8), (25, 4, 36, 12), (19, 3, 22, 10),
                                       (650, 1, 20, 20), (11, 2, 4100, 64)])
def test_layouts_and_partial_heads(T, H, D, rot, layout):
    rng = np.random.default_rng(T + H + D + rot)
    x = rng.standard_normal((T, H * D)).astype(np.float16)
    pos = rng.integers(0, 5000, (1, T))
    table, ms = table_of(0, rot, 10000.0)
    y = rotate(U.dev(x), pos, table, None, ms, H, D, rot, layout)
    ref, bound = B.rotary(x, pos, table, [0] * (rot // 2), ms, H, D, rot, layout)
    B.assert_within(U.host(y), ref, bound, "rotary")
    keep = np.array([c % D >= rot for c in range(H * D)])
    assert np.array_equal(U.host(y)[:, keep], x[:, keep])


@pytest.mark.parametrize("scaling,args", [(1, (8.0, 0, 0, 0)), (2, (4.0, 0, 0, 0)), (3, (16.0, 4096.0, 1.0, 32.0)),
                                          (4, (8.0, 8192.0, 1.0, 4.0))])
def test_far_positions_of_every_scaling(scaling, args):
    T, H, D, rot = 40, 3, 128, 128
    rng = np.random.default_rng(scaling)
    x = rng.standard_normal((T, H * D)).astype(np.float16)
    pos = np.concatenate([rng.integers(0, 2 ** 31 - 1, T - 4), [0, 1, 2 ** 31 - 1, -2 ** 31]])[None]
    table, ms = table_of(scaling, rot, 1e6, *args)
    for layout in (0, 1):
        y = rotate(U.dev(x), pos, table, None, ms, H, D, rot, layout)
        ref, bound = B.rotary(x, pos, table, [0] * 64, float(np.float32(ms)), H, D, rot, layout)
        B.assert_within(U.host(y), ref, bound, "far")


def test_the_angle_is_position_times_frequency():
    # against angles formed in radians in fp64, apart from the table's fixed point
    T, D = 64, 64
    x = np.zeros((T, D), np.float16)
    x[:, :32] = 1
    pos = np.arange(T)[None] * 16001
    table, _ = table_of(0, D, 10000.0)
    y = U.host(rotate(U.dev(x), pos, table, None, 1.0, 1, D, D, 0)).astype(np.float64)
    ang = pos[0][:, None] * 10000.0 ** (-2.0 * np.arange(32) / D)
    err = 2.0 ** -11 + np.abs(ang) * 2.0 ** -51 + 2.0 ** -20
    assert np.all(np.abs(y[:, :32] - np.cos(ang)) <= err) and np.all(np.abs(y[:, 32:] - np.sin(ang)) <= err)


@pytest.mark.parametrize("A", [2, 3, 4])
def test_axes_and_clamped_axis_numbers(A):
    T, H, D = 19, 4, 64
    rng = np.random.default_rng(A)
    x = rng.standard_normal((T, H * D)).astype(np.float16)
    pos = rng.integers(0, 900, (A, T))
    axis = np.arange(32) * A // 32
    table, ms = table_of(0, D, 10000.0)
    ref, bound = B.rotary(x, pos, table, axis, ms, H, D, D, 0)
    B.assert_within(U.host(rotate(U.dev(x), pos, table, axis, ms, H, D, D, 0)), ref, bound, "axes")
    wild = axis.copy()
    wild[0], wild[31] = -5, 99
    clamped = np.clip(wild, 0, A - 1)
    ref, bound = B.rotary(x, pos, table, clamped, ms, H, D, D, 0)
    B.assert_within(U.host(rotate(U.dev(x), pos, table, wild, ms, H, D, D, 0)), ref, bound, "clamped")


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("H,HV,D,rot", [(6, 2, 64, 64), (3, 1, 80, 40), (5, 2, 34, 6), (8, 4, 128, 32), (4, 2, 96, 24), (7, 1, 20, 4)])
def test_packed_projection_in_place_and_out_of_place(H, HV, D, rot, layout):
    T = 21
    rng = np.random.default_rng(D)
    x = rng.standard_normal((T, (H + HV) * D)).astype(np.float16)
    pos = rng.integers(-100, 4000, (1, T))
    table, ms = table_of(0, rot, 10000.0)
    d = U.dev(x)
    y = rotate(d, pos, table, None, ms, H, D, rot, layout)
    rotate(d, pos, table, None, ms, H, D, rot, layout, y=d, y_stride=(H + HV) * D)
    assert np.array_equal(U.host(d)[:, :H * D], U.host(y))
    assert np.array_equal(U.host(d)[:, H * D:], x[:, H * D:])


def test_misaligned_rows_and_nothing_written_between_them():
    import torch
    T, H, D, rot = 7, 3, 64, 32
    rng = np.random.default_rng(1)
    x = rng.standard_normal((T, H * D)).astype(np.float16)
    pos = rng.integers(0, 99, (1, T))
    table, ms = table_of(0, rot, 10000.0)
    for layout in (0, 1):
        for shift, ld in ((1, 195), (2, 198), (8, 200), (0, 193)):
            src = torch.zeros(shift + T * ld, dtype=torch.float16, device="cuda")
            src[shift:].view(T, ld)[:, :H * D] = U.dev(x)
            dst = torch.full((shift + T * ld + 9,), -7.0, dtype=torch.float16, device="cuda")
            rotate(src[shift:].view(T, ld), pos, table, None, ms, H, D, rot, layout, y=dst[shift:], y_stride=ld)
            got = U.host(dst)
            body = got[shift:shift + T * ld].reshape(T, ld)
            ref, bound = B.rotary(x, pos, table, [0] * 16, ms, H, D, rot, layout)
            B.assert_within(body[:, :H * D], ref, bound, "strided")
            assert (body[:, H * D:] == -7).all() and (got[:shift] == -7).all() and (got[shift + T * ld:] == -7).all()


def test_negated_positions_are_the_gradient_and_the_inverse():
    T, H, D, rot = 12, 4, 96, 64
    rng = np.random.default_rng(3)
    x = rng.standard_normal((T, H * D)).astype(np.float16)
    g = rng.standard_normal((T, H * D)).astype(np.float16)
    pos = rng.integers(0, 100000, (1, T))
    table, ms = table_of(3, rot, 10000.0, 4.0, 4096.0, 1.0, 32.0)
    m = float(np.float32(ms))
    for layout in (0, 1):
        axis = [0] * (rot // 2)
        dx = U.host(rotate(U.dev(g), -pos, table, None, ms, H, D, rot, layout)).astype(np.float64)
        # <g, R x> differenced along each element of x: R is linear, so the difference is exact in fp64
        grad = np.zeros_like(dx)
        for j in range(D):
            e = np.zeros((T, H * D))
            e[:, j::D] = 1
            col = B.rotary(e, pos, table, axis, m, H, D, rot, layout)[0]
            grad[:, j::D] = (g.astype(np.float64) * col).reshape(T, H, D).sum(2)
        bound = np.abs(grad) * B.F16_HALF_STEP + B.F16_TINY + 16 * m * 2.0 ** -20
        B.assert_within(dx, grad, bound, "gradient")
        back = U.host(rotate(rotate(U.dev(x), pos, table, None, 1.0, H, D, rot, layout), -pos, table, None, 1.0, H, D, rot, layout))
        # two roundings of values no larger than the pair's magnitude (sqrt 2 times the larger)
        assert np.all(np.abs(back.astype(np.float64) - x) <= 2 * 2 ** 0.5 * np.abs(x).max() * 2.0 ** -11 + 2.0 ** -18)


def test_repeats_captured_and_with_a_long_row_offset():
    import torch
    T, H, D = 300, 4, 64
    rng = np.random.default_rng(9)
    x = rng.standard_normal((T, H * D)).astype(np.float16)
    pos = np.arange(T)[None]
    table, ms = table_of(0, D, 10000.0)
    want = U.host(rotate(U.dev(x), pos, table, None, ms, H, D, D, 0))
    d, y = U.dev(x), U.empty((T, H * D), np.float16)
    t = torch.from_numpy(np.array(table, dtype=np.uint64).view(np.int64)).cuda()
    ps = U.dev(pos.astype(np.int32))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        U.call("hexlib_b200_rope_pos_fp16", U.ptr(d), H * D, U.ptr(ps), 1, U.ptr(t), None, ms, U.ptr(y), H * D, T, H, D, D, 0,
               U.stream())
    for _ in range(2):
        graph.replay()
    assert np.array_equal(U.host(y), want)
    # rows so far apart that the last one's element offset passes 32 bits
    ld = 2 ** 31 // 2 + 8
    big = torch.empty(2 * ld + H * D, dtype=torch.float16, device="cuda")
    for i in range(3):
        big[i * ld:i * ld + H * D] = d[i]
    rotate(big.as_strided((3, H * D), (ld, 1)), pos[:, :3], table, None, ms, H, D, D, 0, y=big, y_stride=ld)
    for i in range(3):
        assert np.array_equal(U.host(big[i * ld:i * ld + H * D]), want[i])
    assert math.isclose(ms, 1.0)


def test_no_tokens_launch_nothing():
    assert U.call_rc("hexlib_b200_rope_pos_fp16", None, 64, None, 1, None, None, 1.0, None, 64, 0, 1, 64, 64, 0, U.stream()) == U.OK
