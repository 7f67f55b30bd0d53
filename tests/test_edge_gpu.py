"""The edge between two blocks (post-norm, gate, residual, pre-norm) against its
64-bit form, and its 8-bit output against the separate quantization, bit for bit."""
from __future__ import annotations

import numpy as np
import pytest

import block_ref as B
import gpu_util as U
from test_e4m3_gpu import quantize, u8

pytestmark = pytest.mark.gpu
EPS = 1e-6


def case(R, C, layer, post, gate_rows, seed=0):
    rng = np.random.default_rng(seed + R * 31 + C)
    n = rng.standard_normal
    c = dict(x=(2 * n((R, C)) + 0.3).astype(np.float16), y=(n((R, C)) + 0.2).astype(np.float16),
             pre_w=(1 + 0.2 * n(C)).astype(np.float32), pre_b=(0.1 * n(C)).astype(np.float32) if layer else None,
             post_w=(1 + 0.2 * n(C)).astype(np.float32) if post else None,
             post_b=(0.1 * n(C)).astype(np.float32) if post and layer else None,
             gate=(2 * n((gate_rows, C))).astype(np.float16) if gate_rows else None)
    return c


def p(t):
    return None if t is None else U.ptr(t)


def run(c, act=0, xs=1.0, ys=1.0, layer=False, eps=EPS, e4m3=False, in_place=None, stream=None):
    """(x', h) on the device; h is (codes, scales) for e4m3. `in_place`: "x" or "y"
    for x_out, "h" for h on y."""
    d = {k: None if v is None else U.dev(v) for k, v in c.items()}
    R, C = c["x"].shape
    xo = None if d.get("y") is None else d[in_place] if in_place in ("x", "y") else U.empty((R, C), np.float16)
    rows = 0 if d["gate"] is None else d["gate"].shape[0]
    s = U.stream() if stream is None else stream
    head = (p(d["x"]), p(d["y"]), p(d["post_w"]), p(d["post_b"]), p(d["gate"]), rows, act, xs, ys, p(xo), p(d["pre_w"]),
            p(d["pre_b"]))
    if e4m3:
        h = u8((R, B.pitch(C))), u8((B.groups(C), R, 4))
        U.call("hexlib_b200_norm_gate_residual_e4m3", *head, U.ptr(h[0]), U.ptr(h[1]), R, C, int(layer), eps, s)
    else:
        h = None if d["pre_w"] is None else d["y"] if in_place == "h" else U.empty((R, C), np.float16)
        U.call("hexlib_b200_norm_gate_residual_fp16", *head, p(h), R, C, int(layer), eps, s)
    return xo, h


def check(c, act=0, xs=1.0, ys=1.0, layer=False, eps=EPS, in_place=None):
    xo, h = run(c, act, xs, ys, layer, eps, in_place=in_place)
    if c["y"] is not None:
        ref, bound = B.edge_x(c["x"], c["y"], c["post_w"], c["post_b"], c["gate"], act, float(np.float32(xs)),
                              float(np.float32(ys)), layer, eps)
        B.assert_within(U.host(xo), ref, bound, "x'")
    stored = U.host(xo) if xo is not None else c["x"]
    if c["pre_w"] is not None:
        ref, bound = B.edge_h(stored, c["pre_w"], c["pre_b"], layer, eps)
        B.assert_within(U.host(h), ref, bound, "h")
        # the 8-bit form: the same x', and exactly the form of the fp16 h
        xo8, (q, s) = run(c, act, xs, ys, layer, eps, e4m3=True)
        if xo is not None:
            assert np.array_equal(U.host(xo8), stored)
        rq, rs = B.quantize(U.host(h))
        assert np.array_equal(U.host(s), rs) and B.same_codes(U.host(q), rq)


WIDTHS = [1, 7, 8, 64, 127, 128, 136, 256, 500, 512, 768, 1000, 1024, 1203, 1280, 1536, 2048, 2304, 2560, 4096, 5000,
          5120, 6144, 8192, 8200, 12288, 16384, 20000]


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("C", WIDTHS)
def test_widths(C, layer):
    check(case(5, C, layer, True, 1), 1, layer=layer)


@pytest.mark.parametrize("R", [1, 2, 3, 8, 65, 1000, 3001])
def test_row_counts(R):
    check(case(R, 768, True, False, 1), layer=True)
    check(case(R, 320, False, True, R), 2)


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("gate_rows", [1, 3, 12])
def test_gates_and_norms(gate_rows, act, post, layer):
    for C in (768, 333, 4096):
        check(case(12, C, layer, post, gate_rows), act, 0.7, -1.5, layer)


@pytest.mark.parametrize("C", [96, 768, 777, 2048])
def test_without_gate_or_block_output_or_next_norm(C):
    c = case(6, C, True, True, 0)
    check(c, layer=True)
    check(dict(c, post_w=None, post_b=None), xs=0.5, ys=2.0, layer=True)
    check(dict(c, y=None, post_w=None, post_b=None), layer=True)
    check(dict(c, pre_w=None, pre_b=None), layer=True)
    check(dict(c, pre_b=None, post_b=None), layer=True)


@pytest.mark.parametrize("C", [768, 1203, 2048, 4096, 17000])
@pytest.mark.parametrize("in_place", ["x", "y", "h"])
def test_in_place(in_place, C):
    c = case(70, C, False, True, 70)
    want = [U.host(t) for t in run(c, 1)]
    got = [U.host(t) for t in run(c, 1, in_place=in_place)]
    assert all(np.array_equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("C", [256, 300, 3000])
def test_rows_of_zeros_and_rows_far_from_zero(C):
    c = case(4, C, True, True, 1)
    c["x"][0], c["y"][0] = 0, 0
    c["x"][1] = np.float16(1000)                     # a constant row: variance 0, the mean exact
    c["y"][1] = 0
    c["post_b"][:] = 0
    xo, h = run(c, layer=True)
    assert np.array_equal(U.host(xo)[:2], c["x"][:2])
    assert np.array_equal(U.host(h)[:2], np.broadcast_to(c["pre_b"].astype(np.float16), (2, C)))
    for layer in (False, True):
        c = case(3, C, layer, False, 0)
        c["x"] = (c["x"].astype(np.float32) + 300).astype(np.float16)
        check(c, layer=layer)


def test_non_finite_rows_stay_their_own():
    for C in (768, 1203):
        c = case(6, C, False, True, 1)
        want, _ = run(c)
        c["x"][2, 5], c["y"][4, 9] = np.inf, np.nan
        xo, h = run(c)
        _, (q, s) = run(c, e4m3=True)
        clean = [0, 1, 3, 5]
        assert np.array_equal(U.host(xo)[clean], U.host(want)[clean])
        assert np.isfinite(U.host(h)[clean].astype(np.float64)).all() and np.isnan(U.host(h)[4]).all()
        assert np.isinf(U.host(xo)[2, 5]) and np.isnan(U.host(xo)[4]).all()
        rq, rs = B.quantize(U.host(h))
        assert np.array_equal(U.host(s), rs) and B.same_codes(U.host(q), rq)


@pytest.mark.parametrize("C", [768, 1203])
def test_misaligned_rows_give_the_same_values(C):
    import torch
    c = case(9, C, True, True, 9)
    want = [U.host(t) for t in run(c, 1, layer=True)]
    d = {}
    for k, v in c.items():
        flat = torch.zeros(v.size + 3, dtype=torch.float16 if v.dtype == np.float16 else torch.float32, device="cuda")
        flat[3:] = U.dev(v).reshape(-1)
        d[k] = flat[3:]
    out = torch.full((2, 9 * C + 16), -7.0, dtype=torch.float16, device="cuda")
    xo, h = out[0][5:5 + 9 * C], out[1][3:3 + 9 * C]
    U.call("hexlib_b200_norm_gate_residual_fp16", p(d["x"]), p(d["y"]), p(d["post_w"]), p(d["post_b"]), p(d["gate"]), 9, 1,
           1.0, 1.0, U.ptr(xo), p(d["pre_w"]), p(d["pre_b"]), U.ptr(h), 9, C, 1, EPS, U.stream())
    # another order of the same sums: each within its own bound of the other
    ref, bound = B.edge_x(c["x"], c["y"], c["post_w"], c["post_b"], c["gate"], 1, 1.0, 1.0, True, EPS)
    B.assert_within(U.host(xo).reshape(9, C), ref, bound, "x'")
    ref, bound = B.edge_h(U.host(xo).reshape(9, C), c["pre_w"], c["pre_b"], True, EPS)
    B.assert_within(U.host(h).reshape(9, C), ref, bound, "h")
    assert want[0].shape == (9, C)
    assert bool((out[0][:5] == -7).all()) and bool((out[0][5 + 9 * C:] == -7).all())
    assert bool((out[1][:3] == -7).all()) and bool((out[1][3 + 9 * C:] == -7).all())


def test_repeats_bit_for_bit_eager_captured_and_on_another_stream():
    import torch
    for C in (768, 1203, 4096):
        c = case(200, C, False, True, 200)
        want = [U.host(t) for t in run(c, 2)]
        other = torch.cuda.Stream()
        with torch.cuda.stream(other):
            got = run(c, 2, stream=other.cuda_stream)
        other.synchronize()
        assert all(np.array_equal(a, U.host(b)) for a, b in zip(want, got))
        d = {k: None if v is None else U.dev(v) for k, v in c.items()}
        xo, h = U.empty((200, C), np.float16), U.empty((200, C), np.float16)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            U.call("hexlib_b200_norm_gate_residual_fp16", p(d["x"]), p(d["y"]), p(d["post_w"]), None, p(d["gate"]), 200, 2,
                   1.0, 1.0, U.ptr(xo), p(d["pre_w"]), None, U.ptr(h), 200, C, 0, EPS, U.stream())
        for _ in range(2):
            graph.replay()
        assert np.array_equal(U.host(xo), want[0]) and np.array_equal(U.host(h), want[1])


def test_the_separate_quantization_agrees_on_the_device():
    c = case(333, 1280, False, True, 333)
    _, h = run(c, 1)
    _, (q, s) = run(c, 1, e4m3=True)
    q2, s2 = quantize(h)
    assert np.array_equal(U.host(q), U.host(q2)) and np.array_equal(U.host(s), U.host(s2))


@pytest.mark.parametrize("act", [1, 2, 3])
@pytest.mark.parametrize("C", [1024, 1203, 17000])
def test_gates_of_every_size(C, act):
    # gates over fp16's whole range on a branch of ones: x' is the gate's function
    rng = np.random.default_rng(act)
    g = (rng.standard_normal((8, C)) * 2.0 ** rng.integers(-12, 5, (8, C))).astype(np.float16)
    g[0, :8] = [0, -0.0, 65504, -65504, 17, -17, 6e-8, -11]
    one = np.ones((8, C), np.float16)
    c = dict(x=one, y=one, post_w=None, post_b=None, gate=g, pre_w=None, pre_b=None)
    xo, _ = run(c, act, xs=0.0)
    ref, bound = B.edge_x(one, one, None, None, g, act, 0.0, 1.0, False, EPS)
    B.assert_within(U.host(xo), ref, bound, "gate")
    g[0, :2] = [np.inf, -np.inf]
    got = U.host(run(c, act, xs=0.0)[0])[0, :2]
    want = {1: [1, 0], 2: [np.inf, np.nan], 3: [1, -1]}[act]
    assert np.array_equal(got.astype(np.float64), np.array(want, np.float64), equal_nan=True)
