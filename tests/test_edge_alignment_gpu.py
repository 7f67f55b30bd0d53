"""The edge between two blocks on tensors that start anywhere: the same bits as from aligned
ones where the rows hold no whole vectors either way, both forms of h from the same
addresses, values within the norms' own bounds elsewhere, and nothing written beside."""
from __future__ import annotations

import numpy as np
import pytest

import block_ref as B
import gpu_util as U
from test_edge_accuracy_gpu import norm, same_form, to_f16
from test_edge_gpu import EPS, case, p, run

pytestmark = pytest.mark.gpu
R = 9


def shifted(c, shift):
    """The tensors of a case, each `shift` elements past an aligned start, and outputs with
    marked elements on both sides."""
    import torch
    d, marked = {}, {}
    for k, v in c.items():
        if v is None:
            d[k] = None
            continue
        flat = torch.zeros(v.size + shift, dtype=torch.float16 if v.dtype == np.float16 else torch.float32, device="cuda")
        flat[shift:] = U.dev(v).reshape(-1)
        d[k] = flat[shift:]
    C = c["x"].shape[1]
    for k in ("xo", "h"):
        marked[k] = torch.full((shift + R * C + 16,), -7.0, dtype=torch.float16, device="cuda")
        d[k] = marked[k][shift:shift + R * C]
    return d, marked


def call(c, d, layer, act, e4m3):
    import torch
    C, rows = c["x"].shape[1], 0 if c["gate"] is None else c["gate"].shape[0]
    head = (p(d["x"]), p(d["y"]), p(d["post_w"]), p(d["post_b"]), p(d["gate"]), rows, act, 1.0, 0.5, p(d["xo"]), p(d["pre_w"]),
            p(d["pre_b"]))
    if not e4m3:
        U.call("hexlib_b200_norm_gate_residual_fp16", *head, p(d["h"]), R, C, int(layer), EPS, U.stream())
        return U.host(d["xo"]).reshape(R, C), U.host(d["h"]).reshape(R, C)
    q = torch.full((R + 1, B.pitch(C)), 0xA5, dtype=torch.uint8, device="cuda")
    s = torch.full((B.groups(C) + 1, R, 4), 0xA5, dtype=torch.uint8, device="cuda")
    U.call("hexlib_b200_norm_gate_residual_e4m3", *head, U.ptr(q), U.ptr(s), R, C, int(layer), EPS, U.stream())
    assert bool((q[R] == 0xA5).all()) and bool((s[-1] == 0xA5).all())
    return U.host(d["xo"]).reshape(R, C), (q[:R], s[:-1])


@pytest.mark.parametrize("layer", [True, False])
@pytest.mark.parametrize("shift", [1, 2, 3, 4])
@pytest.mark.parametrize("C", [7, 285, 768, 1203, 2048, 4100, 16384, 17001])
def test_any_start(C, shift, layer):
    c = case(R, C, layer, True, R)
    xo0, h0 = (U.host(t) for t in run(c, 1, 1.0, 0.5, layer=layer))
    d, marked = shifted(c, shift)
    xo, h = call(c, d, layer, 1, False)
    f64 = lambda a: None if a is None else a.astype(np.float64)  # noqa: E731
    if C % 8:
        # no whole vectors from any start: the same kernel, the same order of every sum
        assert np.array_equal(xo, xo0) and np.array_equal(h, h0)
    else:
        # x' of both is within its bound of the exact value, so within twice that of each other
        u, err = norm(f64(c["y"]), f64(c["post_w"]), f64(c["post_b"]), layer, float(np.float32(EPS)))
        g = B.gate_value(c["gate"], 1)
        v = f64(c["x"]) + 0.5 * u * g
        err = 0.5 * (err * g + np.abs(u) * g * 2.0 ** -21) + (np.abs(f64(c["x"])) + np.abs(u * g)) * 2.0 ** -22
        B.assert_within(xo, *to_f16(v, err), "x'")
        B.assert_within(xo0, *to_f16(v, err), "aligned x'")
    for got, stored in ((h, xo), (h0, xo0)):
        ref, bound = to_f16(*norm(f64(stored), f64(c["pre_w"]), f64(c["pre_b"]), layer, float(np.float32(EPS))))
        B.assert_within(got, ref, bound, "h")
    for m in marked.values():
        assert bool((m[:shift] == -7).all()) and bool((m[shift + R * C:] == -7).all())
    # the 8-bit form from the same addresses
    d, marked = shifted(c, shift)
    xo8, form = call(c, d, layer, 1, True)
    assert np.array_equal(xo8, xo) and same_form(form, h)
