"""The transformer-block operators on tensors of more than 2^31 elements: the last rows,
whose offsets pass 32 bits, against their 64-bit forms."""
from __future__ import annotations

import numpy as np
import pytest

import block_ref as B
import gpu_util as U
from test_e4m3_gpu import u8

pytestmark = pytest.mark.gpu

R, C = 1_050_001, 2048          # 2.15e9 elements
LAST = 5


def rows(seed):
    """fp16 [R, C] on the device, zeros but for its first and last rows."""
    import torch
    x = torch.zeros((R, C), dtype=torch.float16, device="cuda")
    v = np.random.default_rng(seed).standard_normal((LAST, C)).astype(np.float16)
    x[-LAST:] = U.dev(v)
    x[:LAST] = U.dev(v[::-1])
    return x, v


def test_quantize_and_dequant_past_32_bits():
    x, v = rows(1)
    q, s = u8((R, C)), u8((C // 512, R, 4))
    U.call("hexlib_b200_quantize_e4m3_fp16", U.ptr(x), U.ptr(q), U.ptr(s), R, C, U.stream())
    rq, rs = B.quantize(v)
    assert np.array_equal(U.host(q[-LAST:]), rq) and np.array_equal(U.host(s[:, -LAST:]), rs)
    assert np.array_equal(U.host(q[:LAST]), rq[::-1])
    x.zero_()
    U.call("hexlib_b200_dequant_e4m3_fp16", U.ptr(q), U.ptr(s), U.ptr(x), R, C, U.stream())
    want = B.values(rq, rs).astype(np.float16)
    assert np.array_equal(U.host(x[-LAST:]), want) and np.array_equal(U.host(x[:LAST]), want[::-1])


@pytest.mark.parametrize("N", [2048, 2049])
def test_product_past_32_bits(N):
    import torch
    rng = np.random.default_rng(2)
    a = rng.standard_normal((LAST, 128)).astype(np.float16)
    w = (rng.standard_normal((N, 128)) / 11).astype(np.float16)
    (aq, as_), (wq, ws) = B.quantize(a), B.quantize(w)
    q = torch.zeros((R, 128), dtype=torch.uint8, device="cuda")
    s = torch.full((1, R, 4), 127, dtype=torch.uint8, device="cuda")
    q[-LAST:], s[:, -LAST:] = U.dev(aq), U.dev(as_)
    out = torch.empty((R, N), dtype=torch.float16, device="cuda")
    dw, ds = U.dev(wq), U.dev(ws)
    U.call("hexlib_b200_matmul_epilogue_e4m3", U.ptr(q), U.ptr(s), U.ptr(dw), U.ptr(ds), None, U.ptr(out), R, 128, N, 0,
           U.stream())
    U.call("hexlib_b200_stream_status", U.stream())
    ref, bound = B.product(B.values(aq, as_), B.values(wq, ws), None, None, 0)
    B.assert_within(U.host(out[-LAST:]), ref, bound, "last rows")
    assert not bool(out[:-LAST].any())


def test_edge_past_32_bits():
    import torch
    x, v = rows(3)
    y, u = rows(4)
    rng = np.random.default_rng(5)
    pw, w = (1 + 0.1 * rng.standard_normal((2, C))).astype(np.float32)
    h, dpw, dw = torch.empty_like(x), U.dev(pw), U.dev(w)
    U.call("hexlib_b200_norm_gate_residual_fp16", U.ptr(x), U.ptr(y), U.ptr(dpw), None, None, 0, 0, 1.0, 1.0, U.ptr(y),
           U.ptr(dw), None, U.ptr(h), R, C, 0, 1e-6, U.stream())
    ref, bound = B.edge_x(v, u, pw, None, None, 0, 1.0, 1.0, False, 1e-6)
    got = U.host(y[-LAST:])
    B.assert_within(got, ref, bound, "x'")
    ref, bound = B.edge_h(got, w, None, False, 1e-6)
    B.assert_within(U.host(h[-LAST:]), ref, bound, "h")
