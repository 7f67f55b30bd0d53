"""The 8-bit product right after the kernel that writes its operands, all of them carved
from one allocation so that the scales lie in the cache lines the quantization or the
edge has just read."""
from __future__ import annotations

import numpy as np
import pytest

import block_ref as B
import gpu_util as U
from test_e4m3_gpu import operands

pytestmark = pytest.mark.gpu


def carve(sizes):
    """Consecutive pieces of one zeroed buffer, each from the first address after the piece
    before that its alignment allows: [(bytes, alignment)] -> tensors of bytes."""
    import torch
    at, cuts = 0, []
    for n, align in sizes:
        at = -(-at // align) * align
        cuts.append((at, n))
        at += n
    arena = torch.zeros(at + 64, dtype=torch.uint8, device="cuda")
    assert arena.data_ptr() % 16 == 0
    return [arena[a:a + n] for a, n in cuts]


@pytest.mark.parametrize("M,K,N", [(3, 3, 40), (1, 130, 64), (5, 257, 300), (40, 515, 128), (300, 701, 640), (2100, 35, 520)])
@pytest.mark.parametrize("by_edge", [False, True])
def test_scales_in_the_lines_of_the_rows_they_come_from(M, K, N, by_edge):
    import torch
    rng = np.random.default_rng(M + K)
    _, w = operands(rng, 1, K, N)
    kp, g = B.pitch(K), B.groups(K)
    # rows, the scales right behind them, the bias behind those, then codes and output
    x, s, bias, q, out = carve([(2 * M * K, 16), (4 * g * M, 4), (4 * N, 4), (M * kp, 16), (2 * M * N, 16)])
    weight, b = U.dev((1 + 0.1 * rng.standard_normal(K)).astype(np.float32)), rng.standard_normal(N).astype(np.float32)
    bias.view(torch.float32).copy_(U.dev(b))
    xs = [(rng.standard_normal((M, K)) * 4.0 ** i).astype(np.float16) for i in range(3)]
    dev = [U.dev(v) for v in xs]
    outs = []
    for i in range(9):
        x.view(torch.float16).copy_(dev[i % 3].reshape(-1))
        if by_edge:
            U.call("hexlib_b200_norm_gate_residual_e4m3", U.ptr(x), None, None, None, None, 0, 0, 1.0, 1.0, None, U.ptr(weight),
                   None, U.ptr(q), U.ptr(s), M, K, 0, 1.0 + i % 3, U.stream())
        else:
            U.call("hexlib_b200_quantize_e4m3_fp16", U.ptr(x), U.ptr(q), U.ptr(s), M, K, U.stream())
        U.call("hexlib_b200_matmul_epilogue_e4m3", U.ptr(q), U.ptr(s), U.ptr(w[0]), U.ptr(w[1]), U.ptr(bias), U.ptr(out), M, K, N,
               0, U.stream())
        outs.append((out.clone(), q.clone(), s.clone()))
    U.call("hexlib_b200_stream_status", U.stream())
    for i, (y, cq, cs) in enumerate(outs):
        codes, scales = U.host(cq).reshape(M, kp), U.host(cs).reshape(g, M, 4)
        if not by_edge:
            rq, rs = B.quantize(xs[i % 3])
            assert np.array_equal(scales, rs) and B.same_codes(codes, rq)
        ref, bound = B.product(B.values(codes, scales), w[2], b, None, 0)
        B.assert_within(U.host(y.view(torch.float16)).reshape(M, N), ref, bound, f"call {i}")
