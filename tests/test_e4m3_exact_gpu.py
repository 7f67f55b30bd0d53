"""The 8-bit product of small whole numbers: every sum is exact in fp32, so the output is
the exact value rounded once, whatever the tiling and however K is split. A bound of one
rounding for each addition, as random values need it, would hide an accumulator of fewer
bits or a partial sum that is lost or joined twice."""
from __future__ import annotations

import numpy as np
import pytest

import block_ref as B
import gpu_util as U
from test_e4m3_gpu import product

pytestmark = pytest.mark.gpu

CODE = {v: int(np.flatnonzero(B.VALUES == v)[0]) for v in range(-8, 9)}   # (0 stands for +0)
TABLE = np.array([CODE[v] for v in range(-8, 9)], np.uint8)


def form(rng, R, K, low, scales):
    """(codes, scale bytes, values) of R rows of whole numbers low..7 with scales 2^s, s
    drawn for each block."""
    kb = B.pitch(K) // 128
    v = np.zeros((R, kb * 128), np.int64)
    v[:, :K] = rng.integers(low, 8, (R, K))
    s = np.full((R, B.groups(K) * 4), 127, np.uint8)
    s[:, :kb] = 127 + rng.choice(scales, (R, kb))
    s = np.ascontiguousarray(s.reshape(R, -1, 4).transpose(1, 0, 2))
    q = TABLE[v + 8]
    return U.dev(q), U.dev(s), B.values(q, s)


# one token to whole tiles of tokens, one block of K to 129: each width of token tile, each
# split of K over a cluster, and CTA pairs
SHAPES = [(1, 100, 5), (1, 1100, 130), (1, 2048, 640), (3, 4096, 515), (16, 16500, 264), (17, 300, 1000), (33, 1100, 1000),
          (31, 16500, 640), (64, 8200, 777), (100, 4096, 4096), (100, 8200, 777), (130, 16500, 1000), (130, 16500, 2304),
          (257, 5000, 2048), (300, 2048, 640), (700, 8200, 515), (520, 5000, 2304), (1500, 4096, 64), (2600, 300, 777),
          (2600, 4096, 5), (2600, 1100, 1032), (5000, 640, 640), (9500, 130, 770)]


def check(a, w, M, K, N, rng, bias, with_resid):
    av, wv = a[2], w[2]
    assert (np.abs(av).max(1).max() * np.abs(wv).max(1).max() * K) < 2 ** 22   # in quarters, under 24 bits
    resid = rng.integers(-64, 65, (M, N)).astype(np.float16) if with_resid else None
    exact = av @ wv.T + (0 if bias is None else bias) + (0 if resid is None else resid.astype(np.float64))
    assert np.abs(exact).max() < 65504
    y = product(a, w, M, K, N, 0, bias, None if resid is None else U.dev(resid))
    assert np.array_equal(U.host(y), exact.astype(np.float16))


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_sums_of_whole_numbers_are_exact(M, K, N):
    rng = np.random.default_rng(M + K + N)
    a, w = form(rng, M, K, -7, [-1, 0, 1]), form(rng, N, K, -7, [-1, 0, 1])
    check(a, w, M, K, N, rng, None, False)
    check(a, w, M, K, N, rng, rng.integers(-999, 1000, N).astype(np.float32), True)


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_low_bits_of_a_large_sum_are_kept(M, K, N):
    # all products positive, the sum's mean taken off by the bias: a sum of up to 2^20 has
    # to arrive with its last bit
    rng = np.random.default_rng(M * 3 + K + N)
    a, w = form(rng, M, K, 1, [0]), form(rng, N, K, 1, [0])
    check(a, w, M, K, N, rng, np.full(N, -16.0 * K, np.float32), False)
