"""The e4m3 form and the 8-bit product against their 64-bit forms."""
from __future__ import annotations

import numpy as np
import pytest

import block_ref as B
import gpu_util as U

pytestmark = pytest.mark.gpu


def u8(shape, fill=0xA5):
    import torch
    return torch.full(shape, fill, dtype=torch.uint8, device="cuda")


def quantize(x):
    """The library's e4m3 form of an fp16 matrix on the device."""
    R, K = x.shape
    q, s = u8((R, B.pitch(K))), u8((B.groups(K), R, 4))
    U.call("hexlib_b200_quantize_e4m3_fp16", U.ptr(x), U.ptr(q), U.ptr(s), R, K, U.stream())
    return q, s


def rows(rng, R, K):
    """Values over fp16's whole range, a block scale at a time, with rounding ties."""
    x = rng.standard_normal((R, K)) * 2.0 ** rng.integers(-18, 12, (R, 1))
    x.flat[::7] = np.round(x.flat[::7] * 8) / 8
    return np.clip(x, -65504, 65504).astype(np.float16)


@pytest.mark.parametrize("R,K", [(1, 1), (1, 127), (3, 128), (2, 129), (5, 500), (4, 512), (3, 513), (33, 768),
                                 (7, 1203), (130, 1024), (2, 8200), (1, 4096)])
def test_quantize_matches_the_definition_bit_for_bit(R, K):
    x = rows(np.random.default_rng(R * 10007 + K), R, K)
    x[0, K // 2] = 65504
    q, s = quantize(U.dev(x))
    rq, rs = B.quantize(x)
    assert np.array_equal(U.host(s), rs)
    assert B.same_codes(U.host(q), rq)


def test_quantize_every_half_value():
    # all finite fp16 values, each alone in a block and each beside the largest one
    bits = np.arange(65536, dtype=np.uint32).astype(np.uint16).view(np.float16)
    bits = bits[np.isfinite(bits)]
    x = np.zeros((bits.size // 2 + 1, 256), np.float16)
    n = bits.size // 2
    x[:n, 0], x[:n, 128], x[:n, 129] = bits[:n], bits[n:2 * n], np.float16(448)
    q, s = quantize(U.dev(x))
    rq, rs = B.quantize(x)
    assert np.array_equal(U.host(s), rs) and np.array_equal(U.host(q), rq)


def test_quantize_non_finite_values_are_nan_and_leave_the_scale_alone():
    x = rows(np.random.default_rng(5), 4, 300)
    x[1, 3], x[1, 200], x[2, 299], x[3, :128] = np.inf, -np.inf, np.nan, np.inf
    q, s = quantize(U.dev(x))
    rq, rs = B.quantize(x)
    assert np.array_equal(U.host(s), rs) and B.same_codes(U.host(q), rq)


def test_quantize_reads_any_row_start_and_writes_only_its_own():
    import torch
    x = rows(np.random.default_rng(6), 9, 200)
    flat = torch.zeros(1 + x.size, dtype=torch.float16, device="cuda")
    flat[1:] = U.dev(x).reshape(-1)
    q, s = u8((10, 256)), u8((2, 9, 4))
    U.call("hexlib_b200_quantize_e4m3_fp16", U.ptr(flat) + 2, U.ptr(q), U.ptr(s), 9, 200, U.stream())
    rq, rs = B.quantize(x)
    assert np.array_equal(U.host(q)[:9], rq) and np.array_equal(U.host(s)[:1], rs)
    assert (U.host(q)[9] == 0xA5).all() and (U.host(s)[1] == 0xA5).all()


@pytest.mark.parametrize("K,N", [(1, 1), (128, 8), (130, 33), (513, 100), (768, 2304), (1100, 777)])
def test_quantize_weight_is_the_form_of_the_transpose(K, N):
    w = rows(np.random.default_rng(K + N), K, N)
    q, s = u8((N, B.pitch(K))), u8((B.groups(K), N, 4))
    U.call("hexlib_b200_quantize_weight_e4m3_fp16", U.ptr(U.dev(w)), U.ptr(q), U.ptr(s), K, N, U.stream())
    rq, rs = B.quantize(np.ascontiguousarray(w.T))
    assert np.array_equal(U.host(s), rs) and B.same_codes(U.host(q), rq)


@pytest.mark.parametrize("R,K", [(1, 1), (5, 130), (33, 1203), (64, 1024)])
def test_dequant_gives_the_values(R, K):
    x = rows(np.random.default_rng(R + K), R, K)
    q, s = quantize(U.dev(x))
    y = U.empty((R, K), np.float16)
    U.call("hexlib_b200_dequant_e4m3_fp16", U.ptr(q), U.ptr(s), U.ptr(y), R, K, U.stream())
    with np.errstate(over="ignore"):
        ref = B.values(*B.quantize(x))[:, :K].astype(np.float16)
    assert np.array_equal(U.host(y), ref)


def operands(rng, M, K, N, spread=0):
    """Codes and scales of both operands on the device, and their values. With
    `spread`, rows differ by up to 2^spread."""
    def one(R, std):
        x = (rng.standard_normal((R, K)) * std).astype(np.float64)
        if spread:
            x *= 2.0 ** rng.integers(-spread, spread + 1, (R, 1))
        q, s = B.quantize(x.astype(np.float16))
        return U.dev(q), U.dev(s), B.values(q, s)
    return one(M, 1.0), one(N, K ** -0.5)


def product(a, w, M, K, N, act=0, bias=None, resid=None, out=None):
    y = U.empty((M, N), np.float16) if out is None else out
    b = None if bias is None else U.dev(bias.astype(np.float32))
    if resid is None:
        U.call("hexlib_b200_matmul_epilogue_e4m3", U.ptr(a[0]), U.ptr(a[1]), U.ptr(w[0]), U.ptr(w[1]),
               None if b is None else U.ptr(b), U.ptr(y), M, K, N, act, U.stream())
    else:
        U.call("hexlib_b200_matmul_epilogue_residual_e4m3", U.ptr(a[0]), U.ptr(a[1]), U.ptr(w[0]), U.ptr(w[1]),
               None if b is None else U.ptr(b), U.ptr(resid), U.ptr(y), M, K, N, act, U.stream())
    U.call("hexlib_b200_stream_status", U.stream())
    return y


SHAPES = [(1, 1, 1), (1, 128, 8), (1, 4096, 256), (2, 130, 5), (8, 512, 64), (16, 640, 100), (17, 1100, 128),
          (31, 2048, 777), (33, 513, 1000), (64, 768, 768), (65, 256, 192), (100, 384, 264), (127, 128, 136),
          (128, 128, 128), (129, 257, 200), (200, 1024, 2304), (256, 768, 2304), (300, 1100, 777), (513, 896, 1032),
          (1000, 640, 1024), (2100, 300, 520), (4097, 128, 1280)]


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_product_matches_the_64_bit_sum(M, K, N):
    rng = np.random.default_rng(M * 7 + K * 3 + N)
    a, w = operands(rng, M, K, N)
    ref, bound = B.product(a[2], w[2], None, None, 0)
    B.assert_within(U.host(product(a, w, M, K, N)), ref, bound, "product")


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("with_bias,with_resid", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("M,K,N", [(1, 300, 130), (20, 640, 515), (70, 256, 96), (140, 1100, 328), (700, 512, 1000)])
def test_product_epilogues(M, K, N, act, with_bias, with_resid):
    rng = np.random.default_rng(M + K + N + act)
    a, w = operands(rng, M, K, N)
    bias = rng.standard_normal(N).astype(np.float32) if with_bias else None
    resid = rng.standard_normal((M, N)).astype(np.float16) if with_resid else None
    ref, bound = B.product(a[2], w[2], bias, resid, act)
    y = product(a, w, M, K, N, act, bias, None if resid is None else U.dev(resid))
    B.assert_within(U.host(y), ref, bound, "epilogue")


@pytest.mark.parametrize("M,K,N", [(3, 700, 140), (150, 640, 264), (600, 1500, 512)])
def test_product_of_rows_of_very_different_size(M, K, N):
    a, w = operands(np.random.default_rng(M), M, K, N, spread=6)
    ref, bound = B.product(a[2], w[2], None, None, 0)
    B.assert_within(U.host(product(a, w, M, K, N)), ref, bound, "spread")


@pytest.mark.parametrize("M,K,N", [(5, 600, 40), (130, 1024, 256), (600, 1024, 768)])
def test_every_block_has_a_scale_of_its_own(M, K, N):
    # codes of one everywhere and scales drawn block by block: any scale taken from
    # another row, block or operand shows
    rng = np.random.default_rng(M)
    kb = B.pitch(K) // 128

    def form(R):
        s = np.full((R, B.groups(K) * 4), 127, np.uint8)
        s[:, :kb] = rng.integers(121, 130, (R, kb))
        q = np.zeros((R, B.pitch(K)), np.uint8)
        q[:, :K] = 0x38                                        # 1.0
        s = np.ascontiguousarray(s.reshape(R, -1, 4).transpose(1, 0, 2))
        return U.dev(q), U.dev(s), B.values(q, s)
    a, w = form(M), form(N)
    ref, bound = B.product(a[2], w[2], None, None, 0)
    B.assert_within(U.host(product(a, w, M, K, N)), ref, bound, "scales")


@pytest.mark.parametrize("M,N", [(3, 40), (200, 300), (600, 1024)])
def test_nan_codes_reach_their_row_and_column_alone(M, N):
    rng = np.random.default_rng(N)
    a, w = operands(rng, M, 256, N)
    a[0][1, 200] = 0x7F
    w[0][2, 5] = 0xFF
    y = U.host(product(a, w, M, 256, N))
    ref, bound = B.product(a[2], w[2], None, None, 0)
    assert np.isnan(y[1]).all() and np.isnan(y[:, 2]).all()
    keep = np.ix_([i for i in range(M) if i != 1], [j for j in range(N) if j != 2])
    B.assert_within(y[keep], ref[keep], bound[keep], "beside NaN")


@pytest.mark.parametrize("M,N", [(1, 33), (9, 64), (70, 130), (300, 257), (600, 512)])
def test_nothing_is_written_beside_the_output(M, N):
    import torch
    a, w = operands(np.random.default_rng(M + N), M, 384, N)
    for shift in (0, 1, 8):
        flat = torch.full((M * N + 256,), -7.0, dtype=torch.float16, device="cuda")
        y = flat[64 + shift:64 + shift + M * N].view(M, N)
        product(a, w, M, 384, N, out=y)
        ref, bound = B.product(a[2], w[2], None, None, 0)
        B.assert_within(U.host(y), ref, bound, f"shift {shift}")
        assert bool((flat[:64 + shift] == -7).all()) and bool((flat[64 + shift + M * N:] == -7).all())


@pytest.mark.parametrize("M,N", [(4, 100), (40, 512), (333, 264), (1024, 768)])
def test_residual_in_place(M, N):
    rng = np.random.default_rng(M)
    a, w = operands(rng, M, 512, N)
    r = rng.standard_normal((M, N)).astype(np.float16)
    y = U.dev(r)
    product(a, w, M, 512, N, 1, None, y, out=y)
    ref, bound = B.product(a[2], w[2], None, r, 1)
    B.assert_within(U.host(y), ref, bound, "in place")


@pytest.mark.parametrize("M,K,N", [(1, 2048, 520), (48, 1280, 640), (900, 1024, 768)])
def test_product_repeats_bit_for_bit_eager_captured_and_beside_another(M, K, N):
    import torch
    rng = np.random.default_rng(K)
    a, w = operands(rng, M, K, N)
    bias = rng.standard_normal(N).astype(np.float32)
    first = U.host(product(a, w, M, K, N, 2, bias))
    assert np.array_equal(first, U.host(product(a, w, M, K, N, 2, bias)))
    b = U.dev(bias)
    ys = [U.empty((M, N), np.float16) for _ in range(3)]

    def go(y, s):
        U.call("hexlib_b200_matmul_epilogue_e4m3", U.ptr(a[0]), U.ptr(a[1]), U.ptr(w[0]), U.ptr(w[1]), U.ptr(b),
               U.ptr(y), M, K, N, 2, s)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        go(ys[0], U.stream())
    other = torch.cuda.Stream()
    for _ in range(3):
        graph.replay()
        go(ys[1], other.cuda_stream)
        go(ys[2], U.stream())
    torch.cuda.synchronize()
    for y in ys:
        assert np.array_equal(first, U.host(y))
    U.call("hexlib_b200_stream_status", U.stream())


def test_empty_batches_launch_nothing():
    assert U.call_rc("hexlib_b200_quantize_e4m3_fp16", None, None, None, 0, 64, U.stream()) == U.OK
    assert U.call_rc("hexlib_b200_matmul_epilogue_e4m3", None, None, None, None, None, None, 0, 64, 64, 0,
                     U.stream()) == U.OK


# outputs of many 256 x 256 tiles, several to a pair of SMs, with ragged edges in every
# direction and each epilogue
@pytest.mark.parametrize("M,K,N,act,with_bias,with_resid", [
    (2500, 513, 1000, 0, False, False), (4097, 1100, 1032, 0, True, True), (9000, 300, 1288, 1, True, False),
    (9473, 640, 520, 1, False, True), (5000, 128, 2048, 0, True, False), (3000, 2100, 1536, 2, True, True),
    (19000, 1, 264, 0, False, False), (20000, 260, 512, 0, False, False),
    (2600, 1500, 1001, 0, True, True), (2600, 1500, 1002, 1, True, False), (9500, 300, 777, 0, False, True),
    (9500, 300, 770, 2, True, True), (2304, 8200, 1280, 0, True, False)])
def test_product_of_many_tiles(M, K, N, act, with_bias, with_resid):
    rng = np.random.default_rng(M + K)
    a, w = operands(rng, M, K, N, spread=3)
    bias = rng.standard_normal(N).astype(np.float32) if with_bias else None
    resid = rng.standard_normal((M, N)).astype(np.float16) if with_resid else None
    ref, bound = B.product(a[2], w[2], bias, resid, act)
    y = U.dev(resid) if with_resid else U.empty((M, N), np.float16)
    product(a, w, M, K, N, act, bias, y if with_resid else None, out=y)
    first = U.host(y)
    B.assert_within(first, ref, bound, "tiles")
    if not with_resid:
        product(a, w, M, K, N, act, bias, None, out=y)
        assert np.array_equal(first, U.host(y))


@pytest.mark.parametrize("M,K,N", [(3, 2048, 640), (200, 1024, 512), (2600, 640, 1032)])
def test_product_after_copies_events_and_forks(M, K, N):
    # what may stand before a product in a stream: a copy, a fill, a wait for another
    # stream, another product; eager, and as nodes of one captured graph
    import torch
    rng = np.random.default_rng(M)
    a, w = operands(rng, M, K, N)
    want = U.host(product(a, w, M, K, N))
    x = U.dev(rng.standard_normal((M, K)).astype(np.float16))
    xq, xs = quantize(x)
    want2 = U.host(product((xq, xs), w, M, K, N))
    src, scales = a[0].clone(), a[1].clone()
    q, s = torch.zeros_like(src), torch.zeros_like(scales)
    q2, s2 = torch.zeros_like(xq), torch.zeros_like(xs)
    y, y2 = (torch.empty((M, N), dtype=torch.float16, device="cuda") for _ in range(2))
    fork = torch.cuda.Stream()

    def go():
        main = torch.cuda.current_stream()
        y.fill_(-1)
        q.copy_(src)
        fork.wait_stream(main)
        with torch.cuda.stream(fork):
            s.copy_(scales)
            U.call("hexlib_b200_quantize_e4m3_fp16", U.ptr(x), U.ptr(q2), U.ptr(s2), M, K, fork.cuda_stream)
            product((q2, s2), w, M, K, N, out=y2) if not torch.cuda.is_current_stream_capturing() else U.call(
                "hexlib_b200_matmul_epilogue_e4m3", U.ptr(q2), U.ptr(s2), U.ptr(w[0]), U.ptr(w[1]), None, U.ptr(y2), M, K, N, 0,
                fork.cuda_stream)
        main.wait_stream(fork)
        for _ in range(2):
            U.call("hexlib_b200_matmul_epilogue_e4m3", U.ptr(q), U.ptr(s), U.ptr(w[0]), U.ptr(w[1]), None, U.ptr(y), M, K, N, 0,
                   main.cuda_stream)

    def check():
        torch.cuda.synchronize()
        assert np.array_equal(U.host(y), want) and np.array_equal(U.host(y2), want2)
        for t in (q, s, q2, s2):
            t.zero_()
        y.zero_(), y2.zero_()
        torch.cuda.synchronize()
    go()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for _ in range(3):
        graph.replay()
        check()


def test_a_weight_quantized_just_before_its_product():
    import torch
    rng = np.random.default_rng(8)
    for M, K, N in ((1, 4096, 2048), (300, 512, 768)):
        a, _ = operands(rng, M, K, 8)
        ws = [(rng.standard_normal((K, N)) / K ** 0.5).astype(np.float16) for _ in range(2)]
        dev = [U.dev(w) for w in ws]
        q, s = u8((N, B.pitch(K))), u8((B.groups(K), N, 4))
        ys = [torch.empty((M, N), dtype=torch.float16, device="cuda") for _ in range(6)]
        for i, y in enumerate(ys):
            U.call("hexlib_b200_quantize_weight_e4m3_fp16", U.ptr(dev[i % 2]), U.ptr(q), U.ptr(s), K, N, U.stream())
            U.call("hexlib_b200_matmul_epilogue_e4m3", U.ptr(a[0]), U.ptr(a[1]), U.ptr(q), U.ptr(s), None, U.ptr(y), M, K, N,
                   0, U.stream())
        for i, y in enumerate(ys):
            ref, bound = B.product(a[2], B.values(*B.quantize(np.ascontiguousarray(ws[i % 2].T))), None, None, 0)
            B.assert_within(U.host(y), ref, bound, f"call {i}")


@pytest.mark.parametrize("M,K,N,in_place", [(2600, 300, 1001, False), (2600, 300, 1001, True), (9500, 130, 770, False),
                                            (9500, 130, 770, True), (2600, 300, 1032, True), (2600, 300, 259, False)])
def test_residual_from_any_element_reads_only_its_own(M, K, N, in_place):
    import torch
    rng = np.random.default_rng(M + N)
    a, w = operands(rng, M, K, N)
    resid = rng.standard_normal((M, N)).astype(np.float16)
    ref, bound = B.product(a[2], w[2], None, resid, 1)
    first = None
    for shift in (0, 1, 2, 3, 8):
        flat = torch.full((64 + shift + M * N + 64,), float("nan"), dtype=torch.float16, device="cuda")
        view = flat[64 + shift:64 + shift + M * N]
        view.copy_(U.dev(resid).reshape(-1))
        y = product(a, w, M, K, N, 1, None, view, out=view if in_place else None)
        y = U.host(y).reshape(M, N)
        if first is None:
            first = y
            B.assert_within(y, ref, bound, "aligned")
        assert np.array_equal(first, y), shift
        assert bool(flat[:64 + shift].isnan().all()) and bool(flat[64 + shift + M * N:].isnan().all())


def test_residual_and_output_larger_than_l2():
    M, K, N = 4750, 260, 6800
    rng = np.random.default_rng(5)
    a, w = operands(rng, M, K, N)
    r = U.dev(rng.standard_normal((M, N)).astype(np.float16))
    whole = product(a, w, M, K, N, 0, None, r)
    half = M // 2
    s = U.host(a[1]).reshape(-1, M, 4)
    for lo, hi in ((0, half), (half, M)):
        part = (a[0][lo:hi].contiguous(), U.dev(np.ascontiguousarray(s[:, lo:hi])), None)
        y = product(part, w, hi - lo, K, N, 0, None, r[lo:hi].contiguous())
        assert bool((y == whole[lo:hi]).all())
    ref, bound = B.product(a[2][-300:], w[2], None, U.host(r)[-300:], 0)
    B.assert_within(U.host(whole)[-300:], ref, bound, "last rows")
