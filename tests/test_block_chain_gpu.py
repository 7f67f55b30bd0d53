"""A transformer block of the 8-bit operators around the library's attention, as a user
runs it: norm into 8 bits, q|k|v product, rotary positions in place, attention_qkv,
quantization, output product, edge (post-norm, gate, residual, the next norm in 8 bits),
MLP products, last edge. Every stage is held to its 64-bit form on the inputs it had,
then the whole run is captured, replayed and repeated on another stream."""
from __future__ import annotations

import numpy as np
import pytest

import block_ref as B
import gpu_util as U
from test_block_ops_cpu import table_of
from test_e4m3_gpu import u8
from tolerance import assert_close_f16

pytestmark = pytest.mark.gpu
EPS, D = 1e-6, 64


class Block:
    """Weights, workspaces and the calls of one block on images of T tokens."""

    def __init__(self, images, T, H, F, seed):
        rng = np.random.default_rng(seed)
        self.B, self.T, self.H, self.C, self.F = images, T, H, H * D, F
        C, M = self.C, images * T
        self.M = M
        n = rng.standard_normal
        f32 = lambda a: a.astype(np.float32)  # noqa: E731
        self.host = dict(
            x=n((M, C)).astype(np.float16), in_w=f32(1 + 0.1 * n(C)), post_w=f32(1 + 0.1 * n(C)),
            mid_w=f32(1 + 0.1 * n(C)), mid_b=f32(0.1 * n(C)), end_w=f32(1 + 0.1 * n(C)),
            gate=(0.5 * n((images, C))).astype(np.float16), qkv_b=f32(0.1 * n(3 * C)), up_b=f32(0.1 * n(F)),
            down_b=f32(0.1 * n(C)),
            qkv=(n((C, 3 * C)) / C ** 0.5).astype(np.float16), o=(n((C, C)) / C ** 0.5).astype(np.float16),
            up=(n((C, F)) / C ** 0.5).astype(np.float16), down=(n((F, C)) / F ** 0.5).astype(np.float16),
            pos=np.stack([np.arange(M) % T, np.arange(M) // 7 % 5, np.arange(M) % 7]).astype(np.int32),
            axis=(np.arange(D // 2) % 3).astype(np.int32))
        self.table, self.ms = table_of(1, D, 10000.0, 2.0)
        d = self.dev = {k: U.dev(v) for k, v in self.host.items()}
        d["table"] = U.dev(np.array(self.table, np.uint64).view(np.int64))
        self.w = {}
        for k in ("qkv", "o", "up", "down"):
            K, N = self.host[k].shape
            q, s = u8((N, B.pitch(K))), u8((B.groups(K), N, 4))
            U.call("hexlib_b200_quantize_weight_e4m3_fp16", U.ptr(d[k]), U.ptr(q), U.ptr(s), K, N, U.stream())
            self.w[k] = q, s
        f16 = lambda *s: U.empty(s, np.float16)  # noqa: E731
        form = lambda K: (u8((M, B.pitch(K))), u8((B.groups(K), M, 4)))  # noqa: E731
        self.b = dict(h1=form(C), qkv=f16(M, 3 * C), ctx=f16(M, C), ctx8=form(C), attn=f16(M, C), x1=f16(M, C), h2=form(C),
                      up=f16(M, F), up8=form(F), down=f16(M, C), x2=f16(M, C), h3=f16(M, C))

    def run(self, s):
        d, b, M, C, F = self.dev, self.b, self.M, self.C, self.F
        p = U.ptr
        mm = lambda a, w, bias, out, K, N, act: U.call(  # noqa: E731
            "hexlib_b200_matmul_epilogue_e4m3", p(a[0]), p(a[1]), p(self.w[w][0]), p(self.w[w][1]),
            None if bias is None else p(d[bias]), p(out), M, K, N, act, s)
        U.call("hexlib_b200_norm_gate_residual_e4m3", p(d["x"]), None, None, None, None, 0, 0, 1.0, 1.0, None, p(d["in_w"]),
               None, p(b["h1"][0]), p(b["h1"][1]), M, C, 0, EPS, s)
        mm(b["h1"], "qkv", "qkv_b", b["qkv"], C, 3 * C, 0)
        if getattr(self, "keep_raw", False):
            self.raw = U.host(b["qkv"]).copy()
        U.call("hexlib_b200_rope_pos_fp16", p(b["qkv"]), 3 * C, p(d["pos"]), 3, p(d["table"]), p(d["axis"]), self.ms,
               p(b["qkv"]), 3 * C, M, 2 * self.H, D, D, 0, s)
        U.call("hexlib_b200_attention_qkv_fp16", p(b["qkv"]), p(b["ctx"]), self.B, self.T, self.H, D, D ** -0.5, s)
        U.call("hexlib_b200_quantize_e4m3_fp16", p(b["ctx"]), p(b["ctx8"][0]), p(b["ctx8"][1]), M, C, s)
        mm(b["ctx8"], "o", None, b["attn"], C, C, 0)
        U.call("hexlib_b200_norm_gate_residual_e4m3", p(d["x"]), p(b["attn"]), p(d["post_w"]), None, p(d["gate"]), self.B, 1,
               1.0, 0.5, p(b["x1"]), p(d["mid_w"]), p(d["mid_b"]), p(b["h2"][0]), p(b["h2"][1]), M, C, 0, EPS, s)
        mm(b["h2"], "up", "up_b", b["up"], C, F, 1)
        U.call("hexlib_b200_quantize_e4m3_fp16", p(b["up"]), p(b["up8"][0]), p(b["up8"][1]), M, F, s)
        mm(b["up8"], "down", "down_b", b["down"], F, C, 0)
        U.call("hexlib_b200_norm_gate_residual_fp16", p(b["x1"]), p(b["down"]), None, None, None, 0, 0, 1.0, 1.0, p(b["x2"]),
               p(d["end_w"]), None, p(b["h3"]), M, C, 0, EPS, s)


def same_form(form, x):
    q, s = B.quantize(x)
    assert np.array_equal(U.host(form[1]), s) and B.same_codes(U.host(form[0]), q)


@pytest.mark.parametrize("images,T,H,F", [(1, 1, 2, 200), (3, 49, 4, 700), (2, 256, 12, 1536), (5, 130, 3, 264)])
def test_block(images, T, H, F):
    k = Block(images, T, H, F, images + T)
    k.keep_raw = True
    k.run(U.stream())
    k.keep_raw = False
    U.call("hexlib_b200_stream_status", U.stream())
    h, b, C, M = k.host, {n: v if isinstance(v, tuple) else U.host(v) for n, v in k.b.items()}, k.C, k.M
    val = lambda form: B.values(U.host(form[0]), U.host(form[1]))  # noqa: E731
    wv = {n: B.values(U.host(w[0]), U.host(w[1])) for n, w in k.w.items()}
    for n in wv:
        same_form(k.w[n], np.ascontiguousarray(h[n].T))
    # the first norm, whose fp16 h the 8-bit form holds to half a step of e4m3 at its scale
    ref, bound = B.edge_h(h["x"], h["in_w"], None, False, EPS)
    got = val(k.b["h1"])[:, :C]
    assert np.all(np.abs(got - ref) <= bound + (np.abs(ref) + bound) * 2.0 ** -4 + np.abs(ref).max() * 2.0 ** -17)

    def stage(out, a, w, bias, act, what):
        ref, bound = B.product(val(k.b[a]), wv[w], None if bias is None else h[bias], None, act)
        B.assert_within(out, ref, bound, what)
    stage(k.raw, "h1", "qkv", "qkv_b", 0, "q|k|v")
    ref, bound = B.rotary(k.raw, h["pos"], k.table, h["axis"], float(np.float32(k.ms)), 2 * H, D, D, 0)
    B.assert_within(b["qkv"][:, :2 * C], ref, bound, "rotary")
    assert np.array_equal(b["qkv"][:, 2 * C:], k.raw[:, 2 * C:])
    q, kk, v = (b["qkv"].reshape(images, T, 3, H, D)[:, :, i].astype(np.float64).transpose(0, 2, 1, 3) for i in range(3))
    sc = q @ kk.transpose(0, 1, 3, 2) * D ** -0.5
    pr = np.exp(sc - sc.max(-1, keepdims=True))
    ctx = (pr / pr.sum(-1, keepdims=True)) @ v
    assert_close_f16(b["ctx"], ctx.transpose(0, 2, 1, 3).reshape(M, C), what="attention")
    same_form(k.b["ctx8"], b["ctx"])
    stage(b["attn"], "ctx8", "o", None, 0, "output product")
    ref, bound = B.edge_x(h["x"], b["attn"], h["post_w"], None, h["gate"], 1, 1.0, 0.5, False, EPS)
    B.assert_within(b["x1"], ref, bound, "x1")
    ref, bound = B.edge_h(b["x1"], h["mid_w"], h["mid_b"], False, EPS)
    got = val(k.b["h2"])[:, :C]
    assert np.all(np.abs(got - ref) <= bound + (np.abs(ref) + bound) * 2.0 ** -4 + np.abs(ref).max() * 2.0 ** -17)
    stage(b["up"], "h2", "up", "up_b", 1, "up")
    same_form(k.b["up8"], b["up"])
    stage(b["down"], "up8", "down", "down_b", 0, "down")
    ref, bound = B.edge_x(b["x1"], b["down"], None, None, None, 0, 1.0, 1.0, False, EPS)
    B.assert_within(b["x2"], ref, bound, "x2")
    ref, bound = B.edge_h(b["x2"], h["end_w"], None, False, EPS)
    B.assert_within(b["h3"], ref, bound, "h3")


def test_block_captured_replayed_and_on_another_stream():
    import torch
    k = Block(2, 196, 12, 1000, 7)
    k.run(U.stream())
    want = {n: U.host(k.b[n]).copy() for n in ("x1", "x2", "h3")}
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        k.run(U.stream())
    other = torch.cuda.Stream()
    for again in range(3):
        for n in want:
            k.b[n].zero_()
        torch.cuda.synchronize()
        if again == 2:
            k.run(other.cuda_stream)
        else:
            graph.replay()
        torch.cuda.synchronize()
        for n, v in want.items():
            assert np.array_equal(v, U.host(k.b[n])), n
    U.call("hexlib_b200_stream_status", U.stream())


def test_two_blocks_on_two_streams_at_once():
    import torch
    ks = [Block(2, 100 + 60 * i, 4, 520, 20 + i) for i in range(2)]
    want = []
    for k in ks:
        k.run(U.stream())
        want.append(U.host(k.b["h3"]).copy())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ks]
    for _ in range(20):
        for k, s in zip(ks, streams):
            k.run(s.cuda_stream)
    torch.cuda.synchronize()
    for k, w in zip(ks, want):
        assert np.array_equal(U.host(k.b["h3"]), w)
