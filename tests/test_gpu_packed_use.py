"""The operators of packed matrices and of experts as programs call them: captured and replayed, on two streams at once, beside a stream that is not current, with the same
workspace for two graphs, over matrices beyond 4 GiB, and one behind the other as the two products of an 8-bit layer."""
import ctypes as C

import pytest
import torch

import ffn_oracle as O
import packed_oracle as P
from test_gpu_ffn import DEV, Mat, TYPES, randn, stream
from test_gpu_grouped import offsets_of, pack, values
from zluda_amd import abi as K, cublaslt, ffn

pytestmark = pytest.mark.gpu
BF, VEC, BLK = TYPES["bf16"], K.CUBLASLT_MATMUL_MATRIX_SCALE_VEC128_32F, K.CUBLASLT_MATMUL_MATRIX_SCALE_BLK128x128_32F


class Layer:
    """rms -> packed -> product -> gated activation -> packed -> product, 8-bit weights, on the caller's stream"""

    def __init__(self, api, t, d, f, seed):
        self.t, self.d, self.f = t, d, f
        self.x, self.r = randn(seed, t, d).to(BF[0]), randn(seed + 1, t, d).to(BF[0])
        self.w, self.ws, self.sw = pack(2 * f, d, 128, seed + 2, d ** -0.5)
        self.v, self.vs, self.sv = pack(d, f, 128, seed + 3, f ** -0.5)
        self.s, self.z, self.y = (torch.empty((t, n), dtype=BF[0], device=DEV) for n in (d, 2 * f, d))
        self.n8, self.h8 = ffn.packed_buffers(t, d, DEV), ffn.packed_buffers(t, f, DEV)
        self.rms, self.act = ffn.RmsForward(dict(type=BF[1], rows=t, cols=d)), ffn.Activate(dict(type=BF[1], rows=t, cols=f, ldgate=2 * f, ldup=2 * f))
        base = dict(a_type=K.CUDA_R_8F_E4M3, b_type=K.CUDA_R_8F_E4M3, d_type=BF[1], compute_type=K.CUBLAS_COMPUTE_32F, scale_type=K.CUDA_R_32F, transa=1, a_scale_mode=BLK,
                    b_scale_mode=VEC)
        mm = lambda m, k, w, x: cublaslt.MatmulCall(api, dict(base, m=m, n=t, k=k, lda=w.ld, ldb=x[0].shape[1]), max_workspace=8 << 20)  # noqa: E731
        self.up, self.down = mm(2 * f, d, self.w, self.n8), mm(d, f, self.v, self.h8)
        self.up.set_pointers(a_scale=self.ws.ptr, b_scale=self.n8[1].data_ptr())
        self.down.set_pointers(a_scale=self.vs.ptr, b_scale=self.h8[1].data_ptr())
        self.scratch = torch.empty(8 << 20, dtype=torch.uint8, device=DEV)

    def run(self, stream, scratch=None):
        (nc, ns), (hc, hs), ws = self.n8, self.h8, (self.scratch if scratch is None else scratch)
        one, zero = C.c_float(1), C.c_float(0)
        self.rms.run(x=self.x.data_ptr(), residual=self.r.data_ptr(), sum=self.s.data_ptr(), codes=nc.data_ptr(), scales=ns.data_ptr(), stream=stream)
        assert self.up.run(one, self.w.ptr, nc.data_ptr(), zero, self.z.data_ptr(), self.z.data_ptr(), ws.data_ptr(), ws.numel(), stream) == 0
        self.act.run(gate=self.z.data_ptr(), up=self.z[:, self.f:].data_ptr(), codes=hc.data_ptr(), scales=hs.data_ptr(), stream=stream)
        assert self.down.run(one, self.v.ptr, hc.data_ptr(), zero, self.y.data_ptr(), self.y.data_ptr(), ws.data_ptr(), ws.numel(), stream) == 0

    def check(self, what=""):
        """every operator against 64 bits from what the one in front of it left"""
        h = (self.x.float() + self.r.float()).to(BF[0])
        assert torch.equal(self.s, h), what
        ref = P.rms_forward(h, None, 1e-5)
        P.check_packed(self.n8[0], self.n8[1].t(), *ref["y"], self.d, what=what + " n")
        codes = lambda c, n: c.view(torch.float8_e4m3fn).double()[:, :n]  # noqa: E731
        spread = lambda p, n: P.spread(p[1].t().double(), self.t, n)  # noqa: E731
        O.check(self.z, P.scaled_product(codes(self.n8[0], self.d), values(self.w), spread(self.n8, self.d), self.sw), what + " z")
        P.check_packed(self.h8[0], self.h8[1].t(), *P.activated("silu", self.z[:, :self.f], self.z[:, self.f:]), self.f, what=what + " h")
        O.check(self.y, P.scaled_product(codes(self.h8[0], self.f), values(self.v), spread(self.h8, self.f), self.sv), what + " y")

    def close(self):
        self.up.close()
        self.down.close()


@pytest.mark.parametrize("t,d,f", [(1, 2048, 1024), (3, 200, 264), (50, 1000, 1104), (300, 512, 704)])
def test_an_8_bit_layer(gpu_api, t, d, f):
    layer = Layer(gpu_api, t, d, f, 3)
    layer.run(stream())
    torch.cuda.synchronize()
    layer.check()
    layer.close()


def test_graphs_that_share_a_workspace(gpu_api):
    """two layers captured into graphs of their own with one workspace, replayed in turn, inputs changed and eager work between the replays"""
    layers = [Layer(gpu_api, 20, 2048, 512, 1), Layer(gpu_api, 200, 512, 1024, 9)]
    assert any(c.algo.data[2] for layer in layers for c in (layer.up, layer.down))       # (some of them split K)
    shared, side, graphs = torch.empty(8 << 20, dtype=torch.uint8, device=DEV), torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    for layer in layers:
        with torch.cuda.stream(side):
            layer.run(side.cuda_stream, shared)
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                layer.run(torch.cuda.current_stream().cuda_stream, shared)
        graphs.append(g)
    for i in range(4):
        for k, (layer, g) in enumerate(zip(layers, graphs)):
            layer.x.copy_(randn(100 + 10 * i + k, layer.t, layer.d))
            for m in (layer.z, layer.y, layer.s):
                m.zero_()
            g.replay()
        torch.cuda.synchronize()
        for layer in layers:
            layer.check("replay %d" % i)
        layers[i % 2].run(stream(), shared)
        torch.cuda.synchronize()
    for layer in layers:
        layer.close()


def test_two_streams_at_once(gpu_api):
    layers, streams = [Layer(gpu_api, 130, 512, 704, 1), Layer(gpu_api, 9, 2048, 1024, 9)], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for layer, s in zip(layers, streams):          # (neither is the current stream)
            layer.run(s.cuda_stream)
    torch.cuda.synchronize()
    for layer in layers:
        layer.check()
        layer.close()


def grouped_pass(counts, f, d, seed):
    o, dev = offsets_of(counts)
    e, rows = len(counts), o[-1]
    x, w, dy = randn(seed, rows, d).to(BF[0]), randn(seed + 1, e * f, d, std=d ** -0.5).to(BF[0]), randn(seed + 2, rows, f).to(BF[0])
    y, dx, dw = torch.empty_like(dy), torch.empty_like(x), torch.empty_like(w)
    spec = dict(type=BF[1], rows=rows, experts=e, features=f, model=d)
    fwd, bwd = ffn.GroupedForward(spec), ffn.GroupedBackward(spec)
    ws = torch.empty(max(16, bwd.workspace), dtype=torch.uint8, device=DEV)

    def run(stream):
        fwd.run(offsets=dev.data_ptr(), x=x.data_ptr(), w=w.data_ptr(), y=y.data_ptr(), stream=stream)
        bwd.run(offsets=dev.data_ptr(), dy=dy.data_ptr(), x=x.data_ptr(), w=w.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(), workspace=ws.data_ptr(), workspace_size=ws.numel(), stream=stream)

    def check(counts, what):
        at = 0
        for i, n in enumerate(counts):
            r, q, at = slice(at, at + n), slice(i * f, (i + 1) * f), at + n
            if n:
                O.check(y[r], P.product(x[r].double(), w[q].double()), what + " y")
                O.check(dx[r], P.product(dy[r].double(), w[q].double().t()), what + " dx")
            O.check(dw[q], P.product(dy[r].double().t(), x[r].double().t()), what + " dw")
    return run, check, dev, (y, dx, dw)


def test_counts_change_between_replays():
    """a captured pass over experts finds the rows that the offsets hold at its replay"""
    counts = [40, 0, 200, 13, 260]
    run, check, dev, outs = grouped_pass(counts, 264, 328, 5)
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(side.cuda_stream)
        side.synchronize()
        with torch.cuda.graph(g, stream=side):
            run(torch.cuda.current_stream().cuda_stream)
    for c in ([40, 0, 200, 13, 260], [0, 0, 513, 0, 0], [103, 102, 103, 102, 103], [513, 0, 0, 0, 0], [0, 1, 0, 0, 512]):
        dev.copy_(offsets_of(c)[1])
        for m in outs:
            m.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        check(c, str(c))


def test_the_same_bits_again():
    run, _, _, outs = grouped_pass([300, 5, 0, 900], 520, 640, 8)
    run(stream())
    first = [m.clone() for m in outs]
    for _ in range(3):
        run(stream())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, first))


def test_matrices_beyond_4_gib():
    """experts whose matrices, and rows whose offsets, lie past 2^32 bytes and elements"""
    f, d, e = 4096, 8192, 80                                # 5.4 GB of weights
    rows, ld = 2000, 1200000                                # x: 4.8 GB of pitch
    w = torch.zeros((e * f, d), dtype=BF[0], device=DEV)
    last = randn(2, f, d, std=d ** -0.5).to(BF[0])
    w[-f:] = last
    x = Mat(rows, d, BF[0], ld)
    tail = randn(3, 150, d).to(BF[0])
    x.view[-150:] = tail
    o = torch.zeros(e + 1, dtype=torch.int32, device=DEV)
    o[1:e] = rows - 150
    o[e] = rows
    y = torch.empty((rows, f), dtype=BF[0], device=DEV)
    ffn.GroupedForward(dict(type=BF[1], rows=rows, experts=e, features=f, model=d, ldx=ld)).run(offsets=o.data_ptr(), x=x.ptr, w=w.data_ptr(), y=y.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    O.check(y[-150:], P.product(tail.double(), last.double()), "y")
    dy = torch.zeros((rows, f), dtype=BF[0], device=DEV)
    dy[-150:] = randn(4, 150, f).to(BF[0])
    dx, dw = Mat(rows, d, BF[0], ld), torch.empty_like(w)
    bwd = ffn.GroupedBackward(dict(type=BF[1], rows=rows, experts=e, features=f, model=d, ldx=ld, lddx=ld))
    ws = torch.empty(max(16, bwd.workspace), dtype=torch.uint8, device=DEV)
    bwd.run(offsets=o.data_ptr(), dy=dy.data_ptr(), x=x.ptr, w=w.data_ptr(), dx=dx.ptr, dw=dw.data_ptr(), workspace=ws.data_ptr(), workspace_size=ws.numel(), stream=stream())
    torch.cuda.synchronize()
    O.check(dx.view[-150:], P.product(dy[-150:].double(), last.double().t()), "dx")
    O.check(dw[-f:], P.product(dy[-150:].double().t(), tail.double().t()), "dw")
    assert not dw[f:-f].any()


def test_codes_beyond_4_gib(gpu_api):
    """cublasLtMatmul over 8-bit tokens whose offsets pass 2^32"""
    m, n, k, ld = 200, 3000, 256, 1600000
    w, ws, sw = pack(m, k, 128, 1)
    raw = torch.empty(n * ld, dtype=torch.uint8, device=DEV).view(n, ld)
    x = randn(2, n, k).to(torch.float8_e4m3fn)
    raw[:, :k] = x.view(torch.uint8)
    xs = torch.rand((2, n), device=DEV) + 0.5
    y = torch.empty((n, m), dtype=BF[0], device=DEV)
    call = cublaslt.MatmulCall(gpu_api, dict(m=m, n=n, k=k, lda=w.ld, ldb=ld, a_type=K.CUDA_R_8F_E4M3, b_type=K.CUDA_R_8F_E4M3, d_type=BF[1], compute_type=K.CUBLAS_COMPUTE_32F,
                                             scale_type=K.CUDA_R_32F, transa=1, a_scale_mode=BLK, b_scale_mode=VEC))
    assert call.kernel == K.ZLUDA_KERNEL_MFMA_BLK8
    call.set_pointers(a_scale=ws.ptr, b_scale=xs.data_ptr())
    assert call.run(C.c_float(1), w.ptr, raw.data_ptr(), C.c_float(0), y.data_ptr(), y.data_ptr(), None, 0, stream()) == 0
    torch.cuda.synchronize()
    O.check(y, P.scaled_product(x.double(), values(w), P.spread(xs.t().double(), n, k), sw))
    call.close()


def test_gradients_on_two_streams_at_once():
    """two backward passes with shares of K, each with its own workspace, neither on the current stream"""
    passes, streams = [grouped_pass([30, 0, 40], 2816, 520, 3), grouped_pass([64], 4096, 1024, 4)], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(4):
        for (run, _, _, _), s in zip(passes, streams):
            run(s.cuda_stream)
    torch.cuda.synchronize()
    for (_, check, _, _), counts in zip(passes, ([30, 0, 40], [64])):
        check(counts, str(counts))
