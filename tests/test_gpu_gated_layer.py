"""GPU: a training step of a gated-MLP layer with a norm on both sides of its block, through the entry points that stand between its FP8 products: gate + addition + norm + quantize,
the product up, the activation kept in 8 bits, the product down, the next norm; and back, from the 8-bit checkpoints, with both weight gradients.  Every stage against the 64-bit
formula on what the stage before it wrote; then captured into a graph and replayed on other inputs, and on two streams."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

import test_gpu_gated_norm as gn
import test_gpu_swiglu_ckpt as sw
from gpu_util import case, stream

pytestmark = pytest.mark.gpu

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
INPUTS = ("r", "x0", "gate0", "gate1", "wp0", "w0", "wp1", "w1", "dy", "fwd_gu", "bwd_gu", "d_gu", "fwd_d", "bwd_d", "d_d")


class Step:
    def __init__(self, cf, dev, T, H, I, gate_rows, f32, seed):
        self.cf, self.dev, self.T, self.H, self.I, self.gate_rows, self.f32 = cf, dev, T, H, I, gate_rows, f32
        g = torch.Generator(device=dev).manual_seed(seed)
        rn = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
        bf = torch.bfloat16
        self.st = torch.float32 if f32 else bf
        self.r, self.x0 = rn(T, H).to(self.st), rn(T, H).to(bf)
        groups = -(-T // gate_rows)
        self.gate0, self.gate1 = ((0.5 + 0.3 * rn(groups, H)).to(bf) for _ in range(2))
        self.wp0, self.w0, self.wp1, self.w1 = ((1 + 0.1 * rn(H)).to(bf) for _ in range(4))
        self.dy = (1e-2 * rn(T, H)).to(bf)
        u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=dev)  # noqa: E731
        f = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
        b = lambda *s: torch.zeros(*s, dtype=bf, device=dev)  # noqa: E731
        one = lambda v: torch.full((1,), v, device=dev)  # noqa: E731
        # weights: up and gate side by side [2 I, H], down [H, I]; each as rows for the forward and the backward product
        self.fwd_gu, self.bwd_gu, self.d_gu = u8(2 * I, H), u8(H, 2 * I), f(1)
        self.fwd_d, self.bwd_d, self.d_d = u8(H, I), u8(I, H), f(1)
        for w, fwd, bwd, d, i, o in ((0.05 * rn(2 * I, H), self.fwd_gu, self.bwd_gu, self.d_gu, H, 2 * I), (0.05 * rn(H, I), self.fwd_d, self.bwd_d, self.d_d, I, H)):
            cf.cf_fp8_refresh_weight(w.to(bf), fwd, bwd, f(1), f(1), d, i, o, 1, 1, stream())
        # scales that earlier steps left, and their inverses
        self.s_q0, self.d_q0, self.s_a, self.d_a = one(40.0), one(1 / 40.0), one(8.0), one(1 / 8.0)
        self.s_dx, self.d_dx, self.s_gu, self.dd_gu = one(2.0 ** 17), one(2.0 ** -17), one(2.0 ** 17), one(2.0 ** -17)
        like = lambda: torch.zeros_like(self.r)  # noqa: E731
        self.h0, self.prms0, self.rms0, self.x8_0, self.h8_0, self.q0, self.amax_q0 = like(), f(T), f(T), u8(T, H), u8(T, H), u8(T, H), f(1)
        self.gu, gr = b(T, 2 * I), (T, (I + 127) // 128)
        self.g8, self.gd, self.u8, self.ud, self.a8, self.amax_a = u8(T, I), f(*gr), u8(T, I), f(*gr), u8(T, I), f(1)
        self.x1 = b(T, H)
        self.h1, self.normed, self.prms1, self.rms1, self.x8_1, self.h8_1 = like(), b(T, H), f(T), f(T), u8(T, H), u8(T, H)
        self.q1, self.s_q1, self.d_q1 = u8(T, H), f(T), f(T)
        self.dr1, self.dx1, self.dx8, self.dx8_t, self.amax_dx = like(), b(T, H), u8(T, H), u8(H, T), f(1)
        self.dwp1, self.dw1, self.dgate1 = f(H), f(H), f(groups, H)
        self.da, self.grad8, self.grad8_t, self.act8_t, self.amax_gu = b(T, I), u8(T, 2 * I), u8(2 * I, T), u8(I, T), f(1)
        self.q0_t, self.dn = u8(H, T), b(T, H)
        self.dWd, self.dWgu = f(I, H), f(H, 2 * I)
        self.dr, self.dx0, self.dwp0, self.dw0, self.dgate0 = like(), b(T, H), f(H), f(H), f(groups, H)
        n = ctypes.c_size_t(0)
        cf.cf_gated_add_rmsnorm_backward_workspace_bytes(T, H, gate_rows, ctypes.byref(n))
        self.ws, self.ws_bytes = u8(max(n.value, 16)), n.value

    def step(self, st):
        cf, T, H, I, G, f32 = self.cf, self.T, self.H, self.I, self.gate_rows, self.f32
        for t in (self.amax_q0, self.amax_a, self.amax_dx, self.amax_gu, self.dWd, self.dWgu):
            t.zero_()
        cf.cf_gated_add_rmsnorm_quantize_record(self.r, self.x0, f32, 1.25, self.gate0, G, self.wp0, self.w0, T, H, gn.EPS, 0, self.h0, None, self.prms0, self.rms0,
                                                self.x8_0, self.h8_0, self.q0, self.s_q0, self.amax_q0, st)
        cf.cf_fp8_gemm_nt_bf16(T, 2 * I, H, self.q0, H, 0, self.d_q0, self.fwd_gu, self.d_gu, self.gu, 2 * I, st)
        cf.cf_swiglu_ckpt8_quantize_record(self.gu, self.gu[:, I:], 2 * I, T, I, 0, self.g8, self.gd, self.u8, self.ud, self.a8, self.s_a, self.amax_a, st)
        cf.cf_fp8_gemm_nt_bf16(T, H, I, self.a8, I, 0, self.d_a, self.fwd_d, self.d_d, self.x1, H, st)
        cf.cf_gated_add_rmsnorm_quantize_rows(self.h0, self.x1, f32, 1.0, self.gate1, G, self.wp1, self.w1, T, H, gn.EPS, 0, self.h1, self.normed, self.prms1,
                                              self.rms1, self.x8_1, self.h8_1, self.q1, self.s_q1, self.d_q1, st)
        cf.cf_gated_add_rmsnorm_backward_ckpt8(self.dy, self.h8_1, self.x8_1, f32, 1.0, self.gate1, G, self.wp1, self.w1, self.prms1, self.rms1, None, T, H,
                                               self.dr1, self.dx1, self.dx8, self.s_dx, self.amax_dx, self.dwp1, self.dw1, self.dgate1, 0, self.ws, self.ws_bytes, st)
        cf.cf_fp8_gemm_nt_bf16(T, I, H, self.dx8, H, 1, self.d_dx, self.bwd_d, self.d_d, self.da, I, st)
        cf.cf_swiglu_ckpt8_backward_quant_e5m2(self.da, self.g8, self.gd, self.u8, self.ud, T, I, self.grad8, self.grad8_t, self.s_gu, self.amax_gu, self.act8_t,
                                               self.s_a, st)
        cf.cf_transpose_u8(self.dx8, self.dx8_t, T, H, st)
        cf.cf_transpose_u8(self.q0, self.q0_t, T, H, st)
        cf.cf_fp8_gemm_tn_accum_f32(I, H, T, self.act8_t, self.d_a, self.dx8_t, self.d_dx, self.dWd, H, st)
        cf.cf_fp8_gemm_tn_accum_f32(H, 2 * I, T, self.q0_t, self.d_q0, self.grad8_t, self.dd_gu, self.dWgu, 2 * I, st)
        cf.cf_fp8_gemm_nt_bf16(T, H, 2 * I, self.grad8, 2 * I, 1, self.dd_gu, self.bwd_gu, self.d_gu, self.dn, H, st)
        cf.cf_gated_add_rmsnorm_backward(self.dn, self.h0, self.x0, f32, 1.25, self.gate0, G, self.wp0, self.w0, self.prms0, self.rms0, self.dr1, T, H, self.dr,
                                         self.dx0, None, None, None, self.dwp0, self.dw0, self.dgate0, 0, self.ws, self.ws_bytes, st)

    def outputs(self):
        return {k: getattr(self, k) for k in ("h0", "prms0", "rms0", "x8_0", "h8_0", "q0", "amax_q0", "gu", "g8", "gd", "u8", "ud", "a8", "amax_a", "x1", "h1", "normed", "q1", "s_q1",
                                              "dr1", "dx1", "dx8", "amax_dx", "dwp1", "dw1", "dgate1", "da", "grad8", "grad8_t", "act8_t", "amax_gu", "dWd", "dWgu", "dn", "dr",
                                              "dx0", "dwp0", "dw0", "dgate0")}

    def norm_inputs(self, r, x, res, wp, w, gate):
        return SimpleNamespace(rows=self.T, H=self.H, f32=self.f32, gate_rows=self.gate_rows, res=res, r=r.cpu(), x=x.cpu(), wp=wp.cpu(), w=w.cpu(), gate=gate.cpu())

    def check(self):
        c = lambda t: t.cpu()  # noqa: E731
        a0 = self.norm_inputs(self.r, self.x0, 1.25, self.wp0, self.w0, self.gate0)
        a1 = self.norm_inputs(self.h0, self.x1, 1.0, self.wp1, self.w1, self.gate1)
        got = {"sum": c(self.h0), "post_rms": c(self.prms0), "rms": c(self.rms0), "x8": c(self.x8_0), "sum8": c(self.h8_0), "q": c(self.q0), "amax": max(0.125, float(self.amax_q0))}
        h = c(self.h0).double()
        y = h / (h.square().mean(1, keepdim=True) + gn.EPS).sqrt() * a0.w.double()
        gn.check_forward({**got, "normed": y.to(torch.bfloat16)}, a0, "record", 0, float(self.s_q0))
        gn.check_forward({"sum": c(self.h1), "normed": c(self.normed), "post_rms": c(self.prms1), "rms": c(self.rms1), "x8": c(self.x8_1), "sum8": c(self.h8_1), "q": c(self.q1),
                          "scale": c(self.s_q1), "descale": c(self.d_q1)}, a1, "rows", 0)
        I = self.I
        sw.check_forward({"gate8": c(self.g8), "gate8_descale": c(self.gd), "up8": c(self.u8), "up8_descale": c(self.ud), "q": c(self.a8), "amax": max(0.125, float(self.amax_a))},
                         c(self.gu)[:, :I], c(self.gu)[:, I:], "record", 0, float(self.s_a))
        back1 = SimpleNamespace(a=a1, kept=True, rms=c(self.rms1), post_rms=c(self.prms1), dy=c(self.dy), dh=None, h=c(self.h8_1).view(E4M3), x=c(self.x8_1).view(E4M3))
        gn.check_backward({"dr": c(self.dr1), "dx": c(self.dx1), "q": c(self.dx8), "amax": float(self.amax_dx), "out": "both", "qscale": float(self.s_dx), "dwp": c(self.dwp1),
                           "dw": c(self.dw1), "dgate": c(self.dgate1)}, back1)
        back0 = SimpleNamespace(a=a0, kept=False, rms=c(self.rms0), post_rms=c(self.prms0), dy=c(self.dn), dh=c(self.dr1), h=c(self.h0), x=c(self.x0))
        gn.check_backward({"dr": c(self.dr), "dx": c(self.dx0), "out": "bf16", "dwp": c(self.dwp0), "dw": c(self.dw0), "dgate": c(self.dgate0)}, back0)
        glu = sw.Grad.__new__(sw.Grad)
        glu.g8, glu.gd, glu.u8, glu.ud, glu.do = c(self.g8).view(E4M3), c(self.gd), c(self.u8).view(E4M3), c(self.ud), c(self.da)
        sw.check_backward8(([c(self.grad8), c(self.grad8_t), c(self.act8_t)], float(self.amax_gu)), glu, True, float(self.s_gu), float(self.s_a))
        # the products, by the library's own bar for them: 1e-3 of relative L2, and for bf16 the rounding, 2^-8.  An element's own bound would be a multiple of its largest product, to
        # which the matrix cores align the others: with these inputs that is 2/3 of the sum of sizes for some
        v = lambda t, k, d: t.view(k).double() * d.double()  # noqa: E731
        self.near(self.gu, v(self.q0, E4M3, self.d_q0), v(self.fwd_gu, E4M3, self.d_gu), 2.0 ** -8)
        self.near(self.x1, v(self.a8, E4M3, self.d_a), v(self.fwd_d, E4M3, self.d_d), 2.0 ** -8)
        self.near(self.da, v(self.dx8, E5M2, self.d_dx), v(self.bwd_d, E4M3, self.d_d), 2.0 ** -8)
        self.near(self.dn, v(self.grad8, E5M2, self.dd_gu), v(self.bwd_gu, E4M3, self.d_gu), 2.0 ** -8)
        self.near(self.dWd, v(self.act8_t, E4M3, self.d_a), v(self.dx8_t, E5M2, self.d_dx), 0.0)
        self.near(self.dWgu, v(self.q0_t, E4M3, self.d_q0), v(self.grad8_t, E5M2, self.dd_gu), 0.0)

    @staticmethod
    def near(got, a, b, rounding):
        ref = a.mm(b.t().contiguous())
        assert float((got.double() - ref).norm()) <= (1e-3 + rounding) * float(ref.norm())


@pytest.mark.parametrize("T,H,I,gate_rows,f32", [(1, 512, 1024, 1, 0), (48, 512, 704, 48, 1), (300, 1024, 1408, 100, 0), (256, 2048, 2048, 1, 1), (77, 640, 1000, 30, 0)])
def test_a_step(cf, dev, T, H, I, gate_rows, f32):
    case(f"gated layer step {T} x {H} x {I}, gate_rows={gate_rows} f32={f32}")
    s = Step(cf, dev, T, H, I, gate_rows, f32, T)
    s.step(stream())
    torch.cuda.synchronize()
    s.check()


def test_a_captured_step_replayed_on_other_inputs(cf, dev):
    case("gated layer step in a graph")
    make = lambda seed: Step(cf, dev, 272, 1024, 1024, 100, 0, seed)  # noqa: E731
    s, other = make(3), [make(k) for k in (4, 5, 6)]
    s.step(stream())
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        s.step(side.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        s.step(torch.cuda.current_stream().cuda_stream)
    for o in other + other[::-1]:
        o.step(stream())                        # the program's own eager work between the replays
        want = {k: v.clone() for k, v in o.outputs().items()}
        for k in INPUTS:
            getattr(s, k).copy_(getattr(o, k))
        graph.replay()
        torch.cuda.synchronize()
        for k, v in s.outputs().items():
            assert torch.equal(v.view(torch.uint8), want[k].view(torch.uint8)), k


def test_two_streams_at_once(cf, dev):
    """Two steps side by side, each with its own workspace, give what they give one after the other."""
    case("gated layer steps on two streams")
    a, b = Step(cf, dev, 200, 1024, 704, 1, 1, 7), Step(cf, dev, 333, 512, 1000, 111, 0, 8)
    for s in (a, b):
        s.step(stream())
    torch.cuda.synchronize()
    want = [{k: v.clone() for k, v in s.outputs().items()} for s in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for t, s in zip(streams, (a, b)):
            with torch.cuda.stream(t):
                s.step(t.cuda_stream)
    torch.cuda.synchronize()
    for s, w in zip((a, b), want):
        for k, v in s.outputs().items():
            assert torch.equal(v.view(torch.uint8), w[k].view(torch.uint8)), k
