"""GPU: the residual layer's entry points in a run, as a training step makes it: addition + norm + quantize, the experts' block-scaled product on the
bytes, a dense layer's FP8 products both ways, the norm's gradient with the bytes for the next product, and the clipping of what the weight gradients
wrote.  Every stage against the 64-bit formula on what the stage before it wrote; then captured into a graph and replayed on other inputs."""
import ctypes

import pytest
import torch

from gpu_util import case, stream
from test_gpu_add_norm import check_backward, check_forward
from test_gpu_grads import reference_norm, table

pytestmark = pytest.mark.gpu

EPS = 1e-6
ROW_COL, BLOCK, NONE = 1, 2, 0


def sized(fn, dev, *args):
    n = ctypes.c_size_t(0)
    fn(*args, ctypes.byref(n))
    return torch.empty(max(n.value, 16), dtype=torch.uint8, device=dev), n.value


class Layer:
    """y = W q(norm(r + x)) over all tokens, and the experts' products over the routed ones; backward through the dense layer and the norm."""

    def __init__(self, cf, dev, T, H, N, E, top, f32, seed):
        self.cf, self.dev, self.T, self.H, self.N, self.E, self.top, self.f32 = cf, dev, T, H, N, E, top, f32
        g = torch.Generator(device=dev).manual_seed(seed)
        rn = lambda *s: torch.randn(*s, device=dev, generator=g)
        self.st = torch.float32 if f32 else torch.bfloat16
        self.r, self.x, self.gamma = rn(T, H).to(self.st), rn(T, H).to(torch.bfloat16), (1 + 0.1 * rn(H)).to(torch.bfloat16)
        self.dy, self.dh = (1e-2 * rn(T, N)).to(torch.bfloat16), (1e-2 * rn(T, H)).to(self.st)
        u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=dev)
        f = lambda *s: torch.zeros(*s, device=dev)
        b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=dev)
        # dense weights: forward [N, H], backward [H, N]; experts' [E, N, H] with block scales
        w = (0.02 * rn(N, H)).to(torch.bfloat16)
        self.amax_w, self.ws, self.wd, self.fwd8, self.bwd8 = f(1), f(1), f(1), u8(N, H), u8(H, N)
        cf.cf_fp8_refresh_weight(w, self.fwd8, self.bwd8, self.amax_w, self.ws, self.wd, H, N, 1, 1, stream())
        we = (0.02 * rn(E * N, H)).to(torch.bfloat16)
        self.we, es, self.wed = u8(E * N, H), f(E * N // 128, H // 128), f(E * N // 128, H // 128)
        cf.cf_fp8_quantize_block_128x128(we, E * N, H, self.we, es, self.wed, stream())
        self.wd_rows = self.wd.expand(N).contiguous()
        # routing
        scores = torch.softmax(rn(T, E), 1)
        chosen = torch.topk(scores, top, 1).indices.flatten()
        order = torch.sort(chosen, stable=True).indices
        self.index = (order // top).to(torch.int32)
        self.counts = torch.bincount(chosen, minlength=E).to(torch.int32)
        self.offsets = (torch.cumsum(self.counts, 0) - self.counts).to(torch.int32)
        # outputs
        self.h, self.rms, self.normed = torch.zeros_like(self.r), f(T), b(T, H)
        self.q, self.qs, self.qd = u8(T, H), f(T), f(T)
        self.h2, self.qb, self.qbs, self.qbd = torch.zeros_like(self.r), u8(T, H), f(T, H // 128), f(T, H // 128)
        self.y, self.ye = b(T, N), b(T * top, N)
        self.dyq, self.dys, self.dyd, self.damax = u8(T, N), f(1), f(1), f(1)
        self.dn, self.dr, self.dgamma = b(T, H), torch.zeros_like(self.r), f(H)
        self.g8, self.g8s, self.g8amax = u8(T, H), torch.full((1,), 1e5, device=dev), f(1)
        self.dw = f(N, H)
        self.norm, self.coef = f(1), f(1)
        self.grads, self.clipped = [self.dw, self.dgamma], [torch.zeros_like(self.dw), torch.zeros_like(self.dgamma)]
        self.list, self.list_bytes = table(cf, dev, self.grads, self.clipped)
        self.gws, self.gws_bytes = sized(cf.cf_fp8_grouped_gemm_workspace_bytes, dev, T * top, E)
        self.bws, self.bws_bytes = sized(cf.cf_add_rmsnorm_backward_workspace_bytes, dev, T, H)
        self.nws, self.nws_bytes = sized(cf.cf_grad_norm_workspace_bytes, dev)

    def step(self, st):
        cf, T, H, N, E, R = self.cf, self.T, self.H, self.N, self.E, self.T * self.top
        cf.cf_add_rmsnorm_quantize_rows(self.r, self.x, self.f32, self.gamma, T, H, EPS, 0, self.h, self.normed, self.rms, self.q, self.qs, self.qd, st)
        cf.cf_fp8_gemm_nt_bf16_ex(T, N, H, self.q, H, 0, self.qd, self.fwd8, H, self.wd_rows, ROW_COL, NONE, None, None, None, self.y, N, 0, st)
        cf.cf_add_rmsnorm_quantize_block_1x128(self.r, self.x, self.f32, self.gamma, T, H, EPS, self.h2, None, None, self.qb, self.qbs, self.qbd, st)
        cf.cf_fp8_grouped_gemm_nt_bf16_ex(R, N, H, E, self.counts, self.offsets, self.qb, T, H, self.index, self.qbd, self.we, self.wed, BLOCK, NONE,
                                          None, None, self.ye, N, self.gws, self.gws_bytes, st)
        cf.cf_fp8_amax_bf16(self.dy, T * N, self.damax, st)
        cf.cf_fp8_scale_from_amax(self.damax, 57344.0, self.dys, self.dyd, st)
        cf.cf_fp8_quantize_e5m2(self.dy, self.dyq, self.dys, T * N, st)
        cf.cf_fp8_gemm_nt_bf16(T, H, N, self.dyq, N, 1, self.dyd, self.bwd8, self.wd, self.dn, H, st)
        self.dw.zero_()
        self.g8amax.zero_()
        cf.cf_gemm_bf16_tn_accum_f32(N, H, T, self.dy, N, self.normed, H, self.dw, H, st)
        cf.cf_add_rmsnorm_backward_quant_e5m2(self.dn, self.h, self.f32, self.gamma, self.rms, self.dh, T, H, self.dr, self.dgamma, 0, self.g8,
                                              self.g8s, self.g8amax, self.bws, self.bws_bytes, st)
        cf.cf_grad_norm_clip(self.list, self.list_bytes, 0.5, self.norm, self.coef, self.nws, self.nws_bytes, st)

    def outputs(self):
        return {k: getattr(self, k) for k in ("h", "rms", "normed", "q", "qd", "y", "h2", "qb", "qbd", "ye", "dn", "dr", "dgamma", "g8", "g8amax", "dw", "norm", "coef")} | \
            {"clipped0": self.clipped[0], "clipped1": self.clipped[1]}

    def check(self):
        c = lambda t: t.cpu()
        r, x, w = c(self.r), c(self.x), c(self.gamma)
        check_forward({"sum": c(self.h), "rms": c(self.rms), "normed": c(self.normed), "q": c(self.q), "scale": c(self.qs), "descale": c(self.qd)}, r, x, w, "rows", 0)
        check_forward({"sum": c(self.h2), "rms": c(self.rms), "normed": None, "q": c(self.qb), "scale": c(self.qbs), "descale": c(self.qbd)}, r, x, w, "block", 0)
        check_backward({"dr": c(self.dr), "dw": c(self.dgamma), "q": c(self.g8), "amax": float(self.g8amax)}, c(self.h), w, c(self.rms), c(self.dn), c(self.dh), True, 1e5)
        # the products: bf16 rounding 2^-8 and what the matrix cores cut (2^-15 of the sum of sizes, as the other products' tests have it)
        f8 = lambda t, k: t.view(k).double()
        a, wt = f8(self.q, torch.float8_e4m3fn) * self.qd.double()[:, None], f8(self.fwd8, torch.float8_e4m3fn) * self.wd.double()
        self.near(self.y, a, wt)
        ab = (f8(self.qb, torch.float8_e4m3fn).unflatten(1, (-1, 128)) * self.qbd.double()[:, :, None]).flatten(1)
        spread = self.wed.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
        web = (f8(self.we, torch.float8_e4m3fn) * spread).view(self.E, self.N, self.H)
        for e, (n, o) in enumerate(zip(self.counts.tolist(), self.offsets.tolist())):
            self.near(self.ye[o:o + n], ab[self.index[o:o + n].long()], web[e])
        norm = reference_norm([self.dw, self.dgamma])
        assert abs(float(self.norm) - norm) <= (2.0 ** -24 + 1e-11) * norm
        assert float(self.coef) < 1.0
        for g, out in zip(self.grads, self.clipped):
            assert torch.equal(g * self.coef, out)

    @staticmethod
    def near(got, a, b):
        ref, size = a.mm(b.t().contiguous()), a.abs().mm(b.abs().t().contiguous())
        assert bool(((got.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -15 * size).all())


@pytest.mark.parametrize("T,H,N,E,top,f32", [(1, 512, 256, 4, 2, 0), (37, 1024, 384, 8, 2, 1), (300, 2048, 1408, 16, 4, 0), (1000, 512, 512, 6, 2, 1)])
def test_a_step(cf, dev, T, H, N, E, top, f32):
    case(f"residual layer step {T} x {H} -> {N}, {E} experts, f32={f32}")
    layer = Layer(cf, dev, T, H, N, E, top, f32, T)
    layer.step(stream())
    torch.cuda.synchronize()
    layer.check()


def test_a_captured_step_replayed_on_other_inputs(cf, dev):
    case("residual layer step in a graph")
    layer = Layer(cf, dev, 260, 1024, 512, 8, 2, 0, 3)
    other = [Layer(cf, dev, 260, 1024, 512, 8, 2, 0, s) for s in (4, 5, 6)]
    layer.step(stream())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        layer.step(side.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        layer.step(torch.cuda.current_stream().cuda_stream)
    for o in other + other[::-1]:
        o.step(stream())                        # the program's own eager work between the replays
        want = {k: v.clone() for k, v in o.outputs().items()}
        for k in ("r", "x", "gamma", "dy", "dh", "fwd8", "bwd8", "wd", "wd_rows", "we", "wed", "index", "counts", "offsets"):
            getattr(layer, k).copy_(getattr(o, k))
        graph.replay()
        torch.cuda.synchronize()
        for k, v in layer.outputs().items():
            assert torch.equal(v.view(torch.uint8) if v.dim() else v, want[k].view(torch.uint8) if v.dim() else want[k]), k


def test_two_streams_at_once(cf, dev):
    """Two steps side by side, each with its own workspaces, give what they give one after the other."""
    case("residual layer steps on two streams")
    a, b = Layer(cf, dev, 200, 1024, 384, 8, 2, 1, 7), Layer(cf, dev, 333, 512, 256, 4, 2, 0, 8)
    for layer in (a, b):
        layer.step(stream())
    torch.cuda.synchronize()
    want = [{k: v.clone() for k, v in layer.outputs().items()} for layer in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, layer in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                layer.step(s.cuda_stream)
    torch.cuda.synchronize()
    for layer, w in zip((a, b), want):
        assert all(torch.equal(v, w[k]) for k, v in layer.outputs().items() if v.dtype != torch.bfloat16 or not torch.isnan(v).any())
