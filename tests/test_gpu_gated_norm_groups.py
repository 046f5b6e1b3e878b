"""GPU: the gradient of the gated norm where a worker takes whole groups of rows that share a gate, eight and more of them, at each width class: groups of one row and of several, a last one
cut short, adding to what is there, the same bits twice; and adding above H = 8192 with several rows a workgroup.  Formulas and tolerances as in test_gpu_gated_norm, taken on the GPU in 64 bits."""
import ctypes

import pytest
import torch

from gpu_util import case, stream
from test_gpu_add_norm import EPS, STREAM, Out
from test_gpu_gated_norm import E4M3, Layer, check_backward, kept_scale

pytestmark = pytest.mark.gpu


class Grad:
    """The inputs of one call, on the device."""

    def __init__(self, dev, rows, H, f32, gate_rows, res=1.0, kept=False, seed=1):
        g = torch.Generator(device=dev).manual_seed(seed)
        rn = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
        a = self.a = Layer.__new__(Layer)
        a.rows, a.H, a.f32, a.gate_rows, a.res = rows, H, f32, gate_rows, res
        a.r, a.x = ((rn(rows, H) * torch.exp(rn(rows, 1))).to(t) for t in (STREAM[f32], torch.bfloat16))
        a.wp, a.w = ((1.0 + 0.3 * rn(H)).to(torch.bfloat16) for _ in range(2))
        a.gate = rn(-(-rows // gate_rows), H).to(torch.bfloat16) if gate_rows else None
        self.kept = kept
        self.rms, self.post_rms = ((t.double().square().mean(1) + EPS).sqrt().float() for t in (a.r, a.x))
        self.dy, self.dh = (1e-2 * rn(rows, H)).to(torch.bfloat16), (1e-2 * rn(rows, H)).to(STREAM[f32])
        self.h, self.x = a.r, a.x
        if kept:
            self.h, self.x = ((t.double() / p.double()[:, None] * kept_scale(H)).float().to(E4M3) for t, p in ((a.r, self.rms), (a.x, self.post_rms)))


def backward(cf, dev, g, out="both", qscale=2.0e5, start=None, accumulate=0):
    """Its outputs, on the device, with their surroundings looked at."""
    a = g.a
    rows, H = a.rows, a.H
    bits = lambda t: t.view(torch.uint8) if g.kept else t  # noqa: E731
    o = {"dr": Out(dev, (rows, H), a.r.dtype), "dx": Out(dev, (rows, H), torch.bfloat16), "q": Out(dev, (rows, H), torch.uint8), "dwp": Out(dev, (H,), torch.float32),
         "dw": Out(dev, (H,), torch.float32), "dgate": Out(dev, a.gate.shape if a.gate is not None else (1,), torch.float32)}
    for k, v in (start or {}).items():
        o[k].t.copy_(v)
    n = ctypes.c_size_t(0)
    cf.cf_gated_add_rmsnorm_backward_workspace_bytes(rows, H, a.gate_rows, ctypes.byref(n))
    ws = Out(dev, (n.value,), torch.uint8)
    qs, amax = torch.tensor([qscale], device=dev), torch.zeros(1, device=dev)
    call = cf.cf_gated_add_rmsnorm_backward_ckpt8 if g.kept else cf.cf_gated_add_rmsnorm_backward
    call(g.dy, bits(g.h), bits(g.x), a.f32, a.res, a.gate, a.gate_rows, a.wp, a.w, g.post_rms, g.rms, g.dh, rows, H, o["dr"].t, o["dx"].t if out != "e5m2" else None,
         o["q"].t if out != "bf16" else None, qs, amax, o["dwp"].t, o["dw"].t, o["dgate"].t, accumulate, ws.t, n.value, stream())
    torch.cuda.synchronize()
    assert all(v.unharmed() for v in o.values()) and ws.unharmed()
    return {**{k: v.t for k, v in o.items()}, "amax": float(amax), "out": out, "qscale": qscale}


def starts(dev, g):
    line = lambda a, b, n: torch.linspace(a, b, n, device=dev)  # noqa: E731
    gates = line(-1.0, 3.0, 1) if g.a.gate is None else line(-1.0, 3.0, g.a.gate.numel()).view(g.a.gate.shape)
    return {"dw": line(-1.0, 1.0, g.a.H), "dwp": line(2.0, -1.0, g.a.H), "dgate": gates}


def host(t):
    """The same on the host, where check_backward has the gates that are not there."""
    if isinstance(t, torch.Tensor):
        return t.cpu()
    if isinstance(t, dict):
        return {k: host(v) for k, v in t.items()}
    if isinstance(t, (Grad, Layer)):
        other = object.__new__(type(t))
        other.__dict__.update(host(t.__dict__))
        return other
    return t


# rows, H, rows a gate: at least eight groups a worker each, as the plan's test checks
SHAPES = [(16501, 96, 1), (33001, 96, 2), (33000, 511, 2), (8201, 520, 1), (16501, 1001, 2), (4101, 2056, 2), (4101, 4096, 2), (2101, 4096, 1), (6151, 4100, 3), (2101, 7168, 1),
          (4101, 8192, 2), (4101, 8200, 2), (2101, 12288, 1), (2101, 16384, 1)]


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("rows,H,gate_rows", SHAPES)
def test_many_groups(cf, dev, rows, H, gate_rows, f32, kept):
    case(f"gated norm gradient, many groups: rows={rows} H={H} gate_rows={gate_rows} f32={f32} kept={kept}")
    g = Grad(dev, rows, H, f32, gate_rows, -0.75, kept, rows + H)
    got = backward(cf, dev, g)
    check_backward(got, g)
    again = backward(cf, dev, g)
    assert all(torch.equal(got[k], again[k]) for k in ("dr", "dx", "q", "dw", "dwp", "dgate")) and got["amax"] == again["amax"]
    del again
    start = starts(dev, g)
    for accumulate in (1, 2, 3):
        check_backward(backward(cf, dev, g, "e5m2", start=start, accumulate=accumulate), g, start, accumulate)


# no gate, one, pieces of groups that several workers have, several groups a worker, a gate a row; up to 12288 and above
WIDE = [(300, 9216, 0), (300, 9216, 300), (700, 8200, 100), (600, 9001, 3), (2300, 8200, 1), (515, 12288, 2), (300, 12290, 0), (515, 13001, 515), (515, 13001, 250), (600, 16384, 3)]


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("rows,H,gate_rows", WIDE)
def test_wide_rows_accumulate(cf, dev, rows, H, gate_rows, f32, kept):
    case(f"gated norm gradient, adding: rows={rows} H={H} gate_rows={gate_rows} f32={f32} kept={kept}")
    g = Grad(dev, rows, H, f32, gate_rows, 1.25, kept, rows + H)
    start = starts(dev, g)
    for accumulate in (1, 2, 3):
        got = backward(cf, dev, g, start=start, accumulate=accumulate)
        if gate_rows:
            check_backward(got, g, start, accumulate)
        else:
            assert torch.equal(got["dgate"], start["dgate"])
            check_backward(host(got), host(g), host(start), accumulate)


def test_more_groups_than_an_int_times_sixteen(cf, dev):
    """A gate for each of 2^27 rows and a few: the last ones give what they give alone; the rest are zeros, so that the sums over rows are those rows' too."""
    rows, H, n = (1 << 27) + 5, 8, 700
    case(f"gated norm gradient rows={rows} H={H} gate_rows=1")
    g = Grad(dev, n, H, 0, 1, 1.25, True, 3)
    want = backward(cf, dev, g, "both")
    big = object.__new__(Grad)
    big.a = Layer.__new__(Layer)
    a, b = g.a, big.a
    at_the_end = lambda t, fill=0.0: torch.cat([torch.full((rows - n, *t.shape[1:]), fill, dtype=t.dtype, device=dev), t])  # noqa: E731
    bits = lambda t: at_the_end(t.view(torch.uint8)).view(E4M3)  # noqa: E731
    b.rows, b.H, b.f32, b.gate_rows, b.res, b.wp, b.w, b.gate, b.r = rows, H, 0, 1, 1.25, a.wp, a.w, at_the_end(a.gate), a.r
    big.kept, big.rms, big.post_rms, big.dy, big.dh, big.h, big.x = True, at_the_end(g.rms, 1.0), at_the_end(g.post_rms, 1.0), at_the_end(g.dy), at_the_end(g.dh), bits(g.h), bits(g.x)
    got = backward(cf, dev, big, "both")
    for k in ("dr", "dx", "q", "dgate"):
        assert torch.equal(got[k][rows - n:], want[k]) and not bool(got[k][:rows - n].any()), k
    assert got["amax"] == want["amax"]
    for k in ("dw", "dwp"):         # the same terms in other shares, each of which is rounded once, and so is the sum
        assert float((got[k].double() - want[k].double()).abs().max()) <= 2.0 ** -22 * n * float(want[k].abs().max())
