"""GPU: a block's output normed, gated and added to the scaled stream, the next norm and its 8-bit output, and the gradient, against the formulas in 64 bits.

Tolerances.  u = 2^-24.  A row's sum of squares adds at most H / 64 terms per thread and then at most 10 more across threads: relative error below
(H / 64 + 10) u <= 266 u for H = 16384; the root halves it, and the divisions, the root and the products add a few u: R = 150 u bounds the relative error of both rms and of
what is divided by them.  h adds a product and an fma to that.  What follows h is compared with the formulas of h as it was stored.  On top comes the rounding to the output's
type: bf16 2^-8, E4M3 2^-4 or half of its smallest step, E5M2 2^-3 or half of its."""
import ctypes

import pytest
import torch

from gpu_util import case, stream
from test_gpu_add_norm import EPS, F8, R, STREAM, U, Out, gamma_of, rows_of, shifted

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def kept_scale(H):
    return max(2.0 ** e for e in range(9) if 4.0 ** e * H <= 448.0 ** 2)


def gate_of(rows, H, gate_rows, seed):
    """[groups, H] gates of any sign, some of them zero; None without a gate."""
    if not gate_rows:
        return None
    g = torch.randn(-(-rows // gate_rows), H, generator=torch.Generator().manual_seed(seed))
    g[:, ::11] = 0.0
    return g.to(torch.bfloat16)


def gates(gate, gate_rows, rows):
    return gate.double().repeat_interleave(gate_rows, 0)[:rows] if gate is not None else torch.ones(1, 1, dtype=torch.float64)


def put(t, dev, shift):
    return shifted(t, dev, shift)[0] if t is not None else None


class Layer:
    """The inputs of one call."""

    def __init__(self, rows, H, f32, gate_rows, res=1.0, seed=1):
        self.rows, self.H, self.f32, self.gate_rows, self.res = rows, H, f32, gate_rows, res
        self.r, self.x = rows_of(rows, H, seed, STREAM[f32]), rows_of(rows, H, seed + 1, torch.bfloat16, 0.7)
        self.wp, self.w, self.gate = gamma_of(H, seed + 2), gamma_of(H, seed + 3), gate_of(rows, H, gate_rows, seed + 4)


def forward(cf, dev, a, form="rows", e5m2=0, shift=0, in_place=False, kept=True, wanted=True, qscale=12.5):
    rows, H = a.rows, a.H
    r, x, wp, w, gate = (put(t, dev, shift) for t in (a.r, a.x, a.wp, a.w, a.gate))
    o = {"sum": Out(dev, (rows, H), a.r.dtype, shift), "normed": Out(dev, (rows, H), torch.bfloat16, shift), "post_rms": Out(dev, (rows,), torch.float32),
         "rms": Out(dev, (rows,), torch.float32), "x8": Out(dev, (rows, H), torch.uint8, shift), "sum8": Out(dev, (rows, H), torch.uint8, shift),
         "q": Out(dev, (rows, H), torch.uint8, shift)}
    t = {k: v.t for k, v in o.items()}
    if in_place:
        t["sum"], t["normed"] = r, x
    if not kept:
        t["x8"] = t["sum8"] = None
    if not wanted:
        t["sum"] = t["normed"] = t["post_rms"] = t["rms"] = None
    head = (r, x, a.f32, a.res, gate, a.gate_rows, wp, w, rows, H, EPS)
    outs = tuple(t[k] for k in ("sum", "normed", "post_rms", "rms", "x8", "sum8", "q"))
    if form == "record":
        qs, amax = torch.tensor([qscale], device=dev), torch.tensor([0.125], device=dev)
        cf.cf_gated_add_rmsnorm_quantize_record(*head, e5m2, *outs, qs, amax, stream())
    else:
        groups = (rows, (H + 127) // 128) if form == "block" else (rows,)
        for k in ("scale", "descale"):
            o[k] = Out(dev, groups, torch.float32)
            t[k] = o[k].t
        call = cf.cf_gated_add_rmsnorm_quantize_block_1x128 if form == "block" else cf.cf_gated_add_rmsnorm_quantize_rows
        call(*head, *(() if form == "block" else (e5m2,)), *outs, t["scale"], t["descale"], stream())
    torch.cuda.synchronize()
    assert all(v.unharmed() for v in o.values())
    got = {k: v.cpu() if v is not None else None for k, v in t.items()}
    return {**got, "amax": float(amax)} if form == "record" else got


def near8(q, v, half, least, rel):
    """q within one rounding of v, which is known to `rel`."""
    assert torch.all((q - v).abs() <= torch.maximum(half * v.abs(), torch.tensor(least, dtype=torch.float64)) + rel * v.abs())


def check_forward(got, a, form, e5m2, qscale=12.5):
    x, S = a.x.double(), kept_scale(a.H)
    px = (x.square().mean(1, keepdim=True) + EPS).sqrt()
    assert torch.all((got["post_rms"].double()[:, None] - px).abs() <= R * px)
    xh = x / px
    near8(got["x8"].view(E4M3).double(), xh * S, 2.0 ** -4, 2.0 ** -10, 2 * R)
    z = xh * a.wp.double() * gates(a.gate, a.gate_rows, a.rows)
    total = a.res * a.r.double() + z
    store = 2.0 ** -8 if a.r.dtype == torch.bfloat16 else U
    assert torch.all((got["sum"].double() - total).abs() <= (store + U) * total.abs() + 1.01 * (R + 4 * U) * z.abs())
    h = got["sum"].double()
    p = (h.square().mean(1, keepdim=True) + EPS).sqrt()
    assert torch.all((got["rms"].double()[:, None] - p).abs() <= R * p)
    near8(got["sum8"].view(E4M3).double(), h / p * S, 2.0 ** -4, 2.0 ** -10, 2 * R)
    y = h / p * a.w.double()
    assert torch.all((got["normed"].double() - y).abs() <= (2.0 ** -8 + R) * y.abs())
    check_quantized(got, y, form, e5m2, qscale)


def check_quantized(got, y, form, e5m2, qscale, rel=R):
    dtype, top, half, least = F8[e5m2]
    if form == "record":
        m = max(0.125, float(y.abs().max()))
        assert abs(got["amax"] - m) <= rel * m
        v = y * qscale
    else:
        width = 128 if form == "block" else y.shape[1]
        a = torch.stack([part.abs().amax(1) for part in y.split(width, 1)], 1).clamp_min(1e-12)
        assert torch.all((got["scale"].double().view(a.shape) * a / top - 1).abs() <= rel + 2 * U)
        assert torch.all((got["descale"].double().view(a.shape) * top / a - 1).abs() <= rel + 2 * U)
        v = y * (top / a).repeat_interleave(width, 1)[:, :y.shape[1]]
    near8(got["q"].view(dtype).double(), v.clamp(-top, top), half, least, 2 * rel)


FORMS = [("rows", 0), ("rows", 1), ("block", 0), ("record", 0), ("record", 1)]
# rows, H, rows a gate
SHAPES = [(1, 1, 0), (3, 7, 2), (1, 128, 1), (2, 130, 0), (5, 255, 5), (9, 512, 4), (4, 1000, 1), (7, 1001, 3), (33, 1024, 33), (6, 2050, 100), (64, 2048, 7),
          (17, 4096, 0), (1, 4096, 0), (5, 5120, 2), (3, 7168, 3), (13, 8192, 5), (2, 9001, 1), (4, 12288, 4), (3, 16384, 2), (300, 520, 90), (1030, 96, 1)]


@pytest.mark.parametrize("form,e5m2", FORMS)
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("rows,H,gate_rows", SHAPES)
def test_forward(cf, dev, rows, H, gate_rows, f32, form, e5m2):
    case(f"gated norm {form} rows={rows} H={H} gate_rows={gate_rows} f32={f32} e5m2={e5m2}")
    a = Layer(rows, H, f32, gate_rows, 1.0 if rows % 2 else -0.75, rows * 1009 + H)
    check_forward(forward(cf, dev, a, form, e5m2), a, form, e5m2)


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("rows,H,gate_rows", [(300, 2048, 0), (200, 4096, 64), (64, 7168, 1), (40, 12288, 40), (500, 200, 3), (33, 1001, 10)])
def test_forward_stream_has_the_bits_of_the_formula(cf, dev, rows, H, gate_rows, f32):
    """Up to h every operation is one fp32 rounding, in the order in which the formula is written: a bf16 stream next to the border of two values depends on it."""
    case(f"gated norm bits rows={rows} H={H} gate_rows={gate_rows} f32={f32}")
    a = Layer(rows, H, f32, gate_rows, 1.25, rows + H)
    got = forward(cf, dev, a)
    z = a.x.float() / got["post_rms"][:, None] * a.wp.float()
    if a.gate is not None:
        z = a.gate.float().repeat_interleave(gate_rows, 0)[:rows] * z
    assert torch.equal(got["sum"], (1.25 * a.r.float() + z).to(a.r.dtype))
    # a thread's own sum has at most four chains of eight fmas, added up: 12 roundings of u, halved by the root; the rest is in 64 bits, and the result rounded once
    px = (a.x.double().square().mean(1) + EPS).sqrt()
    assert torch.all((got["post_rms"].double() - px).abs() <= 7 * U * px)


@pytest.mark.parametrize("form", ["rows", "block", "record"])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("shift", [0, 1, 2, 4, 8])
def test_forward_in_place_and_any_alignment(cf, dev, form, f32, shift):
    for rows, H, gate_rows in ((5, 1032, 2), (3, 4096, 0), (4, 333, 1)):
        case(f"gated norm in place {form} rows={rows} H={H} f32={f32} shift={shift}")
        a = Layer(rows, H, f32, gate_rows, 1.5, 11)
        check_forward(forward(cf, dev, a, form, 0, shift), a, form, 0)
        check_forward(forward(cf, dev, a, form, 0, shift, in_place=True), a, form, 0)


@pytest.mark.parametrize("form", ["rows", "block", "record"])
def test_forward_outputs_that_are_not_wanted(cf, dev, form):
    a = Layer(6, 1024, 0, 4)
    case(f"gated norm {form} without its optional outputs")
    full, least = forward(cf, dev, a, form), forward(cf, dev, a, form, kept=False, wanted=False)
    for k in ("q", "scale", "descale"):
        assert k not in full or torch.equal(full[k], least[k])


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("H", [96, 1000, 4096])
def test_forward_rows_that_are_zero_infinite_or_nan(cf, dev, H, f32):
    """Zeros give zeros; a NaN or an infinity in either input stays in its own row."""
    case(f"gated norm special rows H={H} f32={f32}")
    a = Layer(7, H, f32, 0, seed=5)
    a.x[1] = 0.0
    a.r[1] = 0.0
    a.x[2, 17] = float("nan")
    a.r[3, 90] = float("inf")
    a.x[4, 3] = float("-inf")
    a.r[5, 0] = float("nan")
    for form in ("rows", "block"):
        got = forward(cf, dev, a, form)
        fine = torch.tensor([0, 6])
        b = Layer(2, H, f32, 0)
        b.r, b.x, b.wp, b.w = a.r[fine], a.x[fine], a.wp, a.w
        check_forward({k: v[fine] for k, v in got.items()}, b, form, 0)
        v = {k: got[k].view(E4M3).float() for k in ("q", "x8", "sum8")}
        assert all(torch.all(t[1] == 0) for t in v.values()) and torch.all(got["normed"][1] == 0)
        for row in (2, 5):
            assert torch.isnan(v["q"][row]).all() and torch.isnan(v["sum8"][row]).all()
        assert torch.isnan(v["x8"][2]).all() and not torch.isnan(v["x8"][5]).any() and not torch.isnan(v["x8"][3]).any()
        assert torch.isnan(v["x8"][4, 3]) and torch.all(v["x8"][4, :3] == 0) and torch.all(v["x8"][4, 4:] == 0)
        assert torch.isnan(v["q"][3, 90]) and torch.all(v["q"][3, :90] == 0) and torch.all(v["q"][3, 91:] == 0)


@pytest.mark.parametrize("H", [96, 1000, 4096])
@pytest.mark.parametrize("size", [1e-30, 1e-18, 1e19, 1e30])
def test_forward_rows_whose_squares_leave_fp32(cf, dev, H, size):
    """Both norms see values whose squares underflow or overflow; eps is far below or above them."""
    case(f"gated norm magnitude {size} H={H}")
    a = Layer(4, H, 1, 0, seed=9)
    a.r, a.x = (a.r * size).float(), (a.x.float() * size).to(torch.bfloat16)
    a.wp = (a.wp.float() * min(size, 1e30)).to(torch.bfloat16)
    got = forward(cf, dev, a, "rows")
    check_forward(got, a, "rows", 0)


# ---- gradient ---------------------------------------------------------------------------------------------------------

class Grad:
    def __init__(self, rows, H, f32, gate_rows, res=1.0, kept=False, seed=1, dh=True):
        a = self.a = Layer(rows, H, f32, gate_rows, res, seed)
        self.kept, S = kept, kept_scale(H)
        self.rms, self.post_rms = ((t.double().square().mean(1) + EPS).sqrt().float() for t in (a.r, a.x))
        g = torch.Generator().manual_seed(seed + 7)
        self.dy = (1e-2 * torch.randn(rows, H, generator=g)).to(torch.bfloat16)
        self.dh = (1e-2 * torch.randn(rows, H, generator=g)).to(STREAM[f32]) if dh else None
        self.h, self.x = a.r, a.x
        if kept:
            self.h, self.x = ((t.double() / p.double()[:, None] * S).float().to(E4M3) for t, p in ((a.r, self.rms), (a.x, self.post_rms)))


def backward(cf, dev, g, out="both", qscale=2.0e5, start=None, shift=0, in_place=False, accumulate=3):
    a = g.a
    rows, H = a.rows, a.H
    bits = lambda t: t.view(torch.uint8) if g.kept else t  # noqa: E731
    dy, dh, gate, wp, w = (put(t, dev, shift) for t in (g.dy, g.dh, a.gate, a.wp, a.w))
    h, x = (put(bits(t), dev, shift) for t in (g.h, g.x))
    rms, post_rms = g.rms.to(dev), g.post_rms.to(dev)
    o = {"dr": Out(dev, (rows, H), a.r.dtype, shift), "dx": Out(dev, (rows, H), torch.bfloat16, shift), "q": Out(dev, (rows, H), torch.uint8, shift),
         "dwp": Out(dev, (H,), torch.float32, shift), "dw": Out(dev, (H,), torch.float32, shift),
         "dgate": Out(dev, a.gate.shape if a.gate is not None else (1,), torch.float32, shift)}
    if start is not None:
        for k, v in start.items():
            o[k].t.copy_(v)
    n = ctypes.c_size_t(0)
    cf.cf_gated_add_rmsnorm_backward_workspace_bytes(rows, H, a.gate_rows, ctypes.byref(n))
    ws = Out(dev, (n.value,), torch.uint8)
    qs, amax = torch.tensor([qscale], device=dev), torch.zeros(1, device=dev)
    dr = dh if in_place else o["dr"].t
    call = cf.cf_gated_add_rmsnorm_backward_ckpt8 if g.kept else cf.cf_gated_add_rmsnorm_backward
    call(dy, h, x, a.f32, a.res, gate, a.gate_rows, wp, w, post_rms, rms, dh, rows, H, dr, o["dx"].t if out != "e5m2" else None,
         o["q"].t if out != "bf16" else None, qs, amax, o["dwp"].t, o["dw"].t, o["dgate"].t, accumulate if start is not None else 0, ws.t, n.value, stream())
    torch.cuda.synchronize()
    assert all(v.unharmed() for v in o.values()) and ws.unharmed()
    got = {k: v.t.cpu() for k, v in o.items()}
    return {**got, "dr": dr.cpu(), "amax": float(amax), "out": out, "qscale": qscale}


def group_sum(t, gate_rows, rows):
    return torch.nn.functional.pad(t, (0, 0, 0, -rows % gate_rows)).unflatten(0, (-1, gate_rows)).sum(1)


def check_backward(got, g, start=None, accumulate=3):
    """A row's mean is a sum of H terms: (H / 64 + 16) u of the sum of their sizes.  D takes 8 roundings besides, e three, dx five; a share of a sum over rows, in 64 bits, is rounded
    once, its terms take four roundings and carry what D is off, and the result is rounded once more."""
    a = g.a
    rows, H, n = a.rows, a.H, (a.H / 64 + 16) * U
    p, px = g.rms.double()[:, None], g.post_rms.double()[:, None]
    if g.kept:
        hh, xh = g.h.double() / kept_scale(H), g.x.double() / kept_scale(H)
    else:
        hh, xh = g.h.double() / p, g.x.double() / px
    dy, w, wp = g.dy.double(), a.w.double(), a.wp.double()
    dh = g.dh.double() if g.dh is not None else torch.zeros_like(hh)
    gg, gate = dy * w, gates(a.gate, a.gate_rows, rows)
    c = (gg * hh).mean(1, keepdim=True)
    D = dh + (gg - hh * c) / p
    off = 1.01 * (8 * U * (dh.abs() + (gg.abs() + (hh * c).abs()) / p) + n * hh.abs() * (gg * hh).abs().mean(1, keepdim=True) / p)
    store = 2.0 ** -8 if a.r.dtype == torch.bfloat16 else U
    dr = a.res * D
    assert torch.all((got["dr"].double() - dr).abs() <= (store + 2 * U) * dr.abs() + 1.01 * abs(a.res) * off)
    gw = (gate * wp).abs()
    e = D * gate * wp
    e_off = gw * off + 3 * U * e.abs()
    m = (e * xh).mean(1, keepdim=True)
    m_off = (xh.abs() * e_off).mean(1, keepdim=True) + n * (e * xh).abs().mean(1, keepdim=True)
    dx = (e - xh * m) / px
    dx_off = 1.01 * (e_off + xh.abs() * m_off + 6 * U * (e.abs() + (xh * m).abs())) / px
    if got["out"] != "e5m2":
        assert torch.all((got["dx"].double() - dx).abs() <= 2.0 ** -8 * dx.abs() + 1.01 * dx_off)
    if got["out"] != "bf16":
        most = float(dx.abs().max())
        assert abs(got["amax"] - most) <= float(dx_off.max()) + U * most
        v = (dx * got["qscale"]).clamp(-57344.0, 57344.0)
        least = torch.tensor(2.0 ** -17, dtype=torch.float64)
        assert torch.all((got["q"].view(torch.float8_e5m2).double() - v).abs() <= torch.maximum(2.0 ** -3 * v.abs(), least) + 1.2 * (dx_off * got["qscale"] + U * v.abs()))

    def near(name, want, size, carried, scales):
        if start is not None and accumulate & (1 if scales else 2):
            want, size = want + start[name].double(), size + start[name].double().abs()
        assert torch.all((got[name].double() - want).abs() <= 8 * U * size + 1.01 * carried + 1e-44), name

    near("dw", (dy * hh).sum(0), (dy * hh).abs().sum(0), 0.0, True)
    t, t_off = D * xh, off * xh.abs()
    near("dwp", (t * gate).sum(0), (t * gate).abs().sum(0), (t_off * gate.abs()).sum(0), True)
    if a.gate is not None:
        sums = [group_sum(v, a.gate_rows, rows) * wp.abs() for v in (t.abs(), t_off)]
        near("dgate", group_sum(t, a.gate_rows, rows) * wp, sums[0], sums[1], False)


GRAD_SHAPES = SHAPES + [(2500, 264, 700), (1100, 1024, 3), (1100, 1024, 1), (1100, 1024, 1100), (4100, 96, 2), (4100, 96, 1000), (600, 264, 1), (40, 16384, 1),
                        (30, 9001, 7), (50, 8192, 20)]


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("rows,H,gate_rows", GRAD_SHAPES)
def test_backward(cf, dev, rows, H, gate_rows, f32, kept):
    case(f"gated norm gradient rows={rows} H={H} gate_rows={gate_rows} f32={f32} kept={kept}")
    g = Grad(rows, H, f32, gate_rows, 1.0 if rows % 2 else -0.75, kept, rows * 31 + H)
    check_backward(backward(cf, dev, g, ["both", "e5m2", "bf16"][(rows + f32) % 3]), g)


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("rows,H,gate_rows", [(300, 9216, 0), (300, 9216, 7), (600, 9001, 1), (700, 8200, 100), (2300, 8200, 1), (515, 12288, 2), (300, 12290, 0), (515, 13001, 250),
                                              (600, 16384, 0), (600, 16384, 3)])
def test_backward_of_wide_rows_with_several_a_workgroup(cf, dev, rows, H, gate_rows, f32, kept):
    case(f"gated norm gradient rows={rows} H={H} gate_rows={gate_rows} f32={f32} kept={kept}")
    g = Grad(rows, H, f32, gate_rows, 1.25, kept, rows + H)
    check_backward(backward(cf, dev, g, ["both", "e5m2", "bf16"][(rows + f32) % 3]), g)


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_backward_accumulates_in_place_at_any_alignment_and_without_a_stream_gradient(cf, dev, f32, shift, kept):
    for rows, H, gate_rows in ((40, 1032, 13), (7, 333, 1), (9, 4096, 9), (1100, 40, 300), (12, 10000, 5)):
        case(f"gated norm gradient in place rows={rows} H={H} f32={f32} shift={shift} kept={kept}")
        g = Grad(rows, H, f32, gate_rows, 1.25, kept, 77)
        start = {"dw": torch.linspace(-1.0, 1.0, H), "dwp": torch.linspace(2.0, -1.0, H), "dgate": torch.linspace(-1.0, 3.0, g.a.gate.numel()).view(g.a.gate.shape)}
        check_backward(backward(cf, dev, g, start=start, shift=shift, in_place=True), g, start)
        for accumulate in (1, 2):
            check_backward(backward(cf, dev, g, start=start, accumulate=accumulate), g, start, accumulate)
        g = Grad(rows, H, f32, gate_rows, 1.25, kept, 78, dh=False)
        check_backward(backward(cf, dev, g, shift=shift), g)


def test_backward_of_no_rows(cf, dev):
    dw, dwp = torch.full((64,), 3.0, device=dev), torch.full((64,), 4.0, device=dev)
    args = (None, None, None, 0, 1.0, None, 0, None, None, None, None, None, 0, 64, None, None, None, None, None, dwp, dw, None)
    cf.cf_gated_add_rmsnorm_backward(*args, 1, None, 0, stream())
    assert torch.all(dw == 3.0) and torch.all(dwp == 4.0)
    cf.cf_gated_add_rmsnorm_backward_ckpt8(*args, 0, None, 0, stream())
    assert torch.all(dw == 0.0) and torch.all(dwp == 0.0)


@pytest.mark.parametrize("gate_rows", [0, 1, 400, 1500])
def test_backward_gives_the_same_bits_twice(cf, dev, gate_rows):
    g = Grad(1500, 1024, 0, gate_rows, kept=True)
    a, b = (backward(cf, dev, g) for _ in range(2))
    assert all(torch.equal(a[k], b[k]) for k in ("dr", "dx", "q", "dw", "dwp", "dgate")) and a["amax"] == b["amax"]


@pytest.mark.parametrize("kept", [False, True])
def test_backward_rows_that_are_nan_or_infinite(cf, dev, kept):
    """A NaN in one row's operands stays in that row; in the sums over rows it reaches its columns, the row's own gradient where the mean carries it there."""
    case(f"gated norm gradient with NaN kept={kept}")
    g = Grad(9, 1000, 0, 4, kept=kept)
    clean = backward(cf, dev, g)
    g.dy[3, 5] = float("nan")
    g.dh[6, 8] = float("inf")
    got = backward(cf, dev, g)
    other = torch.tensor([0, 1, 2, 4, 5, 7, 8])
    for k in ("dr", "dx", "q"):
        assert torch.equal(got[k][other], clean[k][other]), k
    assert torch.isnan(got["dr"][3]).all() and torch.isnan(got["dx"][3]).all() and torch.isnan(got["q"].view(torch.float8_e5m2)[3].float()).all()
    assert torch.isinf(got["dr"][6, 8]) and torch.isfinite(got["dr"][6, :8]).all()
    assert torch.equal(got["dgate"][2], clean["dgate"][2]) and torch.isnan(got["dgate"][0]).all()


@pytest.mark.parametrize("gate_rows", [0, 5, 12])
def test_gradient_against_differences(cf, dev, gate_rows):
    """The directional derivative of sum(y * dy) + sum(h * dh) along random directions of all inputs, by central differences of the forward formula in 64 bits: truncation 1e-8 at a
    step of 1e-4, and the fp32 gradient's own error is below 1e-6 of the sum of sizes; dx is rounded to bf16 once, 2^-8 of each term at most."""
    rows, H = 12, 640
    g = Grad(rows, H, 1, gate_rows, 1.25, seed=91)
    a = g.a
    # h is what the forward pass makes of r, x and the weights
    x, wp, gate = a.x.double(), a.wp.double(), a.gate.double() if a.gate is not None else None

    def stream_of(r, x, wp, gate):
        z = x / (x.square().mean(1, keepdim=True) + EPS).sqrt() * wp
        return 1.25 * r + (z if gate is None else z * gate.repeat_interleave(gate_rows, 0)[:rows])

    r = a.r.double()
    h = stream_of(r, x, wp, gate).float()
    g.h, g.rms = h, (h.double().square().mean(1) + EPS).sqrt().float()
    got = backward(cf, dev, g, "bf16")

    def value(r, x, wp, w, gate):
        h = stream_of(r, x, wp, gate)
        return (h / (h.square().mean(1, keepdim=True) + EPS).sqrt() * w * g.dy.double()).sum() + (h * g.dh.double()).sum()

    gen = torch.Generator().manual_seed(4)
    inputs = [r, x, wp, a.w.double(), gate]
    grads = [got["dr"], got["dx"], got["dwp"], got["dw"], got["dgate"]]
    for _ in range(4):
        d = [torch.randn(t.shape, generator=gen, dtype=torch.float64) if t is not None else None for t in inputs]
        at = lambda t: [i + t * v if i is not None else None for i, v in zip(inputs, d)]  # noqa: E731
        slope = (value(*at(1e-4)) - value(*at(-1e-4))) / 2e-4
        terms = [k.double() * v for k, v in zip(grads, d) if v is not None]
        assert abs(sum(t.sum() for t in terms) - slope) <= 2e-6 * sum(t.abs().sum() for t in terms) + 2.0 ** -8 * terms[1].abs().sum()


def test_more_rows_than_one_launch_holds(cf, dev):
    """Rows of eight, 2^21 and a few, a gate for every thousand: the last ones are as the first."""
    rows, H, gate_rows = (1 << 21) + 7, 8, 1000
    case(f"gated norm {rows} rows of {H}")
    r, x = (torch.randn(rows, H, device=dev).to(torch.bfloat16) for _ in range(2))
    w, gate = torch.ones(H, device=dev).to(torch.bfloat16), torch.randn(-(-rows // gate_rows), H, device=dev).to(torch.bfloat16)
    total, normed = torch.zeros_like(r), torch.zeros_like(r)
    q, x8, sum8 = (torch.zeros(rows, H, dtype=torch.uint8, device=dev) for _ in range(3))
    post_rms, rms, s, d = (torch.zeros(rows, device=dev) for _ in range(4))
    cf.cf_gated_add_rmsnorm_quantize_rows(r, x, 0, 1.0, gate, gate_rows, w, w, rows, H, EPS, 0, total, normed, post_rms, rms, x8, sum8, q, s, d, stream())
    torch.cuda.synchronize()
    a = Layer(7, H, 0, 0)
    tail = slice(rows - 7, rows)
    a.r, a.x, a.wp, a.w = r[tail].cpu(), x[tail].cpu(), w.cpu(), w.cpu()
    a.gate, a.gate_rows = gate[-1:].cpu(), 7
    assert rows % gate_rows >= 7
    check_forward({"sum": total[tail].cpu(), "normed": normed[tail].cpu(), "post_rms": post_rms[tail].cpu(), "rms": rms[tail].cpu(), "x8": x8[tail].cpu(),
                   "sum8": sum8[tail].cpu(), "q": q[tail].cpu(), "scale": s[tail].cpu(), "descale": d[tail].cpu()}, a, "rows", 0)
    assert bool((s > 0).all())
