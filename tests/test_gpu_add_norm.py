"""GPU: residual addition + RMS norm + 8-bit output, and its gradient, against the formulas in 64 bits.

Tolerances.  u = 2^-24.  A row's sum of squares adds at most H / 64 terms per thread and then at most 10 more across threads, so its
relative error is below (H / 64 + 10) u <= 266 u for H = 16384; the root halves it, and the divisions, the root and the products
add a few u: R = 150 u bounds the relative error of rms, y and the scales.  On top comes the rounding to the output's type: bf16 2^-8, E4M3 2^-4 or
half of its smallest step, E5M2 2^-3 or half of its."""
import numpy as np
import pytest
import torch

from gpu_util import case, stream

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
R = 150 * U
EPS = 1e-6
F8 = {0: (torch.float8_e4m3fn, 448.0, 2.0 ** -4, 2.0 ** -10), 1: (torch.float8_e5m2, 57344.0, 2.0 ** -3, 2.0 ** -17)}
STREAM = {0: torch.bfloat16, 1: torch.float32}


def rows_of(rows, H, seed, dtype, sigma=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, H, generator=g) * torch.exp(torch.randn(rows, 1, generator=g)) * sigma
    x[:, ::37] *= 20.0
    return x.to(dtype)


def gamma_of(H, seed):
    return (1.0 + 0.3 * torch.randn(H, generator=torch.Generator().manual_seed(seed))).to(torch.bfloat16)


def shifted(t, dev, elements):
    """The tensor on the device, `elements` elements behind a 256-byte boundary, and the buffer around it (filled with a mark)."""
    n = t.numel()
    buf = torch.full((n + 512,), 7.0, device=dev).to(t.dtype)
    view = buf[elements:elements + n]
    view.copy_(t.reshape(-1))
    return view.view(t.shape), buf


class Out:
    """Output buffers with a mark around them that no kernel may touch."""

    def __init__(self, dev, shape, dtype, shift=0):
        n = int(np.prod(shape))
        self.n, self.at = n, 64 + shift
        self.raw = torch.full((n + 256,), 77, dtype=torch.uint8, device=dev) if dtype == torch.uint8 else torch.full((n + 256,), 77.0, dtype=dtype, device=dev)
        self.t = self.raw[self.at:self.at + n].view(shape)

    def unharmed(self):
        return bool((self.raw[:self.at] == 77).all()) and bool((self.raw[self.at + self.n:] == 77).all())


def forward(cf, dev, r, x, w, f32, form, e5m2, shift=0, with_normed=True, in_place=False, qscale=0.0):
    rows, H = r.shape
    rd, _ = shifted(r, dev, shift)
    xd = shifted(x, dev, shift)[0] if x is not None else None
    wd, _ = shifted(w, dev, shift)
    o = {"sum": Out(dev, r.shape, r.dtype, shift), "rms": Out(dev, (rows,), torch.float32), "q": Out(dev, r.shape, torch.uint8, shift),
         "normed": Out(dev, r.shape, torch.bfloat16, shift)}
    total = rd if in_place else o["sum"].t
    normed = (xd if in_place and xd is not None else o["normed"].t) if with_normed else None
    groups = (rows, (H + 127) // 128) if form == "block" else (rows,)
    if form == "record":
        qs, amax = torch.tensor([qscale], device=dev), torch.tensor([0.125], device=dev)
        cf.cf_add_rmsnorm_quantize_record(rd, xd, f32, wd, rows, H, EPS, e5m2, total, normed, o["rms"].t, o["q"].t, qs, amax, stream())
    else:
        o["scale"], o["descale"] = Out(dev, groups, torch.float32), Out(dev, groups, torch.float32)
        args = (rd, xd, f32, wd, rows, H, EPS) + (() if form == "block" else (e5m2,)) + (total, normed, o["rms"].t, o["q"].t, o["scale"].t, o["descale"].t, stream())
        (cf.cf_add_rmsnorm_quantize_block_1x128 if form == "block" else cf.cf_add_rmsnorm_quantize_rows)(*args)
    torch.cuda.synchronize()
    got = {k: v.t.cpu() for k, v in o.items()}
    assert all(v.unharmed() for v in o.values())
    got["sum"] = total.cpu()
    got["normed"] = normed.cpu() if with_normed else None
    if form == "record":
        got["amax"] = amax.cpu()
    return got


def check_forward(got, r, x, w, form, e5m2, qscale=0.0):
    rows, H = r.shape
    want = (r.float() + x.float()).to(r.dtype) if x is not None else r
    assert torch.equal(got["sum"], want)
    h = want.double()
    rms = (h.square().mean(1) + EPS).sqrt()
    y = h / rms[:, None] * w.double()
    assert torch.all((got["rms"].double() - rms).abs() <= R * rms)
    if got["normed"] is not None:
        assert torch.all((got["normed"].double() - y).abs() <= (2.0 ** -8 + R) * y.abs())
    dtype, top, half, least = F8[e5m2]
    if form == "record":
        m = max(0.125, float(y.abs().max()))
        assert abs(float(got["amax"]) - m) <= R * m
        v = y * qscale
    else:
        width = 128 if form == "block" else H
        a = torch.stack([p.abs().amax(1) for p in y.split(width, 1)], 1).clamp_min(1e-12)
        assert torch.all((got["scale"].double().view(a.shape) * a / top - 1).abs() <= R + 2 * U)
        assert torch.all((got["descale"].double().view(a.shape) * top / a - 1).abs() <= R + 2 * U)
        v = y * (top / a).repeat_interleave(width, 1)[:, :H]
    v = v.clamp(-top, top)
    q = got["q"].view(dtype).double()
    assert torch.all((q - v).abs() <= torch.maximum(half * v.abs(), torch.tensor(least, dtype=torch.float64)) + 2 * R * v.abs())


FORMS = [("rows", 0), ("rows", 1), ("block", 0), ("record", 0), ("record", 1)]
SHAPES = [(1, 1), (3, 7), (1, 128), (2, 130), (5, 255), (9, 512), (4, 1000), (7, 1001), (33, 1024), (6, 2050), (64, 2048), (17, 4096), (1, 4096),
          (5, 5120), (3, 7168), (13, 8192), (2, 9001), (4, 12288), (2, 16384), (300, 520), (1030, 96)]


@pytest.mark.parametrize("form,e5m2", FORMS)
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("rows,H", SHAPES)
def test_forward(cf, dev, rows, H, f32, form, e5m2):
    case(f"add-norm {form} rows={rows} H={H} f32={f32} e5m2={e5m2}")
    r, x, w = rows_of(rows, H, rows * 1009 + H, STREAM[f32]), rows_of(rows, H, rows + H, torch.bfloat16, 0.5), gamma_of(H, H)
    got = forward(cf, dev, r, x, w, f32, form, e5m2, qscale=12.5)
    check_forward(got, r, x, w, form, e5m2, 12.5)


@pytest.mark.parametrize("form", ["rows", "block", "record"])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("shift", [1, 2, 4, 8])
def test_forward_any_alignment(cf, dev, form, f32, shift):
    for rows, H in ((5, 1032), (3, 4096), (4, 333)):
        case(f"add-norm {form} rows={rows} H={H} f32={f32} shift={shift}")
        r, x, w = rows_of(rows, H, 11, STREAM[f32]), rows_of(rows, H, 12, torch.bfloat16), gamma_of(H, 13)
        check_forward(forward(cf, dev, r, x, w, f32, form, 0, shift=shift, qscale=3.0), r, x, w, form, 0, 3.0)


@pytest.mark.parametrize("form", ["rows", "block", "record"])
@pytest.mark.parametrize("f32", [0, 1])
def test_forward_in_place_and_without_an_addend(cf, dev, form, f32):
    for rows, H in ((37, 2048), (5, 777), (1, 7168)):
        case(f"add-norm in place / no addend {form} rows={rows} H={H} f32={f32}")
        r, x, w = rows_of(rows, H, 21, STREAM[f32]), rows_of(rows, H, 22, torch.bfloat16), gamma_of(H, 23)
        got = forward(cf, dev, r, x, w, f32, form, 0, in_place=True, qscale=9.0)
        check_forward(got, r, x, w, form, 0, 9.0)
        got = forward(cf, dev, r, None, w, f32, form, 0, with_normed=False, qscale=9.0)
        check_forward(got, r, None, w, form, 0, 9.0)


def test_forward_outputs_that_are_not_wanted(cf, dev):
    rows, H = 6, 1024
    r, x, w = (t.to(dev) for t in (rows_of(rows, H, 1, torch.bfloat16), rows_of(rows, H, 2, torch.bfloat16), gamma_of(H, 3)))
    q, s, d = torch.empty(rows, H, dtype=torch.uint8, device=dev), torch.empty(rows, device=dev), torch.empty(rows, device=dev)
    q2, s2, d2 = torch.empty_like(q), torch.empty_like(s), torch.empty_like(d)
    cf.cf_add_rmsnorm_quantize_rows(r, x, 0, w, rows, H, EPS, 0, torch.empty_like(r), torch.empty_like(r), torch.empty(rows, device=dev), q, s, d, stream())
    cf.cf_add_rmsnorm_quantize_rows(r, x, 0, w, rows, H, EPS, 0, None, None, None, q2, s2, d2, stream())
    torch.cuda.synchronize()
    assert torch.equal(q, q2) and torch.equal(s, s2) and torch.equal(d, d2)


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("H", [1000, 4096])
def test_forward_rows_that_are_zero_infinite_or_nan(cf, dev, H, f32):
    """A row of zeros gives zeros under the scale of 1e-12; a NaN or an infinity stays in its own row."""
    case(f"add-norm special rows H={H} f32={f32}")
    r, x, w = rows_of(6, H, 5, STREAM[f32]), torch.zeros(6, H, dtype=torch.bfloat16), gamma_of(H, 6)
    r[1] = 0.0
    r[2, 17] = float("nan")
    r[3, 900] = float("inf")
    r[4, 3] = float("-inf")
    for form in ("rows", "block"):
        got = forward(cf, dev, r, x, w, f32, form, 0)
        keep = torch.tensor([0, 5])
        part = {k: v[keep] if k != "scale" and k != "descale" else v[keep] for k, v in got.items()}
        check_forward(part, r[keep], x[keep], w, form, 0)
        q = got["q"].view(torch.float8_e4m3fn).float()
        assert torch.all(q[1] == 0) and torch.all(got["normed"][1] == 0)
        assert torch.all(got["scale"][1].double() == np.float64(np.float32(448.0) / np.float32(1e-12)))
        assert torch.isnan(q[2]).all()                     # the root mean square is NaN
        for row, at in ((3, 900), (4, 3)):                 # it is infinite: 0 everywhere else, and inf / inf
            assert torch.isnan(q[row, at]) and torch.all(q[row, :at] == 0) and torch.all(q[row, at + 1:] == 0)


def test_forward_empty(cf, dev):
    assert cf.raw_cf_add_rmsnorm_quantize_rows(None, None, 0, None, 0, 64, EPS, 0, None, None, None, None, None, None, None) == 0
    assert cf.raw_cf_add_rmsnorm_quantize_block_1x128(None, None, 0, None, 5, 0, EPS, None, None, None, None, None, None, None) == 0


# ---- gradient ---------------------------------------------------------------------------------------------------------

def gradient_inputs(rows, H, f32, seed):
    h, w = rows_of(rows, H, seed, STREAM[f32]), gamma_of(H, seed + 1)
    rms = (h.double().square().mean(1) + EPS).sqrt().float()
    g = torch.Generator().manual_seed(seed + 2)
    dy = (1e-2 * torch.randn(rows, H, generator=g)).to(torch.bfloat16)
    dh = (1e-2 * torch.randn(rows, H, generator=g)).to(STREAM[f32])
    return h, w, rms, dy, dh


def backward(cf, dev, h, w, rms, dy, dh, f32, quant, qscale=1.0, start=None, shift=0, in_place=False):
    import ctypes
    rows, H = h.shape
    hd, wd, dyd, dhd = (shifted(t, dev, shift)[0] if t is not None else None for t in (h, w, dy, dh))
    rd = rms.to(dev)
    dr, dw, q = Out(dev, h.shape, h.dtype, shift), Out(dev, (H,), torch.float32, shift), Out(dev, h.shape, torch.uint8, shift)
    if start is not None:
        dw.t.copy_(start)
    out = dhd if in_place else dr.t
    n = ctypes.c_size_t(0)
    cf.cf_add_rmsnorm_backward_workspace_bytes(rows, H, ctypes.byref(n))
    ws = Out(dev, (n.value,), torch.uint8)
    args = (dyd, hd, f32, wd, rd, dhd, rows, H, out, dw.t, int(start is not None))
    qs, amax = torch.tensor([qscale], device=dev), torch.zeros(1, device=dev)
    if quant:
        cf.cf_add_rmsnorm_backward_quant_e5m2(*args, q.t, qs, amax, ws.t, n.value, stream())
    else:
        cf.cf_add_rmsnorm_backward(*args, ws.t, n.value, stream())
    torch.cuda.synchronize()
    assert dr.unharmed() and dw.unharmed() and q.unharmed() and ws.unharmed()
    return {"dr": out.cpu(), "dw": dw.t.cpu(), "q": q.t.cpu(), "amax": float(amax)}


def formula(h, w, rms, dy, dh):
    """(dr, dw) in 64 bits, and the sums of absolute terms that bound their rounding."""
    h, w, rms, dy = h.double(), w.double(), rms.double()[:, None], dy.double()
    xh, g = h / rms, dy * w
    c = (g * xh).mean(1, keepdim=True)
    dh = dh.double() if dh is not None else torch.zeros_like(h)
    size = dh.abs() + (g.abs() + (xh * c).abs()) / rms
    return dh + (g - xh * c) / rms, (dy * xh).sum(0), size, xh.abs() * (g * xh).abs().mean(1, keepdim=True) / rms, (dy * xh).abs().sum(0)


def check_backward(got, h, w, rms, dy, dh, quant, qscale=1.0, start=None):
    """c sums H terms: (H / 64 + 10) u of the sum of their sizes.  The rest of dr takes 6 roundings, the storage one more.  dw: one rounding for
    each of rows + 1 additions at most, and 3 for a term."""
    rows, H = h.shape
    dr, dw, size, csize, wsize = formula(h, w, rms, dy, dh)
    off = 8 * U * size + (H / 64 + 16) * U * csize
    store = 2.0 ** -8 if h.dtype == torch.bfloat16 else U
    assert torch.all((got["dr"].double() - dr).abs() <= store * dr.abs() + 1.01 * off)
    if start is not None:
        dw, wsize = dw + start.double(), wsize + start.double().abs()
    assert torch.all((got["dw"].double() - dw).abs() <= (rows + 6) * U * wsize)
    if quant:
        m = float(dr.abs().max())
        assert abs(got["amax"] - m) <= float(off.max()) + U * m
        v = (dr * qscale).clamp(-57344.0, 57344.0)
        q = got["q"].view(torch.float8_e5m2).double()
        least = torch.tensor(2.0 ** -17, dtype=torch.float64)
        assert torch.all((q - v).abs() <= torch.maximum(2.0 ** -3 * v.abs(), least) + 1.2 * (off * qscale + U * v.abs()))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("rows,H", SHAPES + [(2500, 264), (1100, 1024)])
def test_backward(cf, dev, rows, H, f32, quant):
    case(f"add-norm gradient rows={rows} H={H} f32={f32} quant={quant}")
    h, w, rms, dy, dh = gradient_inputs(rows, H, f32, rows * 31 + H)
    scale = 2.0e5
    check_backward(backward(cf, dev, h, w, rms, dy, dh, f32, quant, scale), h, w, rms, dy, dh, quant, scale)


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_backward_accumulates_in_place_at_any_alignment_and_without_a_stream_gradient(cf, dev, f32, shift):
    for rows, H in ((40, 1032), (7, 333), (9, 4096)):
        case(f"add-norm gradient in place rows={rows} H={H} f32={f32} shift={shift}")
        h, w, rms, dy, dh = gradient_inputs(rows, H, f32, 77)
        start = torch.linspace(-1.0, 1.0, H)
        check_backward(backward(cf, dev, h, w, rms, dy, dh, f32, True, 1e4, start, shift, True), h, w, rms, dy, dh, True, 1e4, start)
        check_backward(backward(cf, dev, h, w, rms, dy, None, f32, False, 1.0, None, shift), h, w, rms, dy, None, False)


def test_backward_of_no_rows(cf, dev):
    dw = torch.full((64,), 3.0, device=dev)
    args = (None, None, 0, None, None, None, 0, 64, None, dw)
    cf.cf_add_rmsnorm_backward(*args, 1, None, 0, stream())
    assert torch.all(dw == 3.0)
    cf.cf_add_rmsnorm_backward(*args, 0, None, 0, stream())
    assert torch.all(dw == 0.0)


def test_backward_gives_the_same_bits_twice(cf, dev):
    h, w, rms, dy, dh = gradient_inputs(1500, 1024, 0, 5)
    a, b = (backward(cf, dev, h, w, rms, dy, dh, 0, True, 1e4) for _ in range(2))
    assert torch.equal(a["dr"], b["dr"]) and torch.equal(a["dw"], b["dw"]) and torch.equal(a["q"], b["q"]) and a["amax"] == b["amax"]


def test_gradient_against_differences(cf, dev):
    """The directional derivative of sum(y * dy) + sum(h * dh) along random directions, by central differences of the forward formula in 64 bits.
    Truncation: the third derivative is of the order of |v / rms|^3, so step 1e-4 leaves 1e-8; the fp32 gradient's own error is below 1e-6 of the
    sum of sizes."""
    rows, H = 12, 640
    h, w, rms, dy, dh = gradient_inputs(rows, H, 1, 91)
    got = backward(cf, dev, h, w, rms, dy, dh, 1, False)

    def value(h, w):
        return (h / (h.square().mean(1, keepdim=True) + EPS).sqrt() * w * dy.double()).sum() + (h * dh.double()).sum()

    g = torch.Generator().manual_seed(4)
    for _ in range(4):
        v, u, t = torch.randn(rows, H, generator=g, dtype=torch.float64), torch.randn(H, generator=g, dtype=torch.float64), 1e-4
        h64, w64 = h.double(), w.double()
        slope = (value(h64 + t * v, w64 + t * u) - value(h64 - t * v, w64 - t * u)) / (2 * t)
        mine = (got["dr"].double() * v).sum() + (got["dw"].double() * u).sum()
        size = (got["dr"].double() * v).abs().sum() + (got["dw"].double() * u).abs().sum()
        assert abs(mine - slope) <= 2e-6 * size


def test_more_rows_than_one_launch_holds(cf, dev):
    """Rows of eight, 2^21 and a few: the last ones are as the first."""
    rows, H = (1 << 21) + 7, 8
    case(f"add-norm {rows} rows of {H}")
    r = torch.randn(rows, H, device=dev).to(torch.bfloat16)
    x, w = torch.zeros_like(r), torch.ones(H, device=dev).to(torch.bfloat16)
    total, q = torch.zeros_like(r), torch.zeros(rows, H, dtype=torch.uint8, device=dev)
    rms, s, d = (torch.zeros(rows, device=dev) for _ in range(3))
    cf.cf_add_rmsnorm_quantize_rows(r, x, 0, w, rows, H, EPS, 0, total, None, rms, q, s, d, stream())
    torch.cuda.synchronize()
    assert torch.equal(total, r)
    tail = slice(rows - 4000, rows)
    check_forward({"sum": total[tail].cpu(), "rms": rms[tail].cpu(), "normed": None, "q": q[tail].cpu(), "scale": s[tail].cpu(), "descale": d[tail].cpu()},
                  r[tail].cpu(), x[tail].cpu(), w.cpu(), "rows", 0)
    assert bool((s > 0).all())
