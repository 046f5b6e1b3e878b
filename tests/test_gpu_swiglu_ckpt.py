"""GPU: the gated activation with its 8-bit operand and its 8-bit checkpoints, and the gradient from those, against the formulas in 64 bits.

Tolerances.  u = 2^-24.  The checkpoints are compared bit for bit: a group's maximum is a bf16 value, 448 / amax, amax / 448 and the product with the scale are one fp32 rounding each.
The sigmoid s of g is 1 / (1 + e), e = 2^t, t = -g log2(e).  t is rounded once and its constant is off by 0.22 u: 1.22 u |t|, which moves e by ln 2 times
that, 1.22 u |g|; the exponential adds 2 u.  In s these count (1 - s) times, the addition 1 u, the reciprocal 2 u: s is off by (5 + 1.22 |g| (1 - s)) u at most, here
(6 + 2 |g| (1 - s)) u =: sig.  The activation adds two products.  Where e leaves fp32 (g < -87) s is zero, off by 87 e^-87 |u| < 2e-36 |u| in the activation.  On top comes the rounding to the
output's type: bf16 2^-8, E4M3 2^-4 or half of its smallest step, E5M2 2^-3 or half of its."""
import pytest
import torch

from gpu_util import case, stream
from test_gpu_add_norm import F8, U, Out, rows_of, shifted

pytestmark = pytest.mark.gpu

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def activation(g, u):
    """(a, how far it may be off) in 64 bits."""
    g, u = g.double(), u.double()
    s = torch.sigmoid(g)
    a = s * g * u
    return a, a.abs() * U * (9 + 2 * g.abs() * (1 - s)) + 2e-36 * u.abs() * (g < -86)


def check_quantized(got, a, off, form, e5m2, qscale):
    dtype, top, half, least = F8[e5m2]
    if form == "record":
        m = max(0.125, float(a.abs().max()))
        assert abs(got["amax"] - m) <= float(off.max()) + U * m
        scale, rel = torch.full_like(a[:, :1], qscale), torch.zeros_like(a[:, :1])
    else:
        width = 128 if form == "block" else a.shape[1]
        parts = lambda t: torch.stack([p.abs().amax(1) for p in t.split(width, 1)], 1)  # noqa: E731
        m = parts(a).clamp_min(1e-12)
        rel = parts(off) / m + 3 * U            # a maximum is off by the largest of its elements' errors; then a division
        assert torch.all((got["scale"].double().view(m.shape) * m / top - 1).abs() <= 1.01 * rel)
        assert torch.all((got["descale"].double().view(m.shape) * top / m - 1).abs() <= 1.01 * rel)
        spread = lambda t: t.repeat_interleave(width, 1)[:, :a.shape[1]]  # noqa: E731
        scale, rel = spread(top / m), spread(rel)
    v = (a * scale).clamp(-top, top)
    q = got["q"].view(dtype).double()
    assert torch.all((q - v).abs() <= torch.maximum(half * v.abs(), torch.tensor(least, dtype=torch.float64)) + 1.1 * (off * scale + (rel + 2 * U) * v.abs()))



def groups_of(t):
    return torch.nn.functional.pad(t, (0, -t.shape[1] % 128)).unflatten(1, (-1, 128))


def checkpoint(t):
    """(bytes, descale) of bf16 rows, in the same fp32 operations."""
    g = groups_of(t.float())
    a = g.abs().amax(2).clamp_min(1e-12)
    s = torch.tensor(448.0) / a
    return (g * s[:, :, None]).clamp(-448.0, 448.0).to(E4M3).flatten(1)[:, :t.shape[1]], a / torch.tensor(448.0)


def restored(q, d):
    return (groups_of(q.float()) * d[:, :, None]).flatten(1)[:, :q.shape[1]].double()


def inputs(rows, I, seed):
    return rows_of(rows, I, seed, torch.bfloat16), rows_of(rows, I, seed + 1, torch.bfloat16)


def forward(cf, dev, g, u, form="rows", e5m2=0, shift=0, pad=None, qscale=3.0):
    """pad: elements between the rows' ends and beginnings; None: gate and up are the halves of one buffer's rows."""
    rows, I = g.shape
    if pad is None:
        both = shifted(torch.cat([g, u], 1), dev, shift)[0]
        gd, ud = both[:, :I], both[:, I:]
    else:
        gd, ud = (shifted(torch.nn.functional.pad(t, (0, pad), value=float("nan")), dev, shift)[0][:, :I] for t in (g, u))
    ld, groups = gd.stride(0), (rows, (I + 127) // 128)
    if rows == 1:
        ld = max(ld, I)
    o = {"gate8": Out(dev, (rows, I), torch.uint8, shift), "gate8_descale": Out(dev, groups, torch.float32), "up8": Out(dev, (rows, I), torch.uint8, shift),
         "up8_descale": Out(dev, groups, torch.float32), "q": Out(dev, (rows, I), torch.uint8, shift)}
    outs = tuple(v.t for v in o.values())
    if form == "record":
        qs, amax = torch.tensor([qscale], device=dev), torch.tensor([0.125], device=dev)
        cf.cf_swiglu_ckpt8_quantize_record(gd, ud, ld, rows, I, e5m2, *outs, qs, amax, stream())
    else:
        shape = groups if form == "block" else (rows,)
        o["scale"], o["descale"] = Out(dev, shape, torch.float32), Out(dev, shape, torch.float32)
        call = cf.cf_swiglu_ckpt8_quantize_block_1x128 if form == "block" else cf.cf_swiglu_ckpt8_quantize_rows
        call(gd, ud, ld, rows, I, *(() if form == "block" else (e5m2,)), *outs, o["scale"].t, o["descale"].t, stream())
    torch.cuda.synchronize()
    assert all(v.unharmed() for v in o.values())
    got = {k: v.t.cpu() for k, v in o.items()}
    return {**got, "amax": float(amax)} if form == "record" else got


def check_forward(got, g, u, form, e5m2, qscale=3.0):
    for name, t in (("gate8", g), ("up8", u)):
        q, d = checkpoint(t)
        assert torch.equal(got[name + "_descale"], d), name
        assert torch.equal(got[name], q.view(torch.uint8)), name
    check_quantized(got, *activation(g, u), form, e5m2, qscale)


FORMS = [("rows", 0), ("rows", 1), ("block", 0), ("record", 0), ("record", 1)]
SHAPES = [(1, 1), (3, 7), (1, 128), (2, 130), (5, 255), (9, 512), (4, 1000), (7, 1001), (33, 1024), (6, 2050), (64, 1408), (17, 5461), (1, 14336), (3, 8192), (2, 9001),
          (4, 16384), (2, 20000), (1, 32768), (300, 520), (1030, 96), (5000, 8)]


@pytest.mark.parametrize("form,e5m2", FORMS)
@pytest.mark.parametrize("rows,I", SHAPES)
def test_forward(cf, dev, rows, I, form, e5m2):
    case(f"swiglu {form} rows={rows} I={I} e5m2={e5m2}")
    g, u = inputs(rows, I, rows * 7 + I)
    check_forward(forward(cf, dev, g, u, form, e5m2), g, u, form, e5m2)


@pytest.mark.parametrize("form", ["rows", "block", "record"])
@pytest.mark.parametrize("shift", [0, 1, 2, 4, 8])
def test_forward_any_alignment_and_stride(cf, dev, form, shift):
    for rows, I, pad in ((5, 1032, 0), (3, 4096, 24), (4, 333, 3), (3, 3, 0), (2, 1, 0), (4, 5, 1), (6, 128, 128)):
        case(f"swiglu {form} rows={rows} I={I} pad={pad} shift={shift}")
        g, u = inputs(rows, I, 11)
        check_forward(forward(cf, dev, g, u, form, 0, shift, pad), g, u, form, 0)
        check_forward(forward(cf, dev, g, u, form, 0, shift), g, u, form, 0)


@pytest.mark.parametrize("e5m2", [0, 1])
@pytest.mark.parametrize("rows,I", [(3, 16392), (2, 17001), (300, 24576), (2, 24577), (2, 32761)])
def test_forward_wide_rows(cf, dev, rows, I, e5m2):
    case(f"swiglu rows={rows} I={I} e5m2={e5m2}")
    g, u = inputs(rows, I, rows * 7 + I)
    check_forward(forward(cf, dev, g, u, "rows", e5m2), g, u, "rows", e5m2)


@pytest.mark.parametrize("form", ["block", "record"])
def test_forward_wider_than_a_row_in_registers(cf, dev, form):
    g, u = inputs(3, 70001, 5)
    case(f"swiglu {form} I=70001")
    check_forward(forward(cf, dev, g, u, form), g, u, form, 0)


@pytest.mark.parametrize("form", ["rows", "block", "record"])
def test_forward_far_gates(cf, dev, form):
    """Gates from far below zero to far above it, and the type's ends: zero, the line or an infinity, and no NaN."""
    case(f"swiglu {form} far gates")
    g = torch.linspace(-120.0, 120.0, 512).to(torch.bfloat16).view(1, -1).repeat(2, 1)
    u = torch.full((2, 512), 0.5).to(torch.bfloat16)
    u[1] = 1e-3
    got = forward(cf, dev, g, u, form)
    check_quantized(got, *activation(g, u), form, 0, 3.0)
    far = torch.tensor([[-3.38e38, -1e30, -1000.0, -88.0, 1000.0, 88.0, 1e30, 0.0]]).to(torch.bfloat16)
    got = forward(cf, dev, far, torch.full((1, 8), 1e-6).to(torch.bfloat16), "record", qscale=1.0)
    assert not torch.isnan(got["q"].view(E4M3).float()).any() and torch.all(got["q"].view(E4M3).float()[0, :4] == 0)
    assert got["q"].view(E4M3).float()[0, 6] == 448.0


@pytest.mark.parametrize("I", [96, 1000])
@pytest.mark.parametrize("form", ["rows", "block", "record"])
def test_forward_zeros_infinities_and_nans(cf, dev, I, form):
    """Zeros give zeros; a NaN stays itself, an infinity takes its group of the checkpoint with it, and neither reaches other rows."""
    case(f"swiglu special values {form} I={I}")
    g, u = inputs(6, I, 3)
    g[1], u[1] = 0.0, 0.0
    g[2, 17] = float("nan")
    u[3, 40] = float("nan")
    g[4, 90] = float("inf")
    got = forward(cf, dev, g, u, form)
    q = got["q"].view(E4M3).float()
    clean = forward(cf, dev, *inputs(6, I, 3), form)
    for row in (0, 5):
        assert torch.equal(got["q"][row], clean["q"][row]) and torch.equal(got["gate8"][row], clean["gate8"][row])
    assert torch.all(q[1] == 0) and torch.all(got["gate8"][1] == 0) and torch.all(got["up8"][1] == 0)
    for row, at, name in ((2, 17, "gate8"), (3, 40, "up8")):
        kept = got[name].view(E4M3).float()[row]
        assert torch.isnan(q[row, at]) and int(torch.isnan(q[row]).sum()) == 1 and torch.isnan(kept[at]) and int(torch.isnan(kept).sum()) == 1
    back = restored(got["gate8"].view(E4M3), got["gate8_descale"])[4]
    assert torch.isnan(back[:min(I, 128)]).all() and torch.isfinite(back[128:]).all()
    if form == "record":
        assert got["amax"] == float("inf") and q[4, 90] == 448.0 * float(torch.sign(u[4, 90]))


@pytest.mark.parametrize("e5m2", [0, 1])
@pytest.mark.parametrize("I", [96, 1000])
def test_forward_scaled_beyond_fp32(cf, dev, I, e5m2):
    """A finite activation whose product with the given scale leaves fp32 is the format's largest value, as any that the scale takes beyond it."""
    case(f"swiglu record beyond fp32 I={I} e5m2={e5m2}")
    g, u = inputs(6, I, 9)
    g[2, 7], u[2, 7] = 1e20, 1e15
    g[4, 30], u[4, 30] = 1e20, -1e15
    got = forward(cf, dev, g, u, "record", e5m2, qscale=1e10)
    check_forward(got, g, u, "record", e5m2, qscale=1e10)
    dtype, top = F8[e5m2][:2]
    q = got["q"].view(dtype).float()
    assert q[2, 7] == top and q[4, 30] == -top


# ---- gradient ---------------------------------------------------------------------------------------------------------

class Grad:
    def __init__(self, rows, I, seed):
        g, u = inputs(rows, I, seed)
        (self.g8, self.gd), (self.u8, self.ud) = checkpoint(g), checkpoint(u)
        self.do = (1e-2 * torch.randn(rows, I, generator=torch.Generator().manual_seed(seed + 3))).to(torch.bfloat16)

    def formula(self):
        """(dg, du, a), and how far each may be off before its last rounding."""
        g, u, d = restored(self.g8, self.gd), restored(self.u8, self.ud), self.do.double()
        s = torch.sigmoid(g)
        slope = s * (1 + g * (1 - s))
        # 1 - s is off by s sig + u (1 - s), g times that and an fma's rounding by |g| so much more; the decoded values by one rounding each, under which silu and its slope
        # move by 2 u (|g| + 1)
        sig = U * (6 + 2 * g.abs() * (1 - s))
        slope_off = (sig + 2 * U) * slope.abs() + s * (g.abs() * (sig * s + U * (1 - s)) + 2 * U * (1 + g * (1 - s)).abs()) + 2 * U * g.abs()
        dg, du, a = d * u * slope, d * g * s, g * s * u
        drift, far = 2 * U * (1 + g.abs()), 2e-36 * (g < -86)
        return ((dg, (d * u).abs() * (slope_off + far) + 4 * U * dg.abs()), (du, (sig + 4 * U + drift) * du.abs() + far * d.abs()),
                (a, (sig + 4 * U + drift) * a.abs() + far * u.abs()))


def backward(cf, dev, x, shift=0, pad=0, fused=False, with_act=True):
    rows, I = x.do.shape
    do, g8, u8 = (shifted(t, dev, shift)[0] for t in (x.do, x.g8.view(torch.uint8), x.u8.view(torch.uint8)))
    gd, ud = x.gd.to(dev), x.ud.to(dev)
    act = Out(dev, (rows, I), torch.bfloat16, shift)
    if fused:
        both = Out(dev, (rows, 2 * I), torch.bfloat16, shift)
        outs, ld = (both.t[:, :I], both.t[:, I:]), 2 * I
        raw = [both]
    else:
        raw = [Out(dev, (rows, I + pad), torch.bfloat16, shift) for _ in range(2)]
        outs, ld = tuple(o.t[:, :I] for o in raw), I + pad
    cf.cf_swiglu_ckpt8_backward(do, g8, gd, u8, ud, rows, I, *outs, ld, act.t if with_act else None, stream())
    torch.cuda.synchronize()
    assert act.unharmed() and all(o.unharmed() for o in raw)
    if not fused and pad:
        assert all(bool((o.t[:, I:] == 77).all()) for o in raw)
    return [t.cpu() for t in outs] + ([act.t.cpu()] if with_act else [])


def check_backward(got, x):
    for t, (want, off) in zip(got, x.formula()):
        assert torch.all((t.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1.01 * off + 1e-38)


@pytest.mark.parametrize("rows,I", SHAPES)
def test_backward(cf, dev, rows, I):
    case(f"swiglu gradient rows={rows} I={I}")
    x = Grad(rows, I, rows + I)
    check_backward(backward(cf, dev, x, fused=True), x)


@pytest.mark.parametrize("shift", [0, 1, 2, 4, 8])
def test_backward_any_alignment_and_stride(cf, dev, shift):
    for rows, I, pad in ((5, 1032, 0), (3, 4096, 24), (4, 333, 3), (3, 3, 0), (2, 1, 5), (6, 128, 128)):
        case(f"swiglu gradient rows={rows} I={I} pad={pad} shift={shift}")
        x = Grad(rows, I, 12)
        check_backward(backward(cf, dev, x, shift, pad), x)
        check_backward(backward(cf, dev, x, shift, pad, with_act=False), x)


def backward8(cf, dev, x, shift=0, transposed=True, qscale=1e5, act_qscale=3.0):
    rows, I = x.do.shape
    do, g8, u8 = (shifted(t, dev, shift)[0] for t in (x.do, x.g8.view(torch.uint8), x.u8.view(torch.uint8)))
    gd, ud = x.gd.to(dev), x.ud.to(dev)
    o = [Out(dev, s, torch.uint8, shift) for s in ((rows, 2 * I), (2 * I, rows), (I, rows))]
    qs, amax, aqs = (torch.tensor([v], device=dev) for v in (qscale, 0.0, act_qscale))
    cf.cf_swiglu_ckpt8_backward_quant_e5m2(do, g8, gd, u8, ud, rows, I, o[0].t, o[1].t if transposed else None, qs, amax, o[2].t if transposed else None,
                                           aqs if transposed else None, stream())
    torch.cuda.synchronize()
    assert all(v.unharmed() for v in o)
    return [v.t.cpu() for v in o], float(amax)


def check_backward8(got, x, transposed=True, qscale=1e5, act_qscale=3.0):
    (grad8, grad8_t, act8_t), amax = got
    (dg, dg_off), (du, du_off), (a, a_off) = x.formula()
    grad, off = torch.cat([dg, du], 1), torch.cat([dg_off, du_off], 1)
    most = float(grad.abs().max())
    assert abs(amax - most) <= 1.01 * float(off.max()) + U * most
    v = (grad * qscale).clamp(-57344.0, 57344.0)
    least = lambda e: torch.tensor(e, dtype=torch.float64)  # noqa: E731
    assert torch.all((grad8.view(E5M2).double() - v).abs() <= torch.maximum(2.0 ** -3 * v.abs(), least(2.0 ** -17)) + 1.2 * (off * qscale + U * v.abs()))
    if transposed:
        assert torch.equal(grad8_t, grad8.t())
        v = (a * act_qscale).clamp(-448.0, 448.0)
        q = act8_t.t().contiguous().view(E4M3).double()
        assert torch.all((q - v).abs() <= torch.maximum(2.0 ** -4 * v.abs(), least(2.0 ** -10)) + 1.2 * (a_off * act_qscale + U * v.abs()))
    else:
        assert bool((grad8_t == 77).all()) and bool((act8_t == 77).all())


@pytest.mark.parametrize("rows,I", SHAPES + [(128, 128), (256, 384), (16, 8), (144, 264), (130, 1000), (333, 257)])
def test_backward_8_bit(cf, dev, rows, I):
    case(f"swiglu 8-bit gradient rows={rows} I={I}")
    x = Grad(rows, I, rows + I)
    check_backward8(backward8(cf, dev, x), x)


@pytest.mark.parametrize("shift", [1, 2, 4, 8])
def test_backward_8_bit_any_alignment_and_without_the_transposed(cf, dev, shift):
    for rows, I in ((5, 1032), (130, 256), (40, 333), (3, 3), (128, 128)):
        case(f"swiglu 8-bit gradient rows={rows} I={I} shift={shift}")
        x = Grad(rows, I, 12)
        check_backward8(backward8(cf, dev, x, shift), x)
        check_backward8(backward8(cf, dev, x, shift, False), x, False)


@pytest.mark.parametrize("rows,I", [(48, 256), (37, 333)])
def test_backward_nan_and_infinity(cf, dev, rows, I):
    """They stay with their element in both directions."""
    case(f"swiglu gradient with NaN rows={rows} I={I}")
    x = Grad(rows, I, 4)
    clean, clean8 = backward(cf, dev, x, fused=True), backward8(cf, dev, x)[0]
    x.do[3, 5] = float("nan")
    x.do[7, 200] = float("inf")
    got, (got8, amax) = backward(cf, dev, x, fused=True), backward8(cf, dev, x)
    keep = torch.ones(rows, I, dtype=torch.bool)
    keep[3, 5] = keep[7, 200] = False
    for a, b in zip(got, clean):
        assert torch.equal(a[keep], b[keep])
    assert torch.isnan(got[0][3, 5]) and torch.isnan(got[1][3, 5]) and torch.isinf(got[1][7, 200]) and torch.equal(got[2], clean[2])
    both = torch.cat([keep, keep], 1)
    assert torch.equal(got8[0][both], clean8[0][both]) and torch.equal(got8[1], got8[0].t()) and torch.equal(got8[2], clean8[2])
    assert torch.isnan(got8[0].view(E5M2).float()[3, 5]) and abs(float(got8[0].view(E5M2).float()[7, I + 200])) == 57344.0 and amax == float("inf")


@pytest.mark.parametrize("rows,I", [(48, 256), (37, 333)])
def test_backward_8_bit_scaled_beyond_fp32(cf, dev, rows, I):
    """Finite gradients and activations whose products with the given scales leave fp32 are the formats' largest values."""
    case(f"swiglu 8-bit gradient beyond fp32 rows={rows} I={I}")
    x = Grad(rows, I, 6)
    x.do[3, 5], x.do[7, 200] = 1e33, -1e33
    got = backward8(cf, dev, x, qscale=1e10, act_qscale=1e38)
    check_backward8(got, x, qscale=1e10, act_qscale=1e38)
    (dg, _), (du, _), (a, _) = x.formula()
    want = torch.cat([dg, du], 1)
    grad, act = got[0][0].view(E5M2).float(), got[0][2].t().contiguous().view(E4M3).float()
    far = want.abs() * 1e10 > 2.0 ** 129
    assert far.any() and torch.equal(grad[far], 57344.0 * torch.sign(want[far]).float())
    far = a.abs() * 1e38 > 2.0 ** 129
    assert far.any() and torch.equal(act[far], 448.0 * torch.sign(a[far]).float())


def test_gradient_against_differences(cf, dev):
    """The slope of sum(a * dO) along random directions of what the bytes stand for, by central differences in 64 bits (truncation 1e-8 at a step of 1e-4); the bf16 results are off by
    2^-8 of each term at most."""
    x = Grad(24, 384, 9)
    dg, du, _ = (t.double() for t in backward(cf, dev, x, fused=True))
    g, u, d = restored(x.g8, x.gd), restored(x.u8, x.ud), x.do.double()
    value = lambda g, u: (torch.sigmoid(g) * g * u * d).sum()  # noqa: E731
    gen = torch.Generator().manual_seed(4)
    for _ in range(4):
        a, b = (torch.randn(g.shape, generator=gen, dtype=torch.float64) for _ in range(2))
        slope = (value(g + 1e-4 * a, u + 1e-4 * b) - value(g - 1e-4 * a, u - 1e-4 * b)) / 2e-4
        assert abs((dg * a).sum() + (du * b).sum() - slope) <= (2.0 ** -8 + 1e-5) * ((dg * a).abs().sum() + (du * b).abs().sum())


@pytest.mark.parametrize("form", ["rows", "block", "record"])
def test_more_rows_than_one_launch_holds(cf, dev, form):
    """Rows of eight, 2^22 and a few: the last ones are as they are alone, forward and back."""
    rows, I, n = (1 << 22) + 7, 8, 500
    case(f"swiglu {form} {rows} rows of {I}")
    g, u = (torch.randn(rows, I, device=dev).to(torch.bfloat16) for _ in range(2))

    def run(g, u):
        R = g.shape[0]
        b, d = [torch.zeros(R, I, dtype=torch.uint8, device=dev) for _ in range(3)], [torch.zeros(R, 1, device=dev) for _ in range(4)]
        head, kept = (g, u, I, R, I), (b[0], d[0], b[1], d[1], b[2])
        if form == "record":
            cf.cf_swiglu_ckpt8_quantize_record(*head, 0, *kept, torch.full((1,), 20.0, device=dev), torch.zeros(1, device=dev), stream())
        elif form == "block":
            cf.cf_swiglu_ckpt8_quantize_block_1x128(*head, *kept, d[2], d[3], stream())
        else:
            cf.cf_swiglu_ckpt8_quantize_rows(*head, 0, *kept, d[2], d[3], stream())
        o = [torch.zeros(R, I, dtype=torch.bfloat16, device=dev) for _ in range(3)]
        cf.cf_swiglu_ckpt8_backward(u, b[0], d[0], b[1], d[1], R, I, o[0], o[1], I, o[2], stream())
        torch.cuda.synchronize()
        return b + d + o

    for whole, alone in zip(run(g, u), run(g[-n:].contiguous(), u[-n:].contiguous())):
        assert torch.equal(whole[-n:], alone)
