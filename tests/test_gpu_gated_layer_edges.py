"""GPU: the gated norm, the gated activation in 8 bits and their gradients where NaN and infinities lie, in every form and width class: they stay in their rows or elements, and a recorded
maximum is that of the rest.  Tolerances as in test_gpu_gated_norm and test_gpu_swiglu_ckpt."""
import pytest
import torch

from gpu_util import case
from test_gpu_add_norm import F8
from test_gpu_gated_norm import FORMS, Grad, Layer, backward, check_forward, forward
from test_gpu_swiglu_ckpt import FORMS as KEEP_FORMS
from test_gpu_swiglu_ckpt import activation, checkpoint, check_quantized, forward as keep, inputs

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
E4M3 = torch.float8_e4m3fn
# four rows a workgroup, one chunk, two and four a thread; multiples of eight and others
WIDTHS = [264, 511, 1000, 1001, 4096, 5120, 9001, 16384]


def bits(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


@pytest.mark.parametrize("form,e5m2", FORMS)
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("H", WIDTHS)
def test_a_row_that_is_not_finite_stays_by_itself(cf, dev, H, f32, form, e5m2):
    case(f"gated norm special rows {form} H={H} f32={f32} e5m2={e5m2}")
    a = Layer(9, H, f32, 2, seed=H)
    a.r[1], a.x[1] = 0.0, 0.0
    a.r[2, 17] = NAN
    a.r[3, H - 1], a.r[4, 3] = INF, -INF
    a.x[6, 100] = INF
    a.x[7, 0] = NAN
    got = forward(cf, dev, a, form, e5m2)
    fine = torch.tensor([0, 5, 8])
    b = Layer(3, H, f32, 0)
    b.r, b.x, b.wp, b.w, b.gate, b.gate_rows = a.r[fine], a.x[fine], a.wp, a.w, a.gate[fine // 2], 1
    check_forward({k: v if k == "amax" else v[fine] for k, v in got.items()}, b, form, e5m2)          # the recorded maximum too: it is that of the finite rows
    q, x8, sum8 = (got[k].view(t).float() for k, t in (("q", F8[e5m2][0]), ("x8", E4M3), ("sum8", E4M3)))
    assert torch.all(q[1] == 0) and torch.all(x8[1] == 0) and torch.all(sum8[1] == 0) and torch.all(got["normed"][1] == 0)
    for row in (2, 6, 7):               # a NaN, or an infinity of the block's output, whose own quotient is a NaN, in the second norm
        assert torch.isnan(q[row]).all() and torch.isnan(sum8[row]).all() and torch.isnan(got["rms"][row])
    assert not torch.isnan(x8[[2, 3, 4]]).any() and torch.isnan(x8[7]).all()
    assert torch.isnan(x8[6, 100]) and torch.all(x8[6, :100] == 0) and torch.all(x8[6, 101:] == 0) and got["post_rms"][6] == INF
    for row, at in ((3, H - 1), (4, 3)):
        assert got["rms"][row] == INF
        for t in (q, sum8):
            assert torch.isnan(t[row, at]) and torch.all(t[row, :at] == 0) and torch.all(t[row, at + 1:] == 0)


@pytest.mark.parametrize("e5m2", [0, 1])
@pytest.mark.parametrize("H", WIDTHS)
def test_given_scales_that_are_not_finite(cf, dev, H, e5m2):
    """0 times infinity is NaN, everything else saturates; the recorded maximum does not depend on the scale."""
    case(f"gated norm record H={H} e5m2={e5m2}, scales of inf, NaN and 0")
    a = Layer(4, H, 0, 0, seed=8)
    a.r[:, ::5] = 0.0
    a.x[:, ::5] = 0.0
    amax = None
    for scale in (INF, NAN, 0.0, 1.0):
        got = forward(cf, dev, a, "record", e5m2, qscale=scale)
        q, y = got["q"].view(F8[e5m2][0]).float(), got["normed"].float()
        if scale == INF:
            assert torch.isnan(q[y == 0]).all() and torch.equal(q[y != 0], torch.sign(y[y != 0]) * F8[e5m2][1])
        elif scale != scale:
            assert torch.isnan(q).all()
        elif scale == 0.0:
            assert torch.all(q == 0)
        amax = amax or got["amax"]
        assert got["amax"] == amax


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("rows,H,gate_rows", [(37, h, 5) for h in WIDTHS] + [(2100, 511, 0), (2100, 264, 300), (1300, 1001, 1300), (520, 4100, 7), (520, 7168, 100), (300, 9001, 7),
                                              (515, 12288, 0), (300, 16384, 2)])
def test_gradients_that_are_not_finite(cf, dev, rows, H, gate_rows, f32, kept):
    """A NaN of the norm's gradient or of the stream's stays in its row, where the first also reaches the stream's gradient whole; the maximum is that of the other rows.  An infinity is recorded."""
    case(f"gated norm gradient special values rows={rows} H={H} gate_rows={gate_rows} f32={f32} kept={kept}")
    g = Grad(rows, H, f32, gate_rows, kept=kept, seed=55)
    loud = torch.arange(rows) % 3 == 1
    g.dy[loud], g.dh[loud] = g.dy[loud] * 4, g.dh[loud] * 4
    clean = backward(cf, dev, g, qscale=1e3)
    last = rows - 1
    dy, dh = g.dy, g.dh
    g.dy, g.dh = dy.clone(), dh.clone()
    g.dy[4, 9] = NAN
    g.dh[2, 17], g.dh[last, H - 1] = NAN, NAN
    got = backward(cf, dev, g, qscale=1e3)
    bad = torch.zeros(rows, dtype=torch.bool)
    bad[[2, 4, last]] = True
    for k in ("dr", "dx", "q"):
        assert torch.equal(bits(got[k])[~bad], bits(clean[k])[~bad]), k
    assert torch.isnan(got["dr"][4]).all() and torch.isnan(got["dr"][2, 17]) and torch.isnan(got["dr"][last, H - 1])
    others = torch.arange(H) != 17
    assert torch.equal(bits(got["dr"][2][others]), bits(clean["dr"][2][others]))
    # a zero gate keeps no NaN out: the row's mean has it
    assert torch.isnan(got["dx"][bad]).all() and torch.isnan(got["q"].view(torch.float8_e5m2).float()[bad]).all()
    # the maximum is taken before dx is rounded: half a step of bf16 from that of the rounded one at most
    m = float(got["dx"][~bad].float().abs().max())
    assert abs(got["amax"] - m) <= 2.0 ** -8 * m
    others = torch.arange(H) != 9
    assert torch.isnan(got["dw"][9]) and torch.equal(bits(got["dw"])[others], bits(clean["dw"])[others])
    assert torch.isnan(got["dwp"]).all()
    g.dy, g.dh = dy, dh.clone()
    g.dh[2, 17] = -INF
    got = backward(cf, dev, g, qscale=1e3)
    bad[:] = False
    bad[2] = True
    assert got["amax"] == INF and got["dr"][2, 17] == -INF and torch.equal(bits(got["dr"][2][torch.arange(H) != 17]), bits(clean["dr"][2][torch.arange(H) != 17]))
    for k in ("dr", "dx", "q"):
        assert torch.equal(bits(got[k])[~bad], bits(clean[k])[~bad]), k
    assert torch.equal(bits(got["dw"]), bits(clean["dw"]))


@pytest.mark.parametrize("form,e5m2", KEEP_FORMS)
@pytest.mark.parametrize("rows,I", [(9, 96), (9, 511), (9, 1000), (9, 5461), (9, 9001), (9, 17001), (9, 32768), (2100, 1001)])
def test_activations_that_are_not_finite(cf, dev, rows, I, form, e5m2):
    """A NaN stays in its element of the operand and of its checkpoint, and out of every maximum; an infinity takes its group of the checkpoint with it, and its row or group of the operand."""
    case(f"swiglu special values {form} rows={rows} I={I} e5m2={e5m2}")
    g, u = inputs(rows, I, I)
    last = rows - 1
    g[1], u[1] = 0.0, 0.0
    g[2, 17], u[3, I - 1], g[last, 40] = NAN, NAN, NAN
    got = keep(cf, dev, g, u, form, e5m2)
    dtype, top = F8[e5m2][:2]
    bad = torch.zeros(rows, I, dtype=torch.bool)
    bad[2, 17] = bad[3, I - 1] = bad[last, 40] = True
    q = got["q"].view(dtype).float()
    assert torch.equal(torch.isnan(q), bad) and torch.all(q[1] == 0)
    zeroed = lambda t: torch.where(torch.isnan(t), torch.zeros_like(t), t)  # noqa: E731
    for name, t in (("gate8", g), ("up8", u)):
        want, d = checkpoint(zeroed(t))
        assert torch.equal(got[name + "_descale"], d) and torch.equal(got[name][~torch.isnan(t)], want.view(torch.uint8)[~torch.isnan(t)])
        assert torch.isnan(got[name].view(E4M3).float()[torch.isnan(t)]).all()
    # with zeros in place of the NaNs' activations everything else is as the formula has it, maxima too
    got["q"] = torch.where(bad, torch.zeros_like(got["q"]), got["q"])
    a, off = activation(zeroed(g), zeroed(u))
    check_quantized(got, torch.where(bad, torch.zeros_like(a), a), off, form, e5m2, 3.0)
    g[5, 70], u[5, 70] = INF, -1.0
    inf = keep(cf, dev, g, u, form, e5m2)
    q5 = inf["q"].view(dtype).float()[5]
    row = torch.arange(rows) != 5
    same = ["gate8", "gate8_descale", "up8", "up8_descale", "q"] + ([] if form == "record" else ["scale", "descale"])
    again = keep(cf, dev, *(torch.where(row[:, None], t, torch.zeros_like(t)) for t in (g, u)), form, e5m2)
    assert all(torch.equal(bits(inf[k][row]), bits(again[k][row])) for k in same)
    assert torch.isnan(inf["gate8"].view(E4M3).float()[5, 70]) and inf["gate8_descale"][5, 0] == INF
    if form == "record":
        assert inf["amax"] == INF and q5[70] == -top
    else:
        assert torch.isnan(q5[70]) and (inf["descale"][5] if form == "rows" else inf["descale"][5, 0]) == INF
        group = torch.arange(I) // 128 == 0 if form == "block" else torch.ones(I, dtype=torch.bool)
        group[70] = False
        assert torch.all(q5[group] == 0)
