"""GPU: the residual layer where its paths are rare: rows with NaN and infinities in every form and kernel, gradients over several rows a workgroup whose last chunk
is a part or that take two chunks a thread, steps on two streams compared bit by bit.  Tolerances as in test_gpu_add_norm."""
import pytest
import torch

from gpu_util import case, stream
from test_gpu_add_norm import F8, STREAM, backward, check_backward, check_forward, forward, gamma_of, gradient_inputs, rows_of
from test_gpu_residual_layer import Layer

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
# four rows a workgroup, one chunk and two chunks a thread; multiples of eight and others
WIDTHS = [264, 511, 1000, 1001, 4096, 9001, 16384]


def bits(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


@pytest.mark.parametrize("form,e5m2", [("rows", 1), ("block", 0), ("record", 0), ("record", 1)])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("H", WIDTHS)
def test_a_row_that_is_not_finite_stays_by_itself(cf, dev, H, f32, form, e5m2):
    case(f"add-norm special rows {form} H={H} f32={f32} e5m2={e5m2}")
    r, x, w = rows_of(7, H, 5, STREAM[f32]), torch.zeros(7, H, dtype=torch.bfloat16), gamma_of(H, 6)
    r[1] = 0.0
    r[2, 17] = NAN
    r[3, H - 1] = INF
    r[4, 3] = -INF
    x[6, 100] = INF
    got = forward(cf, dev, r, x, w, f32, form, e5m2, qscale=7.0)
    keep = torch.tensor([0, 5])
    part = {k: v if k == "amax" else v[keep] for k, v in got.items()}
    check_forward(part, r[keep], x[keep], w, form, e5m2, 7.0)          # the recorded maximum too: it is that of the finite rows
    q = got["q"].view(F8[e5m2][0]).float()
    assert torch.all(q[1] == 0) and torch.all(got["normed"][1] == 0)
    assert torch.isnan(q[2]).all() and torch.isnan(got["rms"][2])
    for row, at in ((3, H - 1), (4, 3), (6, 100)):
        assert got["rms"][row] == INF
        assert torch.isnan(q[row, at]) and torch.all(q[row, :at] == 0) and torch.all(q[row, at + 1:] == 0)


@pytest.mark.parametrize("e5m2", [0, 1])
@pytest.mark.parametrize("H", WIDTHS)
def test_given_scales_that_are_not_finite(cf, dev, H, e5m2):
    """0 times infinity is NaN, everything else saturates; the recorded maximum does not depend on the scale."""
    case(f"add-norm record H={H} e5m2={e5m2}, scales of inf, NaN and 0")
    r, w = rows_of(4, H, 8, torch.bfloat16), gamma_of(H, 9)
    r[:, ::5] = 0.0
    zero, top = (r == 0), F8[e5m2][1]
    amax = None
    for scale in (INF, NAN, 0.0, 1.0):
        got = forward(cf, dev, r, None, w, 0, "record", e5m2, qscale=scale)
        q = got["q"].view(F8[e5m2][0]).float()
        if scale == INF:
            assert torch.isnan(q[zero]).all() and torch.equal(q[~zero], torch.sign(r.float() * w.float())[~zero] * top)
        elif scale != scale:
            assert torch.isnan(q).all()
        elif scale == 0.0:
            assert torch.all(q == 0)
        amax = amax or float(got["amax"])
        assert float(got["amax"]) == amax


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("rows,H", [(37, h) for h in WIDTHS] + [(2100, 511), (1300, 1001), (1100, 9001)])
def test_gradients_that_are_not_finite(cf, dev, rows, H, f32):
    """NaN and infinities of the stream's gradient stay in their element, those of the norm's gradient in their row and, in the weight's gradient, their column."""
    case(f"add-norm gradient special values rows={rows} H={H} f32={f32}")
    h, w, rms, dy, dh = gradient_inputs(rows, H, f32, 55)
    clean = backward(cf, dev, h, w, rms, dy, dh, f32, True, 1e4)
    last = rows - 1
    dh2, dy2 = dh.clone(), dy.clone()
    dh2[2, 17], dh2[last, H - 1] = NAN, NAN
    dy2[4, 9] = NAN
    got = backward(cf, dev, h, w, rms, dy2, dh2, f32, True, 1e4)
    bad = torch.zeros(rows, H, dtype=torch.bool)
    bad[2, 17] = bad[last, H - 1] = True
    bad[4] = True
    q = got["q"].view(torch.float8_e5m2).float()
    assert torch.isnan(got["dr"][bad]).all() and torch.isnan(q[bad]).all()
    assert torch.equal(bits(got["dr"])[~bad], bits(clean["dr"])[~bad]) and torch.equal(got["q"][~bad], clean["q"][~bad])
    others = torch.arange(H) != 9
    assert torch.isnan(got["dw"][9]) and torch.equal(bits(got["dw"])[others], bits(clean["dw"])[others])
    # the maximum is taken before the stream's type rounds: at most half a step of bf16 from that of the rounded gradient
    m = float(got["dr"][~bad].float().abs().max())
    assert abs(got["amax"] - m) <= 2.0 ** -8 * m and (f32 == 0 or got["amax"] == m)
    dh2 = dh.clone()
    dh2[2, 17], dh2[3, 5] = INF, -INF
    got = backward(cf, dev, h, w, rms, dy, dh2, f32, True, 1e4)
    q = got["q"].view(torch.float8_e5m2).float()
    assert got["amax"] == INF and (got["dr"][2, 17], got["dr"][3, 5]) == (INF, -INF) and (q[2, 17], q[3, 5]) == (57344.0, -57344.0)
    bad[:] = False
    bad[2, 17] = bad[3, 5] = True
    assert torch.equal(bits(got["dr"])[~bad], bits(clean["dr"])[~bad]) and torch.equal(got["q"][~bad], clean["q"][~bad]) and torch.equal(got["dw"], clean["dw"])


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("rows,H", [(4100, 100), (4099, 511), (2600, 1001), (1300, 4095), (1030, 7167), (1100, 8200), (1027, 9001), (769, 16384)])
def test_gradients_over_several_rows_a_workgroup(cf, dev, rows, H, f32, quant):
    case(f"add-norm gradient rows={rows} H={H} f32={f32} quant={quant}")
    h, w, rms, dy, dh = gradient_inputs(rows, H, f32, rows + H)
    start = torch.linspace(-1.0, 1.0, H)
    check_backward(backward(cf, dev, h, w, rms, dy, dh, f32, quant, 2e5), h, w, rms, dy, dh, quant, 2e5)
    check_backward(backward(cf, dev, h, w, rms, dy, dh, f32, quant, 2e5, start, 1, True), h, w, rms, dy, dh, quant, 2e5, start)


def test_two_streams_at_once_bit_by_bit(cf, dev):
    case("residual layer steps on two streams, all bits")
    layers = Layer(cf, dev, 200, 1024, 384, 8, 2, 1, 7), Layer(cf, dev, 333, 512, 256, 4, 2, 0, 8)
    for layer in layers:
        layer.step(stream())
    torch.cuda.synchronize()
    want = [{k: v.clone() for k, v in layer.outputs().items()} for layer in layers]
    assert not any(v.is_floating_point() and bool(torch.isnan(v).any()) for w in want for v in w.values())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, layer in zip(streams, layers):
            with torch.cuda.stream(s):
                layer.step(s.cuda_stream)
    torch.cuda.synchronize()
    for layer, w in zip(layers, want):
        for k, v in layer.outputs().items():
            assert torch.equal(bits(v), bits(w[k])), k
