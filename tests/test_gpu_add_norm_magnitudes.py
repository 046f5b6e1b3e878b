"""GPU: residual addition + RMS norm of rows whose squares leave fp32, and the gradient with the rms they left, against the formulas in 64 bits.

Tolerances as in test_gpu_add_norm: scaling a row by a power of two rounds nothing, but for elements so far below the row's largest that they count for nothing.  The
magnitudes keep rms among the normal fp32 numbers, so that its own rounding is relative."""
import pytest
import torch

import test_gpu_add_norm as base
from gpu_util import case
from test_gpu_add_norm import STREAM, backward, check_backward, check_forward, forward, gamma_of, rows_of

pytestmark = pytest.mark.gpu

# the sizes: four rows a workgroup, one chunk and two a thread; multiples of eight and others
SIZES = [(9, 264), (6, 511), (5, 1032), (7, 4095), (3, 9001), (2, 16384)]


def rows_at(rows, H, f32, size, seed):
    """Rows of magnitude `size` between rows of ordinary ones."""
    r, x = rows_of(rows, H, seed, STREAM[f32]).float(), rows_of(rows, H, seed + 1, torch.bfloat16, 0.5).float()
    r[1::2] *= size
    x[1::2] *= size
    keep = lambda t: t.clamp(-1e38, 1e38)
    return keep(r).to(STREAM[f32]), keep(x).to(torch.bfloat16), gamma_of(H, seed + 2)


@pytest.mark.parametrize("form,e5m2", base.FORMS)
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("size,eps", [(1e17, 1e-6), (1e19, 1e-6), (1e25, 1e-6), (1e37, 1e-6), (1e37, 0.0), (1e-13, 0.0), (1e-17, 0.0), (1e-25, 0.0), (1e-33, 0.0),
                                      (1e-17, 1e-36), (1e-25, 1e-36), (1e-25, 1e-6)])
def test_forward_of_large_and_small_rows(cf, dev, monkeypatch, size, eps, f32, form, e5m2):
    monkeypatch.setattr(base, "EPS", eps)
    for rows, H in SIZES:
        case(f"add-norm {form} rows={rows} H={H} of {size} eps={eps} f32={f32} e5m2={e5m2}")
        r, x, w = rows_at(rows, H, f32, size, H)
        got = forward(cf, dev, r, x, w, f32, form, e5m2, qscale=12.5)
        check_forward(got, r, x, w, form, e5m2, 12.5)


@pytest.mark.parametrize("f32", [0, 1])
def test_rows_of_zeros_under_a_small_eps(cf, dev, monkeypatch, f32):
    monkeypatch.setattr(base, "EPS", 1e-36)
    for rows, H in SIZES:
        r, x, w = rows_at(rows, H, f32, 0.0, H)
        check_forward(forward(cf, dev, r, x, w, f32, "rows", 0), r, x, w, "rows", 0)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("size", [1e25, 1e36, 1e-25])
def test_gradient_with_the_rms_of_the_forward_pass(cf, dev, monkeypatch, size, f32, quant):
    monkeypatch.setattr(base, "EPS", 0.0)
    for rows, H in SIZES:
        case(f"add-norm gradient rows={rows} H={H} of {size} f32={f32} quant={quant}")
        r, x, w = rows_at(rows, H, f32, size, H)
        fwd = forward(cf, dev, r, x, w, f32, "rows", 0)
        g = torch.Generator().manual_seed(H)
        dy = (1e-2 * size * torch.randn(rows, H, generator=g)).to(torch.bfloat16)         # so that dy / rms stays a normal number
        got = backward(cf, dev, fwd["sum"], w, fwd["rms"], dy, None, f32, quant, 1.0)
        check_backward(got, fwd["sum"], w, fwd["rms"], dy, None, quant, 1.0)


@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("size", [3e-38, 1e-39, 1e-40, 3e38])
def test_forward_of_rows_at_the_ends_of_the_type(cf, dev, monkeypatch, size, f32):
    """Rows of subnormal numbers without eps, rows up to the largest number: y and the bytes are as for any other row; rms, where it is subnormal itself, is off by
    half of a subnormal step, 2^-150, at most."""
    monkeypatch.setattr(base, "EPS", 0.0)
    for rows, H in SIZES:
        case(f"add-norm rows={rows} H={H} up to {size} f32={f32}")
        g = torch.Generator().manual_seed(H)
        r, x = size * (2 * torch.rand(rows, H, generator=g, dtype=torch.float64) - 1), 0.0 * torch.rand(rows, H, generator=g, dtype=torch.float64)
        x[:, ::3] = r[:, ::3] * -0.5
        r, x, w = r.to(STREAM[f32]), x.to(torch.bfloat16), gamma_of(H, H + 2)
        r[0, 0] = size
        x[0, 0] = 0.0
        got = forward(cf, dev, r, x, w, f32, "rows", 0)
        h = (r.float() + x.float()).to(r.dtype)
        assert torch.equal(got["sum"], h) and bool(torch.isfinite(h).all())
        rms = h.double().square().mean(1).sqrt()
        assert torch.all((got["rms"].double() - rms).abs() <= base.R * rms + 2.0 ** -150)
        got["rms"] = torch.where(rms < 2.0 ** -126, rms, got["rms"].double())          # looked at above
        check_forward(got, r, x, w, "rows", 0)
