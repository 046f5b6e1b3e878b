"""GPU: the block output's root mean square is the formula's in fp32: the mean of the squares from a 64-bit sum, eps and the root, one rounding each.  Bit for bit: bf16 squares have
sixteen bits, and a sum in 64 bits is off by H 2^-53 at most, too little to move the rounding of the mean for any of these rows.  The root in fp32 is the 64-bit one rounded, which is the
correctly rounded one, as 53 >= 2 x 24 + 2; torch's fp32 root on the CPU is not everywhere (6503 of a million random ones were a unit off)."""
import pytest
import torch

from gpu_util import case
from test_gpu_add_norm import EPS
from test_gpu_gated_norm import Layer, forward

pytestmark = pytest.mark.gpu


def root(mean):
    assert mean.dtype == torch.float32
    return mean.double().sqrt().float()


@pytest.mark.parametrize("form", ["rows", "block", "record"])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("rows,H", [(600, 200), (300, 511), (900, 1024), (300, 2050), (900, 4096), (300, 5120), (600, 7168), (200, 9001), (200, 12288), (300, 16384)])
def test_post_rms_is_the_formulas(cf, dev, rows, H, f32, form):
    case(f"gated norm {form} px rows={rows} H={H} f32={f32}")
    a = Layer(rows, H, f32, 0, seed=rows + H)
    got = forward(cf, dev, a, form)
    mean = (a.x.double().square().sum(1) / H).float()
    assert torch.equal(got["post_rms"], root(mean + torch.tensor(EPS)))


@pytest.mark.parametrize("H", [200, 4096, 9001])
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** 70, 2.0 ** 110])
def test_far_rows_too(cf, dev, H, size):
    """Rows whose squares leave fp32 are scaled by a power of two first, under which the roundings are the same; eps lies far below or far above them."""
    case(f"gated norm px H={H} size={size}")
    a = Layer(50, H, 1, 0, seed=H)
    a.x = (a.x.float() * size).to(torch.bfloat16)
    got = forward(cf, dev, a, "rows")
    if size < 1:
        want = root((a.x.double().square().sum(1) / H).float() + torch.tensor(EPS))
    else:
        want = root((a.x.double().div(size).square().sum(1) / H).float()) * size
    assert torch.equal(got["post_rms"], want)
