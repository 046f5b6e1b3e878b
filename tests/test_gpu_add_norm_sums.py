"""GPU: the sum over the rows in the norm weight's gradient is taken in 64 bits, but for one rounding of each workgroup's share.

h and dy are powers of two times small integers and rms is 1, so every term dy * h is exact: c * 2^24 in the first sixteenth of the rows, c in the others, c in 1..7 by
column.  64 bits hold all sums exactly.  Rounding the shares loses at most 2^-24 of the sum of their sizes, which is the sum itself as all terms have one sign, and the last
rounding 2^-24 of it: 2^-23 in all.  That is an eighth of the rows times c; sums in 32 bits, where each small row falls under half a unit of the large ones before it,
lose fifteen sixteenths."""
import pytest
import torch

from gpu_util import case
from test_gpu_add_norm import STREAM, backward

pytestmark = pytest.mark.gpu


def inputs(rows, H, f32):
    power = torch.ones(rows, 1)
    power[:rows // 16] = 2.0 ** 12
    column = (torch.arange(H) % 7 + 1).float()
    h, dy = (column * power).to(STREAM[f32]), (torch.ones(rows, H) * power).to(torch.bfloat16)
    return h, torch.ones(H).to(torch.bfloat16), torch.ones(rows), dy, None


# up to 512 columns four rows share a workgroup, up to 8192 a thread holds a chunk of a row, beyond it two; multiples of eight and others; all with several
# rows a workgroup
SHAPES = [(40000, 64), (20000, 511), (20000, 512), (17000, 264), (16500, 1000), (17000, 1001), (4200, 4095), (4200, 2048 + 4), (5000, 7168), (4200, 9001), (4100, 16384)]


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("rows,H", SHAPES)
def test_rows_are_summed_in_64_bits(cf, dev, rows, H, f32, quant):
    case(f"add-norm gradient sums rows={rows} H={H} f32={f32} quant={quant}")
    h, w, rms, dy, dh = inputs(rows, H, f32)
    exact = (h.double() * dy.double()).sum(0)
    got = backward(cf, dev, h, w, rms, dy, dh, f32, quant)["dw"].double()
    assert torch.all((got - exact).abs() <= 2.0 ** -23 * exact)
    start = torch.linspace(0.0, 1e9, H)
    total = exact + start.double()
    got = backward(cf, dev, h, w, rms, dy, dh, f32, quant, start=start)["dw"].double()
    assert torch.all((got - total).abs() <= 2.0 ** -24 * (exact + total))
