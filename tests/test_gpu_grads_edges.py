"""GPU: gradients whose norm is not finite stay as they are, bit for bit, in place and in other buffers."""
import pytest
import torch

from gpu_util import case, stream
from test_gpu_grads import packed, table, workspace

pytestmark = pytest.mark.gpu


def bits(t):
    return t.cpu().view(torch.int16 if t.dtype == torch.bfloat16 else torch.int32)


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), 3e38])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("elsewhere", [False, True])
def test_a_norm_that_is_not_finite(cf, dev, bad, dtype, elsewhere):
    case(f"grads {dtype} with {bad}, into other buffers: {elsewhere}")
    sizes = [50_000, 30, 17_001]
    t, _ = packed(dev, sizes, dtype, 8, first=1)
    for i in range(4):
        t[2][1000 + i] = bad
    out = packed(dev, sizes, dtype, 9, first=3)[0] if elsewhere else t
    before = [bits(x).clone() for x in t]
    img, n = table(cf, dev, t, out if elsewhere else None)
    ws, wn = workspace(cf, dev)
    norm, coef = torch.zeros(1, device=dev), torch.zeros(1, device=dev)
    cf.cf_grad_norm_clip(img, n, 0.25, norm, coef, ws, wn, stream())
    torch.cuda.synchronize()
    assert coef.item() == 1.0 and not torch.isfinite(norm).item()
    for b, x, y in zip(before, t, out):
        assert torch.equal(bits(x), b)
        nan = torch.isnan(y.cpu())
        assert torch.equal(bits(y)[~nan], b[~nan]) and torch.equal(nan, torch.isnan(x.cpu()))
