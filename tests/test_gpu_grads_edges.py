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


@pytest.mark.parametrize("sigma", [1e30, 1e-30, 1.0])
def test_a_norm_over_two_lists_joined_in_64_bits(cf, dev, sigma):
    """As over two GPUs: each list's norm, the root of the sum of their squares in 64 bits, both lists clipped by it.  The two norms and the joined one are each rounded
    once: 2^-24 of the norm from each (the squares of the two halve theirs on average, at most they add up to one), twice in all."""
    case(f"grads of {sigma} in two lists")
    lists = [packed(dev, sizes, torch.float32, seed, sigma=sigma)[0] for seed, sizes in ((1, [70_000, 11]), (2, [123_457, 5, 9000]))]
    exact = float(sum(x.double().square().sum() for t in lists for x in t).sqrt())
    before = [[x.clone() for x in t] for t in lists]
    tables = [table(cf, dev, t) for t in lists]
    ws, wn = workspace(cf, dev)
    norms, coefs = torch.zeros(2, device=dev), torch.zeros(2, device=dev)
    for i, (img, n) in enumerate(tables):
        cf.cf_grad_norm(img, n, norms[i:], ws, wn, stream())
    joined = norms.double().square().sum().sqrt().float().reshape(1)
    for i, (img, n) in enumerate(tables):
        cf.cf_grad_clip(img, n, sigma, joined, coefs[i:], stream())
    torch.cuda.synchronize()
    assert abs(joined.item() - exact) <= 2 * 2.0 ** -24 * exact
    assert coefs[0] == coefs[1] < 1
    for t, b in zip(lists, before):
        assert all(torch.equal(x, y * coefs[0]) for x, y in zip(t, b))
