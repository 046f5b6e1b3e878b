"""GPU: the norm of a list of gradients and the gradients clipped by it, against sums in 64 bits.

The norm is the fp32 rounding of a 64-bit root: off by 2^-24 of it, and by the 64-bit sum's 1e-12.  The coefficient follows from the norm that was
returned, and the clipped values from the coefficient, by one division and one product that are rounded as IEEE says: bit for bit."""
import ctypes

import numpy as np
import pytest
import torch

from gpu_util import case, stream

pytestmark = pytest.mark.gpu


def table(cf, dev, tensors, out=None):
    ptrs = torch.tensor([t.data_ptr() for t in tensors], dtype=torch.int64)
    outs = torch.tensor([t.data_ptr() for t in out], dtype=torch.int64) if out is not None else None
    counts = torch.tensor([t.numel() for t in tensors], dtype=torch.int64)
    types = torch.tensor([int(t.dtype == torch.float32) for t in tensors], dtype=torch.int32)
    n = ctypes.c_size_t(0)
    cf.cf_grad_list_bytes(counts, len(tensors), ctypes.byref(n))
    image = torch.zeros(n.value + 16, dtype=torch.uint8)
    cf.cf_grad_list_fill(ptrs, outs, counts, types, len(tensors), image, n.value)
    assert torch.all(image[n.value:] == 0)
    return image.to(dev), n.value


def workspace(cf, dev):
    n = ctypes.c_size_t(0)
    cf.cf_grad_norm_workspace_bytes(ctypes.byref(n))
    return torch.empty(n.value, dtype=torch.uint8, device=dev), n.value


def packed(dev, sizes, dtype, seed, sigma=1e-2, first=0):
    """Tensors back to back in one buffer, the first one `first` elements in, and the buffer."""
    g = torch.Generator().manual_seed(seed)
    buf = torch.full((first + sum(sizes) + 64,), 5.0).to(dtype)
    for at, n in zip(np.cumsum([first] + sizes[:-1]), sizes):
        buf[at:at + n] = (sigma * torch.randn(n, generator=g)).to(dtype)
    d = buf.to(dev)
    return [d[at:at + n] for at, n in zip(np.cumsum([first] + sizes[:-1]), sizes)], d


def reference_norm(tensors):
    return float(sum(t.cpu().double().square().sum() for t in tensors) ** 0.5) if tensors else 0.0


def check(cf, dev, tensors, max_norm, out=None):
    before = [t.cpu().clone() for t in tensors]
    ref = reference_norm(tensors)
    img, n = table(cf, dev, tensors, out)
    ws, wn = workspace(cf, dev)
    norm, coef = torch.full((1,), -1.0, device=dev), torch.full((1,), -1.0, device=dev)
    cf.cf_grad_norm_clip(img, n, max_norm, norm, coef, ws, wn, stream())
    torch.cuda.synchronize()
    got = np.float32(norm.item())
    if ref <= 3.4e38:
        assert abs(float(got) - ref) <= (2.0 ** -24 + 1e-11) * ref + 1e-45
    clips = np.isfinite(got) and got > np.float32(max_norm)
    c = np.float32(np.float64(np.float32(max_norm)) / np.float64(got)) if clips else np.float32(1.0)
    assert np.float32(coef.item()) == c
    for b, t in zip(before, out if out is not None else tensors):
        want = (b.float() * torch.tensor(c)).to(b.dtype)
        same = torch.equal(t.cpu().view(torch.int16 if b.dtype == torch.bfloat16 else torch.int32), want.view(torch.int16 if b.dtype == torch.bfloat16 else torch.int32))
        assert same or bool(torch.isnan(want).any()) and torch.equal(torch.isnan(want), torch.isnan(t.cpu()))
    if out is not None:
        for b, t in zip(before, tensors):
            assert torch.equal(b.view(torch.uint8), t.cpu().view(torch.uint8))
    return float(got), float(c)


SIZES = [[1], [5], [8], [256], [4096, 1, 7, 16384], [16385, 3, 0, 32768, 50000], [2] * 300, [300_001, 77], [1_000_003]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first", [0, 1, 3])
def test_in_place(cf, dev, sizes, dtype, first):
    case(f"grads {len(sizes)} tensors of up to {max(sizes)} {dtype} from element {first}")
    for max_norm in (1e-3, 1e6):
        tensors, buf = packed(dev, sizes, dtype, 3 + first, first=first)
        check(cf, dev, tensors, max_norm)
        assert bool((buf[:first] == 5).all()) and bool((buf[first + sum(sizes):] == 5).all())


@pytest.mark.parametrize("shift", [0, 1, 5])
def test_mixed_types_into_other_buffers(cf, dev, shift):
    """Outputs whose alignment differs from their inputs'."""
    sizes = [1000, 65537, 3, 4096, 20000]
    a, _ = packed(dev, sizes, torch.float32, 1)
    b, _ = packed(dev, sizes, torch.bfloat16, 2, sigma=0.3)
    oa, ba = packed(dev, sizes, torch.float32, 4, first=shift)
    ob, bb = packed(dev, sizes, torch.bfloat16, 5, first=shift)
    for max_norm in (0.5, 1e9):
        check(cf, dev, a + b, max_norm, oa + ob)
        for buf in (ba, bb):
            assert bool((buf[:shift] == 5).all()) and bool((buf[shift + sum(sizes):] == 5).all())


def test_magnitudes_whose_squares_leave_fp32(cf, dev):
    for sigma in (1e30, 1e-30, 3e18, 1e-40):
        case(f"grads of {sigma}")
        t, _ = packed(dev, [70_000, 11], torch.float32, 9, sigma=sigma)
        norm, _ = check(cf, dev, t, sigma)
        assert np.isfinite(norm) and norm > 0


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan"), 3e38])
def test_a_norm_that_is_not_finite_leaves_the_gradients(cf, dev, bad):
    t, _ = packed(dev, [50_000, 30], torch.float32, 8)
    for i in range(4):
        t[0][1000 + i] = bad
    norm, coef = check(cf, dev, t, 1.0)
    assert coef == 1.0 and not np.isfinite(norm) and np.isnan(norm) == np.isnan(bad)


def test_zero_gradients_an_empty_list_and_the_ends_of_max_norm(cf, dev):
    z, _ = packed(dev, [1000, 5], torch.float32, 8, sigma=0.0)
    assert check(cf, dev, z, 0.0) == (0.0, 1.0)
    t, _ = packed(dev, [1000, 5], torch.bfloat16, 8)
    assert check(cf, dev, t, float("inf"))[1] == 1.0
    assert check(cf, dev, t, 0.0)[1] == 0.0 and all(bool((x == 0).all()) for x in t)
    assert check(cf, dev, [], 1.0) == (0.0, 1.0)
    empty, _ = packed(dev, [0, 0], torch.float32, 1)
    assert check(cf, dev, empty, 1.0) == (0.0, 1.0)


def test_two_calls_give_what_one_gives(cf, dev):
    sizes = [123_457, 9, 70_000]
    a, _ = packed(dev, sizes, torch.float32, 6)
    b, _ = packed(dev, sizes, torch.float32, 6)
    ws, wn = workspace(cf, dev)
    ia, n = table(cf, dev, a)
    ib, _ = table(cf, dev, b)
    norm, coef = torch.zeros(2, device=dev), torch.zeros(2, device=dev)
    cf.cf_grad_norm_clip(ia, n, 0.25, norm[:1], coef[:1], ws, wn, stream())
    cf.cf_grad_norm(ib, n, norm[1:], ws, wn, stream())
    cf.cf_grad_clip(ib, n, 0.25, norm[1:], coef[1:], stream())
    torch.cuda.synchronize()
    assert norm[0] == norm[1] and coef[0] == coef[1] and coef[0] < 1
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # a list is read, not consumed; the order of the sum is its own
    again = torch.zeros(1, device=dev)
    for _ in range(3):
        cf.cf_grad_norm(ib, n, again, ws, wn, stream())
        first = again.item()
        cf.cf_grad_norm(ib, n, again, ws, wn, stream())
        assert again.item() == first


def test_more_elements_than_32_bits_count(cf, dev):
    n = (1 << 31) + 12_345
    t = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    t[0], t[n // 2], t[-1] = 3.0, 4.0, 12.0
    img, size = table(cf, dev, [t])
    ws, wn = workspace(cf, dev)
    norm, coef = torch.zeros(1, device=dev), torch.zeros(1, device=dev)
    cf.cf_grad_norm_clip(img, size, 6.5, norm, coef, ws, wn, stream())
    torch.cuda.synchronize()
    assert norm.item() == 13.0 and coef.item() == 0.5
    assert (t[0].item(), t[n // 2].item(), t[-1].item()) == (1.5, 2.0, 6.0)
