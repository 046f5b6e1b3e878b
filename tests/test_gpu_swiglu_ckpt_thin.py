"""GPU: the 8-bit gradient of the gated activation over more 128 x 128 tiles than one launch holds, which thin shapes come to at 2^30 elements.  The tiles at both ends give, bit for bit,
what they give alone; between them are zeros, and the recorded maximum is that of the two ends."""
import pytest
import torch

from gpu_util import case, stream

pytestmark = pytest.mark.gpu

QSCALE, ACT_SCALE = 1e4, 8.0


def backward(cf, dev, do, g8, gd, u8, ud):
    rows, I = do.shape
    o = [torch.full((rows, 2 * I), 77, dtype=torch.uint8, device=dev), torch.full((2 * I, rows), 77, dtype=torch.uint8, device=dev),
         torch.full((I, rows), 77, dtype=torch.uint8, device=dev)]
    amax = torch.zeros(1, device=dev)
    cf.cf_swiglu_ckpt8_backward_quant_e5m2(do, g8, gd, u8, ud, rows, I, o[0], o[1], torch.full((1,), QSCALE, device=dev), amax, o[2], torch.full((1,), ACT_SCALE, device=dev), stream())
    return o, amax


# one row of nearly 2^30 elements, and rows of one element: 2^23 and some more tiles, a whole launch and a few
@pytest.mark.parametrize("rows,I", [(1, (1 << 30) - 1), ((1 << 30) + 200, 1)])
def test_more_tiles_than_one_launch_holds(cf, dev, rows, I):
    case(f"swiglu 8-bit gradient {rows} x {I}")
    n, wide = 1024, I > 1
    ends = [slice(0, n), slice((max(rows, I) - n) // 128 * 128, max(rows, I))]         # both begin where a tile does
    g = torch.Generator(device=dev).manual_seed(3)
    do = torch.zeros(rows, I, dtype=torch.bfloat16, device=dev)
    g8, u8 = (torch.zeros(rows, I, dtype=torch.uint8, device=dev) for _ in range(2))
    gd, ud = (torch.zeros(rows, (I + 127) // 128, device=dev) for _ in range(2))
    alone = []
    for end in ends:
        at = (slice(None), end) if wide else (end, slice(None))
        groups = (slice(None), slice(end.start // 128, None if end.stop == I else end.stop // 128)) if wide else at
        shape = do[at].shape
        do[at] = torch.randn(shape, device=dev, generator=g).to(torch.bfloat16)
        for t in (g8, u8):
            t[at] = torch.randn(shape, device=dev, generator=g).mul_(100.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
        for t in (gd, ud):
            t[groups] = torch.rand(t[groups].shape, device=dev, generator=g).mul_(0.02)
        parts = [t[at].contiguous() for t in (do, g8)] + [gd[groups].contiguous(), u8[at].contiguous(), ud[groups].contiguous()]
        alone.append(backward(cf, dev, *parts))
    (grad, grad_t, act_t), amax = backward(cf, dev, do, g8, gd, u8, ud)
    torch.cuda.synchronize()
    assert float(amax) == max(float(a) for _, a in alone) > 0
    for end, ((one, one_t, one_act), _) in zip(ends, alone):
        length = end.stop - end.start
        if wide:
            assert torch.equal(grad[0, end], one[0, :length]) and torch.equal(grad[0, I + end.start:I + end.stop], one[0, length:])
            assert torch.equal(grad_t[end], one_t[:length]) and torch.equal(grad_t[I + end.start:I + end.stop], one_t[length:]) and torch.equal(act_t[end], one_act)
        else:
            assert torch.equal(grad[end], one) and torch.equal(grad_t[:, end], one_t) and torch.equal(act_t[:, end], one_act)
    for lines in (grad.view(2, I), grad_t.view(2, I), act_t.view(1, I)) if wide else (grad.t(), grad_t, act_t):
        assert not bool(lines[:, n:ends[1].start].any())


@pytest.mark.parametrize("form", ["block", "record"])
@pytest.mark.parametrize("rows,I", [(1, (1 << 30) - 1), ((1 << 30) + 200, 1)])
def test_the_other_forms_run_there(cf, dev, rows, I, form):
    """The forward pass and the bf16 gradient of the same sizes: their ends as alone."""
    case(f"swiglu {form} {rows} x {I}")
    n, wide = 1024, I > 1
    ends = [slice(0, n), slice((max(rows, I) - n) // 128 * 128, max(rows, I))]
    gen = torch.Generator(device=dev).manual_seed(4)
    at = lambda end: (slice(None), end) if wide else (end, slice(None))  # noqa: E731
    slots = lambda end: (slice(None), slice(end.start // 128, -(-end.stop // 128))) if wide else at(end)  # noqa: E731
    g, u, do = (torch.zeros(rows, I, dtype=torch.bfloat16, device=dev) for _ in range(3))
    for end in ends:
        for t in (g, u, do):
            t[at(end)] = torch.randn(t[at(end)].shape, device=dev, generator=gen).to(torch.bfloat16)

    def run(g, u, do):
        rows, I = g.shape
        G = (I + 127) // 128
        b8, d = [torch.zeros(rows, I, dtype=torch.uint8, device=dev) for _ in range(3)], [torch.zeros(rows, G, device=dev) for _ in range(4 if form == "block" else 2)]
        amax = torch.zeros(1, device=dev)
        if form == "block":
            cf.cf_swiglu_ckpt8_quantize_block_1x128(g, u, I, rows, I, b8[0], d[0], b8[1], d[1], b8[2], d[2], d[3], stream())
        else:
            cf.cf_swiglu_ckpt8_quantize_record(g, u, I, rows, I, 0, b8[0], d[0], b8[1], d[1], b8[2], torch.full((1,), ACT_SCALE, device=dev), amax, stream())
        o = [torch.zeros(rows, I, dtype=torch.bfloat16, device=dev) for _ in range(3)]
        cf.cf_swiglu_ckpt8_backward(do, b8[0], d[0], b8[1], d[1], rows, I, o[0], o[1], I, o[2], stream())
        torch.cuda.synchronize()
        return b8 + o, d, float(amax)

    values, scales, amax = run(g, u, do)
    most = 0.0
    for end in ends:
        v, s, m = run(*(t[at(end)].contiguous() for t in (g, u, do)))
        most = max(most, m)
        assert all(torch.equal(a[at(end)], b) for a, b in zip(values, v)) and all(torch.equal(a[slots(end)], b) for a, b in zip(scales, s))
    assert amax == most
