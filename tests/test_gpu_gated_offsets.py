"""GPU: tensors whose elements and bytes are counted beyond 32 bits.  The rows at the end give, bit for bit, what they give alone; the rest are zeros, so that the sums over rows are
those rows' too."""
import ctypes

import pytest
import torch

from gpu_util import case, stream

pytestmark = pytest.mark.gpu

EPS = 1e-6
U = 2.0 ** -24


def put_at_the_end(t, rows):
    """Zeros with the rows of t at the end."""
    big = torch.zeros(rows, t.shape[1], dtype=t.dtype, device=t.device)
    big[rows - t.shape[0]:] = t
    return big


def test_gated_norm_and_its_gradient(cf, dev):
    rows, H, n = 270_000, 8192, 300          # 2.2e9 elements; as many rows alone as take the same kernel
    case(f"gated norm {rows} x {H}")
    g = torch.Generator(device=dev).manual_seed(1)
    bf = lambda *s: torch.randn(*s, device=dev, generator=g).to(torch.bfloat16)  # noqa: E731
    r, x, dy, dh, w, wp, gate = bf(n, H), bf(n, H), bf(n, H), bf(n, H), bf(H), bf(H), bf(1, H)

    def forward(r, x):
        R = r.shape[0]
        o = [torch.empty_like(r), torch.empty(R, device=dev), torch.empty(R, device=dev)] + [torch.empty(R, H, dtype=torch.uint8, device=dev) for _ in range(3)] + \
            [torch.empty(R, device=dev) for _ in range(2)]
        cf.cf_gated_add_rmsnorm_quantize_rows(r, x, 0, 1.25, gate, R, wp, w, R, H, EPS, 0, o[0], None, *o[1:], stream())
        return o

    def backward(dy, dh, h8, x8, rms, prms):
        R = dy.shape[0]
        size = ctypes.c_size_t(0)
        cf.cf_gated_add_rmsnorm_backward_workspace_bytes(R, H, R, ctypes.byref(size))
        ws, qs, amax = torch.empty(size.value, dtype=torch.uint8, device=dev), torch.full((1,), 1e3, device=dev), torch.zeros(1, device=dev)
        o = [torch.empty_like(dh), torch.empty_like(dy), torch.empty(R, H, dtype=torch.uint8, device=dev)]
        sums = [torch.empty(H, device=dev), torch.empty(H, device=dev), torch.empty(1, H, device=dev)]
        cf.cf_gated_add_rmsnorm_backward_ckpt8(dy, h8, x8, 0, 1.25, gate, R, wp, w, prms, rms, dh, R, H, *o, qs, amax, *sums, 0, ws, size.value, stream())
        return o, sums, amax

    small, big = forward(r, x), forward(put_at_the_end(r, rows), put_at_the_end(x, rows))
    torch.cuda.synchronize()
    for a, b in zip(small, big):
        assert torch.equal(a, b[rows - n:])
    assert not bool(big[3][: rows - n].any()) and bool((big[1][: rows - n] > 0).all())
    _, prms, rms, x8, h8 = small[:5]
    want, want_sums, want_amax = backward(dy, dh, h8, x8, rms, prms)
    got, sums, amax = backward(put_at_the_end(dy, rows), put_at_the_end(dh, rows), big[4], big[3], big[2], big[1])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b[rows - n:])
    assert torch.equal(want_amax, amax)
    # the same terms in other shares: each is rounded once, and so is the sum
    for a, b in zip(want_sums, sums):
        assert float((a.double() - b.double()).abs().max()) <= 4 * U * n * float(a.abs().max())


def test_swiglu_and_its_gradient(cf, dev):
    rows, I, n = 140_032, 16384, 112          # 2.3e9 elements, 4.6e9 bytes of gradients; a last tile of 112 rows that begins inside the zeros' tiles
    case(f"swiglu {rows} x {I}")
    g = torch.Generator(device=dev).manual_seed(2)
    bf = lambda *s: torch.randn(*s, device=dev, generator=g).to(torch.bfloat16)  # noqa: E731
    gate, up, do = bf(n, I), bf(n, I), bf(n, I)
    qs, aqs = torch.full((1,), 1e3, device=dev), torch.full((1,), 8.0, device=dev)

    def forward(a, b):
        R = a.shape[0]
        u8 = [torch.empty(R, I, dtype=torch.uint8, device=dev) for _ in range(3)]
        d = [torch.empty(R, I // 128, device=dev) for _ in range(2)]
        amax = torch.zeros(1, device=dev)
        cf.cf_swiglu_ckpt8_quantize_record(a, b, I, R, I, 0, u8[0], d[0], u8[1], d[1], u8[2], aqs, amax, stream())
        return [u8[0], d[0], u8[1], d[1], u8[2]], amax

    def backward(do, kept):
        R = do.shape[0]
        amax = torch.zeros(1, device=dev)
        o = [torch.empty(R, 2 * I, dtype=torch.uint8, device=dev), torch.empty(2 * I, R, dtype=torch.uint8, device=dev), torch.empty(I, R, dtype=torch.uint8, device=dev)]
        cf.cf_swiglu_ckpt8_backward_quant_e5m2(do, *kept, R, I, o[0], o[1], qs, amax, o[2], aqs, stream())
        return o, amax

    small, m = forward(gate, up)
    big, big_m = forward(put_at_the_end(gate, rows), put_at_the_end(up, rows))
    torch.cuda.synchronize()
    assert torch.equal(m, big_m)
    for a, b in zip(small, big):
        assert torch.equal(a, b[rows - n:])
    want, m = backward(do, small[:4])
    got, big_m = backward(put_at_the_end(do, rows), big[:4])
    torch.cuda.synchronize()
    assert torch.equal(m, big_m)
    assert torch.equal(want[0], got[0][rows - n:]) and not bool(got[0][: rows - n].any())
    for a, b in zip(want[1:], got[1:]):
        assert torch.equal(a, b[:, rows - n:]) and not bool(b[:, : rows - n].any())
