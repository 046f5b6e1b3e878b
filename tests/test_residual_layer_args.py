"""What the residual layer's entry points refuse, before anything is launched (no GPU needed)."""
import ctypes

import torch

EPS = 1e-6
P = 0x10000        # an address that is never read: these calls launch nothing


def rows(cf, residual=P, x=P, f32=0, w=P, n=4, H=64, total=P, normed=P, rms=P, q=P, s=P, d=P):
    return cf.raw_cf_add_rmsnorm_quantize_rows(residual, x, f32, w, n, H, EPS, 0, total, normed, rms, q, s, d, None)


def test_forward_refusals(cf):
    assert rows(cf, n=0) == 0 and rows(cf, H=0) == 0
    assert rows(cf, n=-1) == -1 and rows(cf, H=-8) == -1
    assert rows(cf, H=16385) == -2
    for name in ("residual", "w", "q", "s", "d"):
        assert rows(cf, **{name: None}) == -1
    for name in ("residual", "x", "w", "total", "normed", "rms", "s", "d"):
        assert rows(cf, **{name: P + 1}) == -1
    assert rows(cf, f32=1, residual=P + 2) == -1 and rows(cf, f32=1, total=P + 2) == -1
    block = lambda s, d: cf.raw_cf_add_rmsnorm_quantize_block_1x128(P, P, 0, P, 4, 64, EPS, None, None, None, P, s, d, None)
    assert block(None, P) == -1 and block(P, None) == -1 and block(P + 2, P) == -1
    record = lambda s, a: cf.raw_cf_add_rmsnorm_quantize_record(P, P, 0, P, 4, 64, EPS, 0, None, None, None, P, s, a, None)
    assert record(None, P) == -1 and record(P, None) == -1 and record(P, P + 2) == -1


def test_backward_refusals(cf):
    n = ctypes.c_size_t(0)
    assert cf.raw_cf_add_rmsnorm_backward_workspace_bytes(4, 64, ctypes.byref(n)) == 0 and n.value >= 64 * 4
    assert cf.raw_cf_add_rmsnorm_backward_workspace_bytes(-1, 64, ctypes.byref(n)) == -1
    assert cf.raw_cf_add_rmsnorm_backward_workspace_bytes(4, 64, None) == -1
    assert cf.raw_cf_add_rmsnorm_backward_workspace_bytes(4, 20000, ctypes.byref(n)) == -2
    most = ctypes.c_size_t(0)
    assert cf.raw_cf_add_rmsnorm_backward_workspace_bytes(2**31 - 1, 16384, ctypes.byref(most)) == 0 and most.value <= 1 << 30

    def call(dy=P, h=P, f32=0, w=P, rms=P, dh=P, rows=4, H=64, dr=P, dw=P, ws=P, size=1 << 30):
        return cf.raw_cf_add_rmsnorm_backward(dy, h, f32, w, rms, dh, rows, H, dr, dw, 0, ws, size, None)

    assert call(rows=-1) == -1 and call(H=-1) == -1 and call(H=20000) == -2 and call(H=0) == 0
    for name in ("dy", "h", "w", "rms", "dr", "dw", "ws"):
        assert call(**{name: None}) == -1
    for name in ("dy", "h", "w", "rms", "dh", "dr", "dw"):
        assert call(**{name: P + 1}) == -1
    assert call(f32=1, h=P + 2) == -1 and call(f32=1, dr=P + 2) == -1 and call(ws=P + 4) == -1
    assert call(size=64 * 4 - 1) == -1
    quant = lambda q, s, a: cf.raw_cf_add_rmsnorm_backward_quant_e5m2(P, P, 0, P, P, P, 4, 64, P, P, 0, q, s, a, P, 1 << 30, None)
    assert quant(None, P, P) == -1 and quant(P, None, P) == -1 and quant(P, P, None) == -1 and quant(P, P, P + 1) == -1


def test_gradient_list(cf):
    n = ctypes.c_size_t(0)
    counts = torch.tensor([5, 0, 100_000], dtype=torch.int64)
    assert cf.raw_cf_grad_list_bytes(counts.data_ptr(), 3, ctypes.byref(n)) == 0 and n.value > 0
    assert cf.raw_cf_grad_list_bytes(None, 0, ctypes.byref(n)) == 0 and n.value == 0
    assert cf.raw_cf_grad_list_bytes(None, 1, ctypes.byref(n)) == -1
    assert cf.raw_cf_grad_list_bytes(counts.data_ptr(), -1, ctypes.byref(n)) == -1
    assert cf.raw_cf_grad_list_bytes(counts.data_ptr(), 3, None) == -1
    negative = torch.tensor([-1], dtype=torch.int64)      # as a size: more than any address space holds
    assert cf.raw_cf_grad_list_bytes(negative.data_ptr(), 1, ctypes.byref(n)) == -1

    cf.raw_cf_grad_list_bytes(counts.data_ptr(), 3, ctypes.byref(n))
    image = torch.zeros(n.value, dtype=torch.uint8)

    def fill(ptrs=(P, 0, P), outs=None, types=(1, 0, 0), size=n.value, to=image):
        p, t = torch.tensor(ptrs, dtype=torch.int64), torch.tensor(types, dtype=torch.int32)
        o = torch.tensor(outs, dtype=torch.int64) if outs else None
        return cf.raw_cf_grad_list_fill(p.data_ptr(), o.data_ptr() if outs else None, counts.data_ptr(), t.data_ptr(), 3, to.data_ptr() if to is not None else None, size, )

    assert fill() == 0 and int(image.sum()) > 0
    assert fill(size=n.value - 1) == -1 and fill(to=None) == -1
    assert fill(ptrs=(0, 0, P)) == -1 and fill(ptrs=(P + 2, 0, P)) == -1 and fill(ptrs=(P, 0, P + 1)) == -1
    assert fill(types=(2, 0, 0)) == -1 and fill(types=(1, 9, 0)) == 0         # a tensor without elements has nothing to check
    assert fill(outs=(P, 0, 0)) == -1 and fill(outs=(P + 2, 0, P)) == -1 and fill(outs=(P, 0, P)) == 0


def test_gradient_list_stays_in_its_bytes(cf):
    """Whatever the alignment cuts a tensor's first entry to: the bytes that the size names are written, those behind them are not."""
    for count in (1, 7, 8, 4095, 8191, 16377, 16378, 16383, 16384, 16385, 32768, 32769, 49145, 49152, 100_000):
        for kind, el in ((0, 2), (1, 4)):
            for shift in range(0, 16, el):
                n = ctypes.c_size_t(0)
                counts, types = torch.tensor([count, count], dtype=torch.int64), torch.tensor([kind, kind], dtype=torch.int32)
                ptrs = torch.tensor([P + shift, P + shift], dtype=torch.int64)
                assert cf.raw_cf_grad_list_bytes(counts.data_ptr(), 2, ctypes.byref(n)) == 0
                image = torch.full((n.value + 4096,), 0xa5, dtype=torch.uint8)
                assert cf.raw_cf_grad_list_fill(ptrs.data_ptr(), None, counts.data_ptr(), types.data_ptr(), 2, image.data_ptr(), n.value) == 0
                assert bool((image[n.value:] == 0xa5).all())
                # every element of both tensors once, in order, and nothing else: (address, address, count, type, 0) an entry
                at, seen = [P + shift, P + shift], 0
                entries = image[:n.value].view(torch.int64).view(-1, 4)
                for src, dst, what, pad in entries.tolist():
                    length, f32 = what & 0xffffffff, what >> 32
                    if length == 0:
                        continue
                    which = 0 if seen < count else 1
                    assert src == dst == at[which] and f32 == kind and pad == 0
                    at[which] += length * el
                    seen += length
                assert seen == 2 * count


def test_gradient_norm_refusals(cf):
    n = ctypes.c_size_t(0)
    assert cf.raw_cf_grad_norm_workspace_bytes(ctypes.byref(n)) == 0 and cf.raw_cf_grad_norm_workspace_bytes(None) == -1
    norm = lambda l=P, size=64, out=P, ws=P, wn=n.value: cf.raw_cf_grad_norm(l, size, out, ws, wn, None)
    assert norm(l=None) == -1 and norm(l=P + 4) == -1 and norm(size=63) == -1
    assert norm(out=None) == -1 and norm(out=P + 2) == -1 and norm(ws=None) == -1 and norm(ws=P + 8) == -1 and norm(wn=n.value - 1) == -1
    clip = lambda m=1.0, g=P, c=None, l=P: cf.raw_cf_grad_clip(l, 64, m, g, c, None)
    assert clip(m=-1.0) == -1 and clip(m=float("nan")) == -1 and clip(g=None) == -1 and clip(c=P) == -1 and clip(l=None) == -1
    both = lambda m=1.0, g=P, c=None, ws=P: cf.raw_cf_grad_norm_clip(P, 64, m, g, c, ws, n.value, None)
    assert both(m=-1.0) == -1 and both(m=float("nan")) == -1 and both(g=None) == -1 and both(c=P) == -1 and both(ws=None) == -1


def test_block_scaled_experts_refusals(cf):
    n = ctypes.c_size_t(0)
    cf.raw_cf_fp8_grouped_gemm_workspace_bytes(64, 4, ctypes.byref(n))

    def call(scale_mode=2, epi=0, K=512, N=256, up=None, ldc=256, lda=512):
        return cf.raw_cf_fp8_grouped_gemm_nt_bf16_ex(64, N, K, 4, P, P, P, 64, lda, None, P, P, P, scale_mode, epi, up, up, P, ldc, P, n.value, None)

    assert call(scale_mode=3) == -1 and call(scale_mode=-1) == -1
    assert call(epi=2, up=P) == -2                        # no fused epilogue with block scales, as in the dense product
    assert call(K=32896, lda=32896) == -2 and call(K=500) == -2 and call(K=128) == -2
    assert call(N=252) == -2 and call(ldc=260) == -2
