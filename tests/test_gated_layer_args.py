"""What the entry points of the layer with norms on both sides and of the 8-bit gated activation refuse, before anything is launched (no GPU needed)."""
import ctypes

P = 0x10000        # an address that is never read: these calls launch nothing
EPS = 1e-6
INF, NAN = float("inf"), float("nan")


def rows(cf, r=P, x=P, f32=0, res=1.0, gate=P, gate_rows=2, wp=P, w=P, n=4, H=64, total=P, normed=P, prms=P, rms=P, x8=P, sum8=P, q=P, s=P, d=P):
    return cf.raw_cf_gated_add_rmsnorm_quantize_rows(r, x, f32, res, gate, gate_rows, wp, w, n, H, EPS, 0, total, normed, prms, rms, x8, sum8, q, s, d, None)


def test_forward_refusals(cf):
    assert rows(cf, n=0) == 0 and rows(cf, H=0) == 0
    assert rows(cf, n=-1) == -1 and rows(cf, H=-8) == -1
    assert rows(cf, H=16385) == -2
    for name in ("r", "x", "wp", "w", "q", "s", "d"):
        assert rows(cf, **{name: None}) == -1, name
    for name in ("r", "x", "gate", "wp", "w", "total", "normed", "prms", "rms", "s", "d"):
        assert rows(cf, **{name: P + 1}) == -1, name
    assert rows(cf, f32=1, r=P + 2) == -1 and rows(cf, f32=1, total=P + 2) == -1
    assert rows(cf, gate_rows=0) == -1 and rows(cf, gate_rows=-3) == -1
    assert rows(cf, res=INF) == -1 and rows(cf, res=NAN) == -1
    head = (P, P, 0, 1.0, None, 0, P, P, 4, 64, EPS)
    block = lambda s, d: cf.raw_cf_gated_add_rmsnorm_quantize_block_1x128(*head, None, None, None, None, None, None, P, s, d, None)  # noqa: E731
    assert block(None, P) == -1 and block(P, None) == -1 and block(P + 2, P) == -1
    record = lambda s, a: cf.raw_cf_gated_add_rmsnorm_quantize_record(*head, 0, None, None, None, None, None, None, P, s, a, None)  # noqa: E731
    assert record(None, P) == -1 and record(P, None) == -1 and record(P, P + 2) == -1


def test_backward_refusals(cf):
    n = ctypes.c_size_t(0)
    size = lambda *a: cf.raw_cf_gated_add_rmsnorm_backward_workspace_bytes(*a, ctypes.byref(n))  # noqa: E731
    assert size(4, 64, 0) == 0 and n.value >= 2 * 64 * 4
    assert size(-1, 64, 0) == -1 and size(4, -1, 0) == -1 and size(4, 64, -1) == -1 and size(4, 20000, 0) == -2
    assert cf.raw_cf_gated_add_rmsnorm_backward_workspace_bytes(4, 64, 0, None) == -1
    for gate_rows in (0, 1, 2, 1000, 2**30, 2**31 - 1):
        assert size(2**31 - 1, 16384, gate_rows) == 0 and n.value <= 1 << 30
    assert size(0, 64, 3) == 0 and size(4, 0, 3) == 0

    for name in ("cf_gated_add_rmsnorm_backward", "cf_gated_add_rmsnorm_backward_ckpt8"):
        kept = name.endswith("ckpt8")
        fn = getattr(cf, "raw_" + name)

        def call(dy=P, h=P, x=P, f32=0, res=1.0, gate=P, gate_rows=2, wp=P, w=P, prms=P, rms=P, dh=P, rows=4, H=64, dr=P, dx=P, q=P, s=P, a=P, dwp=P, dw=P, dgate=P, acc=0,
                 ws=P, size=1 << 30):
            return fn(dy, h, x, f32, res, gate, gate_rows, wp, w, prms, rms, dh, rows, H, dr, dx, q, s, a, dwp, dw, dgate, acc, ws, size, None)

        assert call(rows=-1) == -1 and call(H=-1) == -1 and call(H=20000) == -2 and call(H=0) == 0
        for k in ("dy", "h", "x", "wp", "w", "prms", "rms", "dr", "s", "a", "dwp", "dw", "dgate", "ws"):
            assert call(**{k: None}) == -1, k
        for k in ("dy", "gate", "wp", "w", "prms", "rms", "dh", "dr", "dx", "s", "a", "dwp", "dw", "dgate", "ws"):
            assert call(**{k: P + 1}) == -1, k
        if not kept:
            assert call(h=P + 1) == -1 and call(x=P + 1) == -1 and call(f32=1, h=P + 2) == -1
        assert call(dx=None, q=None) == -1 and call(f32=1, dr=P + 2) == -1 and call(f32=1, dh=P + 2) == -1
        assert call(gate_rows=0) == -1 and call(gate_rows=-1) == -1 and call(res=INF) == -1 and call(res=NAN) == -1
        assert call(acc=4) == -1 and call(acc=-1) == -1 and call(ws=P + 4) == -1
        cf.raw_cf_gated_add_rmsnorm_backward_workspace_bytes(4, 64, 2, ctypes.byref(n))
        assert call(size=n.value - 1) == -1


def test_workspace_does_not_shrink_what_a_gate_needs(cf):
    """Several gates take room for the rows that several workers share; one gate or none does not."""
    n = ctypes.c_size_t(0)

    def size(rows, H, gate_rows):
        assert cf.raw_cf_gated_add_rmsnorm_backward_workspace_bytes(rows, H, gate_rows, ctypes.byref(n)) == 0
        return n.value

    assert size(8192, 4096, 8192) == size(8192, 4096, 0) < size(8192, 4096, 1000)
    assert size(8192, 4096, 1) == size(8192, 4096, 0)          # whole groups


def test_swiglu_refusals(cf):
    def keep(g=P, u=P, ld=64, rows=4, I=64, g8=P, gd=P, u8=P, ud=P, q=P, s=P, d=P):
        return cf.raw_cf_swiglu_ckpt8_quantize_rows(g, u, ld, rows, I, 0, g8, gd, u8, ud, q, s, d, None)

    assert keep(rows=0) == 0 and keep(I=0) == 0
    assert keep(rows=-1) == -1 and keep(I=-1) == -1 and keep(ld=63) == -1
    assert keep(I=32769, ld=32769) == -2
    for k in ("g", "u", "g8", "gd", "u8", "ud", "q", "s", "d"):
        assert keep(**{k: None}) == -1, k
    for k in ("g", "u", "gd", "ud", "s", "d"):
        assert keep(**{k: P + 1}) == -1, k
    head = (P, P, 64, 4, 64)
    block = lambda s, d, I=64: cf.raw_cf_swiglu_ckpt8_quantize_block_1x128(P, P, I, 4, I, P, P, P, P, P, s, d, None)  # noqa: E731
    assert block(None, P) == -1 and block(P, None) == -1 and block(P + 2, P) == -1 and block(P, P, 1 << 30) == -2
    record = lambda s, a: cf.raw_cf_swiglu_ckpt8_quantize_record(*head, 0, P, P, P, P, P, s, a, None)  # noqa: E731
    assert record(None, P) == -1 and record(P, None) == -1 and record(P, P + 2) == -1


def test_swiglu_gradient_refusals(cf):
    def grad(do=P, g8=P, gd=P, u8=P, ud=P, rows=4, I=64, dg=P, du=P, ld=64, act=P):
        return cf.raw_cf_swiglu_ckpt8_backward(do, g8, gd, u8, ud, rows, I, dg, du, ld, act, None)

    assert grad(rows=0) == 0 and grad(I=0) == 0 and grad(rows=-1) == -1 and grad(I=-1) == -1 and grad(ld=63) == -1 and grad(I=1 << 30, ld=1 << 30) == -2
    for k in ("do", "g8", "gd", "u8", "ud", "dg", "du"):
        assert grad(**{k: None}) == -1, k
    for k in ("do", "gd", "ud", "dg", "du", "act"):
        assert grad(**{k: P + 1}) == -1, k

    def grad8(do=P, g8=P, gd=P, u8=P, ud=P, rows=4, I=64, q=P, qt=P, s=P, a=P, act=P, act_s=P):
        return cf.raw_cf_swiglu_ckpt8_backward_quant_e5m2(do, g8, gd, u8, ud, rows, I, q, qt, s, a, act, act_s, None)

    assert grad8(rows=0) == 0 and grad8(I=0) == 0 and grad8(rows=-1) == -1 and grad8(I=-1) == -1 and grad8(I=1 << 30) == -2
    assert grad8(rows=2**31 - 1, I=(1 << 30) - 1) == -2
    for k in ("do", "g8", "gd", "u8", "ud", "q", "s", "a", "act_s"):
        assert grad8(**{k: None}) == -1, k
    for k in ("do", "gd", "ud", "s", "a", "act_s"):
        assert grad8(**{k: P + 1}) == -1, k
