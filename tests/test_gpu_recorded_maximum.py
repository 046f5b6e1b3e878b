"""GPU: a recorded maximum is that of its own call.  Rows look at copies of it before they raise it, in caches too, so one that was larger before it was cleared must not
keep a call from raising it: calls with large and small rows in turn on one maximum, cleared in between, eager and as one captured graph."""
import pytest
import torch

from gpu_util import case, stream

pytestmark = pytest.mark.gpu

ROWS, H = 9000, 1024


def calls(cf, dev):
    """name -> (function that enqueues the call on a stream, the maximum) for each entry point and size."""
    g = torch.Generator(device=dev).manual_seed(2)
    rn = lambda *s: torch.randn(*s, device=dev, generator=g).to(torch.bfloat16)  # noqa: E731
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=dev)  # noqa: E731
    f = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    r, x, one, qs = rn(ROWS, H), rn(ROWS, H), torch.ones(H, dtype=torch.bfloat16, device=dev), torch.ones(1, device=dev)
    gu, do = rn(ROWS, 2 * H), rn(ROWS, H)
    kept, q, t8 = [u8(ROWS, H), f(ROWS, 8), u8(ROWS, H), f(ROWS, 8)], u8(ROWS, H), u8(ROWS, 2 * H)
    cf.cf_swiglu_ckpt8_quantize_rows(gu, gu[:, H:], 2 * H, ROWS, H, 0, *kept, q, f(ROWS), f(ROWS), stream())
    out = {}
    for name in ("add", "gated", "swiglu", "swiglu gradient"):
        amax = f(1)
        for size in (64.0, 1.0):
            w, xs, dos = (one * size), gu * size, do * size
            if name == "add":
                def call(st, w=w, amax=amax):
                    cf.cf_add_rmsnorm_quantize_record(r, x, 0, w, ROWS, H, 1e-6, 0, None, None, None, q, qs, amax, st)
            elif name == "gated":
                def call(st, w=w, amax=amax):
                    cf.cf_gated_add_rmsnorm_quantize_record(r, x, 0, 1.0, None, 0, one, w, ROWS, H, 1e-6, 0, None, None, None, None, None, None, q, qs, amax, st)
            elif name == "swiglu":
                def call(st, xs=xs, amax=amax):
                    cf.cf_swiglu_ckpt8_quantize_record(xs, xs[:, H:], 2 * H, ROWS, H, 0, *[torch.empty_like(k) for k in kept], q, qs, amax, st)
            else:
                def call(st, dos=dos, amax=amax):
                    cf.cf_swiglu_ckpt8_backward_quant_e5m2(dos, *kept, ROWS, H, t8, None, qs, amax, None, None, st)
            out[name, size] = (call, amax)
    return out


@pytest.mark.parametrize("name", ["add", "gated", "swiglu", "swiglu gradient"])
def test_each_call_has_its_own(cf, dev, name):
    case(f"recorded maximum of {name}")
    all_calls = calls(cf, dev)
    (large, amax), (small, _) = all_calls[name, 64.0], all_calls[name, 1.0]
    amax.zero_()
    small(stream())
    least = float(amax)                     # the maximum's first values
    amax.zero_()
    large(stream())
    most = float(amax)
    assert 0.0 < 8.0 * least < most
    results = torch.zeros(20, device=dev)

    def many(st):
        for i in range(20):
            amax.zero_()
            (small if i % 2 else large)(st)
            results[i:i + 1].copy_(amax)

    want = [most, least] * 10
    many(stream())
    assert results.tolist() == want
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        many(torch.cuda.current_stream().cuda_stream)
    for _ in range(5):
        results.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert results.tolist() == want
        many(stream())
        assert results.tolist() == want
