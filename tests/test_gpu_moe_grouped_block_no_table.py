"""GPU: the experts' product with block scales builds no table of row tiles, so it needs no workspace, and the form without one has neither a limit of row tiles nor
a rule against calls that overlap.  Products and tolerance as in test_gpu_moe_grouped_block."""
import pytest
import torch

from gpu_util import case, stream
from test_gpu_moe_grouped_block import Experts

pytestmark = pytest.mark.gpu


def head(b, dev, C):
    d = lambda t: t.to(dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    return (b.total, b.N, b.K, b.E, i32(b.counts), i32(b.offsets), d(b.a), b.a_rows, b.lda, d(b.index) if b.gather else None, d(b.sa), d(b.w), d(b.sw), 2, 0, None,
            None, C, b.ldc)


@pytest.mark.parametrize("counts", [[5, 0, 9, 2], [64, 90, 200, 130], [900, 20, 600]], ids=str)
def test_without_a_workspace(cf, dev, counts):
    case(f"grouped block GEMM without a workspace counts={counts}")
    b = Experts(dev, counts, 384, 1024, seed=11)
    with_one = b.run(cf).view(torch.int16).clone()
    C = torch.zeros(b.C.shape, dtype=torch.bfloat16, device=dev)
    cf.cf_fp8_grouped_gemm_nt_bf16_ex(*head(b, dev, C), None, 0, stream())
    torch.cuda.synchronize()
    assert torch.equal(C.view(torch.int16)[:b.total], with_one[:b.total])


@pytest.mark.parametrize("counts,N", [([1, 2] * 1700, 8), ([2, 850_000, 0, 31], 8)], ids=["experts", "rows"])
def test_more_row_tiles_than_the_fixed_table_holds(cf, dev, counts, N):
    """3400 experts; 850,000 rows, which are 3320 tiles of 256."""
    case(f"grouped block GEMM of {sum(counts)} rows over {len(counts)} experts in the static form")
    b = Experts(dev, counts, N, 256, seed=12)
    x = b.run(cf).view(torch.int16).clone()
    assert torch.equal(x, b.run(cf, "static").view(torch.int16))
    if len(counts) > 1000:
        b.check(b.C)


def test_static_calls_side_by_side(cf, dev):
    """On two streams at once, with counts that differ: each gives what it gives alone."""
    case("grouped block GEMM, static form, on two streams")
    bs = [Experts(dev, counts, 512, 1024, seed=s) for s, counts in ((13, [300, 20, 600, 8]), (14, [7, 500, 1, 90]))]
    want = [b.run(cf).view(torch.int16).clone() for b in bs]
    outs = [torch.zeros(b.C.shape, dtype=torch.bfloat16, device=dev) for b in bs]
    args = [head(b, dev, C) for b, C in zip(bs, outs)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, a in zip(streams, args):
            cf.cf_fp8_grouped_gemm_nt_bf16_static(*a, s.cuda_stream)
    torch.cuda.synchronize()
    for b, C, w in zip(bs, outs, want):
        assert torch.equal(C.view(torch.int16)[:b.total], w[:b.total])
