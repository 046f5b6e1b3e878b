"""GPU: the experts' product with block scales (cf_fp8_grouped_gemm_nt_bf16_ex, CF_SCALE_BLOCK_128) against 64-bit products of the dequantized operands.

Tolerance: bf16 rounding 2^-8 of the result, and of the sum of absolute terms 2^-24 for each of K / 128 scaled additions, for the
products' own sums of at most 128 terms and for the two factors.  On top of it what the matrix cores cut: v_mfma_f32_16x16x128_f8f6f4 aligns the
products it adds to the largest of them and drops what lies below 2^-13 of that one's power of two (of +2^16 - 2^16 + 2^p it returns 0 up to p = 2 and
2^p from p = 3 on, whatever the order).  An E4M3 product has 8 significant bits, so one that is 2^7 cuts large loses nothing, a smaller one at
most a cut, or itself.  That sum is taken for a sample of rows; for all rows a coarser one, 128 cuts of the largest value of a row times the largest of a column."""
import ctypes

import numpy as np
import pytest
import torch

from gpu_util import case, stream

pytestmark = pytest.mark.gpu

MARK = 0x7fc1          # a bf16 pattern that no product gives


class Experts:
    def __init__(self, dev, counts, N, K, gather=True, lda=None, ldc=None, total=None, seed=0, offsets=None):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.N, self.K, self.E = dev, N, K, len(counts)
        self.counts = list(counts)
        self.filled = sum(counts)
        self.total = total if total is not None else self.filled
        self.offsets = offsets if offsets is not None else [int(v) for v in np.cumsum([0] + self.counts[:-1])]
        self.lda, self.ldc = lda or K, ldc or N
        self.gather = gather
        self.a_rows = 37 if gather else max(self.total, 1)        # a row may be gathered more than once
        kb, nb = K // 128, (N + 127) // 128
        # every finite E4M3 byte occurs; scales spread over several powers of two
        def bytes8(*shape):
            b = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)
            return torch.where((b & 0x7f) == 0x7f, b ^ 1, b)
        self.a = bytes8(self.a_rows, self.lda)
        self.w = bytes8(self.E, N, K)
        self.sa = torch.exp2(torch.randint(-9, -5, (self.a_rows, kb), generator=g).float()) * (1 + torch.rand(self.a_rows, kb, generator=g))
        self.sw = torch.exp2(torch.randint(-9, -5, (self.E, nb, kb), generator=g).float()) * (1 + torch.rand(self.E, nb, kb, generator=g))
        self.index = torch.randint(0, self.a_rows, (max(self.total, 1),), generator=g, dtype=torch.int32)

    def run(self, cf, entry="ex", ws_fill=0xff):
        dev = self.dev
        d = lambda t: t.to(dev)
        self.C = torch.full((max(self.total, 1) + 3, self.ldc), MARK, dtype=torch.int16, device=dev).view(torch.bfloat16)
        n = ctypes.c_size_t(0)
        cf.cf_fp8_grouped_gemm_workspace_bytes(self.total, self.E, ctypes.byref(n))
        ws = torch.full((n.value + 64,), ws_fill, dtype=torch.uint8, device=dev)
        head = (self.total, self.N, self.K, self.E, d(torch.tensor(self.counts, dtype=torch.int32)), d(torch.tensor(self.offsets, dtype=torch.int32)),
                d(self.a), self.a_rows, self.lda, d(self.index) if self.gather else None, d(self.sa), d(self.w), d(self.sw), 2, 0, None, None, self.C, self.ldc)
        if entry == "ex":
            cf.cf_fp8_grouped_gemm_nt_bf16_ex(*head, ws, n.value, stream())
        else:
            cf.cf_fp8_grouped_gemm_nt_bf16_static(*head, stream())
        torch.cuda.synchronize()
        assert bool((ws[n.value:] == ws_fill).all())
        return self.C

    def check(self, C):
        dev, N, K = self.dev, self.N, self.K
        A = (self.a[:, :K].to(dev).view(torch.float8_e4m3fn).double().unflatten(1, (K // 128, 128)) * self.sa.to(dev).double()[:, :, None]).flatten(1)
        bits = C.view(torch.int16)
        written = torch.zeros(C.shape[0], dtype=torch.bool, device=dev)
        for e, (n, o) in enumerate(zip(self.counts, self.offsets)):
            n = min(n, self.total - o)
            if n <= 0:
                continue
            w = self.w[e].to(dev).view(torch.float8_e4m3fn).double()
            w = w * self.sw[e].to(dev).double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)
            rows = A[self.index[o:o + n].to(dev).long()] if self.gather else A[o:o + n]
            ref, size = rows.mm(w.t().contiguous()), rows.abs().mm(w.abs().t().contiguous())
            got = C[o:o + n, :N].double()
            tol = 2.0 ** -8 * ref.abs() + (K / 128 + 130) * 2.0 ** -24 * size
            groups = lambda t: t.unflatten(1, (K // 128, 128)).abs()
            coarse = 2.0 ** -6 * groups(rows).amax(2).mm(groups(w).amax(2).t().contiguous())
            off = (got - ref).abs()
            assert bool((off <= 1.01 * (tol + coarse)).all()), (e, float((off / (tol + coarse)).max()))
            some = torch.unique(torch.tensor([0, 1, 15, 16, 31, 63, 64, 127, 128, n // 2, n - 2, n - 1]).clamp(0, n - 1))
            for r in some.tolist() if e % (1 + self.E // 64) == 0 else []:
                lost = torch.zeros(N, dtype=torch.float64, device=dev)
                for k in range(0, K, 128):
                    product = (rows[r, k:k + 128] * w[:, k:k + 128]).abs()
                    # the scales are the same for a whole group: cuts scale with them.  (Their product is no power of two: one power more.)
                    cut = 2.0 ** -13 * product.amax(1, keepdim=True)
                    lost += torch.where(product < 2.0 ** 8 * cut, torch.minimum(product, cut), 0.0).sum(1)
                assert bool((off[r] <= 1.01 * (tol[r] + lost)).all()), (e, r, float((off[r] / (tol[r] + lost)).max()))
            written[o:o + n] = True
        # rows that belong to no expert and columns behind N are left as they were
        assert bool((bits[~written] == MARK).all())
        assert bool((bits[:, N:] == MARK).all())


def even(total, E):
    return [total // E + (1 if e < total % E else 0) for e in range(E)]


@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("counts,N,K", [
    ([1], 128, 256), ([1, 0, 0, 0], 256, 512), ([0, 3, 0, 2], 8, 256), ([5, 1, 7, 2, 0, 0, 9, 1], 1408, 2048),
    (even(40, 16), 200, 384), (even(96, 64), 384, 1408), ([17, 33, 63, 64, 65], 640, 1024), ([100, 0, 300, 1], 512, 2048),
    ([129, 127, 128, 1, 256, 255, 257], 768, 896), ([1000, 0, 0], 256, 512), ([600, 700], 1416, 640), ([2000, 1, 511], 1024, 1024),
    ([3], 256, 32768), ([70, 200], 136, 20480), ([513, 300, 900, 40], 2048, 256), ([300] * 9, 1408, 384),
], ids=lambda v: str(v) if not isinstance(v, list) else f"{len(v)}x{max(v)}")
def test_block_scaled_experts(cf, dev, counts, N, K, gather):
    case(f"grouped block GEMM counts={counts[:8]} N={N} K={K} gather={gather}")
    b = Experts(dev, counts, N, K, gather, seed=N + K)
    b.check(b.run(cf))


@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("counts,N,K", [
    ([40] * 300, 256, 512),                          # more experts than the table's workgroup has threads
    ([3, 0] * 200, 136, 384),
    ([1536, 1500, 1600, 30, 2000, 257] * 3, 1416, 640),     # last row and column tiles nearly empty, several tiles a workgroup
    ([2500] * 8, 1024 + 8, 384),                     # three K-tiles; eight columns in the last tile
    ([5000, 4000, 6000], 1920, 512),                 # four
    ([300, 420], 264, 32768),                        # all of the weight-block scales' LDS
    ([900, 1, 129, 128, 127, 0, 700] * 4, 1408, 896),
    ([20000], 392, 256),
    ([30] * 2100, 128, 512),                         # more experts than the tile kernels count
], ids=lambda v: str(v) if not isinstance(v, list) else f"{len(v)}x{max(v)}")
def test_block_scaled_experts_of_many_rows(cf, dev, counts, N, K, gather):
    case(f"grouped block GEMM counts={counts[:8]} of {len(counts)} N={N} K={K} gather={gather}")
    b = Experts(dev, counts, N, K, gather, seed=N * 3 + K)
    b.check(b.run(cf))


def test_more_experts_than_the_tile_kernels_count_over_a_long_k(cf, dev):
    case("grouped block GEMM of 2049 experts, K=15488")
    b = Experts(dev, [33] * 2049, 8, 15488, True, seed=4)
    b.check(b.run(cf))


def test_strides_and_rows_behind_the_last_expert(cf, dev):
    """Row strides larger than the rows, a bound above the sum of the counts: the rows behind are left alone."""
    for counts, total in (([3, 0, 5], 64), ([130, 20, 70], 700), ([400, 0, 300, 90], 2000)):
        case(f"grouped block GEMM strides counts={counts} total={total}")
        b = Experts(dev, counts, 264, 640, gather=False, lda=720, ldc=280, total=total, seed=5)
        b.check(b.run(cf))


def test_counts_beyond_the_bound_are_cut(cf, dev):
    for counts, total in (([3, 4, 90], 50), ([300, 500], 450), ([700, 40, 40], 600)):
        case(f"grouped block GEMM cut counts={counts} total={total}")
        b = Experts(dev, counts, 256, 512, gather=False, total=total, seed=6)
        b.check(b.run(cf))


def test_all_rows_on_one_expert_and_none_at_all(cf, dev):
    for counts, total in (([0] * 20 + [640] + [0] * 11, 640), ([0] * 8, 100), ([0] * 63 + [1], 1)):
        case(f"grouped block GEMM on one expert, total={total}")
        b = Experts(dev, counts, 384, 768, total=total, seed=7)
        b.check(b.run(cf))


def test_the_form_without_a_workspace_gives_the_same_bits(cf, dev):
    for counts in ([5, 0, 9, 2], [300, 20, 600]):
        b = Experts(dev, counts, 512, 1024, seed=8)
        x = b.run(cf).view(torch.int16).clone()
        y = b.run(cf, "static").view(torch.int16)
        assert torch.equal(x, y)


def test_the_same_bits_twice(cf, dev):
    for counts in ([5, 0, 9, 2], [64, 90, 200, 130], [900, 20, 600]):
        b = Experts(dev, counts, 1408, 2048, seed=9)
        x = b.run(cf).view(torch.int16).clone()
        assert torch.equal(x, b.run(cf, ws_fill=0).view(torch.int16))
