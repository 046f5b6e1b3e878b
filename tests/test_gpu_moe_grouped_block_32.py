"""GPU: the experts' block-scaled product where its rule takes the 32 x 32 kernel: some ten to thirty rows an expert, too few columns to fill the CUs otherwise.
Products and tolerance as in test_gpu_moe_grouped_block."""
import pytest

from gpu_util import case
from test_gpu_moe_grouped_block import Experts

pytestmark = pytest.mark.gpu

COUNTS_N_K = [
    ([17, 9, 30, 25, 12, 31, 28, 19], 1024, 2048), ([33, 1, 64, 0], 200, 384), ([36], 2048, 512), ([0, 0, 100, 0], 1416, 640), ([16, 15, 32, 31, 1], 8, 256),
    ([30, 30], 136, 32768), ([7, 300, 2, 0, 0, 5, 1, 1, 0, 0], 392, 1024),
]


@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("counts,N,K", COUNTS_N_K, ids=lambda v: str(v) if not isinstance(v, list) else f"{len(v)}x{max(v)}")
def test_block_scaled_experts_of_some_rows(cf, dev, counts, N, K, gather):
    case(f"grouped block GEMM counts={counts} N={N} K={K} gather={gather}")
    b = Experts(dev, counts, N, K, gather, seed=N * 5 + K)
    b.check(b.run(cf))
