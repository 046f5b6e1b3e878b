"""Which kernels the experts' block-scaled product has, which of them its rule takes, and that the GPU tests' sizes reach each (no GPU needed)."""
import re
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
T16, T32, T64, T32X64, T128, T256 = 0, 1, 3, 7, 128, 256
CUS = 256


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """The rule as the library has it, compiled for the host: [(rows, experts, N, K), ...] -> [(shape, beside), ...]."""
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text('#include <cstdio>\n#include "grouped_block_plan.hpp"\n'
                                 "int main() {\n    int r, e, n, k;\n    while (std::scanf(\"%d %d %d %d\", &r, &e, &n, &k) == 4) {\n"
                                 f"        const auto p = cf::grouped_block_plan(r, e, n, k, {CUS});\n"
                                 "        std::printf(\"%d %d\\n\", p.shape, p.beside);\n    }\n}\n")
    subprocess.run(["g++", "-std=c++17", "-O2", "-ffp-contract=off", f"-I{ROOT / 'canopy-foundry_amd' / 'csrc'}", str(at / "plan.cpp"), "-o", str(at / "plan")],
                   check=True, capture_output=True)

    def ask(sizes):
        out = subprocess.run([str(at / "plan")], input="\n".join(" ".join(map(str, s)) for s in sizes), capture_output=True, text=True, check=True)
        return [tuple(map(int, line.split())) for line in out.stdout.splitlines()]
    return ask


def test_no_kernel_that_the_rule_does_not_take(cf):
    """Rows and columns of the small-tile kernels in the library: the four that grouped_gemm_nt_block names."""
    library = (ROOT / "canopy-foundry_amd" / "libcf_fp8.so").read_bytes()
    found = set(re.findall(rb"k_gemm_nt_directILi0ELb0ELb1ELb1ELi(\d)ELi(\d)E", library))
    assert found == {(b"1", b"1"), (b"2", b"2"), (b"4", b"4"), (b"2", b"4")}


def test_what_the_rule_takes(plan):
    """Sizes whose best kernel is far ahead of the next (microseconds beside the rule)."""
    sizes = {(96, 64, 1408, 2048): T32X64, (1280, 64, 1408, 2048): T32X64, (2560, 64, 1408, 2048): T128, (98304, 64, 1408, 2048): T256, (1000, 16, 1536, 4096): T128,
             (4000, 16, 2048, 7168): T256, (500, 8, 1024, 2048): T64, (2000, 8, 1024, 2048): T128, (32768, 8, 1024, 2048): T256, (12, 64, 256, 6144): T16,
             (200, 8, 1024, 2048): T32}
    assert [shape for shape, _ in plan(sizes)] == list(sizes.values())
    # a K of two K-tiles has the 64 x 64 kernel alone, more experts than the tile kernels count and a long K the 32 x 64 one
    assert plan([(5000, 4, 2048, 256), (33 * 2049, 2049, 8, 15488), (30 * 2100, 2100, 128, 512)]) == [(T64, 1), (T32X64, 1), (T64, 2)]


def test_the_gpu_tests_reach_every_kernel(plan):
    """A change of the rule that takes a kernel out of its tests shows here."""
    import test_gpu_moe_grouped_block as t
    from test_gpu_moe_grouped_block_32 import COUNTS_N_K as some_rows
    assert {p[0] for p in plan([(sum(c), len(c), n, k) for c, n, k in some_rows])} == {T32}
    counts = [(c, n, k) for f in (t.test_block_scaled_experts, t.test_block_scaled_experts_of_many_rows) for m in f.pytestmark
              if m.name == "parametrize" and m.args[0] == "counts,N,K" for c, n, k in m.args[1]]
    shapes = [p[0] for p in plan([(sum(c), len(c), n, k) for c, n, k in counts])]
    for kernel, least in ((T16, 3), (T32X64, 2), (T64, 3), (T128, 3), (T256, 3)):
        assert shapes.count(kernel) >= least, (kernel, shapes)
    # the 256 x 256 kernel: a workgroup with several tiles, so that the stores of a whole one are under way when the next begins, a wavefront without an output (64 rows x 128
    # columns), and rows or columns that end inside a wavefront's
    wide = [(c, n, k) for (c, n, k), s in zip(counts, shapes) if s == T256]
    tiles = lambda c, n: sum(-(-r // 256) for r in c) * -(-n // 256)
    assert any(tiles(c, n) > CUS and any(r >= 256 for r in c) for c, n, k in wide)
    assert any(0 < r % 256 <= 192 for c, n, k in wide for r in c) and any(0 < n % 256 <= 128 for c, n, k in wide)
    assert any(r % 64 for c, n, k in wide for r in c) and any(n % 128 for c, n, k in wide)
