"""How the gradient of the gated norm cuts its rows: the plan as the library has it, compiled for the host (no GPU needed)."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
FIELDS = ("parts", "workers", "groups", "several", "segments", "share", "shares", "bytes")


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """[(rows, H, rows a gate), ...] -> the plans as dicts; undefined behaviour ends the program."""
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text('#include <cstdio>\n#include "gated_norm_plan.hpp"\n'
                                 "int main() {\n    int rows, H, gate_rows;\n    while (std::scanf(\"%d %d %d\", &rows, &H, &gate_rows) == 3) {\n"
                                 "        const auto p = cf::grad_plan(rows, H, gate_rows);\n"
                                 "        std::printf(\"%d %d %d %d %d %u %d %zu\\n\", p.parts, p.workers, p.groups, p.several, p.segments, p.share, p.shares, p.bytes);\n    }\n}\n")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", f"-I{ROOT / 'canopy-foundry_amd' / 'csrc'}", str(at / "plan.cpp"),
                    "-o", str(at / "plan")], check=True, capture_output=True)

    def ask(sizes):
        out = subprocess.run([str(at / "plan")], input="\n".join(" ".join(map(str, s)) for s in sizes), capture_output=True, text=True)
        assert out.returncode == 0, out.stderr
        return [dict(zip(FIELDS, map(int, line.split()))) for line in out.stdout.splitlines()]
    return ask


def test_many_groups_stay_in_range(plan):
    """A gate for each of 2^27 rows and more, as many as there are, and widths of every kind."""
    sizes = [(rows, H, gate_rows) for rows in (1 << 27, 1 << 29, (1 << 31) - 1) for H in (1, 8, 512, 513, 4096, 8192, 12288, 16384) for gate_rows in (1, 2, 15, 1 << 20, rows, (1 << 31) - 1)]
    for (rows, H, gate_rows), p in zip(sizes, plan(sizes)):
        assert p["groups"] == -(-rows // gate_rows) and p["workers"] * p["share"] >= rows
        assert p["segments"] == (1 < p["groups"] < 8 * p["workers"])
        assert p["shares"] == (32 if p["workers"] >= 16 * p["groups"] else 8 if p["workers"] >= 4 * p["groups"] else 2)


def width_class(H):
    """A wavefront a row, one chunk a thread, two, two of the wide kernel, the widest."""
    return sum(H > most for most in (512, 4096, 8192, 12288))


def test_the_gpu_tests_reach_both_orders_at_every_width(plan):
    """Whole groups (eight a worker and more), pieces of groups that several workers have, one gate and none; a change of the plan that takes an order out of its tests shows here."""
    import test_gpu_gated_norm_groups as groups
    import test_gpu_gated_norm_sums as sums
    many = plan(groups.SHAPES)
    assert all(p["several"] and not p["segments"] and p["groups"] >= 8 * p["workers"] for p in many)
    assert {width_class(H) for _, H, _ in groups.SHAPES} == set(range(5))
    assert {width_class(H) for rows, H, n in groups.SHAPES if n > 1 and rows % n} >= {0, 1, 2, 3}          # a last group cut short
    for rows, H in sums.SHAPES:
        none, one, some, each = plan([(rows, H, n if n is not None else rows) for n in sums.GATE_ROWS])
        assert not none["several"] and not one["several"] and one["groups"] == 1
        assert some["segments"] and 300 >= 3 * some["share"] and some["share"] >= 30          # pieces, and rows enough for 32 bits to show
        assert each["several"] and not each["segments"]
    assert {width_class(H) for _, H in sums.SHAPES} == set(range(5))
    wide = dict(zip(groups.WIDE, plan(groups.WIDE)))
    assert all(rows > p["parts"] for (rows, _, _), p in wide.items())
    assert {(p["groups"] > 1, p["segments"]) for p in wide.values()} == {(False, 0), (True, 1), (True, 0)}
