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
