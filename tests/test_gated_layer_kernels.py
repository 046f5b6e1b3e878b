"""The library has the kernels of the gated layer that a call can reach, and no others (no GPU needed)."""
import re
from pathlib import Path

LIBRARY = Path(__file__).resolve().parent.parent / "canopy-foundry_amd" / "libcf_fp8.so"


def test_no_kernel_that_no_call_reaches(cf):
    library = LIBRARY.read_bytes()
    # stream fp32, scales, tail, a wavefront a row, chunks a thread: an fp32 row has two at most
    found = {tuple(map(int, m)) for m in re.findall(rb"k_gated_normILb([01])ELi([012])ELb([01])ELb([01])ELi([124])E", library)}
    assert found == {(f32, q, tail, wave, v) for f32 in (0, 1) for q in (0, 1, 2) for tail in (0, 1) for wave, v in [(1, 1), (0, 1), (0, 2)] + ([] if f32 else [(0, 4)])}
    # tail, whole rows of the straight outputs, whole lines of the transposed: whole tiles have no tail
    found = {tuple(map(int, m)) for m in re.findall(rb"k_swiglu_grad8ILb([01])ELb([01])ELb([01])E", library)}
    assert found == {(t, r, w) for t in (0, 1) for r in (0, 1) for w in (0, 1)} - {(1, 1, 1)}
    # scales, tail, a wavefront a row, chunks a thread: several where the scale is the whole row's
    found = {tuple(map(int, m)) for m in re.findall(rb"k_swiglu_keepILi([012])ELb([01])ELb([01])ELi(\d)E", library)}
    assert found == {(0, t, w, v) for t in (0, 1) for w, v in [(1, 1), (0, 1), (0, 2), (0, 3), (0, 4)]} | {(q, t, 0, 1) for q in (1, 2) for t in (0, 1)}
