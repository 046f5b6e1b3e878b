"""Which kernels the experts' block-scaled product has, and which of them its rule takes (no GPU needed)."""
import re


def test_no_kernel_that_the_rule_does_not_take(cf):
    """Rows and columns of the small-tile kernels in the library: the four that grouped_gemm_nt_block names."""
    from pathlib import Path
    library = (Path(__file__).resolve().parent.parent / "canopy-foundry_amd" / "libcf_fp8.so").read_bytes()
    found = set(re.findall(rb"k_gemm_nt_directILi0ELb0ELb1ELb1ELi(\d)ELi(\d)E", library))
    assert found == {(b"1", b"1"), (b"2", b"2"), (b"4", b"4"), (b"2", b"4")}
