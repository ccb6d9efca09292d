"""
What the generation operators' kernels take of a compute unit (the compiler's figures in the
built library): no registers spilled, and the workgroups a CU that their launch rules count on.
"""

import re

import pytest

from tests.test_kernel_resources import _of, kernels  # noqa: F401  (the fixture)


@pytest.mark.parametrize("pattern", [r"prefix_part_kernel", r"prefix_join_kernel",
                                     r"prefix_whole_kernel", r"rope_kernel",
                                     r"evict_(select|move)_kernel", r"logits_kernel"])
def test_nothing_is_spilled(kernels, pattern):  # noqa: F811
    for name, k in _of(kernels, pattern).items():
        assert k["spills"] == 0, (name, k)


def test_attention_parts_run_two_workgroups_a_cu(kernels):  # noqa: F811
    """4 waves each: 2 a CU is 2 waves a SIMD, up to 256 registers a lane; the tiles are dynamic
    shared memory (at most 64 KiB), so the static part has to leave room beside them."""
    for name, k in _of(kernels, r"prefix_part_kernel").items():
        assert k["vgprs"] <= 256 and k["lds"] <= 16 * 1024, (name, k)


def test_every_form_of_the_attention_is_built(kernels):  # noqa: F811
    """Both types and dims; own forms up to the prefix's, or one kind alone (-1 is mangled n1)."""
    found = {tuple(re.search(r"ILi(\d)ELi(\d+)ELi(n?\d)ELi(n?\d)E", n).groups())
             for n in _of(kernels, r"prefix_part_kernel")}
    for dt in "01":
        for d, top in (("64", 4), ("128", 3)):
            for fp in range(top + 1):
                assert (dt, d, str(fp), "n1") in found and (dt, d, "n1", str(fp)) in found
                for fs in range(fp + 1):
                    assert (dt, d, str(fp), str(fs)) in found
