"""Registers of every kernel of a draft model's operators, each by its name: a name
that no built kernel has is a mistake here."""

from __future__ import annotations

import re

import pytest

from tests.test_kernel_registers_cpu import kernels  # noqa: F401  (a fixture)

# how many there are of each: types, vector widths and variants
COUNTS = {
    "forward": 4, "backward": 4, "summarise": 4, "step": 2,
    "lookup": 8, "sort_count": 3, "sort_offsets": 3, "sort_place": 3, "sum_whole_pieces": 4, "sum_larger_pieces": 4,
    "sum_runs": 12, "sum_few": 8, "zeros": 4,
    "narrow_rows": 2, "wide_rows": 2, "join_parts": 2, "gradient": 20,
    "sum_pieces": 2, "locate": 2,
}


def _named(kernels, name):  # noqa: F811
    """Of operators that share a name, those whose types are ``elements.h``'s."""

    types = "Li" if name.startswith("sort_") else "N6myelin"
    return {n: k for n, k in kernels.items() if re.search(rf"_GLOBAL__N_1{len(name)}{name}I{types}", n)}


@pytest.mark.parametrize("name", COUNTS)
def test_no_vector_register_is_spilled(kernels, name):  # noqa: F811
    found = _named(kernels, name)
    assert len(found) == COUNTS[name], sorted(found)
    for n, k in found.items():
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, n
        # forward keeps up to 8 of its scalar registers in lanes of a vector register
        assert k[".sgpr_spill_count"] <= (8 if name == "forward" else 0), (n, k[".sgpr_spill_count"])


@pytest.mark.parametrize("name,most", [("forward", 128), ("backward", 128), ("summarise", 128), ("narrow_rows", 64),
                                       ("wide_rows", 64)])
def test_waves_fit(kernels, name, most):  # noqa: F811
    """A workgroup of 16 waves has 128 vector registers a lane; 8 waves a SIMD have 64."""

    for n, k in _named(kernels, name).items():
        assert k[".vgpr_count"] <= most, (n, k[".vgpr_count"])
