"""Registers of a draft model's built kernels: 16 waves of a workgroup share a CU, so
that more than 128 would not start, and a spilled one is stored and loaded at every
tile."""

from __future__ import annotations

from tests.test_kernel_registers_cpu import kernels  # noqa: F401  (a fixture)

NAMES = ("7forwardIN", "8backwardIN", "9summariseIN", "8sort_oneI", "6lookupIN", "8sum_runsIN", "16sum_whole_piecesIN",
         "9wide_rowsIN", "8gradientIN", "10sum_piecesIN", "6locateIN")


def test_nothing_is_spilled(kernels):  # noqa: F811
    found = {n: k for n, k in kernels.items() if any(name in n for name in NAMES) and "6myelin" in n or "sort_one" in n}
    assert len(found) >= 30
    spilled = {n: k[".vgpr_spill_count"] for n, k in found.items() if k[".vgpr_spill_count"]}
    assert not spilled, spilled
    tight = [k for n, k in found.items() if any(name in n for name in NAMES[:4])]
    assert len(tight) >= 8 and all(k[".vgpr_count"] <= 128 for k in tight)


def test_sorts_fit_two_workgroups(kernels):  # noqa: F811
    found = {n: k for n, k in kernels.items() if "10sort_countI" in n or "10sort_placeI" in n}
    assert len(found) == 6
    for n, k in found.items():
        assert k[".vgpr_count"] <= 64 and not k[".vgpr_spill_count"], (n, k[".vgpr_count"])
        assert k[".group_segment_fixed_size"] <= 80 * 1024, n
