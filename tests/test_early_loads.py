"""Kernels that start while their predecessor still runs do not read its results through the read-only path (checked in
the source): that is for memory which nobody writes during a kernel's whole life, the part before the wait included."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "lplb_b200" / "csrc"
FILES = {p.name: re.sub(r"//[^\n]*", "", p.read_text()) for p in sorted(CSRC.glob("*.cu*"))}
KERNEL = re.compile(r"__global__[^;{]*?\b(\w+_kernel)\s*\(([^{;]*)\)\s*\{")


def _early():
    """(file, kernel, parameters) of every kernel that waits for its predecessors."""
    for name, text in FILES.items():
        for found in KERNEL.finditer(text):
            until = text.find("__global__", found.end())
            if "wait_predecessors();" in text[found.end() : until if until > 0 else len(text)]:
                yield name, found.group(1), found.group(2)


EARLY = list(_early())


def test_all_early_kernels_are_looked_at():
    assert {k for _, k, _ in EARLY} >= {
        "row_fp8_kernel", "row_stream_fp8_kernel", "weight_fp8_kernel", "few_rows_kernel", "moe_few_kernel", "moe_few_plan_kernel",
        "grouped_gemm_kernel", "dispatch_kernel", "route_kernel", "schedule_kernel", "combine_kernel", "tile_solve_kernel",
    }


@pytest.mark.parametrize("file,kernel,parameters", EARLY, ids=[k for _, k, _ in EARLY])
def test_parameters_are_not_promised_to_stay(file, kernel, parameters):
    assert not re.search(r"const\s+\w+\s*\*\s*__restrict__", parameters), f"{kernel} in {file}"


@pytest.mark.parametrize("file", sorted({f for f, _, _ in EARLY} | {"fp8.cuh", "scale_words.cuh"}))
def test_no_loads_by_the_read_only_path(file):
    assert "__ldg(" not in FILES[file] and "ld.global.nc" not in FILES[file]
