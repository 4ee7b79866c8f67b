"""Tensor memory of a CTA pair is allocated once both CTAs have begun (checked in the source: the allocation is a wait without a limit, and one
that was asked for before the peer had begun has left the peer waiting for good)."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "lplb_b200" / "csrc"


def _text(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


KERNELS = {"matmul.cuh": "pair_matmul_kernel(", "moe_gemm.cuh": "cluster_cta_rank()"}  # where a kernel's body begins


def test_these_are_all_that_allocate_for_a_pair():
    using = {p.name for p in CSRC.iterdir() if p.suffix in (".cu", ".cuh") and re.search(r"\btmem_alloc\(smem", _text(p.name))}
    assert using == set(KERNELS)
    pairs = re.findall(r"tcgen05\.(\w+)\.cta_group::2\.sync\.aligned", _text("tcgen05.cuh"))
    assert sorted(pairs) == ["alloc", "dealloc", "relinquish_alloc_permit"]
    for p in CSRC.iterdir():
        if p.name != "tcgen05.cuh" and p.suffix in (".cu", ".cuh"):
            assert "tcgen05.alloc.cta_group::2" not in _text(p.name)


@pytest.mark.parametrize("name", list(KERNELS))
def test_the_cluster_meets_before_the_allocation_and_before_the_permit_is_given_up(name):
    body = _text(name)
    body = body[body.index(KERNELS[name]) :]
    assert body.count("tmem_alloc(") == body.count("tmem_relinquish(") == body.count("tmem_dealloc(") == 1
    steps = [m.group(0) for m in re.finditer(r"cluster_sync\(\)|tmem_alloc\(|tmem_relinquish\(|tmem_dealloc\(", body)]
    assert steps == ["cluster_sync()", "tmem_alloc(", "cluster_sync()", "tmem_relinquish(", "cluster_sync()", "tmem_dealloc("]
    # all threads of both CTAs meet: nothing returns before
    assert "return" not in body[: body.index("tmem_alloc(")].split("{", 1)[-1].replace("[&]", "")
