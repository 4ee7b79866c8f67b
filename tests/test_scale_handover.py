"""Scales that one CTA stages for a matrix instruction of the other are handed over at cluster scope (checked in the source: a
release at CTA scope does not reach the other CTA's thread, which shows now and then at most)."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "lplb_b200" / "csrc"


def _text(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def test_no_arrival_at_another_ctas_barrier_releases_at_cta_scope():
    for path in CSRC.glob("*.cu*"):
        for line in _text(path.name).splitlines():
            if "mbarrier.arrive" in line and "shared::cluster" in line and "tcgen05" not in line:
                assert "release.cluster" in line or "relaxed.cluster" in line, f"{path.name}: {line.strip()}"


def test_arrivals_that_release_nothing_stand_behind_a_fence_at_cluster_scope():
    used = [name for name in sorted(p.name for p in CSRC.glob("*.cu*")) if "mbar_arrive_remote_fenced(" in _text(name)]
    assert used == ["moe_gemm.cuh", "tcgen05.cuh"]
    text = _text("moe_gemm.cuh")
    scales = text[text.index("FP8 && warp == 6") : text.index("go && warp >= 2")]
    assert text.count("mbar_arrive_remote_fenced(") == scales.count("mbar_arrive_remote_fenced(") == 1
    steps = [scales.index(step) for step in ("fetch(chunk);", "fence_proxy_async_shared();", "__syncwarp();", "fence_cluster();", "mbar_arrive_remote_fenced(")]
    assert steps == sorted(steps)
