"""A CTA gives its tensor memory back before it waits for its cluster (checked in the source: the allocation is the one wait
without a limit, and another clustered kernel on the same SMs that wants the columns could hold it up for good)."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "lplb_b200" / "csrc"


def test_few_rows_release_their_columns_before_the_cluster_meets():
    text = re.sub(r"//[^\n]*", "", (CSRC / "matmul_fp8.cuh").read_text())
    body = text[text.index("few_rows_kernel(const __grid_constant__") :]
    assert body.count("tmem_dealloc_single(") == 1
    last_read, release, meet = body.index("tmem_ld_wait();"), body.index("tmem_dealloc_single("), body.index("cluster_sync();")
    assert last_read < body.index("__syncthreads();", last_read) < release < meet
