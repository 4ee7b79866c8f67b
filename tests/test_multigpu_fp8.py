"""The layer in 8 bits over several GPUs: runs tests/dist_fp8_worker.py as one process per GPU."""

import os
import subprocess
import sys

import pytest
import torch

from tests.test_multigpu import _free_port

pytestmark = [pytest.mark.gpu, pytest.mark.multigpu]


@pytest.mark.parametrize("world", [2, 4, 8])
def test_rows_in_8_bits_cross_to_the_peers(world):
    if torch.cuda.device_count() < world:
        pytest.skip(f"needs {world} GPUs")
    env = dict(os.environ, NCCL_NVLS_ENABLE="0")
    worker = os.path.join(os.path.dirname(os.path.abspath(__file__)), "dist_fp8_worker.py")
    cmd = [
        sys.executable, "-m", "torch.distributed.run", "--nnodes=1", f"--nproc-per-node={world}",
        "--master-addr", "127.0.0.1", "--master-port", str(_free_port()), worker,
    ]
    proc = subprocess.run(cmd, env=env, capture_output=True, text=True, timeout=600)
    assert proc.returncode == 0, proc.stdout[-3000:] + proc.stderr[-3000:]
    assert f"DIST_FP8_WORKER_OK {world}" in proc.stdout
