"""CPU: the benchmark's reference arm runs the reference or says that it cannot."""
import json
import os
import subprocess
import sys

import pytest

from conftest import REPO
from oracle.pyoracle import ref_so_path


@pytest.mark.skipif(ref_so_path() is not None, reason="the reference's library is built here")
@pytest.mark.parametrize("config", ["c0", "c2", "c4"])
@pytest.mark.parametrize("rank", ["0", "1"])
def test_reference_arm_without_the_reference(config, rank):
    """No restatement runs under the reference's name: one line on rank 0, nothing on the others."""
    env = dict(os.environ, RANK=rank, LOCAL_RANK=rank, WORLD_SIZE="2", MASTER_ADDR="127.0.0.1", MASTER_PORT="29600")
    got = subprocess.run([sys.executable, os.path.join(REPO, "bench.py"), "--impl", "reference", "--gpus", "2",
                          "--config", config, "--steps", "1"], env=env, capture_output=True, text=True, timeout=120)
    assert got.returncode == 0, got.stderr
    if rank != "0":
        assert got.stdout == ""
        return
    line = json.loads(got.stdout)
    assert set(line) == {"impl", "unavailable"} and line["impl"] == "reference" and "\n" not in line["unavailable"]
