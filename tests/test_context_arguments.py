"""Decoding over a team (rocshmem_b200.parallel.context) refuses queries with a derivative on the CPU backend too, where
the reference that computes a member's part would let autograd into the symmetric buffers."""
import os
import subprocess
import sys

import pytest

from mp_util import HERE, ROOT, assert_all_ok, free_port


@pytest.mark.parametrize("world", [1, 2])
def test_queries_with_a_derivative_are_refused(world):
    port, procs = free_port(), []
    for rank in range(world):
        env = dict(os.environ, RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank), MASTER_ADDR="127.0.0.1",
                   MASTER_PORT=str(port), PYTHONPATH=ROOT + os.pathsep + HERE)
        procs.append(subprocess.Popen([sys.executable, os.path.join(HERE, "context_gradient_worker.py")], env=env,
                                      stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True))
    results = []
    for p in procs:
        try:
            out, _ = p.communicate(timeout=180)
        except subprocess.TimeoutExpired:
            p.kill()
            out = p.communicate()[0] + "\n[killed: timeout]"
        results.append((p.returncode, out))
    assert_all_ok(results)
