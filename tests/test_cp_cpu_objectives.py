"""Policy and preference passes with dropout on CPU ranks (gloo): every way to shard a sequence gives the unsharded losses and gradients."""
import json
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
_PORT = [29860]


def run_worker(nproc, *args):
    _PORT[0] += 1
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", f"--nproc-per-node={nproc}", "--master-addr", "127.0.0.1",
           "--master-port", str(_PORT[0] + (os.getpid() % 200)), os.path.join(HERE, "mp_objectives_worker.py"), *map(str, args)]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600, env=dict(os.environ, OMP_NUM_THREADS="1"))
    line = [v for v in r.stdout.splitlines() if v.startswith("{")]
    assert r.returncode == 0 and line, f"worker failed rc={r.returncode}\nstdout:\n{r.stdout[-3000:]}\nstderr:\n{r.stderr[-3000:]}"
    assert json.loads(line[-1])["ok"], line[-1]


@pytest.mark.parametrize("nproc,args", [
    (2, ("--mode", "ring")), (2, ("--mode", "ring", "--recompute", "full", "--family", "gpt2")), (2, ("--mode", "ulysses", "--rotator", "alltoall")),
    (4, ("--mode", "hybrid", "--ulysses", 2)), (4, ("--mode", "ring", "--cp", 2, "--recompute", "selective"))])
def test_sharded(nproc, args):
    run_worker(nproc, *args)
