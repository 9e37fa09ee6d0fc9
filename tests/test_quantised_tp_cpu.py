"""8-bit linears and a 4-bit cache on two tensor-parallel ranks (gloo)."""
import json
import os
import subprocess
import sys

from tests.conftest import scratch_dir

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(ranks, port):
    out = os.path.join(scratch_dir("gllm_b200_q_"), "q.json")
    script = os.path.join(ROOT, "tests", "mp_quantised_tp_cpu.py")
    launch = [] if ranks == 1 else ["-m", "torch.distributed.run", "--nnodes=1", f"--nproc-per-node={ranks}", "--master-addr", "127.0.0.1",
                                    "--master-port", str(port)]
    r = subprocess.run([sys.executable, *launch, script, out], capture_output=True, text=True, timeout=300, cwd=ROOT,
                       env=dict(os.environ, PYTHONPATH=ROOT, GLLM_B200_LOG="WARNING"))
    assert r.returncode == 0 and os.path.exists(out), r.stdout[-2000:] + r.stderr[-3000:]
    with open(out) as f:
        return json.load(f)


def test_two_ranks():
    """Shards are the checkpoint's codes and scales, a block of them gives the definition's value, and with a 4-bit cache two ranks generate one
    rank's tokens (a rank holds whole heads, which are coded by themselves)."""
    assert _run(2, 29961) == _run(1, 29981)
