"""bench.py::supervise_ranks and a start that takes long: the ranks' children are replaced by a few lines that write the progress marks a rank writes."""
import json
import os
import socket
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CHILD = """
import json, os, sys, time
rank, transport = int(os.environ["RANK"]), sys.argv[sys.argv.index("--transport") + 1]
def beat(what, seconds):
    open(os.environ["FBHIP_BENCH_HEARTBEAT"], "w").write(f"{time.time():.3f} {what}\\n")
    time.sleep(seconds)
plan = json.loads(os.environ["CHILD_PLAN"]).get(transport, {}).get(str(rank), {})
for what in ("started", "process group up", "agent and replay shard built", "warm-up done", "timed repeat 1 of 1 done"):
    beat(what, plan.get(what, 0.2))
if rank == 0:
    print(json.dumps({"metric": "none", "value": 1.0, "data_parallel": {"transport": transport}}), flush=True)
"""


def _supervise(plan):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    env = {k: v for k, v in os.environ.items() if k not in ("WORLD_SIZE", "RANK", "LOCAL_RANK", "MASTER_PORT", "FBHIP_BENCH_CHILD")}
    env.update(FBHIP_BENCH_CHILD_CMD=json.dumps([sys.executable, "-c", CHILD]), CHILD_PLAN=json.dumps(plan))
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", "2", "--master-addr", "127.0.0.1", "--master-port", str(port),
           str(ROOT / "bench.py"), "--gpus", "2", "--steps", "4", "--stall-timeout", "4"]
    out = subprocess.run(cmd, capture_output=True, text=True, timeout=300, cwd=str(ROOT), env=env)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-3000:]
    line, = [x for x in out.stdout.splitlines() if x.startswith("{")]
    return json.loads(line)["data_parallel"]["attempts"], out.stderr


def test_a_slow_build_of_the_agent_is_no_stall():
    """between these two marks a rank only computes (the networks' orthogonal initialisation, on as many threads as the other ranks want too): it takes
    longer than the limit between two marks of the run, on both ranks or on one"""
    attempts, _ = _supervise({"rccl": {"0": {"process group up": 9.0}, "1": {"process group up": 7.0}}})
    assert [a["transport"] for a in attempts] == ["rccl"] and [r["outcome"] for r in attempts[0]["ranks"]] == ["ok", "ok"], attempts


@pytest.mark.parametrize("mark", ["started", "agent and replay shard built"])
def test_a_stall_elsewhere_is_still_one(mark):
    attempts, err = _supervise({"rccl": {"1": {mark: 60.0}}})
    assert [a["transport"] for a in attempts] == ["rccl", "rccl", "c10d"], attempts
    assert all(a["ranks"][1] == {"outcome": "failed (no progress on rank 1)", "last_progress": mark} for a in attempts[:2]), attempts
    # each attempt's end, with every rank's last mark, is on the supervisor's own output too
    assert err.count(f"'last_progress': '{mark}'") == 2 and err.count("transport rccl did not finish") == 2, err
