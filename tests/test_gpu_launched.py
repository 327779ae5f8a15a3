"""Launched train iterations: with and without the library's second stream, run to run, and through a live RCCL group.  Needs a GPU."""
import json
import os
import subprocess
import sys

import pytest
import torch

from tests.test_gpu_fused_step import _trainer
from tests.test_gpu_step_ops import _trained_flats

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("cfg", ["cfg2_nerf_inn_llff_hier", "dtu"])
def test_the_second_stream_changes_no_bit(cfg):
    runs = []
    for overlap in (False, True):
        tr, var0 = _trainer(cfg, True)
        tr.overlap = overlap
        losses = [{k: float(v.detach()) for k, v in tr.train_iteration(type(var0)(var0)).items()} for _ in range(6)]
        torch.cuda.synchronize()
        assert tr.fused.desc.overlap == int(overlap)
        runs.append((losses, [f.clone() for f in tr._flats()]))
    assert runs[0][0] == runs[1][0]
    assert all(torch.equal(x, y) for x, y in zip(runs[0][1], runs[1][1]))


def test_training_is_bit_reproducible():
    a, la = _trained_flats(False)
    b, lb = _trained_flats(False)
    assert la == lb and all(torch.equal(x, y) for x, y in zip(a, b))


def test_bench_line_through_a_live_rccl_group():
    """bench.py --force-dist: the rank check and the flat gradient all-reduce through a ONE-rank RCCL process group"""
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT="29633")
    for k in ("RANK", "WORLD_SIZE", "LOCAL_RANK"):
        env.pop(k, None)
    cmd = [sys.executable, os.path.join(ROOT, "bench.py"), "--config", "cfg3", "--lean", "--force-dist", "--steps", "4", "--warmup", "16", "--kernel-steps", "0"]
    r = subprocess.run(cmd, cwd=ROOT, env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    line = json.loads([l for l in r.stdout.splitlines() if l.startswith("{")][-1])
    assert line["ranks_seen"] == 1 and line["backend"] == "nccl" and line["hip_graph"] is False and line["comm_ms"] is not None


def test_the_benchmark_refuses_to_replay():
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--hip-graph", "on", "--lean", "--steps", "1"], cwd=ROOT, capture_output=True, text=True,
                       timeout=600)
    assert r.returncode != 0 and "switched off" in r.stderr
