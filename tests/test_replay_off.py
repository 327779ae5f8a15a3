"""Replay of captured train iterations is switched off (engine.REPLAY_OFF): it is refused before anything is built, and bench.py launches."""
import os
import re

import pytest

from neural_invertible_warp_amd import configs, engine
from neural_invertible_warp_amd._lib import NiwError

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_trainer_refuses_to_replay():
    for device in ("cpu", "cuda:0"):
        with pytest.raises(NiwError, match="switched off.*segmentation fault.*hip_graph=False"):
            engine.INNTrainer(configs.cfg3_barf_inn_llff(device=device), 5, hip_graph=True)


def test_the_benchmark_builds_launched_trainers_by_default():
    import inspect
    import bench
    assert inspect.signature(bench.build_workloads).parameters["hip_graph"].default is False


def test_every_test_that_replays_a_trainer_is_listed():
    """no test builds a replayed trainer outside the list of skipped ones"""
    from tests import conftest
    for name in sorted(os.listdir(os.path.join(ROOT, "tests"))):
        if not re.match(r"test_.*\.py$", name) or name == os.path.basename(__file__):
            continue
        source = open(os.path.join(ROOT, "tests", name)).read()
        for body in re.split(r"^(?=def |@pytest)", source, flags=re.M):
            test = re.match(r"(?:@pytest[^\n]*\n(?:[^d\n][^\n]*\n)*)?def (test_\w+)", body)
            if test and re.search(r"hip_graph=True|hip_graph=graph|hip_graph=hip_graph|_flats\(True\)|FAIL_CAPTURE_RANK|\"--hip-graph\", mode", body):
                assert test[1] in conftest.REPLAYS_A_TRAINER.get(name, ()), (name, test[1])
