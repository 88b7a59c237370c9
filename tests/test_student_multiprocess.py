"""Sandwich norms, gates and distillation with tensor parallelism: the parameters of the new norms and gates are replicas whose
gradients come from every rank's tokens, and the teacher's tensors are split as the labels are."""
import os

import pytest

from jaxpp_b200.launch import launch

WORKER = os.path.join(os.path.dirname(os.path.abspath(__file__)), "student_worker.py")


@pytest.mark.parametrize("scenario,nproc", [("tp2", 2), ("pp2_tp2", 4)])
def test_student_sharded(scenario, nproc):
    assert launch([WORKER, scenario], nproc, env={"CUDA_VISIBLE_DEVICES": "", "OMP_NUM_THREADS": "1"}, timeout_s=300) == 0
