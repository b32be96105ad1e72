"""TokenStep's batches without tokens, and what becomes of rows that have no request or no page."""
import pytest
import torch

import mlora
from gpu_common import say
from test_gpu_token_step_refused import batch, i32, runs_as_alone, scene  # noqa: F401  (scene is a fixture)

pytestmark = pytest.mark.gpu


def test_a_batch_without_tokens(scene):  # noqa: F811
    say("token step: no tokens")
    step = scene()
    e = i32([])
    for _ in range(2):
        step.begin(mlora.KVBatch(e, e, i32([[0]])), e)
        assert step.layer(0, torch.empty((0, 128), device="cuda", dtype=torch.float16)).shape == (0, 4, 64)
        runs_as_alone(step, scene, batch(3, 2), i32([0, -1, 2]), "after a batch without tokens")
