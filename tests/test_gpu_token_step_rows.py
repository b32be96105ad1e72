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


def test_rows_without_a_request_are_zeros(scene):  # noqa: F811
    """Whatever batch of a size up to the same power of two ran before, and captured as well."""
    say("token step: rows without a request")
    step = scene()
    x = torch.randn((4, 128), device="cuda").half()
    step.begin(batch(4, 2), i32([0, 1, 2, 0]))
    assert (step.layer(0, x) != 0).any(-1).all()
    for T, gone in ((4, 2), (3, 0), (4, 3)):
        b = batch(T, 1)
        b.tok_req[gone] = -1
        step.begin(b, i32([0] * T))
        out = step.layer(0, x[:T])
        assert (out[gone] == 0).all() and (out[[t for t in range(T) if t != gone]] != 0).any(-1).all()
    full = batch(4, 2)
    step.begin(full, i32([0, 1, 2, 0]))
    step.layer(0, x)
    torch.cuda.synchronize()
    b, slots = batch(4, 1), i32([1, 1, 0, 2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.begin(b, slots)
        out = step.layer(0, x)
    for gone in (1, 3, 0):
        step.begin(full, i32([0, 1, 2, 0]))
        step.layer(0, x)
        b.tok_req.copy_(i32([-1 if t == gone else t for t in range(4)]))
        graph.replay()
        torch.cuda.synchronize()
        assert (out[gone] == 0).all() and (out[[t for t in range(4) if t != gone]] != 0).any(-1).all()


def test_tokens_that_no_page_holds_are_counted(scene):  # noqa: F811
    say("token step: missing pages")
    step = scene()
    x = torch.randn((4, 128), device="cuda").half()
    for missing in (1, 3, 0):
        b = batch(4, 1)
        b.pages[:missing] = -1
        b.tok_req[3] = -1                                      # a row without a request is not missing anything
        step.begin(b, i32([0] * 4))
        assert int(step.bad) == 0
        for _ in range(2):
            step.layer(0, x)
        assert int(step.bad) == 2 * missing
    slots = i32([0] * 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.begin(b, slots)
        step.layer(0, x)
    for missing in (2, 0, 1):
        b.pages.copy_(i32([[-1 if t < missing else t] for t in range(4)]))
        graph.replay()
        assert int(step.bad) == missing
