"""TokenStep on the GPU after a refused batch: the next ones give what a step of their own gives, bit for bit."""
import pytest
import torch

import mlora
from gpu_common import say
from test_gpu_token_step import build

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.fixture
def scene():
    pool, weights, cache, g = build(1, 128, 4, 2, 64, 3, F16, 40, 1)
    packed = [{n: mlora.W4Weight(*w, group=32) for n, w in layer.items()} for layer in weights]
    rope = mlora.RopeTable(128, 64)
    return lambda: mlora.TokenStep(pool, cache, packed, 4, rope)


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def batch(T, n_prefix, prefix_pages=True):
    """Tokens at the first place behind prefixes of 20 + 3 f keys, on pages of their own; prefixes on pages 20 and up."""
    if not n_prefix:
        return mlora.KVBatch(i32(range(T)), i32([5] * T), i32([[t] for t in range(T)]))
    lens = [20 + 3 * f for f in range(n_prefix)]
    of = [t % n_prefix for t in range(T)]
    return mlora.KVBatch(i32(range(T)), i32([lens[f] for f in of]), i32([[t] for t in range(T)]), i32(of),
                         i32([[20 + 2 * f, 21 + 2 * f] for f in range(n_prefix)]) if prefix_pages else None, i32(lens))


def runs_as_alone(step, scene, b, slots, what):
    x = torch.randn((b.T, 128), device="cuda").half()
    alone = scene()
    out = []
    for s in (alone, step):
        s.begin(b, slots)
        out.append(s.layer(0, x).clone())
    assert torch.equal(out[0], out[1]), what


def test_a_refused_batch_leaves_nothing_behind(scene):
    say("token step: refused batches")
    T = 6
    step = scene()
    x = torch.randn((T, 128), device="cuda").half()
    first, second = i32([0, 1, 2, -1, 0, 0]), i32([2, 2, -1, 0, 1, 1])
    with pytest.raises(ValueError, match="prefix_pages"):
        step.begin(batch(T, 2, prefix_pages=False), first)
    with pytest.raises(RuntimeError, match="begin"):
        step.layer(0, x)
    runs_as_alone(step, scene, batch(T, 0), first, "after a refused first batch")
    with pytest.raises(ValueError, match="prefix_pages"):
        step.begin(batch(T, 2, prefix_pages=False), second)
    with pytest.raises(RuntimeError, match="begin"):
        step.layer(0, x)
    runs_as_alone(step, scene, batch(T, 1), first, "after a refused batch of the same size")
    many = batch(T, 1)
    many.prefix_len, many.prefix_pages = i32([20] * 4097), i32([[20, 21]] * 4097)
    with pytest.raises(mlora.MloraError):
        step.begin(many, second)
    runs_as_alone(step, scene, batch(T, 3), second, "after a refused growth in prefixes")
    with pytest.raises(TypeError):
        step.begin(batch(T, 3), first.long())
    with pytest.raises(RuntimeError, match="begin"):
        step.layer(0, x)
    runs_as_alone(step, scene, batch(T, 3), first, "after refused adapters")
