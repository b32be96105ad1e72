"""TokenStep after a batch that was refused: nothing of it is used, and the next batch is as if it had not been there.  The launches are stood
in for, so no GPU is needed."""
from types import SimpleNamespace

import pytest
import torch

import mlora
from mlora import token_step as ts


@pytest.fixture
def step(monkeypatch):
    """A step whose plans are records: what they were made from, and for an attention plan how many prefixes its buffer holds."""
    calls = SimpleNamespace(refuse_attention=False, refuse_decode=False, seen=[])

    def plan_decode(tok, pool, out=None, n_proj=None):
        if calls.refuse_decode:
            raise TypeError("tok_adapter must be int32")
        out = out if out is not None else SimpleNamespace()
        out.tok_adapter = tok
        return out

    def plan_attention(batch, cache, n_q_heads, out=None, room=0):
        n = 0 if batch.prefix_len is None else batch.prefix_len.numel()
        if calls.refuse_attention or (n and batch.prefix_pages is None):
            raise ValueError("attention over shared prefixes needs prefix_pages")
        if out is None:
            out = SimpleNamespace(holds=max(n, room))
        if n > out.holds:
            raise mlora.MloraError(mlora._ext.MLORA_ENOSPACE, "plan too small")
        out.batch = batch
        return out

    monkeypatch.setattr(ts.ops, "plan_decode", plan_decode)
    monkeypatch.setattr(ts, "plan_attention", plan_attention)
    monkeypatch.setattr(ts.ops, "bgmv", lambda ys, xs, pool, layer, names, tok, plan, accumulate: calls.seen.append((tok, plan.tok_adapter)))
    monkeypatch.setattr(ts, "kv_append", lambda q, k, v, cache, layer, batch, rope, **kw: calls.seen.append(batch))
    monkeypatch.setattr(ts, "prefix_attention", lambda q, cache, layer, plan, scale, out: calls.seen.append(plan.batch) or out)
    pool = mlora.AdapterPool(1, {"q": (64, 256), "k": (64, 128), "v": (64, 128)}, 2, 4, max_rank=16, device="cpu")
    s = mlora.TokenStep(pool, mlora.KVCache(1, 4, 2, 64, device="cpu"), None, 4)
    s.calls = calls
    return s


def batch(T, n_prefix=0, pages=True):
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32)      # noqa: E731
    if not n_prefix:
        return mlora.KVBatch(i(T), i(T), i(T, 1))
    return mlora.KVBatch(i(T), i(T), i(T, 1), i(T), i(n_prefix, 1) if pages else None, i(n_prefix))


def adapters(T):
    return torch.zeros(T, dtype=torch.int32)


def runs(step, b, tok):
    """One layer of the batch: every operator meets this batch, its adapters and the plans made from them."""
    step.begin(b, tok)
    step.calls.seen.clear()
    step.layer(0, torch.zeros((b.T, 64), dtype=torch.float16))
    (given, planned), appended, attended = step.calls.seen
    assert given is tok and planned is tok and appended is b and attended is b


def test_a_refused_first_batch(step):
    with pytest.raises(ValueError):
        step.begin(batch(3, 2, pages=False), adapters(3))
    with pytest.raises(RuntimeError, match="begin"):
        step.layer(0, torch.zeros((3, 64), dtype=torch.float16))
    runs(step, batch(3), adapters(3))
    runs(step, batch(3, 2), adapters(3))


def test_a_refused_batch_of_the_same_size(step):
    runs(step, batch(3), adapters(3))
    with pytest.raises(ValueError):
        step.begin(batch(3, 2, pages=False), adapters(3))
    with pytest.raises(RuntimeError, match="begin"):
        step.layer(0, torch.zeros((3, 64), dtype=torch.float16))
    runs(step, batch(3), adapters(3))


def test_refused_adapters_of_the_same_size(step):
    runs(step, batch(3), adapters(3))
    step.calls.refuse_decode = True
    with pytest.raises(TypeError):
        step.begin(batch(3), adapters(3).long())
    with pytest.raises(RuntimeError, match="begin"):
        step.layer(0, torch.zeros((3, 64), dtype=torch.float16))
    step.calls.refuse_decode = False
    runs(step, batch(3), adapters(3))


def test_refused_adapters_of_a_first_batch(step):
    step.calls.refuse_decode = True
    with pytest.raises(TypeError):
        step.begin(batch(3, 1), adapters(3).long())
    step.calls.refuse_decode = False
    runs(step, batch(3, 1), adapters(3))


@pytest.mark.parametrize("n", [3, 4097])
def test_a_refused_growth_in_prefixes(step, n):
    runs(step, batch(3, 1), adapters(3))
    step.calls.refuse_attention = True
    with pytest.raises(ValueError):
        step.begin(batch(3, n), adapters(3))
    step.calls.refuse_attention = False
    runs(step, batch(3, 3), adapters(3))
    runs(step, batch(3, 1), adapters(3))


def test_a_batch_and_adapters_of_unlike_length(step):
    runs(step, batch(3), adapters(3))
    with pytest.raises(ValueError, match="every token"):
        step.begin(batch(4), adapters(3))
    with pytest.raises(RuntimeError, match="begin"):
        step.layer(0, torch.zeros((3, 64), dtype=torch.float16))
    runs(step, batch(4), adapters(4))


def test_a_batch_without_tokens(step):
    runs(step, batch(0), adapters(0))
    runs(step, batch(2), adapters(2))
    runs(step, batch(0), adapters(0))


def test_rows_without_a_request_hold_nothing_of_earlier_batches(step):
    """Batches of three and four tokens share a buffer; what a row without a request holds of it is zeros."""
    step.begin(batch(4), adapters(4))
    step.out.fill_(5.0)
    for T in (3, 4, 4):
        step.begin(batch(T), adapters(T))
        assert (step.out == 0).all()
        step.out.fill_(5.0)


def test_tokens_left_out_are_counted_per_step(step, monkeypatch):
    given = []
    monkeypatch.setattr(ts, "kv_append", lambda *a, bad: given.append(bad) or bad.add_(3))
    for _ in range(2):
        step.begin(batch(4), adapters(4))
        assert int(step.bad) == 0 and step.bad.dtype == torch.int32
        for _ in range(2):
            step.layer(0, torch.zeros((4, 64), dtype=torch.float16))
        assert int(step.bad) == 6 and all(b is step.bad for b in given)
