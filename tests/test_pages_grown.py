"""The rows that the last resize made longer, as the host sees them before any launch: no GPU is needed."""
import torch

import mlora


def test_no_row_may_be_written_before_a_resize():
    cache = mlora.KVCache(1, 70, 1, 64, device="cpu")
    p = mlora.KVPages(cache, 5, 4)
    assert p.grown.dtype == torch.int32 and p.grown.tolist() == [-1] * 5
    # behind the managed pages' bytes, a byte for each of 128 pages, and apart from what a snapshot holds
    assert p.grown.data_ptr() - p.scratch.data_ptr() == 128
    assert not p.state.data_ptr() <= p.grown.data_ptr() < p.state.data_ptr() + p.state.numel() * 4
    assert p._managed.sum() == 70 and not p.scratch[32 + 5:].any()


def test_adopted_tables_name_no_row():
    cache = mlora.KVCache(1, 20, 1, 64, device="cpu")
    p = mlora.KVPages(cache, 3, 4)
    p.grown.copy_(torch.arange(3))
    p.adopt(torch.full((3, 4), -1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    assert p.grown.tolist() == [-1] * 3
