"""How finely the plan cuts prefixes, and the attention over ranges of every length it takes."""
import pytest
import torch

import mlora
from gpu_common import say
from step_ref import Scene

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("heads, kv, requests, prefixes, prefix", [(32, 8, 64, 8, 1500), (64, 8, 32, 8, 1500), (64, 8, 8, 1, 8000)])
def test_ranges_of_256_keys_are_not_halved_for_smaller_heads(heads, kv, requests, prefixes, prefix):
    """The plan's items (its first word) for 64 and for 128 elements a head, where a range is two steps of 128 keys."""
    n = prefix // 64 + 1
    batch = mlora.KVBatch(i32(range(requests)), i32([prefix + 10] * requests), i32([[0, 1]] * requests), i32([r % prefixes for r in range(requests)]),
                          i32([list(range(n))] * prefixes), i32([prefix] * prefixes))
    items = [int(mlora.plan_attention(batch, mlora.KVCache(1, n, kv, D, page_tokens=64), heads).buf[:4].view(torch.int32)) for D in (64, 128)]
    assert items[0] == items[1]


@pytest.mark.parametrize("own", [20, 400, 900])
@pytest.mark.parametrize("requests, prefix", [(9, 3000), (40, 1500)])
def test_ranges_of_many_lengths(requests, prefix, own):
    say(f"attention ranges {requests} {prefix} {own}")
    s = Scene([(r % 3 - 1, 1 + (r * 7919) % own) for r in range(requests)], [prefix, prefix // 2 + 7], 16, 8, 64, 16, torch.bfloat16, seed=own)
    plan = mlora.plan_attention(s.batch, s.cache, 16)
    s.compare(mlora.prefix_attention(s.dev_q, s.cache, 0, plan), tokens=[0, 1, 2, 5, requests - 1], heads=[0, 15])
