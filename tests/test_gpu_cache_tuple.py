"""A cache given as a plain pair (values, scales): the same through every way that a call can take."""
import pytest
import torch

from tests.cache_inputs import random_cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_plain_pair_is_a_cache():
    from test_operator_b200 import op
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    kv = torch.randn(3, 1152, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0)).bfloat16()[:, 576:]
    q = torch.randn(3, 16, 576, device=DEV, dtype=torch.bfloat16)
    table, idx, meta = i32(1, 0, 2).view(1, 3), i32(*range(12)).view(3, 4), i32(0, 40, 39, 4, 0, 40, 38, 4, 0, 40, 2, 4).view(3, 4)
    results = []
    for make in (op.LatentCache, lambda *pair: pair):
        cache = make(*random_cache(4, 16, DEV, 3))
        op.cache_append(kv, cache, i32(0, 17, 40))                       # strided rows
        op.cache_append(kv.contiguous(), cache, i32(1, 18, 41))
        need = op._fwd_cached_workspace_bytes(3, 16, 4, 4, 16, 1, 3, 0)
        for kwargs in ({}, {"workspace": op.Workspace(need, DEV)}, {"check_device_status": True}, {"workspace_budget": 1 << 20}):
            results.append(op.mla_fwd_cached(q, cache, table, idx, meta, **kwargs))
        results[-1] = (*results[-1], *cache)
    half = len(results) // 2
    for a, b in zip(results[:half], results[half:]):
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))
