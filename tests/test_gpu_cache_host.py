"""The cache's calls through the compiled host module and the Python way: the same results; what the module leaves to the other way still runs."""
import pytest
import torch

from tests.cache_inputs import random_cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _step():
    """Everything that the three entries return and change."""
    from test_operator_b200 import op
    table = torch.full((3, 4), -1, dtype=torch.int32, device=DEV)
    table[1, 0] = 9
    free = torch.arange(12, dtype=torch.int32, device=DEV)
    plan = op.cache_plan(_i32(0, 5, 0), _i32(20, 3, 1), table, free, _i32(8), 16, 27, 6)
    values, scales = random_cache(12, 16, DEV, seed=1)
    cache = op.LatentCache(values, scales)
    gen = torch.Generator(device=DEV).manual_seed(2)
    kv = torch.randn(27, 576, generator=gen, device=DEV, dtype=torch.bfloat16)
    assert op.cache_append(kv, cache, plan.slots) is None
    q = torch.randn(27, 16, 576, generator=gen, device=DEV, dtype=torch.bfloat16)
    idx = torch.randint(-1, 20, (27, 6), generator=gen, device=DEV, dtype=torch.int32)
    o, lse = op.mla_fwd_cached(q, cache, table, idx, plan.query_meta)
    o2, lse2 = op.mla_fwd_cached(q, cache, table, idx, plan.query_meta, sm_scale=0.1, causal=False, lse_is_base2=False)
    return [*plan, table, free, values.view(torch.uint8), scales, o, lse, o2, lse2]


def test_both_ways_agree(monkeypatch):
    from test_operator_b200 import op
    native = op._host()
    if native is op._NoNativeHost:
        pytest.skip("no compiled host module here")
    got = _step()
    monkeypatch.setattr(op, "_native", op._NoNativeHost)
    want = _step()
    assert all(a.shape == b.shape and a.dtype == b.dtype and a.is_contiguous() and torch.equal(a, b) for a, b in zip(got, want))


def test_plain_calls_take_the_module():
    from test_operator_b200 import op
    native = op._host()
    if native is op._NoNativeHost:
        pytest.skip("no compiled host module here")
    values, scales = random_cache(4, 16, DEV)
    cache = op.LatentCache(values, scales)
    kv = torch.zeros(2, 576, dtype=torch.bfloat16, device=DEV)
    table, meta, idx = torch.zeros(1, 4, dtype=torch.int32, device=DEV), torch.zeros(2, 4, dtype=torch.int32, device=DEV), torch.zeros(2, 5, dtype=torch.int32, device=DEV)
    q = torch.zeros(2, 8, 576, dtype=torch.bfloat16, device=DEV)
    assert type(native.cache_plan(_i32(0), _i32(1), table, _i32(1, 2), _i32(2), 16, 1, 5)) is tuple
    assert native.cache_append(kv, cache, _i32(0, 1)) == 0
    assert type(native.fwd_cached(q, cache, table, idx, meta, None, 1, 1)) is tuple
    # and what they do not take
    assert native.cache_plan(_i32(0), _i32(1), table, _i32(1, 2), _i32(2), 16, 0, 5) is None
    assert native.cache_plan(_i32(0, 0), _i32(1), table, _i32(1, 2), _i32(2), 16, 1, 5) is None
    assert native.cache_append(torch.zeros(2, 600, dtype=torch.bfloat16, device=DEV)[:, :576], cache, _i32(0, 1)) is None
    assert native.cache_append(kv, (values,), _i32(0, 1)) is None
    assert native.cache_append(kv, (values, scales.double()), _i32(0, 1)) is None
    assert native.fwd_cached(q, cache, table, idx.long(), meta, None, 1, 1) is None
    assert native.fwd_cached(q, cache, table, idx, meta[:1], None, 1, 1) is None
    assert native.fwd_cached(q.cpu(), cache, table, idx, meta, None, 1, 1) is None


def test_outputs_of_a_plan_are_tensors_of_their_own():
    from test_operator_b200 import op
    table, free = torch.zeros(1, 4, dtype=torch.int32, device=DEV), torch.arange(4, dtype=torch.int32, device=DEV)
    plan = op.cache_plan(_i32(0), _i32(3), table, free, _i32(4), 16, 5, 7)
    assert plan.query_meta.data_ptr() % 16 == 0
    keep = [t.clone() for t in plan]
    for k, t in enumerate(plan):
        t.fill_(77)
        assert all(torch.equal(u, w) for u, w in list(zip(plan, keep))[k + 1:])
    assert plan.slots[1:].add(1).tolist() == [78] * 4 and plan.kv_len.cpu().tolist() == [77]
