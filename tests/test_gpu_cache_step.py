"""The three together as a server uses them: every step plans, appends and attends; captured once and replayed for later steps."""
import numpy as np
import pytest
import torch

from oracle.latent_cache_ref import append_ref, attend_ref, plan_ref
from tests.cache_inputs import share_of_bound

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("captured", [False, True])
def test_steps_of_a_server(captured):
    from test_operator_b200 import op
    page, n, width, n_pages, rows, heads, topk = 16, 6, 12, 40, 64, 16, 24
    rng = np.random.default_rng(17)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    cache = op.LatentCache.empty(n_pages, page, DEV)
    kv_len, new_len, table = i32([0] * n), i32([0] * n), torch.full((n, width), -1, dtype=torch.int32, device=DEV)
    free, count = i32(rng.permutation(n_pages)), i32([n_pages])
    kv = torch.zeros(rows, 576, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(rows, heads, 576, dtype=torch.bfloat16, device=DEV)
    picks = torch.zeros(rows, topk, device=DEV)
    got = {}

    def step():
        plan = op.cache_plan(kv_len, new_len, table, free, count, page, rows, topk)
        op.cache_append(kv, cache, plan.slots)
        indices = (picks * (plan.query_meta[:, 2:3] + 1)).to(torch.int32)
        got["o"], got["lse"] = op.mla_fwd_cached(q, cache, table, indices, plan.query_meta)
        got["indices"], got["plan"] = indices, plan
        kv_len.copy_(plan.kv_len)
        count.copy_(plan.free_count)

    if captured:
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()                                  # (no new tokens yet: changes nothing)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    ref_v, ref_s = np.zeros((n_pages, page, 576)), np.zeros(n_pages)
    state = (np.zeros(n, dtype=np.int64), table.cpu().numpy(), free.cpu().numpy(), n_pages)
    steps = [[7, 16, 3, 0, 0, 1], [1, 1, 1, 0, 20, 1], [1, -1, 1, 1, 1, 1], [1, 9, -1, 1, 1, -1], [1, 1, 1, 1, 1, 1], [2, 2, 2, 2, 2, 2]] + [[1] * n] * 4
    for k, lens in enumerate(steps):
        new_len.copy_(i32(lens))
        kv.copy_(torch.from_numpy(rng.standard_normal((rows, 576)) * (1 + 2 * (k % 3))))
        q.copy_(torch.from_numpy(rng.standard_normal((rows, heads, 576))))
        picks.copy_(torch.from_numpy(rng.random((rows, topk))))
        graph.replay() if captured else step()
        torch.cuda.synchronize()
        want = plan_ref(state[0], lens, state[1], state[2], state[3], page, rows, topk)
        ref_v, ref_s = append_ref(kv.double().cpu().numpy(), ref_v, ref_s, want.slots)
        assert np.array_equal(got["plan"].slots.cpu().numpy(), want.slots) and np.array_equal(table.cpu().numpy(), want.block_table)
        assert np.array_equal(kv_len.cpu().numpy(), want.kv_len) and count.tolist() == [want.free_count]
        assert np.array_equal(cache.values.float().cpu().numpy(), ref_v) and np.array_equal(cache.scales.cpu().numpy(), ref_s)
        ref = attend_ref(q, cache.values, cache.scales, table, got["indices"], got["plan"].query_meta)
        assert torch.equal(got["lse"].isposinf(), ref.lse.isposinf()) and got["lse"].isfinite().any(1).sum() == want.admitted.sum()
        assert share_of_bound(got["o"], ref.o, ref.o_bound) <= 1
        state = (want.kv_len, want.block_table, want.free_pages, want.free_count)


def test_stored_rows_give_what_bf16_rows_give():
    # over rows that e4m3 holds exactly the cached forward and the bf16 one are the same function
    from test_operator_b200 import op
    n, heads, topk = 300, 64, 200
    gen = torch.Generator(device=DEV).manual_seed(0)
    kv = torch.randn(n, 576, generator=gen, device=DEV).mul(64).clamp(-448, 448).to(torch.float8_e4m3fn).to(torch.bfloat16) / 64
    q = torch.randn(n, heads, 576, generator=gen, device=DEV, dtype=torch.bfloat16)
    cache = op.LatentCache.empty(8, 64, DEV)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    table = torch.full((1, 6), -1, dtype=torch.int32, device=DEV)
    plan = op.cache_plan(i32([0]), i32([n]), table, i32(list(range(8))), i32([8]), 64, n, topk)
    op.cache_append(kv, cache, plan.slots)
    indices = torch.randint(0, n, (n, topk), generator=gen, device=DEV, dtype=torch.int32)
    o, lse = op.mla_fwd_cached(q, cache, table, indices, plan.query_meta, check_device_status=True)
    o2, lse2 = op.mla_fwd(q, kv, indices)
    some = lse2.isfinite()
    assert torch.equal(lse.isfinite(), some)
    assert (o - o2).float().norm() <= 2 ** -7 * o2.float().norm() and (lse - lse2)[some].abs().max() <= 1e-4
