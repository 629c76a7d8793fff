"""Steps whose draft tokens are dropped again: the plan gives their pages back, none is lost and none handed out twice."""
import numpy as np
import pytest
import torch

from oracle.latent_cache_ref import append_ref, attend_ref, plan_ref
from tests.cache_inputs import on, requests, share_of_bound

DEV = "cuda:0"


def _state(n, ctx, page, spare, seed, width=3):
    rng = np.random.default_rng(seed)
    kv_len = rng.integers(0, ctx + 1, n).astype(np.int32)
    table, n_pages = requests(kv_len, page, spare, rng)
    table = np.concatenate([table, np.full((n, width), -1, dtype=np.int32)], 1)
    free = rng.permutation(np.setdiff1d(np.arange(n_pages), table))
    stack = np.full(n_pages, -7, dtype=np.int32)
    stack[:len(free)] = free
    return rng, kv_len, table, stack, len(free), n_pages


def _step(rng, kv_len, new, drop, ending=0.1):
    n = len(kv_len)
    new_len = rng.integers(0, new + 1, n)
    new_len[rng.random(n) < ending] = -1
    rejected = np.where(rng.random(n) < 0.6, rng.integers(0, drop + 1, n), 0)
    rejected[::7] = 10 ** 6                      # more than there are
    rejected[3::7] = -5
    return new_len.astype(np.int32), rejected.astype(np.int32)


def _held(p, page):
    return [int(p.block_table[i, k]) for i in range(len(p.kv_len)) for k in range(-(-int(p.kv_len[i]) // page))]


@pytest.mark.parametrize("seed", range(6))
def test_no_page_is_lost(seed):
    page = 16
    rng, kv_len, table, stack, count, n_pages = _state(30, 90, page, 25, seed)
    for _ in range(12):
        new_len, rejected = _step(rng, kv_len, 20, 40)
        p = plan_ref(kv_len, new_len, table, stack, count, page, int(np.maximum(new_len, 0).sum()) - 3, 5, rejected)
        assert sorted(_held(p, page) + list(p.free_pages[:p.free_count])) == list(range(n_pages))
        used = p.slots[p.slots >= 0]
        assert len(set(used)) == len(used) == p.admitted.sum()
        kv_len, table, stack, count = p.kv_len, p.block_table, p.free_pages, p.free_count


def test_kv_len_set_back_by_hand_loses_them():
    # what the definition says: a request's pages are those of kv_len tokens
    table, stack = np.array([[0, -1, -1, -1]]), np.arange(7, 0, -1)
    by_hand, dropped = (15, table, stack, 7), (15, table, stack, 7)
    for _ in range(3):
        p = plan_ref([by_hand[0]], [2], *by_hand[1:], 16, 2, 5)
        by_hand = (int(p.kv_len[0]) - 2, p.block_table, p.free_pages, p.free_count)
        p = plan_ref([dropped[0]], [2], *dropped[1:], 16, 2, 5, [0 if dropped[0] == 15 else 2])
        dropped = (int(p.kv_len[0]), p.block_table, p.free_pages, p.free_count)
    assert by_hand[3] == 4 and dropped[3] == 6


def _same(want, p, d):
    got = (p.slots, p.query_meta, p.kv_len, p.free_count, p.admitted, d[2], d[3])
    return [name for name, g, w in zip(want._fields, got, want) if not np.array_equal(g.cpu().numpy(), np.atleast_1d(w))]


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("n, ctx, new, drop", [(1, 1, 1, 1), (7, 64, 3, 5), (33, 300, 5, 200), (513, 90, 3, 4), (1500, 400, 1, 40), (8192, 40, 1, 2), (3, 5000, 3000, 4000)])
def test_steps(n, ctx, new, drop, page):
    from test_operator_b200 import op
    rng, kv_len, table, stack, count, _ = _state(n, ctx, page, n * (new // 16 + 1), n + page, width=new // 16 + 2)
    new_len, rejected = _step(rng, kv_len, new, drop)
    for max_tokens in (int(np.maximum(new_len, 0).sum()) + 13, int(np.maximum(new_len, 0).sum()) // 2 + 1):
        want = plan_ref(kv_len, new_len, table, stack, count, page, max_tokens, 9, rejected)
        d = on(DEV, kv_len, new_len, table, stack, np.array([count], dtype=np.int32))
        rej = on(DEV, rejected)[0]
        for _ in range(2):                       # the same call again does the same
            assert _same(want, op.cache_plan(*d, page, max_tokens, 9, rej), d) == []
        assert np.array_equal(rej.cpu().numpy(), rejected)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(4))
def test_too_few_pages(seed):
    from test_operator_b200 import op
    rng, kv_len, table, stack, _, _ = _state(60, 100, 16, 15, seed, width=12)
    new_len, rejected = _step(rng, kv_len, 150, 30, ending=0.0)
    count = 3
    want = plan_ref(kv_len, new_len, table, stack, count, 16, 6000, 9, rejected)
    short = (want.admitted == 0) & (new_len > 0)
    assert short.any() and np.array_equal(want.kv_len[short], kv_len[short])       # (dropped tokens of those stay for the next step to drop)
    d = on(DEV, kv_len, new_len, table, stack, np.array([count], dtype=np.int32))
    assert _same(want, op.cache_plan(*d, 16, 6000, 9, rejected=on(DEV, rejected)[0]), d) == []


@pytest.mark.gpu
def test_lengths_that_make_no_sense():
    from test_operator_b200 import op
    big = 2 ** 31 - 1
    kv_len = np.array([20, -3, big, 7, 40, 80, 33], dtype=np.int32)
    new_len = np.array([3, 2, 1, big, -(2 ** 31), 0, 1], dtype=np.int32)
    rejected = np.array([-(2 ** 31), big, big, big, big, big, 33], dtype=np.int32)
    table, stack = np.arange(7 * 5, dtype=np.int32).reshape(7, 5), np.arange(100, 140, dtype=np.int32)
    d = on(DEV, kv_len, new_len, table, stack, np.array([10], dtype=np.int32))
    p = op.cache_plan(*d, page_size=16, max_tokens=64, topk=1, rejected=on(DEV, rejected)[0])
    # (request 3 asks for more rows than there can be, and what stands behind it has none)
    assert p.kv_len.tolist() == [23, -3, big, 7, 0, 80, 33] and p.admitted.tolist() == [3, 0, 0, 0, 0, 0, 0]
    assert p.slots.tolist() == [20, 21, 22] + [-1] * 61 and p.free_count.tolist() == [13]
    assert d[3][:13].tolist() == list(range(100, 110)) + [20, 21, 22]


@pytest.mark.gpu
def test_refusals_and_both_ways(monkeypatch):
    from test_operator_b200 import op
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    call = lambda rejected: [t.tolist() for t in op.cache_plan(i32(40, 20), i32(2, -1), torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4), i32(9, 8, 0, 0, 0, 0),  # noqa: E731,E501
                                                               i32(2), 16, 4, 7, rejected)]
    for bad in (i32(1), i32(1, 1).long(), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32, device=DEV), i32(0, 0, 0, 0)[::2], [1, 1]):
        with pytest.raises(RuntimeError, match="rejected"):
            call(bad)
    want = call(i32(25, 1))
    assert want[0] == [15, 1 * 16, -1, -1] and want[2] == [17, 0] and want[3] == [5]
    assert call(None) == call(i32(0, 0)) != want
    monkeypatch.setattr(op, "_native", op._NoNativeHost)
    assert call(i32(25, 1)) == want and call(None) == call(i32(0, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_drafts_of_a_server(captured):
    """Each step appends a token and three drafts of every request, attends, and drops some of the drafts in the next one."""
    from test_operator_b200 import op
    page, n, width, n_pages, drafts, heads, topk = 16, 5, 8, 36, 4, 16, 40
    rng = np.random.default_rng(5)
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)  # noqa: E731
    rows = n * drafts + 3
    cache = op.LatentCache.empty(n_pages, page, DEV)
    kv_len, new_len, rejected, table = i32([0] * n), i32([0] * n), i32([0] * n), torch.full((n, width), -1, dtype=torch.int32, device=DEV)
    free, count = i32(rng.permutation(n_pages)), i32([n_pages])
    kv, q = (torch.zeros(rows, *shape, dtype=torch.bfloat16, device=DEV) for shape in ((576,), (heads, 576)))
    picks = torch.zeros(rows, topk, device=DEV)
    got = {}

    def step():
        plan = op.cache_plan(kv_len, new_len, table, free, count, page, rows, topk, rejected)
        op.cache_append(kv, cache, plan.slots)
        indices = (picks * (plan.query_meta[:, 2:3] + 1)).to(torch.int32)
        got["o"], got["lse"] = op.mla_fwd_cached(q, cache, table, indices, plan.query_meta)
        got["indices"], got["plan"] = indices, plan
        kv_len.copy_(plan.kv_len)
        count.copy_(plan.free_count)

    step()                                       # (no new tokens: changes nothing)
    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    ref_v, ref_s = np.zeros((n_pages, page, 576)), np.zeros(n_pages)
    state = (np.zeros(n, dtype=np.int64), table.cpu().numpy(), free.cpu().numpy(), n_pages)
    for k in range(14):
        lens = [drafts] * n if k != 9 else [drafts, -1, drafts, 0, drafts]
        drop = rng.integers(0, drafts, n) if k else np.zeros(n, dtype=np.int64)
        new_len.copy_(i32(lens))
        rejected.copy_(i32(drop))
        kv.copy_(torch.from_numpy(rng.standard_normal((rows, 576)) * (1 + 2 * (k % 3))))
        q.copy_(torch.from_numpy(rng.standard_normal((rows, heads, 576))))
        picks.copy_(torch.from_numpy(rng.random((rows, topk))))
        graph.replay() if captured else step()
        torch.cuda.synchronize()
        want = plan_ref(state[0], lens, state[1], state[2], state[3], page, rows, topk, drop)
        assert _same(want, got["plan"], (None, None, table, free)) == [] and count.tolist() == [want.free_count]
        assert sorted(_held(want, page) + list(want.free_pages[:want.free_count])) == list(range(n_pages))
        ref_v, ref_s = append_ref(kv.double().cpu().numpy(), ref_v, ref_s, want.slots)
        assert np.array_equal(cache.values.float().cpu().numpy(), ref_v) and np.array_equal(cache.scales.cpu().numpy(), ref_s)
        ref = attend_ref(q, cache.values, cache.scales, table, got["indices"], got["plan"].query_meta)
        assert share_of_bound(got["o"], ref.o, ref.o_bound) <= 1
        state = (want.kv_len, want.block_table, want.free_pages, want.free_count)
