"""Tables of a serving step against plain loops: whole numbers, equal."""
import numpy as np
import pytest
import torch

from oracle.latent_cache_ref import plan_ref
from tests.cache_inputs import on, requests

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _inputs(n, ctx, new, page, spare_pages, ending, seed, width=4):
    rng = np.random.default_rng(seed)
    kv_len = rng.integers(0, ctx + 1, n)
    table, n_pages = requests(kv_len, page, spare_pages, rng)
    table = np.concatenate([table, np.full((n, width), -1, dtype=np.int32)], 1)
    free = rng.permutation(np.setdiff1d(np.arange(n_pages), table))
    stack = np.full(n_pages, -7, dtype=np.int32)
    stack[:len(free)] = free
    new_len = rng.integers(0, new + 1, n)
    new_len[rng.random(n) < ending] = -1
    return kv_len.astype(np.int32), new_len.astype(np.int32), table, stack, len(free)


def _check(kv_len, new_len, table, stack, free_count, page, max_tokens, topk=9):
    from test_operator_b200 import op
    want = plan_ref(kv_len, new_len, table, stack, min(max(free_count, 0), len(stack)), page, max_tokens, topk)
    d = on(DEV, kv_len, new_len, table, stack, np.array([free_count], dtype=np.int32))
    first = None
    for _ in range(2):          # the same call again does the same
        p = op.cache_plan(*d, page_size=page, max_tokens=max_tokens, topk=topk)
        got = (p.slots, p.query_meta, p.kv_len, p.free_count, p.admitted, d[2], d[3])
        for name, g, w in zip(want._fields, got, want):
            assert np.array_equal(g.cpu().numpy(), np.atleast_1d(w)), name
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, got))
        first = [t.clone() for t in got]
    assert torch.equal(d[0].cpu(), torch.from_numpy(kv_len)) and torch.equal(d[1].cpu(), torch.from_numpy(new_len)) and int(d[4]) == free_count
    return want


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("n, ctx, new", [(1, 0, 1), (1, 1, 1), (7, 64, 1), (33, 300, 5), (511, 128, 2), (512, 90, 1), (513, 90, 3), (1500, 400, 1), (8192, 40, 1), (3, 5000, 3000)])
def test_steps(n, ctx, new, page):
    kv_len, new_len, table, stack, free = _inputs(n, ctx, new, page, n * (new // 16 + 2), 0.1, n + page, width=new // 16 + 2)
    _check(kv_len, new_len, table, stack, free, page, int(np.maximum(new_len, 0).sum()) + 13)


@pytest.mark.parametrize("seed", range(6))
def test_too_few_pages(seed):
    # requests that do not fit get nothing, later ones that need no page still get their rows; pages of the ones that end are at hand at once
    kv_len, new_len, table, stack, free = _inputs(60, 100, 40, 16, 15, 0.2 if seed % 2 else 0.0, seed)
    want = _check(kv_len, new_len, table, stack, free, 16, 2000)
    assert (want.admitted[new_len > 0] == 0).any() or (new_len < 0).any()      # (with what comes back there may be enough)


def test_rows_and_table_too_narrow():
    kv_len, new_len, table, stack, free = _inputs(40, 100, 60, 16, 400, 0.0, 1, width=1)      # some would need more pages than the table is wide
    want = _check(kv_len, new_len, table, stack, free, 16, 1000)
    assert (want.admitted[new_len > 0] == 0).any()
    _check(kv_len, new_len, table, stack, free, 16, 100)                                      # most rows do not fit


def test_lengths_that_make_no_sense():
    kv_len = np.array([5, -3, 2 ** 31 - 1, 7, 40, -1], dtype=np.int32)
    new_len = np.array([3, 2, 2 ** 31 - 1, 2 ** 31 - 1, -(2 ** 31), -1], dtype=np.int32)
    table = np.arange(6 * 5, dtype=np.int32).reshape(6, 5)
    stack = np.arange(100, 140, dtype=np.int32)
    from test_operator_b200 import op
    d = on(DEV, kv_len, new_len, table, stack, np.array([10], dtype=np.int32))
    p = op.cache_plan(*d, page_size=16, max_tokens=64, topk=1)
    # the first one fits; the others ask for more than there can be, and what stands behind them has no row
    assert p.admitted.tolist() == [3, 0, 0, 0, 0, 0] and p.kv_len.tolist() == [8, -3, 2 ** 31 - 1, 7, 0, 0]
    assert p.slots.tolist() == [5, 6, 7] + [-1] * 61
    assert p.free_count.tolist() == [13] and d[3][:13].tolist() == list(range(100, 110)) + [20, 21, 22]


def test_step_of_endings_alone_and_a_stack_that_is_full():
    kv_len, new_len, table, stack, free = _inputs(20, 90, 1, 16, 5, 1.0, 4)
    _check(kv_len, new_len, table, stack, free, 16, 0)
    _check(kv_len, new_len, table, stack[:free + 3], free, 16, 0)          # no room for all pages: the rest is dropped, nothing is written behind the end
    for count in (-5, 2 ** 31 - 1):                                        # a count outside the stack is taken as its nearest end
        _check(kv_len, np.zeros_like(new_len), table, stack, count, 16, 3)


def test_on_another_stream_and_in_a_graph():
    from test_operator_b200 import op
    kv_len, new_len, table, stack, free = _inputs(50, 200, 3, 32, 60, 0.1, 5)
    d = on(DEV, kv_len, new_len, table, stack, np.array([free], dtype=np.int32))
    want = plan_ref(kv_len, new_len, table, stack, free, 32, 160, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p = op.cache_plan(*d, page_size=32, max_tokens=160, topk=9)
    side.synchronize()
    assert np.array_equal(p.slots.cpu().numpy(), want.slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = op.cache_plan(*d, page_size=32, max_tokens=160, topk=9)
    for shift in (0, 1):
        lens = np.maximum(kv_len - shift, 0)
        d[0].copy_(torch.from_numpy(lens))
        d[2].copy_(torch.from_numpy(table))
        d[3].copy_(torch.from_numpy(stack))
        graph.replay()
        torch.cuda.synchronize()
        want = plan_ref(lens, new_len, table, stack, free, 32, 160, 9)
        assert np.array_equal(p.slots.cpu().numpy(), want.slots) and np.array_equal(p.query_meta.cpu().numpy(), want.query_meta)


def test_steps_queued_one_behind_the_other():
    # each plan takes what the one before left, with nothing between the calls
    from test_operator_b200 import op
    n, page, calls, rows = 700, 16, 20, 800
    rng = np.random.default_rng(8)
    table, n_pages = np.full((n, 4), -1, dtype=np.int32), 1500
    stack = rng.permutation(n_pages).astype(np.int32)
    news = [np.where(rng.random(n) < 0.1, -1, 1).astype(np.int32) for _ in range(calls)]
    d_table, d_stack, d_len, d_count = on(DEV, table, stack, np.zeros(n, dtype=np.int32), np.array([n_pages], dtype=np.int32))
    d_news = on(DEV, *news)
    torch.cuda.synchronize()
    plans = []
    for new in d_news:
        plans.append(op.cache_plan(d_len, new, d_table, d_stack, d_count, page, rows, 5))
        d_len, d_count = plans[-1].kv_len, plans[-1].free_count
    state = (np.zeros(n, dtype=np.int64), table, stack, n_pages)
    for new, plan in zip(news, plans):
        want = plan_ref(state[0], new, state[1], state[2], state[3], page, rows, 5)
        assert np.array_equal(plan.slots.cpu().numpy(), want.slots) and np.array_equal(plan.kv_len.cpu().numpy(), want.kv_len)
        state = (want.kv_len, want.block_table, want.free_pages, want.free_count)
    assert np.array_equal(d_table.cpu().numpy(), state[1]) and np.array_equal(d_stack.cpu().numpy(), state[2])
