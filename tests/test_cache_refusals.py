"""What the entries of the paged cache refuse, before anything runs: the C ABI's checks (no GPU needed) and the Python entries' messages."""
import ctypes

import pytest
import torch

from test_operator_b200 import op

BAD, WORKSPACE = 1, 3
A = 1 << 20         # an address that is aligned and never used: every call here is turned away on the host


def _plan(**changes):
    v = dict(kv_len=A, new_len=A, free_count=A, block_table=A, free_pages=A, slots=A, query_meta=A, kv_len_out=A, free_count_out=A, admitted=A,
             n_requests=4, max_pages=8, n_free=16, page_size=64, max_tokens=4, topk=5)
    v.update(changes)
    return op.load_library().smla_cache_plan(ctypes.byref(op._CachePlanParams(**v)), None)


@pytest.mark.parametrize("changes", [
    {"kv_len": 0}, {"new_len": 0}, {"free_count": 0}, {"block_table": 0}, {"free_pages": 0}, {"slots": 0}, {"query_meta": 0}, {"query_meta": A + 8},
    {"kv_len_out": 0}, {"free_count_out": 0}, {"admitted": 0}, {"n_requests": 0}, {"n_requests": 8193}, {"max_pages": 0}, {"n_free": 0}, {"page_size": 0},
    {"page_size": 48}, {"page_size": 8}, {"page_size": 256}, {"page_size": -64}, {"max_tokens": -1}, {"max_tokens": 1 << 30}, {"topk": -1},
    {"max_pages": (1 << 24) + 1}, {"n_requests": 8192, "max_pages": 1 << 18, "page_size": 16}])
def test_plan_refuses(changes):
    assert _plan(**changes) == BAD


def _append(workspace=A, workspace_bytes=1 << 30, **changes):
    v = dict(kv=A, slots=A, values=A, scales=A, kv_stride=576, n_rows=4, n_pages=4, page_size=64)
    v.update(changes)
    return op.load_library().smla_cache_append(ctypes.byref(op._CacheAppendParams(**v)), workspace, workspace_bytes, None)


@pytest.mark.parametrize("changes", [
    {"kv": 0}, {"kv": A + 8}, {"slots": 0}, {"values": 0}, {"values": A + 4}, {"scales": 0}, {"kv_stride": 580}, {"kv_stride": -576}, {"n_rows": 0},
    {"n_rows": -1}, {"n_pages": 0}, {"page_size": 63}, {"n_pages": 1 << 25}, {"n_rows": 9000, "workspace": None}, {"n_rows": 9000, "workspace": A + 16}])
def test_append_refuses(changes):
    assert _append(**changes) == BAD


def test_append_asks_for_its_workspace():
    lib = op.load_library()
    assert lib.smla_cache_append_workspace_size(8192) == 0
    need = lib.smla_cache_append_workspace_size(9000)
    assert need >= 9000 * 8 and _append(n_rows=9000, workspace_bytes=need - 1) == WORKSPACE


def _cached(workspace=A, workspace_bytes=1 << 30, **changes):
    v = dict(q=A, values=A, scales=A, block_table=A, indices=A, query_meta=A, o=A, lse=A, s_q=4, h_q=16, topk=7, n_pages=4, page_size=64, n_requests=2, max_pages=2,
             sm_scale=0.0, causal=1, lse_is_base2=1)
    v.update(changes)
    p = op._FwdCachedParams(**v)
    return op.load_library().smla_fwd_cached_run(ctypes.byref(p), workspace, workspace_bytes, None), op.load_library().smla_fwd_cached_workspace_size(ctypes.byref(p), 0)


@pytest.mark.parametrize("changes", [
    {"s_q": 0}, {"h_q": 0}, {"h_q": 12}, {"h_q": 136}, {"topk": 0}, {"n_pages": 0}, {"page_size": 24}, {"n_requests": 0}, {"n_requests": -1}, {"max_pages": 0},
    {"max_pages": 1 << 25}, {"query_meta": A + 4}, {"n_pages": 1 << 26}, {"s_q": 1 << 27}])
def test_forward_refuses_shapes(changes):
    assert _cached(**changes) == (BAD, 0)


@pytest.mark.parametrize("changes", [{n: 0} for n in ("q", "values", "scales", "block_table", "indices", "query_meta", "o", "lse")] +
                         [{"q": A + 8}, {"values": A + 8}, {"o": A + 8}, {"workspace": None}, {"workspace": A + 16}])
def test_forward_refuses_pointers(changes):
    assert _cached(**changes)[0] == BAD


def test_forward_asks_for_its_workspace():
    status, need = _cached(workspace_bytes=100)
    assert status == WORKSPACE and need > 100


def test_tensors_on_the_cpu_are_refused():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA"):
        op.cache_plan(i32(2), i32(2), i32(2, 4), i32(8), i32(1), 64, 2, 5)
    cache = op.LatentCache.empty(4, 64, "cpu")
    assert cache.page_size == 64 and cache.values.shape == (4, 64, 576) and cache.values.dtype == torch.float8_e4m3fn
    with pytest.raises(RuntimeError, match="CUDA"):
        op.cache_append(torch.zeros(2, 576, dtype=torch.bfloat16), cache, i32(2))
    with pytest.raises(RuntimeError, match="CUDA"):
        op.mla_fwd_cached(torch.zeros(2, 16, 576, dtype=torch.bfloat16), cache, i32(2, 4), i32(2, 5), i32(2, 4))
    with pytest.raises(RuntimeError, match="page_size"):
        op.LatentCache.empty(4, 48, "cpu")


@pytest.mark.gpu
def test_python_entries_name_what_is_wrong():
    dev = "cuda:0"
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    ok = dict(kv_len=i32(2), new_len=i32(2), block_table=i32(2, 4), free_pages=i32(8), free_count=i32(1), page_size=64, max_tokens=2, topk=5)
    op.cache_plan(**ok)
    for name, bad in [("kv_len", i32(2, 1)), ("kv_len", i32(0)), ("new_len", i32(3)), ("new_len", i32(2).long()), ("block_table", i32(3, 4)),
                      ("block_table", i32(4, 2).t()), ("free_pages", i32(0)), ("free_count", i32(2)), ("page_size", 65), ("max_tokens", -1), ("topk", -1)]:
        with pytest.raises(RuntimeError):
            op.cache_plan(**{**ok, name: bad})
    cache = op.LatentCache.empty(4, 64, dev)
    kv = torch.zeros(2, 576, dtype=torch.bfloat16, device=dev)
    op.cache_append(kv, cache, i32(2))
    wide = torch.zeros(2, 580, dtype=torch.bfloat16, device=dev)
    other = op.LatentCache(cache.values.view(torch.uint8), cache.scales)
    halves = op.LatentCache(cache.values[:, :32], cache.scales)
    for args in [(kv.float(), cache, i32(2)), (kv[:, :512], cache, i32(2)), (wide[:, :576], cache, i32(2)), (wide[:, 4:], cache, i32(2)), (kv, cache, i32(3)),
                 (kv, cache, i32(2).long()), (kv, other, i32(2)), (kv, halves, i32(2)), (kv, op.LatentCache(cache.values, cache.scales[:3]), i32(2)),
                 (kv, op.LatentCache(cache.values, cache.scales.double()), i32(2)), (kv, cache.values, i32(2))]:
        with pytest.raises(RuntimeError):
            op.cache_append(*args)
    q = torch.zeros(2, 16, 576, dtype=torch.bfloat16, device=dev)
    good = dict(q=q, cache=cache, block_table=i32(2, 4), indices=i32(2, 5), query_meta=i32(2, 4))
    op.mla_fwd_cached(**good)
    for name, bad in [("q", q.half()), ("q", q[:, :12].contiguous()), ("q", q[:, ::2]), ("q", q[0]), ("cache", other), ("cache", None), ("block_table", i32(2)), ("block_table", i32(0, 4)),
                      ("indices", i32(3, 5)), ("indices", i32(2, 0)), ("indices", i32(2, 5).long()), ("query_meta", i32(2, 3)), ("query_meta", i32(3, 4)),
                      ("query_meta", i32(9)[1:].view(2, 4)), ("block_table", i32(2, 1 << 25))]:
        with pytest.raises(RuntimeError):
            op.mla_fwd_cached(**{**good, name: bad})
    with pytest.raises(RuntimeError, match="small|workspace|status 3"):
        op.mla_fwd_cached(**good, workspace=op.Workspace(256, dev))
