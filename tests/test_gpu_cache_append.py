"""Rows into the paged cache against plain loops in 64 bits: stored numbers and scales are equal, for every order of slots."""
import numpy as np
import pytest
import torch

from oracle.latent_cache_ref import append_ref
from tests.cache_inputs import on, random_cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _kv(n, seed, grow=0.2):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, 576)) * np.where(rng.random((n, 1)) < grow, 9.0, 1.0)
    return torch.from_numpy(x).bfloat16()


def _check(kv, values, scales, slots):
    """kv on the host (bf16), the cache on the device; returns the cache after the call."""
    from test_operator_b200 import op
    want_v, want_s = append_ref(kv.double().numpy(), values.float().cpu().numpy(), scales.cpu().numpy(), slots)
    cache = op.LatentCache(values, scales)
    before = values.view(torch.uint8).clone()
    op.cache_append(kv.to(DEV), cache, on(DEV, np.asarray(slots, dtype=np.int32))[0])
    got = values.float().cpu().numpy()
    assert np.array_equal(scales.cpu().numpy(), want_s)
    assert np.array_equal(got, want_v, equal_nan=True)
    n_pages, page = values.shape[:2]
    named = np.zeros(n_pages, dtype=bool)
    for s in slots:
        if 0 <= s < n_pages * page:
            named[s // page] = True
    assert torch.equal(values.view(torch.uint8)[torch.from_numpy(~named)], before[torch.from_numpy(~named)])       # not a bit of the other pages
    return cache


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("n", [1, 3, 77])
def test_single_tokens(n, page):
    rng = np.random.default_rng(n * page)
    values, scales = random_cache(n + 5, page, DEV, seed=n)
    slots = rng.permutation(n + 5)[:n] * page + rng.integers(0, page, n)
    _check(_kv(n, n), values, scales, slots)


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("n", [2047, 8192, 8193, 9000, 20001])
def test_prompts(n, page):
    # runs of tokens that begin and end inside pages, some rows left out, the last ones behind the end
    rng = np.random.default_rng(n + page)
    n_pages = n // page + 60
    pages, slots = list(rng.permutation(n_pages)), []
    while len(slots) < n and len(pages) > 1:
        length = int(rng.integers(1, 5 * page))
        at = int(rng.integers(0, page))
        for _ in range(length):
            if at == page:
                if len(pages) <= 1:
                    break
                at = 0
                pages.pop()
            slots.append(pages[-1] * page + at)
            at += 1
        pages.pop()
        slots += [-1] * int(rng.integers(0, 3))
    slots = np.array((slots + [-1] * n)[:n])
    values, scales = random_cache(n_pages, page, DEV, seed=n)
    _check(_kv(n, page), values, scales, slots)


@pytest.mark.parametrize("n", [300, 3000, 9001, 20011])
def test_any_order_and_slots_named_twice(n):
    # pages come up again and again, slots twice and more often (the last row stays), numbers outside the cache are left out
    rng = np.random.default_rng(n)
    n_pages = max(4, n // 40)
    slots = rng.integers(-20, n_pages * 32 + 20, n)
    slots[::50] = 2 ** 31 - 1
    slots[7::50] = -(2 ** 31)
    values, scales = random_cache(n_pages, 32, DEV, seed=1)
    _check(_kv(n, 2), values, scales, slots)


@pytest.mark.parametrize("n", [500, 5000, 9000])
def test_every_row_to_one_slot(n):
    values, scales = random_cache(3, 64, DEV)
    _check(_kv(n, 3), values, scales, [64 + 5] * n)


def test_scale_grows_and_never_shrinks():
    values, scales = random_cache(2, 16, DEV)
    for k, mult in enumerate((1.0, 100.0, 1e-3, 3e4, 2.0 ** 90, 2.0 ** -120)):
        _check(_kv(1, k, grow=0) * mult, values, scales, [16 + 1 + k])
    assert scales[1].item() > 2.0 ** 80
    _check(_kv(1, 9, grow=0), values, scales, [16])          # row 0: the page starts anew
    assert scales[1].item() < 1


@pytest.mark.parametrize("kind", ["zeros", "tiny", "largest", "nonfinite", "all_nan", "at_448", "ties"])
def test_numbers_at_the_ends(kind):
    kv = _kv(4, 5)
    if kind == "zeros":
        kv.zero_()
        kv[1] = -0.0
    elif kind == "tiny":
        kv[:] = torch.ldexp(torch.ones(576), -torch.arange(576) % 40 - 94).bfloat16()
    elif kind == "largest":
        kv[0, 5], kv[3, 1] = torch.finfo(torch.bfloat16).max, -torch.finfo(torch.bfloat16).max
    elif kind == "nonfinite":
        kv[0, 3], kv[1, 570], kv[2, 0], kv[2, 575] = float("inf"), float("-inf"), float("nan"), 50.0
    elif kind == "all_nan":
        kv[:] = float("nan")
    elif kind == "at_448":
        kv[0, 0] = 448 * 2.0 ** -9
        kv[1:] *= 1e-3
    else:                   # halfway between two stored numbers
        kv[:] = (torch.arange(576) % 16 * 2 + 17).bfloat16()
        kv[0, 0] = 448
    for slots in ([0, 1, 2, 3], [5, 17, 6, 31]):
        values, scales = random_cache(2, 16, DEV, seed=3)
        _check(kv, values, scales, slots)


def test_nan_that_is_kept_stays_one():
    values, scales = random_cache(1, 16, DEV)
    values.view(torch.uint8)[0, 3, 7], values.view(torch.uint8)[0, 4, 8] = 0x7f, 0xff
    _check(_kv(1, 1, grow=1.0), values, scales, [9])
    assert values.float()[0, 3, 7].isnan() and values.float()[0, 4, 8].isnan()


def test_strided_rows_and_an_extra_dimension():
    from test_operator_b200 import op
    kv = _kv(9, 4)
    slots = np.array([3, 4, 5, 40, 41, 16, 17, 18, 0])
    want_v, want_s = append_ref(kv.double().numpy(), np.zeros((3, 16, 576)), np.zeros(3), slots)
    wide = torch.full((9, 1600), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 1024:] = kv.to(DEV)
    for rows in (wide[:, 1024:], wide[:, None, 1024:], kv.to(DEV)[:, None]):
        cache = op.LatentCache.empty(3, 16, DEV)
        op.cache_append(rows, cache, on(DEV, slots.astype(np.int32))[0])
        assert np.array_equal(cache.values.float().cpu().numpy(), want_v) and np.array_equal(cache.scales.cpu().numpy(), want_s)


def test_no_rows():
    from test_operator_b200 import op
    cache = op.LatentCache.empty(3, 16, DEV)
    op.cache_append(torch.zeros(0, 576, dtype=torch.bfloat16, device=DEV), cache, torch.zeros(0, dtype=torch.int32, device=DEV))


def test_pages_behind_two_to_the_32_bytes():
    from test_operator_b200 import op
    n_pages = 2 ** 32 // (64 * 576) + 100
    cache = op.LatentCache.empty(n_pages, 64, DEV)
    kv = _kv(70, 6)
    slots = np.concatenate([np.arange(64) + (n_pages - 1) * 64, (n_pages - 50) * 64 + np.arange(6)])
    op.cache_append(kv.to(DEV), cache, on(DEV, slots.astype(np.int32))[0])
    tail = cache.values[n_pages - 100:].float().cpu().numpy()
    want_v, want_s = append_ref(kv.double().numpy(), np.zeros((100, 64, 576)), np.zeros(100), slots - (n_pages - 100) * 64)
    assert np.array_equal(tail, want_v) and np.array_equal(cache.scales[n_pages - 100:].cpu().numpy(), want_s)
    assert not cache.values[:n_pages - 100].view(torch.uint8).any()


@pytest.mark.parametrize("n", [5000, 9000])
def test_replayed_in_a_graph(n):
    from test_operator_b200 import op
    kv, slots = _kv(n, 7).to(DEV), on(DEV, np.random.default_rng(1).permutation(12800)[:n].astype(np.int32))[0]
    cache = op.LatentCache.empty(200, 64, DEV)
    op.cache_append(kv, cache, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.cache_append(kv, cache, slots)
    kv.copy_(_kv(n, 8).to(DEV))
    again = op.LatentCache(cache.values.clone(), cache.scales.clone())
    graph.replay()
    op.cache_append(kv, again, slots)
    torch.cuda.synchronize()
    assert torch.equal(cache.values.view(torch.uint8), again.values.view(torch.uint8)) and torch.equal(cache.scales, again.scales)


@pytest.mark.parametrize("n", [64, 9000])
def test_calls_queued_one_behind_the_other(n):
    # nothing between the calls: a later one may come up under an earlier one's tail, on the same pages
    from test_operator_b200 import op
    page, calls = 16, 12
    pages = -(-n // 8)
    cache = op.LatentCache.empty(pages, page, DEV)
    want_v, want_s = np.zeros((pages, page, 576)), np.zeros(pages)
    kvs, slot_maps = [], []
    for k in range(calls):
        kvs.append(_kv(n, k, grow=0) * float(2.0 ** (k % 5)))
        slot_maps.append(np.array([(t // 8) * page + (t + k) % 8 + (8 if k % 2 else 0) for t in range(n)]))
    device = [(kv.to(DEV), on(DEV, s.astype(np.int32))[0]) for kv, s in zip(kvs, slot_maps)]
    torch.cuda.synchronize()
    for kv, slots in device:
        op.cache_append(kv, cache, slots)
    for kv, slots in zip(kvs, slot_maps):
        want_v, want_s = append_ref(kv.double().numpy(), want_v, want_s, slots)
    assert np.array_equal(cache.scales.cpu().numpy(), want_s) and np.array_equal(cache.values.float().cpu().numpy(), want_v)
