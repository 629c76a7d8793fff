"""The oracle of the paged 8-bit cache against torch's own conversions and by its invariants."""
import numpy as np
import pytest
import torch

from oracle.latent_cache_ref import append_ref, attend_ref, plan_ref, round_e4m3, scale_ref
from tests.cache_inputs import on, queries, random_cache, requests


def test_rounding_is_the_formats():
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    x = x[x.isfinite() & (x.abs() <= 448)]
    assert np.array_equal(round_e4m3(x.numpy()), x.to(torch.float8_e4m3fn).double().numpy())
    assert np.isnan(round_e4m3([np.inf, -np.inf, np.nan])).all()


@pytest.mark.parametrize("amax, scale", [(0.0, 2.0 ** -100), (448.0, 1.0), (449.0, 2.0), (224.0, 0.5), (225.0, 1.0), (2.0 ** -130, 2.0 ** -100), (3e38, 2.0 ** 120)])
def test_scale_is_the_smallest_that_holds(amax, scale):
    assert scale_ref(amax) == scale


def test_rescaling_loses_nothing_but_small_numbers():
    # rows that are stored and then brought over to a larger scale are what they would be had the scale been larger from the start, but for subnormals
    rng = np.random.default_rng(0)
    x = torch.from_numpy(rng.standard_normal((4, 576))).bfloat16().double().numpy()
    big = x[3] * 64
    v, s = append_ref(x[:3], np.zeros((1, 16, 576)), np.zeros(1), [0, 1, 2])
    v, s = append_ref(big[None], v, s, [3])
    w, t = append_ref(np.concatenate([x[:3], big[None]]), np.zeros((1, 16, 576)), np.zeros(1), [0, 1, 2, 3])
    assert s[0] == t[0]
    normal = np.abs(w) >= 2.0 ** -6
    assert normal.any() and np.array_equal(v[normal], w[normal]) and np.abs(v - w).max() <= 2.0 ** -9


@pytest.mark.parametrize("seed", range(8))
def test_plan_keeps_pages_apart(seed):
    rng = np.random.default_rng(seed)
    page, n = 16, 9
    kv_len = rng.integers(0, 70, n)
    table, n_pages = requests(kv_len, page, 12, rng)
    table = np.concatenate([table, np.full((n, 4), -1, dtype=np.int32)], 1)
    free = np.setdiff1d(np.arange(n_pages), table)
    stack = np.zeros(n_pages, dtype=np.int32)
    stack[:len(free)] = free
    new = rng.integers(-1, 30, n)
    p = plan_ref(kv_len, new, table, stack, len(free), page, int(np.maximum(new, 0).sum()) - 3, 7)
    live = [p.block_table[i, k] for i in range(n) for k in range(-(-int(p.kv_len[i]) // page))]
    assert sorted(live + list(p.free_pages[:p.free_count])) == list(range(n_pages))         # every page is somebody's, once
    used = p.slots[p.slots >= 0]
    assert len(set(used)) == len(used) == p.admitted.sum()
    assert ((p.slots >= 0) == p.query_meta.any(1)).all()


def test_attention_is_a_softmax_over_the_stored_rows():
    rng = np.random.default_rng(3)
    kv_len, new = [40, 5, 23], [1, 2, 3]
    table, n_pages = requests(kv_len, 16, 2, rng)
    meta, idx = queries(kv_len, new, 20, rng, pad=2)
    values, scales = random_cache(n_pages, 16, "cpu")
    q = torch.from_numpy(rng.standard_normal((len(meta), 8, 576))).bfloat16()
    got = attend_ref(q, values, scales, *on("cpu", table, idx, meta))
    rows = values.double() * scales.double()[:, None, None]
    for i, (r, tokens, pos, use) in enumerate(meta):
        chosen = [int(j) for j in idx[i, :use] if 0 <= j < tokens and j <= pos]
        if not chosen:
            assert got.lse[i].isposinf().all() and not got.o[i].any()
            continue
        k = torch.stack([rows[table[r, j // 16], j % 16] for j in chosen])
        x = q[i].double() @ k.T / 24
        assert torch.allclose(got.o[i], torch.softmax(x, 1) @ k[:, :512]) and torch.allclose(got.lse[i], torch.log2(torch.exp(x).sum(1)))
