"""Attention over the paged 8-bit cache: the largest scales that rows are stored with, and pages whose scales lie as far apart as is allowed."""
import numpy as np
import pytest
import torch

from oracle.latent_cache_ref import attend_ref
from tests.cache_inputs import on, queries, random_cache, requests, share_of_bound

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _check(case):
    from test_operator_b200 import op
    ref = attend_ref(*case)
    o, lse = op.mla_fwd_cached(case[0], op.LatentCache(case[1], case[2]), *case[3:], check_device_status=True)
    assert bool(ref.lse.isfinite().all()) and bool(lse.isfinite().all()) and bool(o.isfinite().all())
    assert share_of_bound(o, ref.o, ref.o_bound) <= 1 and share_of_bound(lse, ref.lse, ref.lse_bound) <= 1
    return o, lse, ref


@pytest.mark.parametrize("s_q", [1, 60])
@pytest.mark.parametrize("exps", [(120, 121), (105, 121)])
def test_largest_scales(s_q, exps):
    # kv up to the largest bf16 numbers; q so small that the logits are ordinary
    rng = np.random.default_rng(0)
    table, n_pages = requests([900], 32, 1, rng)
    meta, idx = queries([900], [s_q], 500, rng)
    values, scales = random_cache(n_pages, 32, DEV, 1, exps=exps)
    values = values.float().clamp(-128, 128).to(torch.float8_e4m3fn)
    q = torch.randn(s_q, 64, 576, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0)) * 2.0 ** -126
    q[:, ::2] *= 2.0 ** 4
    _, lse, ref = _check((q.bfloat16(), values, scales, *on(DEV, table, idx, meta)))
    assert float(lse.std(dim=1).min()) > 0.01           # (not all logits are nothing)


@pytest.mark.parametrize("large", [4, 64, 120])
@pytest.mark.parametrize("first", ["small", "large", "mixed"])
@pytest.mark.parametrize("s_q", [1, 40, 200])
def test_scales_far_apart(large, first, s_q):
    # half of the keys in pages of scale 2^large, half in pages of 2^104 less; logits of about the same size, so that all keys weigh something
    page, n = 16, 1600
    rng = np.random.default_rng(3)
    table, n_pages = requests([n], page, 1, rng)
    table_d = torch.from_numpy(table).to(DEV)
    values, scales = random_cache(n_pages, page, DEV, 2)
    values = values.float().clamp(-112, 112).to(torch.float8_e4m3fn)
    scales[table_d[0].long()[0::2]] = 2.0 ** large
    small = table_d[0].long()[1::2]
    scales[small] = 2.0 ** (large - 104)
    if large == 4:
        values.view(torch.uint8)[small] = 0             # pages of zeros, as they are stored: 2^-100
    order = np.arange(n)
    is_large = (order // page) % 2 == 0
    order = {"small": np.concatenate([order[~is_large], order[is_large]]), "large": np.concatenate([order[is_large], order[~is_large]]),
             "mixed": rng.permutation(n)}[first]
    idx = np.repeat(order[None], s_q, 0).astype(np.int32)
    meta = np.array([[0, n, n - 1, n]] * s_q, dtype=np.int32)
    q = torch.randn(s_q, 64, 576, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0)) * 2.0 ** (-5 - large)
    o, lse, ref = _check((q.bfloat16(), values, scales, table_d, *on(DEV, idx, meta)))
    assert float((lse - np.log2(n)).abs().max()) < 6
