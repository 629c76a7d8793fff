"""Attention over the paged 8-bit cache: one NaN in a key makes the whole row NaN wherever the key counts, and nothing else."""
import numpy as np
import pytest
import torch

from oracle.latent_cache_ref import attend_ref
from tests.cache_inputs import on, queries, random_cache, requests, share_of_bound

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("s_q", [1, 5, 90, 300])
@pytest.mark.parametrize("column", [0, 300, 511, 512, 575])
def test_all_columns_of_a_row(s_q, column):
    # one query over several clusters, queries cut between two of them, whole ones
    rng = np.random.default_rng(s_q)
    table, n_pages = requests([3000], 64, 1, rng)
    meta, idx = queries([3000], [s_q], 1500, rng, unused=0.0)
    values, scales = random_cache(n_pages, 64, DEV, 2)
    values.view(torch.uint8)[int(table[0, 3]), 7, column] = 0x7f if column % 2 else 0xff
    idx[::2][idx[::2] == 3 * 64 + 7] = 5
    q = torch.randn(s_q, 64, 576, generator=torch.Generator(device=DEV).manual_seed(s_q), device=DEV, dtype=torch.bfloat16)
    case = (q, values, scales, *on(DEV, table, idx, meta))
    from test_operator_b200 import op
    hit = (case[4] == 3 * 64 + 7).any(1)
    assert s_q < 90 or bool(hit.any()) and not bool(hit.all())
    o, lse = op.mla_fwd_cached(q, op.LatentCache(values, scales), *case[3:], check_device_status=True)
    assert torch.equal(o.isnan(), hit[:, None, None].expand_as(o)) and torch.equal(lse.isnan(), hit[:, None].expand_as(lse))
    ref = attend_ref(*case)
    assert share_of_bound(o[~hit], ref.o[~hit], ref.o_bound[~hit]) <= 1
