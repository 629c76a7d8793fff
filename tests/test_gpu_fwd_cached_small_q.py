"""Attention over the paged 8-bit cache: columns of q that are far smaller than the row's largest, where the largest meets zeros in the cache."""
import math

import pytest
import torch

from oracle.latent_cache_ref import attend_ref
from tests.cache_inputs import on, queries, random_cache, requests, share_of_bound

import numpy as np

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _case(bits, largest, n=600, s_q=5, h_q=64, topk=300, page=32):
    """Column 3 of q is `largest` alone, `bits` above the others (one to two times a power of two, all eight bits of them), and 0 in the cache."""
    rng = np.random.default_rng(bits)
    table, n_pages = requests([n], page, 1, rng)
    meta, idx = queries([n], [s_q], topk, rng)
    values, scales = random_cache(n_pages, page, DEV, bits)
    values.view(torch.uint8)[:, :, 3] = 0
    gen = torch.Generator(device=DEV).manual_seed(bits)
    q = (1 + torch.randint(0, 128, (s_q, h_q, 576), generator=gen, device=DEV) / 128) * (1 - 2 * torch.randint(0, 2, (s_q, h_q, 576), generator=gen, device=DEV))
    q[:, :, 3] = largest * 2.0 ** bits
    return q.bfloat16(), values, scales, *on(DEV, table, idx, meta)


@pytest.mark.parametrize("bits", [4, 9, 11, 13])
@pytest.mark.parametrize("largest", [1.0, 1.7578125, 1.9921875])
def test_columns_below_the_largest_are_exact(bits, largest):
    # q in two parts is q: what is left are the fp32 sums (2^-18 of the products' magnitudes), ex2 and logarithm
    from test_operator_b200 import op
    q, values, scales, table, idx, meta = _case(bits, largest)
    ref = attend_ref(q, values, scales, table, idx, meta)
    o, lse = op.mla_fwd_cached(q, op.LatentCache(values, scales), table, idx, meta, check_device_status=True)
    k = (values.double() * scales.double()[:, None, None])[table[0].long()].flatten(0, 1)
    products = (q.double().abs() @ k.abs().T).amax(2) / 24
    logits = (q.double() @ k.T).abs().amax(2) / 24
    bound = 2 * (2 ** -18 * products + 2 ** -20 + logits * 2 ** -22 + 2 ** -20) + ref.lse.abs() * 2 ** -22
    assert share_of_bound(lse, ref.lse, bound / math.log(2)) <= 1
    assert share_of_bound(o, ref.o, ref.o_bound) <= 1


@pytest.mark.parametrize("bits", [16, 20])
def test_smaller_ones_are_within_2_to_the_minus_21(bits):
    from test_operator_b200 import op
    q, values, scales, table, idx, meta = _case(bits, 1.0)
    q[:, :, 4:] *= 2.0 ** 6                    # (so that the logits are not all about 0)
    q[:, :, 3] *= 2.0 ** 6
    ref = attend_ref(q, values, scales, table, idx, meta)
    o, lse = op.mla_fwd_cached(q, op.LatentCache(values, scales), table, idx, meta, check_device_status=True)
    k = (values.double() * scales.double()[:, None, None])[table[0].long()].flatten(0, 1)
    products = (q.double().abs() @ k.abs().T).amax(2) / 24
    cut = q.double().abs().amax(2) * 2 ** -21 * k.abs().sum(1).amax() / 24
    logits = (q.double() @ k.T).abs().amax(2) / 24
    bound = 2 * (2 ** -18 * products + cut + logits * 2 ** -22 + 2 ** -20) + ref.lse.abs() * 2 ** -22
    assert share_of_bound(lse, ref.lse, bound / math.log(2)) <= 1
