"""Attention over the paged 8-bit cache with logits so large that fp32 holds them in steps of more than a bit: one key takes all."""
import math

import pytest
import torch

from tests.cache_inputs import on

import numpy as np

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("exponent", [10, 20, 24, 25, 26, 27, 28, 29, 30, 40, 60, 100])
@pytest.mark.parametrize("order", ["up", "down", "any"])
@pytest.mark.parametrize("s_q", [1, 100])
def test_the_largest_takes_all(exponent, order, s_q):
    # logit of key j: (1 + j % 7 / 8) 2^exponent bits and one key of 15 / 8; apart by 2^(exponent - 3) bits at least: weights of the others are 0
    from test_operator_b200 import op
    page, n, h_q = 16, 800, 16
    gen = torch.Generator(device=DEV).manual_seed(exponent)
    rows = torch.randn(n, 576, generator=gen, device=DEV)
    rows[:, 512:] = 0
    rows[:, 512] = (1 + torch.arange(n, device=DEV) % 7 / 8)
    rows[417, 512] = 15 / 8
    values = (rows * 64).to(torch.float8_e4m3fn).view(n // page, page, 576)
    scales = torch.full((n // page,), 2.0 ** -6, device=DEV)
    q = torch.zeros(s_q, h_q, 576, device=DEV, dtype=torch.bfloat16)
    q[:, :, 512] = 1
    rank = torch.argsort(rows[:, 512], stable=True)
    idx = {"up": rank, "down": rank.flip(0), "any": torch.randperm(n, generator=gen, device=DEV)}[order].int()[None].expand(s_q, n).contiguous()
    table, meta = on(DEV, np.arange(n // page, dtype=np.int32)[None], np.array([[0, n, n - 1, n]] * s_q, dtype=np.int32))
    sm_scale = 2.0 ** exponent * math.log(2)
    o, lse = op.mla_fwd_cached(q, op.LatentCache(values, scales), table, idx, meta, sm_scale=sm_scale, check_device_status=True)
    want = (values.float() * 2.0 ** -6).view(n, 576)[417, :512].bfloat16()
    # (a number of the format is one of bf16, and the key's weight is 1 whatever P is)
    assert torch.equal(o, want.expand_as(o))
    # the scale in log2 units, its product with the logit and the sum: a few halves of 2^-23
    assert float((lse.double() / (15 / 8 * 2.0 ** exponent) - 1).abs().max()) <= 2 ** -21
