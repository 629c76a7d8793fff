"""Attention over the paged 8-bit cache where one key outweighs the rest: the tail of such a row counts, key by key."""
import math

import numpy as np
import pytest
import torch

from oracle.latent_cache_ref import attend_ref
from tests.cache_inputs import on, share_of_bound

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 2.0 ** -6
BIT = 24 * math.log(2)          # q * c that is one bit of a logit


def _sink(n, v_sink, mean, spread, slots_of_sink, h_q=128, gaps=(12, 20), page=64, seed=0, sink_scale=1.0):
    """One request of n tokens, whose token 0 outweighs each of the others by `gaps` bits (over the heads).  Its V is v_sink of theirs, theirs have
    a common mean; their logits are alike, or vary by `spread` bits.  Query i names the sink in slot slots_of_sink[i]."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n_pages = -(-n // page) + 1                     # page 0 holds the sink alone
    v = torch.randn(n, 576, generator=gen, device=DEV) + mean
    v[0] *= v_sink / sink_scale
    v[:, 512:] = 0
    v[0, 512] = 7 / sink_scale
    v[1:, 513] = torch.randn(n - 1, generator=gen, device=DEV)
    rows = torch.zeros(n_pages * page, 576, device=DEV)
    rows[0], rows[page:page + n - 1] = v[0], v[1:]
    values = (rows / SCALE).clamp(-448, 448).to(torch.float8_e4m3fn).view(n_pages, page, 576)
    scales = torch.full((n_pages,), SCALE, device=DEV)
    scales[0] *= sink_scale
    # positions: the sink is position 0, the others begin with the second page
    table, meta = on(DEV, np.arange(n_pages, dtype=np.int32)[None], np.array([[0, n_pages * page, n_pages * page - 1, n]] * len(slots_of_sink), dtype=np.int32))
    idx = torch.stack([torch.randperm(n - 1, generator=gen, device=DEV) for _ in slots_of_sink]) + page
    idx = torch.stack([torch.cat([i[:at], i.new_zeros(1), i[at:]]) for i, at in zip(idx, slots_of_sink)]).to(torch.int32)
    q = torch.zeros(len(slots_of_sink), h_q, 576, device=DEV)
    q[:, :, 512] = torch.linspace(*gaps, h_q, device=DEV) * BIT / 7
    q[:, :, 513] = spread * BIT
    return q.bfloat16(), values, scales, table, idx, meta


def _bound(q, values, scales, table, idx, meta, ref):
    """What roundings may amount to.  As in attend_ref, but for P, the heaviest of which is 2^11 to 2^12: half a step of eight significant bits, 2^-8, from
    2^-6 on (2^-17 of the heaviest), and 2^-25 of the heaviest below: there P is a whole number of 2^-9 and three bits of what that leaves, at most
    2^-10, whose half step is 2^-14."""
    n_pages, page = values.shape[:2]
    k = (values.view(torch.uint8).view(-1, 576).view(torch.float8_e4m3fn).double(), scales.double())
    bound = torch.zeros_like(ref.o)
    for i in range(len(q)):
        pos = idx[i].long()
        pages = table[0].long()[pos // page]
        code, s = k[0][pages * page + pos % page], k[1][pages][:, None]
        logits = q[i].double() @ (code * s).T / 24
        p = torch.softmax(logits, 1)
        off = 2 ** -18 * (q[i].double().abs() @ (code * s).abs().T).amax(1, keepdim=True) / 24 + 2 ** -19 + logits.abs().amax(1, keepdim=True) * 2 ** -22
        heavy = (p * s[:, 0]).amax(1, keepdim=True)
        bound[i] = (2 ** -8 + 2 * off) * (p @ (code * s)[:, :512].abs()) + 2 ** -25 * heavy * code[:, :512].abs().sum(0) + 2 ** -8 * ref.o[i].abs()
    return bound


def _run(*case):
    from test_operator_b200 import op
    return op.mla_fwd_cached(case[0], op.LatentCache(case[1], case[2]), *case[3:], check_device_status=True)


def _worst(case):
    """Largest difference as a share of the bound; relative error of o by head (norms over queries and columns)."""
    ref = attend_ref(*case)
    o, lse = _run(*case)
    assert share_of_bound(lse, ref.lse, ref.lse_bound) <= 1
    off = (o.double() - ref.o).transpose(0, 1).flatten(1)
    return share_of_bound(o, ref.o, _bound(*case, ref)), off.norm(dim=1) / ref.o.transpose(0, 1).flatten(1).norm(dim=1)


@pytest.mark.parametrize("n", [256, 700, 2048])
@pytest.mark.parametrize("v_sink", [1.0, 0.05])
@pytest.mark.parametrize("spread", [0.0, 2.0])
def test_tail_under_a_sink(n, v_sink, spread):
    # the sink in every tile, and at its first and last slot; P and the output each a half step of bf16 off at most
    at = [k for k in range(0, n, 256)] + [n - 1]
    share, relative = _worst(_sink(n, v_sink, 0.5, spread, at))
    assert share <= 1 and float(relative.max()) <= 2 ** -7


@pytest.mark.parametrize("h_q", [16, 64, 128])
@pytest.mark.parametrize("spread", [0.0, 2.0])
def test_tail_alone_in_the_output(h_q, spread):
    # nothing of the sink in o: what is left is the tail, each of its P within a half step of bf16 up to 17 bits below
    share, relative = _worst(_sink(2048, 0.0, 0.5, spread, [0, 1000, 2047], h_q=h_q, gaps=(12, 16.9)))
    assert share <= 1 and float(relative.max()) <= 2 ** -7


def test_sink_in_a_page_of_a_larger_scale():
    # what is rounded is p s: a sink whose page has 2^4 of the others' scale stands that much higher
    share, relative = _worst(_sink(2048, 0.05, 0.5, 0.0, [0, 1500], gaps=(8, 16.9), sink_scale=16.0))
    assert share <= 1 and float(relative.max()) <= 2 ** -7


def test_many_queries():
    share, relative = _worst(_sink(1000, 0.05, 0.5, 1.0, [(37 * k) % 1000 for k in range(250)], h_q=64))
    assert share <= 1 and float(relative.max()) <= 2 ** -7
