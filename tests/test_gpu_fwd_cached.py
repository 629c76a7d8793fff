"""Attention over the paged 8-bit cache against the definition in 64 bits; each element within the bounds that the oracle derives."""
import numpy as np
import pytest
import torch

from oracle.latent_cache_ref import attend_ref
from tests.cache_inputs import on, queries, random_cache, requests, share_of_bound

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAN = 0x7f


def _case(kv_len, new, h_q, topk, page, seed=0, pad=0, unused=0.1, spare=3):
    rng = np.random.default_rng(seed)
    table, n_pages = requests(kv_len, page, spare, rng)
    meta, idx = queries(kv_len, new, topk, rng, pad, unused)
    values, scales = random_cache(n_pages, page, DEV, seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(len(meta), h_q, 576, generator=gen, device=DEV, dtype=torch.bfloat16)
    table, idx, meta = on(DEV, table, idx, meta)
    # pages that are nobody's, and rows behind a request's last token, hold what they may: NaN here
    codes = values.view(torch.uint8)
    free = np.setdiff1d(np.arange(n_pages), table.cpu().numpy())
    codes[free] = NAN
    scales[torch.from_numpy(free).to(DEV)] = float("nan")
    for r, n in enumerate(kv_len):
        if n % page:
            codes[int(table[r, n // page]), n % page:] = NAN
    return q, values, scales, table, idx, meta


def _run(q, values, scales, table, idx, meta, **kwargs):
    from test_operator_b200 import op
    return op.mla_fwd_cached(q, op.LatentCache(values, scales), table, idx, meta, check_device_status=True, **kwargs)


def _compare(o, lse, ref):
    none = ref.lse.isposinf()
    assert int((lse.isposinf() != none).sum()) == 0 and int(o[none].count_nonzero()) == 0
    assert share_of_bound(o, ref.o, ref.o_bound) <= 1
    fine = ~none
    assert share_of_bound(lse[fine], ref.lse[fine], ref.lse_bound[fine]) <= 1
    # roundings are of either sign: together they come to less than one of them (half a step of bf16 and of P, each at most 2^-8 and 2^-9 on average)
    off = (o.double() - ref.o)[~ref.o.isnan()]
    assert off.norm() <= 2 ** -8 * ref.o[~ref.o.isnan()].norm()


@pytest.mark.parametrize("h_q", [8, 16, 64, 72, 128])
@pytest.mark.parametrize("topk", [1, 31, 256, 257, 700])
def test_single_tokens(h_q, topk):
    case = _case([1, 2, 17, 300, 1000, 64, 65], [1] * 7, h_q, topk, 64, seed=topk + h_q, pad=2)
    _compare(*_run(*case), attend_ref(*case))


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("kv_len, new, topk", [([5000], [1], 2048), ([3000, 2500], [2, 3], 2047), ([40, 700, 3], [40, 300, 3], 100), ([900], [900], 520)])
def test_prompts_and_steps(kv_len, new, topk, page):
    case = _case(kv_len, new, 128 if topk > 2000 else 64, topk, page, seed=page, pad=1)
    _compare(*_run(*case), attend_ref(*case))


@pytest.mark.parametrize("h_q", [16, 128])
def test_many_queries(h_q):
    # ranges of several queries per cluster, queries cut between two of them; every length of the last tile
    case = _case([600] * 40, [9] * 40, h_q, 600, 32, seed=2)
    case[5][:, 3] = torch.randint(0, 601, (360,), device=DEV)
    _compare(*_run(*case), attend_ref(*case))


@pytest.mark.parametrize("s_q", [3, 200])
def test_what_takes_no_part(s_q):
    q, values, scales, table, idx, meta = _case([500] * 3, [s_q // 3 + 1] * 3, 64, 300, 16, seed=5)
    n_pages = scales.numel()
    idx[0::5, ::3] = 2 ** 31 - 1
    idx[1::5, ::3] = -(2 ** 31)
    idx[2::5] = -1                                          # no slot at all
    idx[3::5, :] = idx[3::5, :1]                            # one position many times
    for k, bad in enumerate((-1, n_pages, 2 ** 31 - 1, -(2 ** 31))):
        table[k % 3, 2 + 5 * k] = bad                       # pages that are none
    meta[4::15, 0] = 3                                      # no such request
    meta[9::15, 0] = -1
    meta[14::15, 1] = 10 ** 9                               # more tokens than the table has pages for
    meta[14::15, 2] = 10 ** 9
    idx[14::15, 5::2] += 16 * table.shape[1]
    meta[5::15, 3] = 0
    meta[6::15, 3] = -4
    meta[7::15, 3] = 10 ** 6
    meta[8::15, 2] = -1                                     # before the request's first token
    case = (q, values, scales, table, idx, meta)
    ref = attend_ref(*case)
    assert ref.lse.isposinf().any() and ref.lse.isfinite().any()
    _compare(*_run(*case), ref)


def test_causal_rule_can_be_left_out():
    case = _case([400, 90], [60, 90], 16, 80, 16, seed=6)
    case[4].copy_(torch.randint(-5, 400, case[4].shape, device=DEV))
    for causal in (True, False):
        _compare(*_run(*case, causal=causal), attend_ref(*case, causal=causal))


def test_scale_and_units():
    case = _case([400], [5], 64, 200, 64, seed=7)
    ref = attend_ref(*case, sm_scale=0.11)
    o, lse = _run(*case, sm_scale=0.11)
    _compare(o, lse, ref)
    o_e, lse_e = _run(*case, sm_scale=0.11, lse_is_base2=False)
    assert torch.equal(o, o_e) and torch.allclose(lse_e, lse * np.log(2), rtol=2 ** -22, atol=0)


@pytest.mark.parametrize("kind", ["one_page_large", "one_page_small", "spread", "large", "tiny", "zero_pages"])
def test_scales_of_pages(kind):
    # a key weighs p times its page's scale in the output: pages whose scales are far apart
    q, values, scales, table, idx, meta = _case([900, 600], [4, 3], 128, 500, 16, seed=8)
    live = table[table >= 0].long()
    if kind == "one_page_large":
        scales[live[::7]] *= 2.0 ** 9
        values.view(torch.uint8)[live[::7]] = values.view(torch.uint8)[live[::7]] & 0x87 | 0x10      # their numbers small, but for the scale
    elif kind == "one_page_small":
        scales[live[::7]] *= 2.0 ** -14
    elif kind == "spread":
        scales[live] *= torch.ldexp(torch.ones(live.numel(), device=DEV), torch.randint(-6, 3, (live.numel(),), device=DEV))
    elif kind == "large":
        scales[live] *= 2.0 ** 70
        q *= 2.0 ** -60
        q *= 2.0 ** -10
    elif kind == "tiny":
        scales[live] = 2.0 ** -90
    else:
        scales[live[::3]] = 0
        values.view(torch.uint8)[live[::3]] = 0
    case = (q, values, scales, table, idx, meta)
    _compare(*_run(*case), attend_ref(*case))


def test_a_scale_counts_by_its_exponent():
    q, values, scales, table, idx, meta = _case([300], [3], 64, 100, 32, seed=9)
    plain = _run(q, values, scales, table, idx, meta)
    uneven = _run(q, values, scales * (1 + torch.rand_like(scales) * 0.99), table, idx, meta)
    assert all(torch.equal(a, b) for a, b in zip(plain, uneven))


@pytest.mark.parametrize("kind", ["outlier", "large", "tiny", "zero", "sharp"])
def test_queries(kind):
    q, values, scales, table, idx, meta = _case([900, 20], [4, 3], 128, 400, 64, seed=10)
    if kind == "outlier":
        q[:, :, 17] *= 60
    elif kind == "large":
        q *= 2.0 ** 100
        scales *= 2.0 ** -95
    elif kind == "tiny":
        q *= 2.0 ** -120
    elif kind == "zero":
        q[:, ::2] = 0
    else:
        q *= 16
    case = (q, values, scales, table, idx, meta)
    _compare(*_run(*case), attend_ref(*case))


@pytest.mark.parametrize("s_q", [1, 90])
@pytest.mark.parametrize("kind", ["kv_nan", "q_nan", "q_inf"])
def test_what_is_not_a_number_stays_none(kind, s_q):
    q, values, scales, table, idx, meta = _case([2000], [s_q], 64, 1500, 64, seed=11, unused=0.0)
    hit = torch.zeros(s_q, 64, dtype=torch.bool, device=DEV)
    if kind == "kv_nan":
        values.view(torch.uint8)[int(table[0, 3]), 7, 100] = 0xff
        hit |= (idx == 3 * 64 + 7).any(1)[:, None]
    else:
        q[0, 5, 575] = float("nan") if kind == "q_nan" else float("-inf")
        hit[0, 5] = True
    ref = attend_ref(q, values, scales, table, idx, meta)
    o, lse = _run(q, values, scales, table, idx, meta)
    assert torch.equal(o.isnan().any(2), hit) and torch.equal(o.isnan().all(2), hit if kind != "kv_nan" else o.isnan().all(2)) and torch.equal(lse.isnan(), hit)
    fine = ~hit
    assert share_of_bound(o[fine], ref.o[fine], ref.o_bound[fine]) <= 1


def test_same_bits_every_time_and_on_every_stream():
    case = _case([3000] * 6, [20] * 6, 128, 1000, 64, seed=12)
    want = _run(*case)
    from test_operator_b200 import op
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for k in range(6):
        with torch.cuda.stream(streams[k % 2]):
            got.append(op.mla_fwd_cached(case[0], op.LatentCache(case[1], case[2]), *case[3:]))
    torch.cuda.synchronize()
    for o, lse in got:
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


def test_smaller_workspaces_and_an_unaligned_output():
    from test_operator_b200 import op
    case = _case([3000, 100], [3, 70], 64, 1000, 64, seed=13)
    ref = attend_ref(*case)
    for budget in (1, 1 << 20, 3 << 20):
        _compare(*_run(*case, workspace_budget=budget), ref)
    need = op._fwd_cached_workspace_bytes(73, 64, 1000, case[2].numel(), 64, 2, case[3].shape[1], 0)
    _compare(*_run(*case, workspace=op.Workspace(need, DEV)), ref)
    # indices that start anywhere, of one more dimension
    one = torch.empty(case[4].numel() + 1, dtype=torch.int32, device=DEV)[1:].view(73, 1, 1000)
    one.copy_(case[4][:, None])
    _compare(*_run(*case[:4], one, case[5]), ref)


def test_no_queries():
    case = _case([30], [2], 16, 10, 16)
    o, lse = _run(case[0][:0], *case[1:4], case[4][:0], case[5][:0])
    assert o.shape == (0, 16, 512) and lse.shape == (0, 16)


def test_cache_of_more_than_two_to_the_32_bytes():
    page, n = 128, 2 ** 32 // 576 + 100000
    table, n_pages = requests([n], page, 1, np.random.default_rng(0))
    values, scales = random_cache(n_pages, page, DEV, seed=14)
    rng = np.random.default_rng(1)
    meta, idx = queries([n], [5], 500, rng)
    q = torch.randn(5, 64, 576, device=DEV, dtype=torch.bfloat16)
    case = (q, values, scales, *on(DEV, table, idx, meta))
    _compare(*_run(*case), attend_ref(*case))


def test_replayed_in_a_graph_beside_another():
    from test_operator_b200 import op
    cases = [_case([2000] * 3, [n] * 3, 64, 900, 64, seed=15 + n) for n in (1, 30)]
    graphs, outs = [], []
    for case in cases:
        call = lambda: op.mla_fwd_cached(case[0], op.LatentCache(case[1], case[2]), *case[3:])  # noqa: B023,E731
        call()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call())
    for case in cases:
        case[0].normal_()
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for case, (o, lse) in zip(cases, outs):
        _compare(o, lse, attend_ref(*case))


@pytest.mark.parametrize("s_q", [2, 150])
def test_padding_queries_may_hold_anything(s_q):
    case = _case([700], [s_q], 64, 600, 32, seed=16, pad=40)
    plain = _run(*case)
    case[0][s_q:] = float("nan")
    case[0][s_q + 1::3] = float("inf")
    o, lse = _run(*case)
    assert torch.equal(o, plain[0]) and torch.equal(lse, plain[1])
    assert int(o[s_q:].count_nonzero()) == 0 and bool(lse[s_q:].isposinf().all())
