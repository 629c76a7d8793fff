"""Inputs of the cache tests: a random cache, block tables of requests whose pages lie anywhere, ragged queries."""
import numpy as np
import torch

D_QK = 576


def random_cache(n_pages, page, device, seed=0, exps=(-7, -4)):
    gen = torch.Generator(device=device).manual_seed(seed)
    codes = (torch.randn(n_pages, page, D_QK, generator=gen, device=device, dtype=torch.bfloat16) * 64).clamp_(-448, 448)
    e = torch.randint(exps[0], exps[1], (n_pages,), generator=gen, device=device)
    return codes.to(torch.float8_e4m3fn), torch.ldexp(torch.ones(n_pages, device=device), e)


def requests(kv_len, page, spare, rng):
    """Block table (int32) for requests of these lengths, entries behind their pages -1; number of pages of the cache."""
    pages = [-(-int(n) // page) for n in kv_len]
    n_pages = sum(pages) + spare
    order = rng.permutation(n_pages)
    table = np.full((len(pages), max(1, max(pages))), -1, dtype=np.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    return table, n_pages


def queries(kv_len, new, topk, rng, pad=0, unused=0.1):
    """query_meta and indices [sum(new) + pad, topk] of requests whose last `new` tokens are the queries; some slots -1."""
    rows = [(r, int(k), int(k) - int(n) + j, topk) for r, (k, n) in enumerate(zip(kv_len, new)) for j in range(int(n))]
    meta = np.array(rows + [(0, 0, 0, 0)] * pad, dtype=np.int32).reshape(-1, 4)
    idx = (rng.random((len(meta), topk)) * (meta[:, 2:3] + 1)).astype(np.int32)
    idx[rng.random(idx.shape) < unused] = -1
    return meta, idx


def on(device, *arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).to(device) for a in arrays]


def share_of_bound(got, want, bound):
    """The largest difference as a share of what it may be; above 1 where only one of the two is a NaN."""
    if not got.numel():
        return 0.0
    share = torch.where((got.double() == want) | (got.isnan() & want.isnan()), 0.0, (got.double() - want).abs() / bound)
    return float(share.nan_to_num(nan=1e9, posinf=1e9).max())
