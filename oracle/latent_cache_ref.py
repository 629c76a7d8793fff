"""CPU restatement of the paged 8-bit cache: tables of a step, rows into the cache, attention over it.  TEST INFRASTRUCTURE ONLY: imported by
tests/, never by the product path.

The reference project has no such operators (parity unpinned: there are no reference outputs); the definitions are the ones that
include/smla_bwd.h gives, in plain loops and 64 bits.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import numpy as np
import torch

D_QK, D_V = 576, 512
MIN_EXP = -100


class Plan(NamedTuple):
    slots: np.ndarray
    query_meta: np.ndarray
    kv_len: np.ndarray
    free_count: int
    admitted: np.ndarray
    block_table: np.ndarray
    free_pages: np.ndarray


def plan_ref(kv_len, new_len, block_table, free_pages, free_count, page_size, max_tokens, topk, rejected=None) -> Plan:
    table, free = np.array(block_table), np.array(free_pages)
    kv_len, new_len = [int(v) for v in kv_len], [int(v) for v in new_len]
    stack = [int(v) for v in free[:free_count]]
    n = len(kv_len)
    room = table.shape[1] * page_size
    pages = lambda tokens: -(-tokens // page_size)  # noqa: E731
    keep = [k - min(max(int(r), 0), max(k, 0)) for k, r in zip(kv_len, [0] * n if rejected is None else rejected)]
    row_end = np.cumsum([max(m, 0) for m in new_len])
    fits = lambda i: new_len[i] >= 0 and 0 <= kv_len[i] <= room and keep[i] + new_len[i] <= room and row_end[i] <= max_tokens  # noqa: E731
    for i in range(n):
        if new_len[i] < 0 or fits(i):          # all pages of a request that ends, those behind the last token of one that goes on
            for k in range(0 if new_len[i] < 0 else pages(keep[i] + new_len[i]), pages(min(max(kv_len[i], 0), room))):
                stack.append(int(table[i, k]))
                if len(stack) <= len(free):
                    free[len(stack) - 1] = table[i, k]
    slots = np.full(max_tokens, -1)
    meta = np.zeros((max_tokens, 4), dtype=np.int64)
    after, admitted = list(kv_len), [0] * n
    first, short = 0, False
    for i in range(n):
        if new_len[i] < 0:
            after[i] = 0
            continue
        row0, first = first, first + new_len[i]
        if not fits(i):
            continue
        have, want = pages(kv_len[i]), pages(keep[i] + new_len[i])
        if want > have and (short or want - have > len(stack)):
            short = True
            continue
        for k in range(have, want):
            table[i, k] = stack.pop()
        after[i], admitted[i] = keep[i] + new_len[i], new_len[i]
        for j in range(new_len[i]):
            pos = keep[i] + j
            slots[row0 + j] = table[i, pos // page_size] * page_size + pos % page_size
            meta[row0 + j] = (i, after[i], pos, topk)
    return Plan(slots, meta, np.array(after), min(len(stack), len(free)), np.array(admitted), table, free)


def round_e4m3(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 number, ties to even, for |x| <= 448: four significant bits, steps of 2^-9 below 2^-6.  NaN for what is not finite."""
    x = np.asarray(x, dtype=np.float64)
    fine = np.isfinite(x)
    _, e = np.frexp(np.where(fine, x, 0.0))
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.where(fine, np.rint(np.where(fine, x, 0.0) / step) * step, np.nan)


def scale_ref(amax: float) -> float:
    e = MIN_EXP
    while 448.0 * 2.0 ** e < amax:
        e += 1
    return 2.0 ** e


def append_ref(kv, values, scales, slots):
    """kv [n, 576], values [n_pages, page, 576], scales [n_pages] in numpy floats -> (values, scales)."""
    values, scales = np.array(values, dtype=np.float64), np.array(scales, dtype=np.float64)
    n_pages, page = values.shape[:2]
    pages = {}
    for t, slot in enumerate(slots):
        if 0 <= slot < n_pages * page:
            pages.setdefault(int(slot) // page, {})[int(slot) % page] = t          # (the last one stays)
    for p, rows in pages.items():
        x = np.stack([np.asarray(kv[t], dtype=np.float64) for t in rows.values()])
        wanted = scale_ref(np.abs(x[np.isfinite(x)]).max(initial=0.0))
        if 0 not in rows:
            wanted = max(wanted, scales[p])
            if wanted > scales[p]:
                values[p] = round_e4m3(values[p] * (scales[p] / wanted))
        values[p, list(rows)] = round_e4m3(x / wanted)
        scales[p] = wanted
    return values, scales


class Attention(NamedTuple):
    o: torch.Tensor         # [s_q, h_q, 512] fp64
    lse: torch.Tensor       # [s_q, h_q] base 2
    o_bound: torch.Tensor   # how far rounding may take o and lse
    lse_bound: torch.Tensor


def attend_ref(q, values, scales, block_table, indices, query_meta, sm_scale=None, causal=True) -> Attention:
    """In 64 bits, query by query, on q's device, with bounds on what the roundings of the product path can amount to:

    logits   fp32 sums of 576 products (2 x 576 with q in two parts): 2^-18 of the sum of magnitudes covers their alignment to the largest
             one in every step (probed: 2.5e-6 where one product dominates); q within 2^-9 where its row's largest magnitude is 224 to 448 (more than the product path takes, 2^-14).
    P        half a step of eight significant bits, 2^-8, and 2^-16 of the largest P of the row (more than the product path takes, 2^-25: the tests of
             rows with one heavy key have a bound of their own).
    o        half a step of bf16, 2^-8.   ex2, the division and the sums in fp32: a few 2^-22.
    log2 s   is added to the logits and taken out again by way of the sum's logarithm: numbers of size |log2 s|, each of three roundings half of
             2^-23 of it (the logit, the logarithm and its own error), 2^-22 together.
    """
    sm_scale = 1 / math.sqrt(D_QK) if sm_scale is None else sm_scale
    n_pages, page = values.shape[:2]
    store = values.view(torch.uint8).reshape(-1, D_QK)
    s_q, h_q, _ = q.shape
    new = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device=q.device)  # noqa: E731
    out = Attention(new(s_q, h_q, D_V), new(s_q, h_q) + math.inf, new(s_q, h_q, D_V), new(s_q, h_q))
    for i, (r, tokens, pos, use) in enumerate(query_meta.tolist()):
        idx = indices[i].reshape(-1)[:max(use, 0)].long()
        ok = (idx >= 0) & (idx < tokens) & (idx // page < block_table.shape[1])
        if causal:
            ok &= idx <= pos
        if not 0 <= r < block_table.shape[0]:
            continue
        idx = idx[ok]
        at = block_table[r].long()[idx // page]
        inside = (at >= 0) & (at < n_pages)
        at, idx = at[inside], idx[inside]
        if not at.numel():
            continue
        s = torch.ldexp(torch.ones_like(scales[at]), torch.frexp(scales[at])[1] - 1).double().clamp(min=2.0 ** MIN_EXP)[:, None]       # the exponent alone
        code = store[at * page + idx % page].view(torch.float8_e4m3fn).double()
        k, x = code * s, q[i].double()
        logits = x @ k.T * sm_scale
        out.lse[i] = torch.logsumexp(logits, 1) / math.log(2)
        p = torch.softmax(logits, 1)
        out.o[i] = p @ k[:, :D_V]
        size = (x.abs() @ k.abs().T * 2.0 ** -18 + x.abs().amax(1, keepdim=True) * k.abs().sum(1) * 2.0 ** -9 / 224) * abs(sm_scale)
        off = size.amax(1, keepdim=True) + 2.0 ** -20 + logits.abs().amax(1, keepdim=True) * 2.0 ** -22 + float(s.log2().abs().max()) * 2.0 ** -24
        heavy = (p * s[:, 0]).amax(1, keepdim=True)
        out.o_bound[i] = (2.0 ** -8 + 2 * off) * (p @ k[:, :D_V].abs()) + 2.0 ** -16 * heavy * code[:, :D_V].abs().sum(0) + 2.0 ** -8 * out.o[i].abs()
        out.lse_bound[i] = off[:, 0] * 2 + (out.lse[i].abs() + s.log2().abs().max()) * 2.0 ** -22
    return out
