"""The attention block's operators from their definitions, in 64 bits on the CPU, and what their results may be off by."""
import math

import torch


def rows_of(table, b, length, page, n_pages):
    """Pool rows of a request's cached tokens, and which of them lie in the pool."""
    j = torch.arange(length)
    pages = table[b].long()[j // page]
    ok = (pages >= 0) & (pages < n_pages)
    return torch.where(ok, pages, torch.zeros_like(pages)) * page + j % page, ok


def attend(q, kb, vb, table, starts, news, lens, page, window, scale, max_kv=None):
    """``(out, weights, bound)``: out [T, hq, d] in 64 bits, nan where no request has a row; weights [requests, tokens]; bound: what
    an element of out may be off by (see ``bound_of``)."""
    q, table = q.detach().cpu(), table.cpu()
    kb, vb = kb.detach().cpu(), vb.detach().cpu()
    T, hq, d = q.shape
    hkv = kb.shape[1]
    group = hq // hkv
    n_pages = kb.shape[0] // page
    out = torch.full((T, hq, d), math.nan, dtype=torch.float64)
    bound = torch.full((T, hq, d), math.nan, dtype=torch.float64)
    weights = torch.zeros(len(news), table.shape[1] * page, dtype=torch.float64)
    w_bound = torch.zeros_like(weights)
    u = torch.finfo(q.dtype).eps / 2
    for b, (at, n, length) in enumerate(zip(starts, news, lens)):
        if n < 1:
            continue
        if max_kv is not None:
            length = min(length, max_kv)
        rows, ok = rows_of(table, b, length, page, n_pages)
        p = torch.arange(length - n, length)[:, None]
        j = torch.arange(length)[None]
        sees = (j <= p) & ok[None]
        if window:
            sees = sees & (j > p - window)
        for h in range(hq):
            K, V = kb[rows, h // group].double(), vb[rows, h // group].double()
            Q = q[at:at + n, h].double()
            s = (Q @ K.T) * scale
            s = torch.where(sees, s, torch.full_like(s, -math.inf))
            m = s.amax(-1, keepdim=True) if length else torch.full((n, 1), -math.inf, dtype=torch.float64)
            e = torch.where(torch.isneginf(m), torch.zeros_like(s), torch.exp(s - m))
            total = e.sum(-1, keepdim=True)
            w = torch.where(total == 0, torch.zeros_like(e), e / total)
            # a token that is not seen does not show, whatever it holds
            seen_by_all = sees.all(0)
            o = w[:, seen_by_all] @ V[seen_by_all]
            for t in torch.nonzero(~seen_by_all).flatten().tolist():
                o = o + torch.where(sees[:, t, None], w[:, t, None] * V[t][None], torch.zeros_like(o))
            out[at:at + n, h] = o
            weights[b, :length] += w.sum(0)
            # off by: scores in 32 bits (d products and their sum, the scaling, the exponent's argument), the exponential
            absolute = (Q.abs() @ K.abs().T) * scale
            absolute = torch.where(sees, absolute, torch.zeros_like(absolute))
            rel = (2 * d + 8) * 2.0 ** -24 * torch.nan_to_num(absolute, nan=0.0, posinf=0.0).amax(-1, keepdim=True) + 2.0 ** -20 if length else torch.zeros(n, 1).double()
            size = w @ torch.nan_to_num(V, nan=0.0, posinf=0.0, neginf=0.0).abs() + torch.nan_to_num(o, nan=0.0, posinf=0.0, neginf=0.0).abs()
            # weights that the second product takes are rounded (u each, none below the type's least step), its sum is in 32 bits,
            # the result is rounded
            least = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
            top = torch.nan_to_num(V, nan=0.0, posinf=0.0, neginf=0.0).abs().amax() if length else 0.0
            bound[at:at + n, h] = size * (u * (1 + u) ** 2 + 2 * rel + (length + 64) * 2.0 ** -24) + u * size + 2 * length * least * top + 2.0 ** -24
            w_bound[b, :length] += (w * (2 * rel + (length + 64) * 2.0 ** -24)).sum(0) + n * 2.0 ** -100
    return out, weights, bound, w_bound


def check_out(got, want, bound, what=""):
    got, mine = got.detach().cpu().double(), ~torch.isnan(bound)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    err = torch.where(same, torch.zeros_like(got), (got - want).abs())
    over = mine & ~(err <= bound) & ~same
    assert not bool(over.any()), (f"{what}: {int(over.sum())} of {int(mine.sum())} over, the worst by a factor "
                                  f"{float(torch.nan_to_num(err / bound, nan=math.inf)[over].max())}, at {over.nonzero()[:3].tolist()}")
