"""The operators between a decoder layer's linears from their definitions, in 64 bits on the CPU, one row at a time."""
from __future__ import annotations

import math

import torch

# half a unit in the last place of a 16- or 32-bit type, as a share of the value, and the smallest step's half
HALF_ULP = {torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.float32: (2.0 ** -24, 2.0 ** -150)}


def norm_ref(x, residual, weight, eps):
    """(y in fp64, the residual in its type): the residual's sum is rounded to its type, and normed as it is kept."""
    x = x.cpu()
    h = x if residual is None else (x.double() + residual.cpu().double()).to(residual.dtype)
    hd = h.double()
    y = hd / torch.sqrt((hd * hd).mean(-1, keepdim=True) + eps)
    return (y if weight is None else y * weight.cpu().double()), h


def rotate_ref(x, positions, table, interleaved):
    """x [T, heads, dim] in fp64 with its first rot columns turned."""
    x, table = x.cpu().double().clone(), table.cpu().double()
    half = table.shape[1] // 2
    for t, pos in enumerate(positions.tolist()):
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            c, s = table[pos, i], table[pos, half + i]
            u, w = x[t, :, a].clone(), x[t, :, b].clone()
            x[t, :, a], x[t, :, b] = u * c - w * s, w * c + u * s
    return x


def cached(cache, name, pages, n):
    """[heads, n, dim] in fp64: the first n tokens of a list of page ids; a page outside the cache has none (None)."""
    x, scale = getattr(cache, name).cpu(), getattr(cache, name + "_scale")
    rows = []
    for t in range(n):
        page = pages[t // x.shape[2]]
        rows.append(x[page, :, t % x.shape[2]].double() if 0 <= page < x.shape[0] else None)
    keep = [r for r in rows if r is not None]
    got = torch.stack(keep, 1) if keep else torch.zeros(x.shape[1], 0, x.shape[3], dtype=torch.float64)
    present = torch.tensor([r is not None for r in rows], dtype=torch.bool)
    return (got if scale is None else got * scale.cpu().double().view(-1, 1, 1)), present


def attention_ref(q, cache, page_table, seq_lens, prefix_pages, prefix_len, query_start, scale):
    """(out, lse, sum of p |v|) in fp64; rows that see nothing give zeros and -inf."""
    q = q.cpu().double()
    t, h, d = q.shape
    hk = cache.k.shape[1]
    out, mag = torch.zeros(t, h, d, dtype=torch.float64), torch.zeros(t, h, d, dtype=torch.float64)
    lse = torch.full((t, h), -math.inf, dtype=torch.float64)
    starts = list(range(len(seq_lens) + 1)) if query_start is None else query_start.tolist()
    pk, pv = (cached(cache, n, prefix_pages.tolist() if prefix_len else [], prefix_len) for n in ("k", "v"))
    for b, n in enumerate(seq_lens.tolist()):
        k, present = cached(cache, "k", page_table[b].tolist(), n)
        v, _ = cached(cache, "v", page_table[b].tolist(), n)
        count = starts[b + 1] - starts[b]
        where = torch.nonzero(present).flatten()
        for i in range(count):
            own = int((where < n - count + i + 1).sum())
            kk, vv = torch.cat((pk[0], k[:, :own]), 1), torch.cat((pv[0], v[:, :own]), 1)
            if kk.shape[1] == 0:
                continue
            row = starts[b] + i
            for head in range(h):
                s = kk[head // (h // hk)] @ q[row, head] * scale
                lse[row, head] = torch.logsumexp(s, 0)
                p = torch.exp(s - lse[row, head])
                out[row, head], mag[row, head] = p @ vv[head // (h // hk)], p @ vv[head // (h // hk)].abs()
    return out, lse, mag


def assert_attention(got, lse, ref, dtype):
    """Each probability and the result are rounded once to ``dtype``; scores, exponents and sums are fp32, of which the scores'
    rounding (2^-22 of sums of up to a few hundred, twice) is the largest."""
    out, ref_lse, mag = ref
    u, tiny = HALF_ULP[dtype]
    err = (got.cpu().double() - out).abs()
    tol = (u + 2.0 ** -12) * mag + u * out.abs() + tiny
    assert bool((err <= tol).all()), f"off by {(err / tol.clamp_min(1e-300)).max().item():.3g} of the tolerance"
    if lse is not None:
        lse = lse.cpu().double()
        fine = torch.isfinite(ref_lse)
        assert torch.equal(fine, torch.isfinite(lse)) and torch.equal(lse[~fine], ref_lse[~fine])
        assert bool(((lse - ref_lse)[fine].abs() <= 2.0 ** -13 * (1 + ref_lse[fine].abs())).all())


def attention_ref_fast(q, cache, page_table, seq_lens, prefix_pages, prefix_len, query_start, scale):
    """attention_ref with a sequence's rows at once, in fp64 where q is (for sizes that row by row would take minutes); pages
    are all in the cache."""
    t, h, d = q.shape
    hk = cache.k.shape[1]
    out, mag = torch.zeros(t, h, d, dtype=torch.float64, device=q.device), torch.zeros(t, h, d, dtype=torch.float64, device=q.device)
    lse = torch.full((t, h), -math.inf, dtype=torch.float64, device=q.device)

    def tokens(name, pages, n):
        x, s = getattr(cache, name), getattr(cache, name + "_scale")
        pages = pages[:-(-n // x.shape[2])].long()
        rows = x.view(torch.uint8)[pages].view(x.dtype) if x.element_size() == 1 else x[pages]
        rows = rows.double().transpose(0, 1).reshape(hk, -1, d)[:, :n]
        return rows if s is None else rows * s.double().view(-1, 1, 1)

    starts = list(range(len(seq_lens) + 1)) if query_start is None else query_start.tolist()
    for b, n in enumerate(seq_lens.tolist()):
        k, v = (torch.cat((tokens(x, prefix_pages, prefix_len), tokens(x, page_table[b], n)), 1) for x in ("k", "v"))
        a, c = starts[b], starts[b + 1]
        if a == c or k.shape[1] == 0:
            continue
        own = (n - (c - a) + 1 + torch.arange(c - a, device=q.device)).clamp_min(0)
        sees = torch.arange(k.shape[1], device=q.device) < (prefix_len + own).view(-1, 1)
        for head in range(h):
            s = (q[a:c, head].double() @ k[head // (h // hk)].t() * scale).masked_fill(~sees, -math.inf)
            z = torch.logsumexp(s, 1)
            p = torch.exp(s - z.view(-1, 1)).nan_to_num(0.0)
            lse[a:c, head], out[a:c, head] = z, p @ v[head // (h // hk)]
            mag[a:c, head] = p @ v[head // (h // hk)].abs()
    return out.cpu(), lse.cpu(), mag.cpu()
