"""Plain 64-bit forms of the paged-cache and position-bias operators, and how far a correct 32-bit
implementation may be from them."""
import math

import torch

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16, torch.float32)}
TINY = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for t in HALF_STEP}     # half a step of the smallest numbers


def bucket(n: int, side: int, max_distance: int) -> int:
    """Bucket of a distance, in whole numbers: the largest one that n has reached."""
    half = side // 2
    if n < half:
        return n
    rest, k = side - half, 0
    while k + 1 < rest and n ** rest >= half ** (rest - k - 1) * max_distance ** (k + 1):
        k += 1
    return half + k


def bucket_row(differences, buckets, bidirectional, max_distance):
    """Buckets of key position - query position."""
    side = buckets // 2 if bidirectional else buckets
    out = []
    for x in differences:
        n = abs(x) if bidirectional else max(-x, 0)
        out.append(bucket(n, side, max_distance) + (side if bidirectional and x > 0 else 0))
    return torch.tensor(out, dtype=torch.int64)


def relbias(weight, tq, tk, bidirectional, max_distance, offset):
    row = bucket_row([x - offset for x in range(1 - tq, tk)], weight.shape[0], bidirectional, max_distance)
    at = torch.arange(tk)[None, :] - torch.arange(tq)[:, None] + tq - 1
    return weight.double()[row[at]].permute(2, 0, 1)[None], row[at]


def relbias_grad(dbias, which, buckets):
    out = torch.zeros(buckets, dbias.shape[1], dtype=torch.float64)
    for k in range(buckets):
        out[k] = (dbias[0].double() * (which == k)).sum((1, 2))
    return out


def locate(page_table, b, p, page_size, pages):
    """(page, slot) of position p of sequence b, None when there is none."""
    if p < 0 or p // page_size >= page_table.shape[1]:
        return None
    page = int(page_table[b, p // page_size])
    return (page, p % page_size) if 0 <= page < pages else None


def append(key, value, k_cache, v_cache, page_table, lengths, pos_emb=None, query=None, counts=None):
    """Returns (k_cache, v_cache, query) in 64 bits and, of each, the size of the terms that were added."""
    kc, vc = k_cache.double().clone(), v_cache.double().clone()
    ks, q = kc.abs(), None if query is None else query.double().clone()
    qs = None if q is None else q.abs()
    page_size, pages = k_cache.shape[1], k_cache.shape[0]

    def turn(x, p):
        y, size = x.double().clone(), x.double().abs()
        if pos_emb is not None:
            R = pos_emb.shape[2]
            sin, cos = pos_emb[0, p].double(), pos_emb[1, p].double()
            a, b = x[..., 0:R:2].double(), x[..., 1:R:2].double()
            y[..., 0:R:2], y[..., 1:R:2] = a * cos[0::2] - b * sin[0::2], b * cos[1::2] + a * sin[1::2]
            size[..., 0:R:2] = (a * cos[0::2]).abs() + (b * sin[0::2]).abs()
            size[..., 1:R:2] = (b * cos[1::2]).abs() + (a * sin[1::2]).abs()
        return y, size

    for b in range(key.shape[0]):
        for i in range(key.shape[1] if counts is None else max(0, min(key.shape[1], int(counts[b])))):
            p = int(lengths[b]) + i
            at = locate(page_table, b, p, page_size, pages)
            if at is None or (pos_emb is not None and p >= pos_emb.shape[1]):
                continue
            kc[at], ks[at] = turn(key[b, i], p)
            vc[at] = value[b, i].double()
            if q is not None:
                q[b, i], qs[b, i] = turn(query[b, i], p)
    return (kc, vc, q), (ks, vc.abs(), qs)


def assert_rotated(got, want, size, what):
    """Two fp32 products (half a step each) and their sum (another), then one rounding to the output's type."""
    t = got.dtype
    slack = HALF_STEP[t] * want.abs() + 2.0 ** -22 * size + TINY[t]
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert (off <= slack).all(), f"{what}: off by {off.max():.3e}, {int((off > slack).sum())} elements over their bound"


def attention(q, k_cache, v_cache, page_table, lengths, scale, weight=None, bidirectional=False, max_distance=128):
    """(o, lse, bound on o's error, bound on lse's error) of a 32-bit implementation before o's last rounding.

    Each score is a sum of d products: off by at most (d + 8) half steps of fp32 of the sum of their sizes, the 8 for
    scale, log2 e, the bias and their rounding.  With e that of the largest, a weight exp(s - max) is off by a factor
    of 1 + 2 e + 2^-20 (the 2^-20 is the base-2 exponential's and the running rescales') and, split into two 16-bit
    numbers, by another 2^-18 of its own and 2^-25 of the largest; numerator and denominator each have that."""
    B, _, H, d = q.shape
    page_size, pages, Hk = k_cache.shape[1], k_cache.shape[0], k_cache.shape[2]
    o, bound = torch.zeros(B, 1, H, d, dtype=torch.float64), torch.zeros(B, 1, H, d, dtype=torch.float64)
    lse, lse_bound = torch.full((B, H), -math.inf, dtype=torch.float64), torch.zeros(B, H, dtype=torch.float64)
    for b in range(B):
        n = max(0, min(int(lengths[b]), page_table.shape[1] * page_size))
        at = [(j, locate(page_table, b, j, page_size, pages)) for j in range(n)]
        at = [(j, x) for j, x in at if x is not None]
        if not at:
            continue
        j, where = torch.tensor([j for j, _ in at]), tuple(torch.tensor(x) for x in zip(*[x for _, x in at]))
        k, v = (c[where].double().repeat_interleave(H // Hk, 1) for c in (k_cache, v_cache))
        s = torch.einsum("hd,khd->hk", q[b, 0].double(), k) * scale
        size = torch.einsum("hd,khd->hk", q[b, 0].double().abs(), k.abs()) * abs(scale)
        if weight is not None:
            side = weight.shape[0] // 2 if bidirectional else weight.shape[0]
            rows = torch.tensor([bucket(n - 1 - int(x), side, max_distance) for x in j])
            add = weight.double()[rows].t()
            s, size = s + add, size + add.abs()
        finite = torch.where(torch.isfinite(size), size, torch.zeros_like(size))
        e = (d + 8) * 2.0 ** -24 * finite.amax(-1)
        m = s.amax(-1, keepdim=True)
        m = torch.where(m == -math.inf, torch.zeros_like(m), m)
        w = (s - m).exp()
        total = w.sum(-1, keepdim=True)
        empty = total[:, 0] == 0
        total = torch.where(total == 0, torch.ones_like(total), total)
        o[b, 0] = torch.einsum("hk,khd->hd", w / total, v)
        spread = torch.einsum("hk,khd->hd", w / total, v.abs())
        least = torch.einsum("hk,khd->hd", torch.ones_like(w) / total, v.abs())
        bound[b, 0] = (2 * (2 * e + 2.0 ** -20) + 2.0 ** -18)[:, None] * spread + 2.0 ** -25 * least
        lse[b] = torch.where(empty, torch.full_like(m[:, 0], -math.inf), m[:, 0] + total[:, 0].log())
        lse_bound[b] = 2 * e + 2.0 ** -19 + 2.0 ** -22 * lse[b].abs().nan_to_num(posinf=0)
    return o, lse, bound, lse_bound


def assert_attention(got, got_lse, want, what):
    o, lse, bound, lse_bound = want
    off = (got.double().cpu() - o).abs()
    slack = HALF_STEP[got.dtype] * (o.abs() + bound) + bound + TINY[got.dtype]
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert (off <= slack).all(), f"{what}: off by {off.max():.3e}, {int((off > slack).sum())} of {off.numel()} over their bound"
    if got_lse is not None:
        got_lse = got_lse.double().cpu()
        assert torch.equal(got_lse == -math.inf, lse == -math.inf), f"{what}: rows without a key"
        live = lse > -math.inf
        assert ((got_lse - lse).abs()[live] <= lse_bound[live]).all(), f"{what}: log-sum-exp"


def assert_grad(got, want, size, terms, what):
    """A sum of `terms` fp32 numbers, each partial sum over at most 2^10 of them in fp32 (and the sums of those in fp32
    or more): off by at most 2^10 half steps of the sum of the sizes, one rounding at the end."""
    off = (got.double().cpu() - want).abs()
    slack = HALF_STEP[got.dtype] * want.abs() + min(terms, 1 << 10) * 2.0 ** -24 * size + TINY[got.dtype]
    assert (off <= slack).all(), f"{what}: off by {off.max():.3e}"
