"""Timed cases of the serving and position-bias operators: appending keys and values to a paged cache with the
rotation applied on the way, attention of one new token over such a cache, and a learned relative position bias with
its gradient.

``run`` computes a pass either in plain torch operations or, with ``own`` true, through the entry points of
``rgd_triton_b200.functional``; ``exact`` computes it in 64 bits from the definitions.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MOST_SLOTS = 1 << 28        # elements of the largest key cache, and of the keys that the plain form gathers densely


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # Append: one new token of each of four conversations far into their context (latency counts) ...
        _append("append_decode_small_bf16", "bf16", 4, 1, 32, 8, 128, 16, past=30000),
        # ... one new token of each sequence of a large serving batch ...
        _append("append_decode_batch_f16", "f16", 256, 1, 32, 8, 128, 16, past=8000, heads_second=True),
        # ... the prompts of a batch, all of one length, right after the projection ...
        _append("append_prompt_bf16", "bf16", 4, 4096, 16, 16, 128, 64, past=500),
        # ... and ragged pieces of prompts, partial rotation by an fp32 table, an odd page size.
        _append("append_ragged_f16", "f16", 7, 333, 12, 4, 96, 24, past=1000, R=48, table="f32", ragged=True),
        # One new token: a single short conversation (latency) ...
        _attn("paged_short_bf16", "bf16", 1, 16, 16, 128, 300, 16),
        # ... a serving batch of grouped heads and mixed lengths ...
        _attn("paged_batch_bf16", "bf16", 64, 32, 8, 128, 8192, 16, ragged=True),
        # ... one document of 131 thousand tokens ...
        _attn("paged_long_bf16", "bf16", 1, 32, 8, 128, 131079, 64),
        # ... ungrouped heads of 64 channels, odd lengths and pages, the cache head by head ...
        _attn("paged_ragged_f16", "f16", 48, 24, 24, 64, 2500, 24, ragged=True, heads_second=True),
        # ... and a decoder with a learned position bias instead of a rotation.
        _attn("paged_bias_bf16", "bf16", 16, 16, 16, 64, 1500, 16, ragged=True, buckets=32),
        # Position bias: between the few tokens of a small encoder, at inference ...
        _bias("relbias_infer_odd_bf16", "bf16", "f32", False, 12, 197, 333, 32, True),
        # ... the training step of an encoder at 4096 tokens, for the attention with a matrix bias ...
        _bias("relbias_train_f16", "f16", "f32", True, 24, 4096, 4096, 32, True),
        # ... and of a decoder of ordinary size, looking back only.
        _bias("relbias_train_back_bf16", "bf16", "bf16", True, 16, 1024, 1023, 32, False),
    ]


def _append(name, dtype, B, N, Hq, Hkv, d, page, past, R=None, table=None, ragged=False, heads_second=False):
    """N new tokens (up to N when ragged) of each of B sequences that hold up to `past` tokens already."""
    return {"name": name, "op": "append", "dtype": dtype, "table": table or dtype, "B": B, "N": N, "Hq": Hq, "Hkv": Hkv, "d": d,
            "R": d if R is None else R, "page": page, "past": past, "ragged": ragged, "heads_second": heads_second}


def _attn(name, dtype, B, Hq, Hkv, d, longest, page, ragged=False, heads_second=False, buckets=0):
    return {"name": name, "op": "attn", "dtype": dtype, "B": B, "Hq": Hq, "Hkv": Hkv, "d": d, "longest": longest, "page": page,
            "ragged": ragged, "heads_second": heads_second, "buckets": buckets}


def _bias(name, dtype, wdtype, train, H, tq, tk, buckets, both):
    return {"name": name, "op": "bias", "dtype": dtype, "wdtype": wdtype, "train": train, "H": H, "tq": tq, "tk": tk,
            "buckets": buckets, "both": both, "max_distance": 128, "offset": 0}


def _spread(rng, lo, hi):
    """A whole number, uniform over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op, dtype = rng.choice(("append", "attn", "attn", "bias")), rng.choice(("f16", "bf16"))
    largest = {c["op"]: max(work(x)["bytes"] for x in listed() if x["op"] == c["op"]) for c in listed()}
    while True:
        Hkv, G, d = rng.choice((1, 2, 4, 5, 8, 12, 16)), rng.choice((1, 1, 2, 3, 4, 7, 8, 16)), rng.choice((40, 64, 64, 96, 128, 128))
        page, heads_second = rng.choice((8, 16, 16, 24, 32, 64, 100)), rng.random() < 0.3
        if op == "append":
            N = 1 if rng.random() < 0.4 else _spread(rng, 2, 4096)
            case = _append("", dtype, _spread(rng, 1, 256), N, rng.choice((0, Hkv * G)), Hkv, d, page, _spread(rng, 10, 30000),
                           rng.choice((0, d // 2, d)), rng.choice((dtype, "f32")), N > 1 and rng.random() < 0.5, heads_second)
            fits = case["B"] * (N + 2 * page) * Hkv * d <= MOST_SLOTS
            if case["R"] == 0:
                case["Hq"] = 0
        elif op == "attn":
            longest = _spread(rng, 16, 131079)
            case = _attn("", dtype, _spread(rng, 1, 256), Hkv * G, Hkv, d, longest, page, rng.random() < 0.7, heads_second,
                         rng.choice((0, 0, 0, 32, 64)))
            fits = case["B"] * (longest + page) * Hkv * d <= MOST_SLOTS
        else:
            tq = _spread(rng, 16, 4608)
            case = _bias("", rng.choice(("f32", "f16", "bf16")), rng.choice(("f32", "f16", "bf16")), rng.random() < 0.6,
                         rng.randint(1, 24), tq, tq if rng.random() < 0.5 else _spread(rng, 16, 4608), rng.choice((8, 32, 32, 64)),
                         rng.random() < 0.5)
            case["max_distance"], case["offset"] = rng.choice((64, 128, 128, 200)), rng.choice((0, 0, 1, 77))
            fits = True
        if fits and work(case)["bytes"] <= largest[op]:
            del case["name"]
            return case


def _lengths(case):
    """Cached tokens of each sequence: sizes, so they go by the case and not by the seed."""
    longest = case["past"] if case["op"] == "append" else case["longest"]
    rng = random.Random("%d %d %d" % (case["B"], longest, case["page"]))
    if case["op"] == "append":
        return [rng.randint(0, longest) for _ in range(case["B"])]
    if not case["ragged"]:
        return [longest] * case["B"]
    return [longest] + [_spread(rng, min(16, longest), longest) for _ in range(case["B"] - 1)]


def _counts(case):
    """New tokens of each sequence."""
    rng = random.Random("%d %d" % (case["B"], case["N"]))
    return [rng.randint(0, case["N"]) if case["ragged"] else case["N"] for _ in range(case["B"])]


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "append":
        tokens = sum(_counts(case))
        values = tokens * case["d"] * 2 * case["Hkv"] + case["B"] * case["N"] * case["d"] * case["Hq"]
        rotated = tokens * case["R"] * (case["Hkv"] + case["Hq"])
        return {"bytes": 2 * values * size + tokens * (2 * case["R"] * (4 if case["table"] == "f32" else 2) + 4), "flops": 3 * rotated}
    if case["op"] == "attn":
        keys = sum(_lengths(case))
        cache = 2 * keys * case["Hkv"] * case["d"] * size
        return {"bytes": cache + 2 * case["B"] * case["Hq"] * case["d"] * size, "flops": 4 * keys * case["Hq"] * case["d"]}
    elements = case["H"] * case["tq"] * case["tk"]
    weight = case["buckets"] * case["H"] * (4 if case["wdtype"] == "f32" else 2)
    passes = 2 if case["train"] else 1
    return {"bytes": passes * (elements * size + weight), "flops": elements if case["train"] else 0}


# ---------------------------------------------------------------------------------------------------- inputs
def _rotary_table(positions, R, dtype):
    """[2, positions, R]: sin, cos of t * 10000^(-2i/R), each angle repeated for its pair."""
    inv = 1.0 / (10000.0 ** (torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R))
    ang = (torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv).repeat_interleave(2, dim=-1)
    return torch.stack([ang.sin(), ang.cos()]).to(dtype)


def _pool(case, g, pages):
    """Keys and values of `pages` pages (a recycled pool: every slot holds something), as (page, slot, head, channel)."""
    page, Hkv, d = case["page"], case["Hkv"], case["d"]
    shape = (pages, Hkv, page, d) if case["heads_second"] else (pages, page, Hkv, d)
    pool = [torch.randn(*shape, generator=g, device="cuda", dtype=DTYPES[case["dtype"]]) for _ in range(2)]
    return [t.transpose(1, 2) for t in pool] if case["heads_second"] else pool


def _page_table(case, g, first, last):
    """Pages scattered over the pool for logical pages [first, last) of each sequence; -1 where there is none.
    Returns the table and the pages of the pool."""
    width, used = max(max(last), 1), [max(0, b - a) for a, b in zip(first, last)]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    at = torch.arange(width, device="cuda")[None, :]
    lo, hi = (torch.tensor(x, device="cuda")[:, None] for x in (first, last))
    before = torch.tensor([sum(used[:b]) for b in range(len(used))], device="cuda")[:, None]
    index = (before + at - lo).clamp(0, pages - 1)
    return torch.where((at >= lo) & (at < hi), order[index], torch.full_like(order[:1], -1)), pages


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    if case["op"] == "bias":
        return _prepare_bias(case, g)
    dtype, page, B = DTYPES[case["dtype"]], case["page"], case["B"]
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
    lengths = _lengths(case)
    state = {"case": case, "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
    if case["op"] == "attn":
        state["page_table"], pages = _page_table(case, g, [0] * B, [-(-n // page) for n in lengths])
        state["k_cache"], state["v_cache"] = _pool(case, g, pages)
        state["query"] = randn(B, 1, case["Hq"], case["d"])
        state["weight"] = torch.randn(case["buckets"], case["Hq"], generator=g, device="cuda") if case["buckets"] else None
        return state
    counts = _counts(case)
    state["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda") if case["ragged"] else None
    # which of the B * N tokens are new ones: a program that packs its batch has the list
    token = torch.arange(case["N"], device="cuda")[None, :] < torch.tensor(counts, device="cuda")[:, None]
    state["tokens"] = token.flatten().nonzero().flatten()
    # the pages that hold earlier tokens alone are not in the pool here: no append touches them
    state["page_table"], pages = _page_table(case, g, [n // page for n in lengths], [-(-(n + c) // page) for n, c in zip(lengths, counts)])
    state["k_cache"], state["v_cache"] = _pool(case, g, pages)
    state["key"], state["value"] = randn(B, case["N"], case["Hkv"], case["d"]), randn(B, case["N"], case["Hkv"], case["d"])
    state["query"] = randn(B, case["N"], case["Hq"], case["d"]) if case["Hq"] else None
    state["pos_emb"] = _rotary_table(case["past"] + case["N"] + 1, case["R"], DTYPES[case["table"]]) if case["R"] else None
    return state


def _prepare_bias(case, g):
    H, tq, tk, dtype = case["H"], case["tq"], case["tk"], DTYPES[case["dtype"]]
    weight = torch.randn(case["buckets"], H, generator=g, device="cuda").to(DTYPES[case["wdtype"]])
    # the upstream gradient of an attention's bias: probabilities times differences, small
    grad = torch.randn(1, H, tq, tk, generator=g, device="cuda", dtype=dtype) * 0.01 if case["train"] else None
    return {"case": case, "weight": weight.requires_grad_(case["train"]), "grad": grad}


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"append": _run_append, "attn": _run_attn, "bias": _run_bias}[state["case"]["op"]](state)


def _run_append(s):
    if own:
        from rgd_triton_b200 import functional
        q = functional.paged_cache_append_fn(s["key"], s["value"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"],
                                             pos_emb=s["pos_emb"], query=s["query"], counts=s["counts"])
        out = {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        return out if q is None else {**out, "query": q}
    B, N, page = s["case"]["B"], s["case"]["N"], s["case"]["page"]
    pos = (s["lengths"].long()[:, None] + torch.arange(N, device="cuda")).flatten()[s["tokens"]]
    where = (s["page_table"].long()[s["tokens"] // N, pos // page], pos % page)
    out = {}
    for name, x in (("k_cache", s["key"]), ("v_cache", s["value"]), ("query", s["query"])):
        if x is None:
            continue
        rows = x.flatten(0, 1)
        new = rows[s["tokens"]]
        if name != "v_cache" and s["pos_emb"] is not None:
            new = _rotate(new.float(), s["pos_emb"].float(), pos).to(x.dtype)
        if name == "query":
            out[name] = rows.index_copy(0, s["tokens"], new).view(x.shape)
        else:
            out[name] = s[name].index_put_(where, new)
    return out


def _rotate(x, table, pos):
    """Pairs of neighbouring channels turned by the angles of their token's position; channels past the table's as they are."""
    R = table.shape[2]
    sin, cos = table[0, pos][:, None, :], table[1, pos][:, None, :]
    turned = torch.stack([-x[..., 1:R:2], x[..., 0:R:2]], dim=-1).flatten(-2)
    return torch.cat([x[..., :R] * cos + turned * sin, x[..., R:]], dim=-1)


def _run_attn(s):
    if own:
        from rgd_triton_b200 import functional
        return functional.paged_attention_func(s["query"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"],
                                               rel_weight=s["weight"], bidirectional=False, max_distance=128)
    c = s["case"]
    B, Hkv, d = c["B"], c["Hkv"], c["d"]
    table = s["page_table"].long().clamp(min=0)
    k = s["k_cache"][table].flatten(1, 2).float()
    v = s["v_cache"][table].flatten(1, 2).float()
    q = s["query"].float().view(B, Hkv, -1, d)
    score = torch.einsum("bhgd,bkhd->bhgk", q, k) / math.sqrt(d)
    key = torch.arange(k.shape[1], device="cuda")
    length = s["lengths"].long()[:, None]
    if s["weight"] is not None:
        bias = s["weight"][_bucket(length - 1 - key, c["buckets"], 128).clamp(min=0)]
        score = score + bias.permute(0, 2, 1).reshape(score.shape)
    score = score.masked_fill((key >= length)[:, None, None, :], -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    return torch.einsum("bhgk,bkhd->bhgd", p, v).reshape(s["query"].shape).to(s["query"].dtype)


def _bucket(n, buckets, max_distance):
    """Bucket of a distance n >= 0: one each for the first half, then even steps of the logarithm up to max_distance.
    In 64 bits, with borders that fall on whole numbers counted to the upper bucket."""
    half = buckets // 2
    step = (n.double().clamp(min=half) / half).log() / math.log(max_distance / half) * (buckets - half)
    return torch.where(n < half, n, (half + (step + 1e-9).floor().long()).clamp(max=buckets - 1))


def _buckets_of(case, difference):
    """Bucket of (key position - query position): forward distances use the upper half of the buckets."""
    n = case["buckets"]
    if not case["both"]:
        return _bucket((-difference).clamp(min=0), n, case["max_distance"])
    return _bucket(difference.abs(), n // 2, case["max_distance"]) + torch.where(difference > 0, n // 2, 0)


def _run_bias(s):
    c = s["case"]
    H, tq, tk = c["H"], c["tq"], c["tk"]
    if own:
        from rgd_triton_b200 import functional
        bias = functional.relative_position_bias_fn(s["weight"], tq, tk, bidirectional=c["both"], max_distance=c["max_distance"],
                                                    offset=c["offset"], dtype=DTYPES[c["dtype"]])
        if not c["train"]:
            return bias
        return {"bias": bias.detach(), "dweight": torch.autograd.grad(bias, s["weight"], s["grad"])[0]}
    # element (i, j) depends on j - i alone: windows of one row of tk + tq - 1 differences
    row = _buckets_of(c, torch.arange(1 - tq, tk, device="cuda") - c["offset"])
    i, j = torch.arange(tq, device="cuda")[:, None], torch.arange(tk, device="cuda")
    weight = s["weight"].detach()
    bias = weight.float()[row].to(DTYPES[c["dtype"]]).t().contiguous()[:, j - i + tq - 1][None]
    if not c["train"]:
        return bias
    # sums along the diagonals: rows written one element further each come under one another when read one shorter
    wide = torch.zeros(H, tq, tk + tq, device="cuda")
    wide[:, :, :tk] = s["grad"][0].flip(1)
    sums = wide.view(H, -1)[:, :tq * (tk + tq - 1)].view(H, tq, tk + tq - 1).sum(1, dtype=torch.float64)
    which = (row[:, None] == torch.arange(c["buckets"], device="cuda")).double()
    return {"bias": bias, "dweight": (sums @ which).t().to(weight.dtype)}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "bias": _exact_bias}[case["op"]](s)


def _exact_append(s):
    c, lengths, counts = s["case"], _lengths(s["case"]), _counts(s["case"])
    out = {"k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double()}
    if s["query"] is not None:
        out["query"] = s["query"].double()
    for b in range(c["B"]):
        n = counts[b]
        at = torch.arange(lengths[b], lengths[b] + n, device="cuda")
        pages = s["page_table"][b].long()[at // c["page"]]
        new = {"k_cache": s["key"][b, :n].double(), "v_cache": s["value"][b, :n].double()}
        if s["query"] is not None:
            new["query"] = s["query"][b, :n].double()
        if s["pos_emb"] is not None:
            sin, cos = s["pos_emb"].double()[:, lengths[b]:lengths[b] + n, None, :]
            for name in set(new) - {"v_cache"}:
                x = new[name][..., :c["R"]].clone()
                new[name][..., 0:c["R"]:2] = x[..., 0::2] * cos[..., 0::2] - x[..., 1::2] * sin[..., 0::2]
                new[name][..., 1:c["R"]:2] = x[..., 1::2] * cos[..., 1::2] + x[..., 0::2] * sin[..., 1::2]
        out["k_cache"][pages, at % c["page"]], out["v_cache"][pages, at % c["page"]] = new["k_cache"], new["v_cache"]
        if s["query"] is not None:
            out["query"][b, :n] = new["query"]
    return out


def _borders(buckets, max_distance):
    """The least distance of each bucket from 1 on, by whole numbers: bucket half + j begins where
    (n / half)^(buckets - half) reaches (max_distance / half)^j."""
    half = buckets // 2
    rest, found = buckets - half, list(range(1, half + 1))
    for j in range(1, rest):
        n = found[-1]
        while n ** rest * half ** j < half ** rest * max_distance ** j:
            n += 1
        found.append(n)
    return torch.tensor(found, device="cuda")


def _exact_attn(s):
    c, lengths = s["case"], _lengths(s["case"])
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        where = (s["page_table"][b].long()[at // c["page"]], at % c["page"])
        k, v = s["k_cache"][where].double().transpose(0, 1), s["v_cache"][where].double().transpose(0, 1)
        q = s["query"][b, 0].double().view(c["Hkv"], -1, c["d"])
        score = q @ k.transpose(1, 2) * c["d"] ** -0.5
        if s["weight"] is not None:
            which = torch.searchsorted(_borders(c["buckets"], 128), n - 1 - at, right=True)
            score = score + s["weight"].double()[which].t().reshape(score.shape)
        out[b, 0] = (torch.softmax(score, dim=-1) @ v).view(c["Hq"], c["d"])
    return out


def _exact_bias(s):
    c, H, tq, tk = s["case"], s["case"]["H"], s["case"]["tq"], s["case"]["tk"]
    side = c["buckets"] // 2 if c["both"] else c["buckets"]
    borders = _borders(side, c["max_distance"])
    difference = torch.arange(tk, device="cuda")[None, :] - torch.arange(tq, device="cuda")[:, None] - c["offset"]
    which = torch.searchsorted(borders, difference.abs(), right=True)
    which = which + side * (difference > 0) if c["both"] else which.masked_fill(difference > 0, 0)
    bias = torch.empty(1, H, tq, tk, dtype=torch.float64, device="cuda")
    for h in range(H):
        bias[0, h] = s["weight"].detach()[:, h].double()[which]
    if not c["train"]:
        return bias
    dweight = torch.zeros(c["buckets"], H, dtype=torch.float64, device="cuda")
    for k in range(c["buckets"]):
        dweight[k] = (s["grad"][0] * (which == k)).sum((1, 2), dtype=torch.float64)
    return {"bias": bias, "dweight": dweight}
