"""Paged key-value cache: appending with rotation, and attention of one new token, against their 64-bit forms."""
import math

import pytest
import torch

from rgd_triton_b200 import _lib, functional as F_, ops
from tests import _plain as P
from tests._util import DTYPES, gen, randn, rotary_table

pytestmark = pytest.mark.gpu


def _pool(g, pages, page, Hk, d, dtype, layout="tokens"):
    """A (page, slot, head, channel) view of each of the two caches, filled."""
    def one():
        if layout == "tokens":
            return randn(g, pages, page, Hk, d, dtype=dtype)
        if layout == "heads":
            return randn(g, pages, Hk, page, d, dtype=dtype).transpose(1, 2)
        if layout == "odd":         # rows that no 16-byte access reaches
            return randn(g, pages, page, Hk, d + 3, dtype=dtype)[..., 1:1 + d]
        return randn(g, pages, 2, page, Hk, d, dtype=dtype)[:, 1]       # keys and values side by side
    return one(), one()


def _table(g, lengths, page, spare=2, width=None):
    """Pages scattered over the pool, -1 past each sequence's last one."""
    need = [max(0, -(-n // page)) for n in lengths]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(need + [1]) if width is None else width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def _gpu(t):
    """The same values and strides on the GPU."""
    if t is None:
        return None
    if t.is_contiguous():
        return t.cuda()
    out = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda")
    return out.copy_(t)


# ------------------------------------------------------------------------------------------- append
APPEND = [
    # B, N, Hq, Hk, d, R, page, layout
    (1, 1, 0, 1, 64, 64, 16, "tokens"), (3, 1, 8, 2, 128, 128, 16, "heads"), (2, 37, 12, 4, 96, 48, 24, "tokens"),
    (2, 5, 3, 3, 40, 0, 1, "beside"), (4, 19, 5, 5, 17, 8, 7, "odd"), (1, 130, 16, 1, 128, 64, 100, "odd"),
    (2, 9, 6, 2, 8, 2, 16, "heads"), (1, 3, 2, 1, 1, 0, 4, "tokens"), (5, 64, 40, 8, 80, 80, 32, "tokens"), (300, 1, 4, 4, 64, 64, 16, "heads"),
    (2, 6, 70, 70, 128, 96, 16, "tokens"), (2, 11, 3, 1, 120, 6, 16, "tokens"),
]


@pytest.mark.parametrize("B,N,Hq,Hk,d,R,page,layout", APPEND)
@pytest.mark.parametrize("dtype,table", [("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "bf16")])
def test_append(B, N, Hq, Hk, d, R, page, layout, dtype, table):
    g = gen(B * N + d)
    dt = DTYPES[dtype]
    lengths = torch.randint(0, 3 * page + 2, (B,), generator=g, dtype=torch.int32)
    counts = torch.randint(0, N + 1, (B,), generator=g, dtype=torch.int32)
    page_table, pages = _table(g, [int(n) + N for n in lengths], page)
    kc, vc = _pool(g, pages, page, Hk, d, dt, layout)
    key, value = randn(g, B, N, Hk, d, dtype=dt), randn(g, B, Hk, N, d, dtype=dt).transpose(1, 2)
    query = randn(g, B, N, Hq + 1, d, dtype=dt)[:, :, 1:] if Hq and R else None
    pos = rotary_table(4 * page + N + 2, R, DTYPES[table]) if R else None
    for cnt in (None, counts):
        (wk, wv, wq), (sk, sv, sq) = P.append(key, value, kc, vc, page_table, lengths, pos, query, cnt)
        k_gpu, v_gpu = _gpu(kc), _gpu(vc)
        version = k_gpu._version
        q = F_.paged_cache_append_fn(_gpu(key), _gpu(value), k_gpu, v_gpu, page_table.cuda(), lengths.cuda(), _gpu(pos), _gpu(query), _gpu(cnt))
        assert k_gpu._version > version and v_gpu._version > 0
        P.assert_rotated(k_gpu.cpu(), wk, sk, "k_cache")
        assert torch.equal(v_gpu.cpu(), wv.to(dt))
        untouched = wk == kc.double()
        assert torch.equal(k_gpu.cpu()[untouched], kc[untouched])       # every slot but the new tokens' as it was
        if query is None:
            assert q is None
        else:
            P.assert_rotated(q.cpu(), wq, sq, "query")
            if cnt is not None:
                for b in range(B):
                    assert torch.equal(q[b, int(cnt[b]):].cpu(), query[b, int(cnt[b]):])
    assert _lib.load().rgd_device_status() == 0


def test_append_around_the_cache_changes_nothing():
    """The memory between and around strided slots stays as it was."""
    g = gen(1)
    store = randn(g, 2, 6, 8, 3, 2, 70, dtype=torch.float16)
    mine = store.cuda()
    kc, vc = mine[0][:, :, 1, :, 3:67], mine[1][:, :, 1, :, 3:67]
    key, value = randn(g, 2, 5, 2, 64, dtype=torch.float16), randn(g, 2, 5, 2, 64, dtype=torch.float16)
    table = torch.tensor([[4, 0], [1, 3]], dtype=torch.int32)
    F_.paged_cache_append_fn(key.cuda(), value.cuda(), kc, vc, table.cuda(), torch.tensor([6, 2], dtype=torch.int32).cuda())
    want = store.clone()
    for b, first in ((0, 6), (1, 2)):
        for i in range(5):
            at = P.locate(table, b, first + i, 8, 6)
            want[0][at[0], at[1], 1, :, 3:67], want[1][at[0], at[1], 1, :, 3:67] = key[b, i], value[b, i]
    assert torch.equal(mine.cpu(), want)


@pytest.mark.parametrize("R", [6, 12, 20, 34])
def test_channels_past_the_rotated_ones_are_copied_bit_for_bit(R):
    """Infinities, NaN and negative zeros there, next to rotated channels in one 16-byte group."""
    g = gen(R)
    d, page = 64, 16
    key = randn(g, 2, 7, 3, d, dtype=torch.float16)
    special = torch.tensor([math.inf, -math.inf, math.nan, -0.0, 0.0, -2.5], dtype=torch.float16)
    key[..., R:] = special[torch.randint(0, 6, key[..., R:].shape, generator=g)]
    table, lengths = torch.tensor([[1, 0], [3, 2]], dtype=torch.int32), torch.tensor([3, 12], dtype=torch.int32)
    kc, vc = (torch.zeros(4, page, 3, d, dtype=torch.float16) for _ in range(2))
    k_gpu, v_gpu = kc.cuda(), vc.cuda()
    q = F_.paged_cache_append_fn(key.cuda(), key.cuda(), k_gpu, v_gpu, table.cuda(), lengths.cuda(), rotary_table(64, R, torch.float32).cuda(), key.cuda())
    bits = lambda t: t.cpu().contiguous().view(torch.int16)
    assert torch.equal(bits(q[..., R:]), bits(key[..., R:]))
    for b in range(2):
        for i in range(7):
            at = P.locate(table, b, int(lengths[b]) + i, page, 4)
            assert torch.equal(bits(k_gpu[at][..., R:]), bits(key[b, i][..., R:])) and torch.equal(bits(v_gpu[at]), bits(key[b, i]))
            assert torch.isfinite(k_gpu[at][..., :R]).all()


def test_append_of_many_tokens_with_few_and_many_heads():
    """Grids of the caches and of the query that differ by more than a hundred times, and tokens that cross sequences."""
    g = gen(77)
    B, N, Hq, Hk, d = 3, 1500, 96, 1, 8
    lengths = torch.tensor([0, 7, 100], dtype=torch.int32)
    table, pages = _table(g, [int(n) + N for n in lengths], 32)
    kc, vc = _pool(g, pages, 32, Hk, d, torch.bfloat16)
    key, value, query = (randn(g, B, N, h, d, dtype=torch.bfloat16) for h in (Hk, Hk, Hq))
    pos = rotary_table(1700, d, torch.bfloat16)
    k_gpu, v_gpu = kc.cuda(), vc.cuda()
    q = F_.paged_cache_append_fn(key.cuda(), value.cuda(), k_gpu, v_gpu, table.cuda(), lengths.cuda(), pos.cuda(), query.cuda())
    (wk, wv, wq), (sk, _, sq) = P.append(key, value, kc, vc, table, lengths, pos, query)
    P.assert_rotated(k_gpu.cpu(), wk, sk, "k_cache")
    assert torch.equal(v_gpu.cpu().double(), wv)
    P.assert_rotated(q.cpu(), wq, sq, "query")


def test_append_leaves_out_what_has_no_place():
    """Bad pages, positions past the table or the rotary table, negative lengths: not written, and reported."""
    g = gen(2)
    lib = _lib.load()
    assert lib.rgd_device_status() == 0
    page, pages, N = 4, 6, 6
    kc, vc = _pool(g, pages, page, 2, 64, torch.bfloat16)
    key, value, query = (randn(g, 4, N, h, 64, dtype=torch.bfloat16) for h in (2, 2, 4))
    for name, table, lengths, P_rows in (
            ("page past the pool", [[0, 6, 1], [2, 3, 4], [5, -1, -1], [1, 7, 2 ** 31 - 1]], [0, 1, 0, 30], 64),
            ("negative page", [[0, -5, 1], [2, 3, 4], [5, -2 ** 31, -1], [-1, -1, -1]], [0, 1, 0, 0], 64),
            ("position past the table", [[0, 1, 2], [3, 4, 5], [-1, -1, -1], [-1, -1, -1]], [9, 4, 12, 2 ** 31 - 1], 64),
            ("negative length", [[0, 1, 2], [3, 4, 5], [-1, -1, -1], [-1, -1, -1]], [-3, 4, -2 ** 31, -6], 64),
            ("position past the rotary table", [[0, 1, 2], [3, 4, 5], [-1, -1, -1], [-1, -1, -1]], [2, 5, 0, 0], 7)):
        table, lengths = torch.tensor(table, dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32)
        counts = torch.tensor([N, N, N if "rotary" not in name else 0, N if "rotary" not in name else 0], dtype=torch.int32)
        pos = rotary_table(P_rows, 64, torch.float32)
        (wk, wv, wq), (sk, _, sq) = P.append(key, value, kc, vc, table, lengths, pos, query, counts)
        k_gpu, v_gpu = kc.cuda(), vc.cuda()
        q = F_.paged_cache_append_fn(key.cuda(), value.cuda(), k_gpu, v_gpu, table.cuda(), lengths.cuda(), pos.cuda(), query.cuda(), counts.cuda())
        P.assert_rotated(k_gpu.cpu(), wk, sk, name)
        assert torch.equal(v_gpu.cpu().double(), wv), name
        P.assert_rotated(q.cpu(), wq, sq, name)
        assert lib.rgd_device_status() == _lib.RGD_E_PAGE, name
        assert lib.rgd_device_status() == 0


# ------------------------------------------------------------------------------------------- attention
ATTN = [
    # lengths, Hq, Hk, d, page, layout
    ([1], 1, 1, 64, 16, "tokens"), ([1, 2, 15, 16, 17, 63, 64, 65], 4, 2, 128, 16, "tokens"), ([300, 0, 129, 1], 8, 8, 64, 16, "heads"),
    ([1000, 7, 640], 32, 8, 128, 24, "tokens"), ([257, 511], 7, 1, 96, 100, "beside"), ([77, 140], 6, 3, 17, 7, "odd"),
    ([129], 16, 1, 128, 64, "heads"), ([200, 90], 40, 2, 64, 32, "tokens"), ([65, 128], 64, 1, 80, 16, "tokens"),
    ([5000], 4, 1, 128, 16, "tokens"), ([2049, 3, 1500], 12, 12, 40, 1, "tokens"), ([31, 100], 2, 2, 1, 16, "tokens"), ([444], 5, 5, 128, 33, "odd"),
]


def _case(lengths, Hq, Hk, d, page, layout, dtype, seed, scale=1.0):
    g = gen(seed)
    table, pages = _table(g, lengths, page)
    kc, vc = _pool(g, pages, page, Hk, d, dtype, layout)
    q = randn(g, len(lengths), 1, Hq, d, dtype=dtype, scale=scale)
    return q, kc, vc, table, torch.tensor(lengths, dtype=torch.int32)


@pytest.mark.parametrize("lengths,Hq,Hk,d,page,layout", ATTN)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bias", [None, (32, False, 128), (8, True, 20)])
def test_attention(lengths, Hq, Hk, d, page, layout, dtype, bias):
    q, kc, vc, table, n = _case(lengths, Hq, Hk, d, page, layout, DTYPES[dtype], sum(lengths) + d)
    w, args = None, {}
    if bias:
        w = randn(gen(9), bias[0], Hq)
        args = {"rel_weight": w.cuda(), "bidirectional": bias[1], "max_distance": bias[2]}
    o, lse = F_.paged_attention_func(q.cuda(), _gpu(kc), _gpu(vc), table.cuda(), n.cuda(), return_lse=True, **args)
    assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == (len(lengths), Hq)
    want = P.attention(q, kc, vc, table, n, d ** -0.5, w, *(bias[1:] if bias else ()))
    P.assert_attention(o, lse, want, "o")
    assert _lib.load().rgd_device_status() == 0


@pytest.mark.parametrize("B,Hq,Hk,longest", [(70, 8, 8, 700), (200, 4, 2, 300), (3, 16, 2, 20000), (600, 1, 1, 64), (33, 24, 24, 64)])
def test_attention_of_many_sequences(B, Hq, Hk, longest):
    """Units that are split between CTAs, CTAs with many units, many empty sequences."""
    g = gen(B)
    lengths = torch.randint(0, longest + 1, (B,), generator=g)
    lengths[torch.rand(B, generator=g) < 0.2] = 0
    lengths[B // 2] = longest
    q, kc, vc, table, n = _case(lengths.tolist(), Hq, Hk, 64, 16, "tokens", torch.bfloat16, B)
    o, lse = F_.paged_attention_func(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda(), return_lse=True)
    P.assert_attention(o, lse, P.attention(q, kc, vc, table, n, 64 ** -0.5), "o")
    again = F_.paged_attention_func(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda())
    assert torch.equal(o, again)


@pytest.mark.parametrize("scale", [0.0, -0.3, 0.02, 5.0])
def test_attention_scales_and_wide_views(scale):
    q, kc, vc, table, n = _case([333, 64, 2], 6, 2, 64, 16, "tokens", torch.float16, 5)
    wide = torch.full((3, 9), 77, dtype=torch.int32)
    wide[:, :table.shape[1] if table.shape[1] < 9 else 9] = table[:, :9]
    big = torch.full((3, table.shape[1] + 5), -9, dtype=torch.int32)
    big[:, 2:2 + table.shape[1]] = table
    qw = randn(gen(6), 3, 2, 8, 64, dtype=torch.float16)
    qw[:, 1:, 1:7] = q
    o, lse = F_.paged_attention_func(qw.cuda()[:, 1:, 1:7], kc.cuda(), vc.cuda(), big.cuda()[:, 2:2 + table.shape[1]], n.cuda(),
                                     softmax_scale=scale, return_lse=True)
    P.assert_attention(o, lse, P.attention(q, kc, vc, table, n, scale), "o")


def test_attention_ignores_what_lies_past_a_sequence():
    """NaN and infinities in unused slots, pages and table entries; lengths of zero with a table of rubbish."""
    q, kc, vc, table, n = _case([70, 0, 1, 129], 8, 4, 128, 16, "tokens", torch.bfloat16, 6)
    want = P.attention(q, kc, vc, table, n, 128 ** -0.5)
    used = torch.zeros(kc.shape[:2], dtype=torch.bool)
    for b in range(4):
        for j in range(int(n[b])):
            used[P.locate(table, b, j, 16, kc.shape[0])] = True
    for rubbish in (math.nan, math.inf, -math.inf, torch.finfo(torch.bfloat16).max):
        k2, v2 = kc.clone(), vc.clone()
        k2[~used], v2[~used] = rubbish, rubbish
        t2 = torch.where(table < 0, torch.full_like(table, 2 ** 31 - 1), table)
        o, lse = F_.paged_attention_func(q.cuda(), k2.cuda(), v2.cuda(), t2.cuda(), n.cuda(), return_lse=True)
        P.assert_attention(o, lse, want, str(rubbish))
        assert (o[1] == 0).all()
    assert _lib.load().rgd_device_status() == 0


def test_attention_leaves_out_bad_pages_and_cuts_lengths():
    lib = _lib.load()
    assert lib.rgd_device_status() == 0
    q, kc, vc, table, n = _case([200, 333, 48], 4, 2, 64, 16, "tokens", torch.float16, 8)
    table[0, 3], table[0, 12], table[1, 0], table[2, :3] = -7, kc.shape[0], 2 ** 31 - 1, -1
    for lengths in (n, torch.tensor([200, 2 ** 31 - 1, -4], dtype=torch.int32)):
        t = table.clone()
        t[1, 21:] = 3
        o, lse = F_.paged_attention_func(q.cuda(), kc.cuda(), vc.cuda(), t.cuda(), lengths.cuda(), return_lse=True)
        P.assert_attention(o, lse, P.attention(q, kc, vc, t, lengths, 64 ** -0.5), "o")
        assert (o[2] == 0).all() and (lse[2] == -math.inf).all()
        assert lib.rgd_device_status() == _lib.RGD_E_PAGE
        assert lib.rgd_device_status() == 0


@pytest.mark.parametrize("longest", [40, 3000])
@pytest.mark.parametrize("entry", [-1, -2 ** 31, 2 ** 31 - 1, "pages"])
def test_every_bad_entry_is_reported(longest, entry):
    """One bad entry of a live page, in a table for few and for many keys; the same entry past the sequence is fine."""
    lib = _lib.load()
    assert lib.rgd_device_status() == 0
    q, kc, vc, table, n = _case([longest, 33], 2, 2, 64, 16, "tokens", torch.float16, 21)
    value = kc.shape[0] if entry == "pages" else entry
    for at, status in ((2, _lib.RGD_E_PAGE), (3, 0)):
        t = table.clone()
        t[1, min(at, t.shape[1] - 1)] = value
        if at < t.shape[1]:
            o = F_.paged_attention_func(q.cuda(), kc.cuda(), vc.cuda(), t.cuda(), n.cuda())
            P.assert_attention(o, None, P.attention(q, kc, vc, t, n, 64 ** -0.5), "o")
            assert lib.rgd_device_status() == status


def test_a_pool_without_pages():
    lib = _lib.load()
    q = randn(gen(22), 2, 1, 4, 64, dtype=torch.float16).cuda()
    empty = torch.empty(0, 16, 2, 64, dtype=torch.float16, device="cuda")
    table, n = torch.zeros(2, 200, dtype=torch.int32, device="cuda"), torch.tensor([3000, 5], dtype=torch.int32, device="cuda")
    for t in (table, table[:, :1]):
        o, lse = F_.paged_attention_func(q, empty, empty, t, n, return_lse=True)
        assert (o == 0).all() and (lse == -math.inf).all()
        assert lib.rgd_device_status() == _lib.RGD_E_PAGE
    key = q[:, :, :2]
    F_.paged_cache_append_fn(key, key, empty, empty, table, torch.zeros_like(n))
    assert lib.rgd_device_status() == _lib.RGD_E_PAGE


def test_attention_bias_of_the_types_lowest_value():
    """Buckets masked with -inf and with the lowest finite value; a row that is masked whole."""
    q, kc, vc, table, n = _case([100, 9], 2, 1, 64, 16, "tokens", torch.bfloat16, 9)
    for wdtype in (torch.float32, torch.bfloat16, torch.float16):
        low = torch.finfo(wdtype).min
        w = randn(gen(10), 8, 2).to(wdtype)
        w[3:, 0], w[:4, 1] = -math.inf, low
        o, lse = F_.paged_attention_func(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda(), rel_weight=w.cuda(), max_distance=20, return_lse=True)
        want = P.attention(q, kc, vc, table, n, 64 ** -0.5, w, False, 20)
        for b, h in ((0, 0), (0, 1), (1, 0), (1, 1)):
            P.assert_attention(o[b:b + 1, :, h:h + 1], None, [x[b:b + 1, :, h:h + 1] if x.ndim == 4 else x for x in want], f"{b} {h}")
        if wdtype != torch.float16:         # every key masked with it: the scores are lost in its rounding, the mean of v is left
            w[:, 1] = low
            o = F_.paged_attention_func(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda(), rel_weight=w.cuda(), max_distance=20)
            flat = vc[table.long().clamp(min=0)].flatten(1, 2)[:, :, 0].double()
            for b in range(2):
                mean, size = flat[b, :n[b]].mean(0), flat[b, :n[b]].abs().mean(0)
                assert ((o[b, 0, 1].cpu().double() - mean).abs() <= 2.0 ** -8 * mean.abs() + 2.0 ** -16 * size).all()
        w[:, 0] = -math.inf
        o, lse = F_.paged_attention_func(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda(), rel_weight=w.cuda(), max_distance=20, return_lse=True)
        assert (o[:, :, 0] == 0).all() and (lse[:, 0] == -math.inf).all()


def test_nan_and_infinity_of_live_keys_reach_the_output():
    q, kc, vc, table, n = _case([80, 80], 2, 2, 64, 16, "tokens", torch.float16, 11)
    at = P.locate(table, 0, 70, 16, kc.shape[0])
    kc[at[0], at[1], 0] = math.nan
    o = F_.paged_attention_func(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda())
    assert o[0, 0, 0].isnan().all() and torch.isfinite(o[0, 0, 1]).all() and torch.isfinite(o[1]).all()


def test_shared_pages_and_64_bit_offsets():
    """Sequences that share their first pages; a cache of more than 2^32 elements, pages at both ends."""
    page, Hk, d, pages = 64, 8, 128, 66000
    assert pages * page * Hk * d > 1 << 32
    kc = torch.zeros(pages, page, Hk, d, dtype=torch.float16, device="cuda")
    vc = torch.zeros(pages, page, Hk, d, dtype=torch.float16, device="cuda")
    g = gen(12)
    table = torch.tensor([[pages - 1, 5, 0], [pages - 1, 5, pages - 2], [pages - 1, 65999, 65537]], dtype=torch.int32)
    small = sorted(set(table.flatten().tolist()))
    place = {x: i for i, x in enumerate(small)}
    near = torch.tensor([[place[int(x)] for x in row] for row in table], dtype=torch.int32)
    lengths = torch.tensor([100, 128, 64], dtype=torch.int32)
    key, value, query = randn(g, 3, 64, Hk, d, dtype=torch.float16), randn(g, 3, 64, Hk, d, dtype=torch.float16), randn(g, 3, 1, 16, d, dtype=torch.float16)
    kn, vn = _pool(g, len(small), page, Hk, d, torch.float16)
    kc[small], vc[small] = kn.cuda(), vn.cuda()
    counts = torch.tensor([60, 64, 0], dtype=torch.int32)
    wide = (kc, vc, table.cuda())
    close = (kn.cuda(), vn.cuda(), near.cuda())
    for caches in (wide, close):
        F_.paged_cache_append_fn(key.cuda(), value.cuda(), *caches, lengths.cuda(), counts=counts.cuda())
    assert torch.equal(kc[small], close[0]) and torch.equal(vc[small], close[1])
    total = (lengths + counts).cuda()
    o = F_.paged_attention_func(query.cuda(), *wide, total)
    assert torch.equal(o, F_.paged_attention_func(query.cuda(), *close, total))
    P.assert_attention(o, None, P.attention(query, close[0].cpu(), close[1].cpu(), near, lengths + counts, d ** -0.5), "o")
    del kc, vc, wide
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("d,Hq,Hk,page", [(64, 8, 2, 16), (128, 4, 4, 24)])
def test_prompt_then_tokens_equals_attention_over_the_whole(d, Hq, Hk, page):
    """A prompt is appended, then tokens one at a time with the attention over the cache; every step against the
    attention over all rotated keys, and the prompt's own against FlashAttention's last row."""
    g = gen(13)
    B, prompt, steps, dt = 3, 50, 40, torch.bfloat16
    total = prompt + steps
    q, k, v = (randn(g, B, total, h, d, dtype=dt).cuda() for h in (Hq, Hk, Hk))
    pos = rotary_table(total + 1, d, torch.float32).cuda()
    table = torch.randperm(B * -(-total // page), generator=g).to(torch.int32).view(B, -1).cuda()
    kc, vc = (torch.zeros(table.numel(), page, Hk, d, dtype=dt, device="cuda") for _ in range(2))
    append, attend = ops.PagedCacheAppend(), ops.PagedAttention()
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        q0 = append(k[:, :prompt], v[:, :prompt], kc, vc, table, lengths, pos, q[:, :prompt])
        lengths += prompt
        flat = lambda c: c[table.long()].flatten(1, 2)
        share = lambda t: t.repeat_interleave(Hq // Hk, 2)
        whole = ops.FlashAttention()(q0, share(flat(kc)[:, :prompt]), share(v[:, :prompt]), causal=True)
        last = attend(q0[:, -1:], kc, vc, table, lengths)
        # both round the same exact value; the first also rounds its weights to 16 bits
        assert (last.float() - whole[:, -1:].float()).abs().max() <= 4 * 2.0 ** -8 * whole.float().abs().max()
        for i in range(prompt, total):
            qi = append(k[:, i:i + 1], v[:, i:i + 1], kc, vc, table, lengths, pos, q[:, i:i + 1])
            lengths += 1
            o, lse = F_.paged_attention_func(qi, kc, vc, table, lengths, return_lse=True)
            if i in (prompt, prompt + 13, total - 1):
                want = P.attention(qi.cpu(), kc.cpu(), vc.cpu(), table.cpu(), lengths.cpu(), d ** -0.5)
                P.assert_attention(o, lse, want, f"token {i}")
    assert torch.equal(flat(vc)[:, :total], v)
    assert _lib.load().rgd_device_status() == 0


@pytest.mark.parametrize("G", [1, 2, 7, 8, 9, 15, 16, 17, 24, 25, 33])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 24), (100, 16)])
def test_attention_of_any_number_of_heads_to_a_cache_head(G, d, page):
    """One and two column tiles of heads, whole and not, groups of 16; with and without a schedule; twice the same bits."""
    for lengths in ([300, 1, 77], [3000, 20, 500]):
        q, kc, vc, table, n = _case(lengths, 2 * G, 2, d, page, "tokens", torch.bfloat16, G + d)
        w = randn(gen(G), 32, 2 * G)
        for bias in (None, w):
            args = {} if bias is None else {"rel_weight": bias.cuda()}
            call = lambda: F_.paged_attention_func(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda(), return_lse=True, **args)
            o, lse = call()
            P.assert_attention(o, lse, P.attention(q, kc, vc, table, n, d ** -0.5, bias, *(() if bias is None else (False, 128))), (lengths, G))
            again = call()
            assert torch.equal(o, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("buckets,both,most", [(32, False, 5000), (512, True, 1000), (6, False, 200), (256, False, 129), (4, True, 1 << 20)])
@pytest.mark.parametrize("wdtype", ["f32", "f16", "bf16"])
def test_attention_bias_of_near_and_far_distances(buckets, both, most, wdtype):
    """Borders on either side of where the kernel stops looking buckets up, for weights of every type."""
    lengths = [4000, 255, 256, 257, 258, 1]
    q, kc, vc, table, n = _case(lengths, 6, 3, 64, 16, "tokens", torch.bfloat16, buckets)
    w = randn(gen(buckets), buckets, 6, dtype={"f32": torch.float32, **DTYPES}[wdtype])
    o, lse = F_.paged_attention_func(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda(), rel_weight=w.cuda(), bidirectional=both,
                                     max_distance=most, return_lse=True)
    P.assert_attention(o, lse, P.attention(q, kc, vc, table, n, 64 ** -0.5, w, both, most), "o")


def test_position_bias_of_a_token_is_the_matrix_form_s_last_row():
    g = gen(14)
    m = ops.RelativePositionBias(32, 6, bidirectional=False).cuda()
    q, kc, vc, table, n = _case([300], 6, 6, 64, 16, "tokens", torch.float16, 14)
    with torch.no_grad():
        o = ops.PagedAttention()(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda(), rel_bias=m)
        k = kc[table.long()].flatten(1, 2)[:, :300].cuda()
        v = vc[table.long()].flatten(1, 2)[:, :300].cuda()
        full = ops.FlashAttention()(q.cuda(), k, v, bias=m(1, 300, offset=299))
    assert (o.float() - full.float()).abs().max() <= 4 * 2.0 ** -11 * full.float().abs().max()


def test_captured_steps_replay_for_other_lengths_and_two_graphs():
    """Two graphs of a whole step, replayed in turns after the lengths grew; eager calls in between."""
    g = gen(15)
    B, Hq, Hk, d, page = 4, 8, 2, 128, 16
    table = torch.randperm(B * 40, generator=g).to(torch.int32).view(B, 40).cuda()
    pos = rotary_table(700, d, torch.bfloat16).cuda()
    pools = [[t.cuda() for t in _pool(g, B * 40, page, Hk, d, torch.bfloat16)] for _ in range(2)]
    lengths = torch.tensor([1, 100, 350, 16], dtype=torch.int32, device="cuda")
    new = [[randn(g, B, 1, h, d, dtype=torch.bfloat16).cuda() for h in (Hk, Hk, Hq)] for _ in range(2)]

    def step(i):
        k, v, q = new[i]
        q = F_.paged_cache_append_fn(k, v, *pools[i], table, lengths, pos, q)
        return F_.paged_attention_func(q, *pools[i], table, lengths + 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0), step(1)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(step(i))
    for grow in (0, 37, 150):
        lengths += grow
        for a in new:
            for t in a:
                t.copy_(torch.randn_like(t))
        for i in (0, 1, 0):
            graphs[i].replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for i in range(2):
            assert torch.equal(got[i], step(i))
    assert _lib.load().rgd_device_status() == 0


def test_calls_on_two_streams_at_once():
    q, kc, vc, table, n = _case([3000, 20, 1000], 8, 2, 128, 16, "tokens", torch.bfloat16, 16)
    dev = [t.cuda() for t in (q, kc, vc, table, n)]
    q2, k2, v2, t2, n2 = [t.cuda() for t in _case([500, 4000], 16, 4, 64, 24, "tokens", torch.bfloat16, 17)]
    want, want2 = F_.paged_attention_func(*dev), F_.paged_attention_func(q2, k2, v2, t2, n2)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(20):
        with torch.cuda.stream(a):
            got.append((F_.paged_attention_func(*dev), want))
        with torch.cuda.stream(b):
            got.append((F_.paged_attention_func(q2, k2, v2, t2, n2), want2))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in got)


def test_inference_mode_and_empty_calls():
    q, kc, vc, table, n = [t.cuda() for t in _case([30, 3], 4, 2, 64, 16, "tokens", torch.float16, 18)]
    with torch.inference_mode():
        k2, v2 = kc.clone(), vc.clone()
        assert F_.paged_cache_append_fn(q[:, :, :2], q[:, :, :2], k2, v2, table, n - 1) is None
        o = F_.paged_attention_func(q, k2, v2, table, n)
    assert o.shape == q.shape
    assert F_.paged_cache_append_fn(k2.new_empty(2, 0, 2, 64), k2.new_empty(2, 0, 2, 64), kc, vc, table, n) is None
    empty = F_.paged_attention_func(q[:0], kc, vc, table[:0], n[:0])
    assert empty.shape == (0, 1, 4, 64)
    nothing = F_.paged_attention_func(q, kc[:0], vc[:0], table[:, :0], torch.zeros_like(n))
    assert (nothing == 0).all()
    assert _lib.load().rgd_device_status() == 0


@pytest.mark.parametrize("Hq,Hk,d", [(1, 1, 64), (16, 1, 64), (6, 2, 128), (3, 1, 40)])
@pytest.mark.parametrize("B,n", [(1200, 8192), (2, 800)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_many_keys_far_below_one_count(Hq, Hk, d, B, n, dtype):
    """One key with a value of 0, and all the others with one score far below it: the output is their weight alone.  With
    a run of one warp as long as a sequence (more units than warps), and with few keys (a CTA per unit).

    The products are exact (one channel).  A score in base 2 is scale * log2(e) (half a step of fp32) times that, rounded:
    off by 2^-23 of itself, the base-2 exponential by 2^-22, the two 16-bit numbers by 2^-18 of the weight (bf16) or
    2^-22 and 2^-40 of the largest (fp16).  Two sums for 16 keys, each off by at most a step: 2 n / 16 * 2^-23; the row
    sum, in 8 lanes: n / 8 * 2^-24.  The output's rounding at the end."""
    dt, page = DTYPES[dtype], 64
    pages = -(-n // page)
    v = torch.rand(pages, page, Hk, d, generator=gen(23)).to(dt)
    v[0, 0] = 0
    table = torch.arange(pages, dtype=torch.int32).cuda()[None].expand(B, -1)       # all sequences read the same pages
    lengths = torch.full((B,), n, dtype=torch.int32, device="cuda")
    q = torch.zeros(B, 1, Hq, d, dtype=dt)
    q[..., 0] = 8
    for gap in (9.0, 12.0, 15.0, 17.0, 17.375, 19.0):       # exact in both types
        k = torch.zeros(pages, page, Hk, d, dtype=dt)
        k[0, 0, :, 0] = gap
        o, lse = F_.paged_attention_func(q.cuda(), k.cuda(), v.cuda(), table, lengths, softmax_scale=0.125, return_lse=True)
        weight = math.exp(-gap)
        total = 1 + (n - 1) * weight
        want = (v.flatten(0, 1)[:n].double().sum(0) * weight / total).repeat_interleave(Hq // Hk, 0)
        split = 2.0 ** -18 if dtype == "bf16" else 2.0 ** -22 + 2.0 ** -40 / weight
        off = 2.0 ** -23 * gap / math.log(2) + 2.0 ** -22 + split + n / 8 * 2.0 ** -23 + n / 8 * 2.0 ** -24
        slack = (2 * off + P.HALF_STEP[dt]) * want + P.TINY[dt]
        assert ((o[:, 0].double().cpu() - want).abs() <= slack).all(), f"gap {gap}: {((o[:, 0].double().cpu() - want).abs() / want).max():.2e}"
        assert (lse.double().cpu() - (gap + math.log(total))).abs().max() <= 2 * off + 2.0 ** -22 * gap


@pytest.mark.parametrize("d", [64, 128])
def test_sums_over_a_long_run_do_not_drift(d):
    """131 thousand keys in one warp's run (more units than warps; all sequences read the same pages), values of one sign.

    Each output: its rounding (half a step), the weights (as in the plain form's bound) and two sums, of the products and of
    the weights, of n / 16 and n / 8 terms that are rounded each (half a step of fp32).  Together: these errors have either
    sign, and the mean over the outputs, of which the rounding to fp16 is by far the largest and uniform in its step, stays
    within six times half a step / sqrt(3 outputs)."""
    n, page, Hk, B, dt = 131072, 64, 512 // d, 1 + 1200 * d // 512, torch.float16
    g = gen(d)
    k, v = randn(g, n // page, page, Hk, d, dtype=dt).cuda(), torch.rand(n // page, page, Hk, d, generator=g).to(dt).cuda()
    q = randn(g, 1, 1, Hk, d, dtype=dt).cuda()
    table = torch.arange(n // page, dtype=torch.int32, device="cuda")[None].expand(B, -1)
    lengths = torch.full((B,), n, dtype=torch.int32, device="cuda")
    o = F_.paged_attention_func(q.expand(B, 1, Hk, d), k, v, table, lengths)[:, 0].double()
    kd, vd, qd = k.flatten(0, 1).double(), v.flatten(0, 1).double(), q[0, 0].double()
    want = torch.einsum("hk,khd->hd", torch.softmax(torch.einsum("hd,khd->hk", qd, kd) * d ** -0.5, -1), vd)
    e = (d + 8) * 2.0 ** -24 * (torch.einsum("hd,khd->hk", qd.abs(), kd.abs()) * d ** -0.5).max()
    weights = 2 * (2 * e + 2.0 ** -20) + 2.0 ** -18
    off = o / want - 1
    assert off.abs().max() <= P.HALF_STEP[dt] + weights + 3 * n / 16 * 2.0 ** -24
    assert off.mean((1, 2)).abs().max() <= 6 * P.HALF_STEP[dt] / math.sqrt(3 * Hk * d) + weights


@pytest.mark.parametrize("layout", ["tokens", "heads"])
def test_attention_of_a_padded_prompt_over_its_gathered_keys(layout):
    """A padded batch of prompts with grouped heads: the append rotates the query, the rotated keys are gathered from the
    pages, and the causal attention of the real rows is that of the rotated tokens.  FlashAttention rounds its weights
    and its output to bf16: two half steps of the largest value, twice that for the second product's own rounding."""
    g = gen(24)
    B, n, heads, heads_k, d, page, dt = 3, 37, 8, 2, 64, 16, torch.bfloat16
    counts = torch.tensor([37, 5, 20], dtype=torch.int32)
    table, pages = _table(g, counts.tolist(), page)
    kc, vc = (_gpu(t) for t in _pool(g, pages, page, heads_k, d, dt, layout))
    key, value, query = (randn(g, B, n, h, d, dtype=dt) for h in (heads_k, heads_k, heads))
    pos = rotary_table(n, d, torch.float32)
    lengths, page_table = torch.zeros(B, dtype=torch.int32).cuda(), table.cuda()
    _, _, rotated = P.append(key, value, torch.zeros(pages, page, heads_k, d), torch.zeros(pages, page, heads_k, d), table, torch.zeros(B, dtype=torch.int32), pos, query, counts)[0]
    q = F_.paged_cache_append_fn(key.cuda(), value.cuda(), kc, vc, page_table, lengths, pos.cuda(), query.cuda(), counts.cuda())
    used = page_table[:, :(n + page - 1) // page].long().clamp(min=0)
    k = kc[used].flatten(1, 2)[:, :n]
    share = heads // heads_k
    o = F_.flash_attn_func(q, k.repeat_interleave(share, 2), value.cuda().repeat_interleave(share, 2), causal=True).double().cpu()
    sin, cos = pos.double()
    for b in range(B):
        m = int(counts[b])
        x = key[b, :m].double()
        kr = torch.stack([x[..., 0::2] * cos[:m, None, 0::2] - x[..., 1::2] * sin[:m, None, 0::2],
                          x[..., 1::2] * cos[:m, None, 1::2] + x[..., 0::2] * sin[:m, None, 1::2]], -1).flatten(-2).to(dt).double()
        kr, v = kr.repeat_interleave(share, 1), value[b, :m].double().repeat_interleave(share, 1)
        s = torch.einsum("ihd,jhd->hij", rotated[b, :m].to(dt).double(), kr) * d ** -0.5
        s = s.masked_fill(torch.ones(m, m, dtype=torch.bool).triu(1), -math.inf)
        want = torch.einsum("hij,jhd->ihd", s.softmax(-1), v)
        assert (o[b, :m] - want).abs().max() <= 4 * 2.0 ** -8 * v.abs().max()
