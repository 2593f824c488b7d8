"""Paged cache and position bias without a GPU: bucket borders, addressing, refusals, the C ABI's argument checks."""
import ctypes as C
import inspect

import pytest
import torch

from rgd_triton_b200 import _lib, functional as F_, ops
from tests import _plain as P


@pytest.mark.parametrize("side,most", [(2, 2), (2, 100), (3, 7), (8, 20), (16, 128), (32, 128), (5, 1000), (32, 20), (256, 129), (16, 1 << 20), (128, (1 << 28) - 1)])
def test_borders_are_exact(side, most):
    borders = F_.relative_position_borders(side, most)
    assert len(borders) == side - 1 and list(borders) == sorted(borders) and borders[0] == 1
    near = {n + d for n in borders for d in (-1, 0, 1)} | {0, 1, 2, most - 1, most, most + 1, 2 * most}
    for n in sorted(near):
        if n >= 0:
            assert sum(x <= n for x in borders) == P.bucket(n, side, most), n
    if side == 16 and most == 128:
        assert {16, 32, 64} < set(borders)         # powers that a rounded logarithm gets wrong


def _paged(table, page=16, pages=10, sp=1000, ss=60, k=1):
    return _lib.Paged(k, k, sp, ss, 1, sp * 2, ss, 1, pages, page, table.data_ptr(), table.stride(0), table.shape[1], 1)


def test_slots_are_found_and_bad_pages_are_not_followed():
    lib = _lib.load()
    table = torch.tensor([[3, 0, 9, -1], [10, 2 ** 31 - 1, -2 ** 31, 4]], dtype=torch.int32)
    k, v = C.c_int64(0), C.c_int64(0)
    at = lambda c, row, p: lib.rgd_paged_slot(C.byref(c), row, p, C.byref(k), C.byref(v))
    for page in (1, 3, 7, 16, 100, 1 << 20):
        c = _paged(table, page)
        for row in range(2):
            for p in sorted({x for i in range(4) for x in (i * page, i * page + page // 2, (i + 1) * page - 1)}):
                entry = int(table[row, p // page])
                if 0 <= entry < 10:
                    assert at(c, row, p) == 0
                    assert k.value == entry * 1000 + p % page * 60 and v.value == entry * 2000 + p % page * 60
                else:
                    assert at(c, row, p) == _lib.RGD_E_PAGE
        for p in (-1, -2 ** 31, 4 * page, 2 ** 31, 2 ** 40):
            assert at(c, 0, p) == _lib.RGD_E_PAGE
    # offsets past 32 bits
    big = torch.tensor([[2 ** 31 - 2]], dtype=torch.int32)
    c = _paged(big, 128, 2 ** 31 - 1, sp=128 * 8 * 128, ss=1024)
    assert at(c, 0, 127) == 0 and k.value == (2 ** 31 - 2) * 131072 + 127 * 1024
    assert at(_paged(table, 1 << 29), 0, 5) == _lib.RGD_E_SIZE           # positions are 31-bit
    assert at(_paged(table, 0), 0, 5) == _lib.RGD_E_INVALID
    assert at(_paged(table, ss=-60), 0, 5) == _lib.RGD_E_STRIDE


def test_c_abi_argument_checks():
    lib = _lib.load()
    h = lambda p=1: C.byref(_lib.Heads(p, 8, 8, 8))
    table = torch.zeros(1, 4, dtype=torch.int32)
    cache = _paged(table)
    app = lambda dt=_lib.RGD_F16, d=64, R=64, pos=1, c=cache, k=None, q=None, pdt=0, B=1, N=1: lib.rgd_paged_append(
        k or h(), h(), q, q, C.byref(c), None, pos, 64, 64, 100, R, B, N, 4, 2, d, dt, pdt, None)
    assert app(dt=_lib.RGD_F32) == _lib.RGD_E_DTYPE and app(pdt=7) == _lib.RGD_E_DTYPE
    assert app(d=256) == _lib.RGD_E_SIZE and app(B=1 << 20, N=1 << 20) == _lib.RGD_E_SIZE
    assert app(R=63) == _lib.RGD_E_INVALID and app(R=66) == _lib.RGD_E_INVALID and app(R=-2) == _lib.RGD_E_INVALID
    assert app(k=h(None)) == _lib.RGD_E_NULL
    assert app(c=_paged(table, k=None)) == _lib.RGD_E_NULL
    assert app(N=0) == 0 and app(B=0) == 0
    att = lambda dt=_lib.RGD_F16, d=64, Hq=4, Hkv=2, c=cache, q=None, bias=None, ws=None, n=0: lib.rgd_paged_attn(
        q or h(), C.byref(c), bias, h(), None, 1, Hq, Hkv, d, 1.0, dt, ws, n, None)
    assert att(dt=_lib.RGD_F32) == _lib.RGD_E_DTYPE and att(d=136) == _lib.RGD_E_SIZE
    assert att(Hq=5) == _lib.RGD_E_INVALID and att(Hkv=0) == _lib.RGD_E_INVALID
    assert att(q=h(None)) == _lib.RGD_E_NULL and att(d=0) == 0
    borders = (C.c_int32 * 3)(1, 5, 4)
    bias = lambda **kw: C.byref(_lib.RelBias(*[{"weight": 1, "sb": 4, "sh": 1, "dtype": 0, "n": 4, "both": 0, "at": borders, **kw}[x]
                                               for x in ("weight", "sb", "sh", "dtype", "n", "both", "at")]))
    assert att(bias=bias()) == _lib.RGD_E_INVALID                       # borders that fall
    borders[2] = 9
    assert att(bias=bias(weight=None)) == _lib.RGD_E_NULL and att(bias=bias(dtype=9)) == _lib.RGD_E_DTYPE
    assert att(bias=bias(n=3, both=1)) == _lib.RGD_E_INVALID and att(bias=bias(n=600)) == _lib.RGD_E_SIZE
    assert lib.rgd_paged_attn_workspace_bytes(-1, 4, 4, 64, 4, 16) == _lib.RGD_E_INVALID
    fwd = lambda b=None, out=16, sh=64, sq=8, H=4, tq=8, tk=8, off=0, dt=0: lib.rgd_relbias_fwd(b or bias(), out, sh, sq, H, tq, tk, off, dt, None)
    assert fwd(out=8) == _lib.RGD_E_STRIDE and fwd(sq=7) == _lib.RGD_E_STRIDE and fwd(tk=9) == _lib.RGD_E_STRIDE and fwd(sh=2) == _lib.RGD_E_STRIDE
    assert fwd(dt=5) == _lib.RGD_E_DTYPE and fwd(H=-1) == _lib.RGD_E_INVALID and fwd(off=1 << 40) == _lib.RGD_E_SIZE
    assert fwd(out=None) == _lib.RGD_E_NULL and fwd(tq=0) == 0
    bwd = lambda g=16, dw=16, ws=16, n=1 << 20, tq=8, tk=8, dt=0: lib.rgd_relbias_bwd(bias(), g, 64, 8, dt, dw, 4, tq, tk, 0, ws, n, None)
    assert bwd(g=None) == _lib.RGD_E_NULL and bwd(dw=None) == _lib.RGD_E_NULL and bwd(n=8) == _lib.RGD_E_WORKSPACE
    assert bwd(ws=8) == _lib.RGD_E_STRIDE and bwd(dt=4) == _lib.RGD_E_DTYPE
    assert lib.rgd_relbias_bwd_workspace_bytes(1, 1 << 40, 4, 32) == _lib.RGD_E_SIZE


def _append_args(**kw):
    a = {"key": torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16), "k_cache": torch.zeros(5, 16, 4, 64, dtype=torch.bfloat16),
         "page_table": torch.zeros(2, 3, dtype=torch.int32), "lengths": torch.zeros(2, dtype=torch.int32)}
    a["value"], a["v_cache"] = a["key"], a["k_cache"].clone()
    a.update(kw)
    return a


@pytest.mark.parametrize("change", [
    {"key": torch.zeros(3, 4, 64, dtype=torch.bfloat16)}, {"value": torch.zeros(2, 3, 4, 32, dtype=torch.bfloat16)},
    {"key": torch.zeros(2, 3, 4, 64), "value": torch.zeros(2, 3, 4, 64)}, {"k_cache": torch.zeros(5, 16, 4, 64, dtype=torch.float16)},
    {"k_cache": torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16)}, {"v_cache": torch.zeros(4, 16, 4, 64, dtype=torch.bfloat16)},
    {"k_cache": torch.zeros(5, 4, 64, dtype=torch.bfloat16)}, {"k_cache": torch.zeros(5, 16, 4, 128, dtype=torch.bfloat16)[..., ::2]},
    {"k_cache": torch.zeros(1, 16, 4, 64, dtype=torch.bfloat16).expand(5, 16, 4, 64)},
    {"page_table": torch.zeros(2, 3, dtype=torch.int64)}, {"page_table": torch.zeros(1, 3, dtype=torch.int32)},
    {"lengths": torch.zeros(3, dtype=torch.int32)}, {"lengths": torch.zeros(2, dtype=torch.int64)},
    {"query": torch.zeros(2, 3, 8, 64, dtype=torch.bfloat16)},                                   # nothing to rotate it with
    {"query": torch.zeros(2, 4, 8, 64, dtype=torch.bfloat16), "pos_emb": torch.zeros(2, 9, 64)},
    {"query": torch.zeros(2, 3, 8, 64, dtype=torch.float16), "pos_emb": torch.zeros(2, 9, 64)},
    {"pos_emb": torch.zeros(2, 9, 63)}, {"pos_emb": torch.zeros(2, 9, 66)}, {"pos_emb": torch.zeros(3, 9, 64)}, {"pos_emb": torch.zeros(2, 9, 64).long()},
    {"counts": torch.zeros(3, dtype=torch.int32)}, {"counts": torch.zeros(2, dtype=torch.int64)},
    {"key": torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16, requires_grad=True)},
    {},                                                                                          # on the CPU: there is no such path
])
def test_append_refusals(change):
    args = _append_args(**change)
    before = {k: t.clone() for k, t in args.items() if k in ("k_cache", "v_cache")}
    with pytest.raises(AssertionError):
        F_.paged_cache_append_fn(**args)
    with pytest.raises(AssertionError):
        ops.PagedCacheAppend()(**args)
    assert all(torch.equal(args[k], t) for k, t in before.items())


@pytest.mark.parametrize("change", [
    {"q": torch.zeros(2, 2, 8, 64, dtype=torch.bfloat16)}, {"q": torch.zeros(2, 8, 64, dtype=torch.bfloat16)},
    {"q": torch.zeros(2, 1, 6, 64, dtype=torch.bfloat16)}, {"q": torch.zeros(2, 1, 8, 64)}, {"q": torch.zeros(2, 1, 8, 64, dtype=torch.float16)},
    {"q": torch.zeros(2, 1, 8, 136, dtype=torch.bfloat16)}, {"q": torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16, requires_grad=True)},
    {"lengths": torch.zeros(2, 1, dtype=torch.int32)}, {"page_table": torch.zeros(6, dtype=torch.int32)},
    {"rel_weight": torch.zeros(32, 4)}, {"rel_weight": torch.zeros(1, 8)}, {"rel_weight": torch.zeros(32, 8), "max_distance": 16},
    {"rel_weight": torch.zeros(31, 8), "bidirectional": True}, {"rel_weight": torch.zeros(32, 8, dtype=torch.int32)}, {"rel_weight": torch.zeros(300, 8)},
    {},
])
def test_attention_refusals(change):
    args = _append_args()
    for k in ("key", "value"):
        del args[k]
    args["q"] = torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16)
    args.update(change)
    with pytest.raises(AssertionError):
        F_.paged_attention_func(**args)


def test_position_bias_module():
    m = ops.RelativePositionBias(32, 4, max_distance=100, bidirectional=False, dtype=torch.bfloat16)
    assert list(m.state_dict()) == ["weight"] and m.weight.shape == (32, 4) and m.weight.dtype == torch.bfloat16
    assert 0 < m.weight.float().std() < 0.1
    with pytest.raises(AssertionError):
        m(4, 4)                                     # CPU weights: there is no such path
    for bad in ((31, 4), (2, 4), (600, 4), (32, 4, 8)):
        with pytest.raises(AssertionError):
            ops.RelativePositionBias(*bad)
    sig = lambda f: list(inspect.signature(f).parameters)
    assert sig(ops.RelativePositionBias.forward) == ["self", "seqlen_q", "seqlen_k", "offset", "dtype"]
    assert sig(ops.PagedAttention.forward) == ["self", "q", "k_cache", "v_cache", "page_table", "lengths", "softmax_scale", "rel_bias"]


def test_registered_operators_give_the_kernels_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from rgd_triton_b200 import library  # noqa: F401
    bf = torch.bfloat16
    with FakeTensorMode():
        w = torch.empty(32, 5, device="cuda")
        b = torch.ops.rgd_b200.relbias(w, 10, 21, True, 128, 0, bf)
        assert b.shape == (1, 5, 10, 21) and b.dtype == bf and b.stride() == (5 * 10 * 24, 10 * 24, 24, 1)
        dw = torch.ops.rgd_b200.relbias_bwd(b, 32, True, 128, 0, torch.float32)
        assert dw.shape == w.shape and dw.dtype == w.dtype
        kc = torch.empty(7, 16, 2, 64, device="cuda", dtype=bf)
        table, n = torch.empty(3, 4, device="cuda", dtype=torch.int32), torch.empty(3, device="cuda", dtype=torch.int32)
        key, q = torch.empty(3, 9, 2, 64, device="cuda", dtype=bf), torch.empty(3, 9, 8, 64, device="cuda", dtype=bf)
        pos = torch.empty(2, 64, 32, device="cuda")
        assert torch.ops.rgd_b200.paged_append(key, key, kc, kc, table, n, pos, q, None).shape == q.shape
        assert torch.ops.rgd_b200.paged_append(key, key, kc, kc, table, n, None, None, n).numel() == 0
        o, lse = torch.ops.rgd_b200.paged_attn(q[:, :1], kc, kc, table, n, None, None, False, 128)
        assert o.shape == (3, 1, 8, 64) and o.dtype == bf and lse.shape == (3, 8) and lse.dtype == torch.float32


def test_workspaces_follow_the_plan():
    """None where every unit has a CTA, a part of a 16-row tile for every warp otherwise, refusals past 32-bit schedules."""
    lib = _lib.load()
    size = lambda B, Hq, Hk, d, pages, page: lib.rgd_paged_attn_workspace_bytes(B, Hq, Hk, d, pages, page)
    assert size(1, 16, 16, 128, 19, 16) == 0 and size(16, 16, 16, 64, 28, 32) == 0
    per_warp = lambda D: 20 + 2 * 16 * (D + 2) * 4
    for args, D in (((1, 1, 1, 128, 64, 16), 128), ((64, 24, 24, 64, 1000, 16), 64), ((1, 32, 8, 96, 5000, 24), 128)):
        assert size(*args) > 0 and size(*args) % (4 * per_warp(D)) == 0
    assert size(1 << 20, 64, 64, 128, 1 << 16, 16) == _lib.RGD_E_SIZE
    assert size(4, 5, 2, 64, 4, 16) == _lib.RGD_E_INVALID and size(4, 0, 0, 64, 4, 16) == 0



def test_one_tensor_for_both_caches_is_refused():
    both = torch.zeros(5, 16, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="share memory"):
        F_.paged_cache_append_fn(**_append_args(k_cache=both, v_cache=both))


def test_c_abi_refuses_negative_gradient_strides_and_too_many_sequences():
    lib = _lib.load()
    borders = (C.c_int32 * 3)(1, 5, 9)
    bias = C.byref(_lib.RelBias(1, 4, 1, 0, 4, 0, borders))
    for sh, sq in ((-64, 8), (64, -8)):
        assert lib.rgd_relbias_bwd(bias, 16, sh, sq, 0, 16, 4, 8, 8, 0, 16, 1 << 20, None) == _lib.RGD_E_STRIDE
    h = C.byref(_lib.Heads(1, 8, 8, 8))
    cache = _paged(torch.zeros(1, 0, dtype=torch.int32))                # no page: nothing else bounds the sequences
    assert lib.rgd_paged_attn(h, C.byref(cache), None, h, None, (1 << 30) + 1, 1, 1, 64, 1.0, _lib.RGD_F16, None, 0, None) == _lib.RGD_E_SIZE
    assert lib.rgd_paged_attn_workspace_bytes((1 << 30) + 1, 1, 1, 64, 0, 16) == _lib.RGD_E_SIZE


def test_c_abi_refuses_one_cache_for_keys_and_values():
    lib = _lib.load()
    h = C.byref(_lib.Heads(16, 8, 8, 8))
    table = torch.zeros(1, 4, dtype=torch.int32)
    append = lambda cache, N=1, Hkv=2: lib.rgd_paged_append(h, h, None, None, C.byref(cache), None, None, 0, 0, 0, 0, 1, N, 0, Hkv, 64,
                                                            _lib.RGD_F16, _lib.RGD_F16, None)
    assert append(_paged(table, k=16)) == _lib.RGD_E_INVALID
    assert append(_paged(table, k=16), N=0) == 0 and append(_paged(table, k=16), Hkv=0) == 0        # nothing to write
