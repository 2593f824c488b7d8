"""Learned relative position bias against its 64-bit form: values, gradients, refusals, and a run through the attention."""
import pytest
import torch

from rgd_triton_b200 import _lib, functional as F_, ops
from tests import _plain as P
from tests._util import DTYPES, assert_attn, gen, randn

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 1), (2, 1, 300), (3, 300, 1), (12, 197, 333), (5, 64, 64), (2, 65, 129), (1, 513, 4099), (2, 1030, 260), (3, 7, 8), (16, 130, 128)]


def _weight(g, buckets, H, dtype):
    return randn(g, buckets, H, dtype=dtype)


@pytest.mark.parametrize("H,tq,tk", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16"), ("f16", "bf16"), ("bf16", "bf16")])
def test_values_and_gradient(H, tq, tk, dtype, wdtype):
    g = gen(tq + tk)
    for buckets, both, most, offset in ((32, True, 128, 0), (32, False, 128, 5), (6, True, 20, -3), (2, False, 40, 0)):
        w = _weight(g, buckets, H, DTYPES[wdtype])
        wd = w.cuda().requires_grad_(True)
        out = F_.relative_position_bias_fn(wd, tq, tk, both, most, offset, DTYPES[dtype])
        want, which = P.relbias(w, tq, tk, both, most, offset)
        assert out.shape == (1, H, tq, tk) and out.dtype == DTYPES[dtype]
        assert torch.equal(out.detach().cpu(), want.to(DTYPES[dtype]))      # a copy, rounded once
        assert out.stride(2) % 8 == 0 and out.data_ptr() % 16 == 0
        dy = randn(g, 1, H, tq, tk, dtype=DTYPES[dtype])
        dw, = torch.autograd.grad(out, wd, dy.cuda())
        assert dw.dtype == w.dtype and dw.shape == w.shape
        terms = int(torch.bincount(which.flatten(), minlength=buckets).max())
        P.assert_grad(dw, P.relbias_grad(dy, which, buckets), P.relbias_grad(dy.abs(), which, buckets), terms, "dweight")
    assert _lib.load().rgd_device_status() == 0


@pytest.mark.parametrize("make", ["expanded", "heads_last", "offset", "rows_apart", "channel_stride"])
def test_gradients_of_any_layout(make):
    H, tq, tk = 4, 70, 133
    g = gen(3)
    if make == "expanded":
        dy = randn(g, 1, 1, 1, 1).cuda().expand(1, H, tq, tk)
    elif make == "heads_last":
        dy = randn(g, 1, tq, H, tk).cuda().transpose(1, 2)
    elif make == "offset":
        dy = randn(g, H * tq * tk + 1).cuda()[1:].view(1, H, tq, tk)
    elif make == "rows_apart":
        dy = randn(g, 1, H, tq, tk + 11).cuda()[..., 3:3 + tk]
    else:
        dy = randn(g, 1, H, tk, tq).cuda().transpose(2, 3)
    w = _weight(g, 32, H, torch.float32).cuda().requires_grad_(True)
    dw, = torch.autograd.grad(F_.relative_position_bias_fn(w, tq, tk), w, dy)
    _, which = P.relbias(w.detach().cpu(), tq, tk, True, 128, 0)
    dyc = dy.cpu()
    P.assert_grad(dw, P.relbias_grad(dyc, which, 32), P.relbias_grad(dyc.abs(), which, 32), tq * tk, make)


def test_gradient_is_the_same_every_time_and_matches_differences():
    g = gen(4)
    w = _weight(g, 32, 6, torch.float32).cuda().requires_grad_(True)
    dy = randn(g, 1, 6, 500, 700).cuda()
    first = torch.autograd.grad(F_.relative_position_bias_fn(w, 500, 700), w, dy)[0]
    for _ in range(3):
        assert torch.equal(first, torch.autograd.grad(F_.relative_position_bias_fn(w, 500, 700), w, dy)[0])
    # the bias is linear in w, so a difference is exact but for rounding: dy . bias(direction) = dw . direction
    direction = randn(g, 32, 6).cuda()
    left = (dy.double() * F_.relative_position_bias_fn(direction, 500, 700).double()).sum()
    right = (first.double() * direction.double()).sum()
    size = (dy.double() * F_.relative_position_bias_fn(direction, 500, 700).double()).abs().sum()
    assert (left - right).abs() <= (1 << 10) * 2.0 ** -24 * size


def test_strided_weight_values_far_apart_and_empty_sizes():
    g = gen(5)
    wide = randn(g, 64, 10).cuda()
    for w in (wide[::2, 1:5], wide.t()[:8, :8].t(), wide[:32, :1].expand(32, 4)):
        want, _ = P.relbias(w.cpu(), 90, 90, True, 128, 0)
        assert torch.equal(F_.relative_position_bias_fn(w, 90, 90).cpu(), want.float())
    w = torch.tensor([[-torch.inf], [torch.finfo(torch.float32).min], [torch.nan], [1.0]]).cuda()
    out = F_.relative_position_bias_fn(w, 9, 9, False, 16).cpu()
    want, _ = P.relbias(w.cpu(), 9, 9, False, 16, 0)
    assert torch.equal(out.nan_to_num(nan=7.0), want.float().nan_to_num(nan=7.0))
    for tq, tk in ((0, 5), (5, 0), (0, 0)):
        v = wide[:32].clone().requires_grad_(True)
        out = F_.relative_position_bias_fn(v, tq, tk)
        assert out.shape == (1, 10, tq, tk)
        dw, = torch.autograd.grad(out, v, torch.zeros_like(out))
        assert torch.equal(dw, torch.zeros_like(v))
    far = F_.relative_position_bias_fn(wide[:32], 3, 3, True, 128, 1 << 29)
    assert torch.equal(far[0, :, 0, 0], wide[15])          # every key lies far before the queries


def test_large_matrix_offsets_past_32_bits():
    """2^31 elements and more: rows at the end against the same rows of a short matrix."""
    H, tq, tk = 9, 16384, 16384
    w = randn(gen(6), 32, H, dtype=torch.bfloat16).cuda()
    out = F_.relative_position_bias_fn(w, tq, tk)
    assert out.numel() > 1 << 31
    part = F_.relative_position_bias_fn(w, 200, tk, offset=tq - 200)
    assert torch.equal(out[:, :, -200:], part)
    leaf = w.clone().requires_grad_(True)
    counts, = torch.autograd.grad(F_.relative_position_bias_fn(leaf, tq, tk, dtype=torch.float32), leaf,
                                  torch.ones(1, device="cuda").expand(1, H, tq, tk))
    which = P.bucket_row(range(1 - tq, tk), 32, True, 128)
    many = tq - (torch.arange(1 - tq, tk)).abs()
    want = torch.zeros(32, dtype=torch.int64).index_add_(0, which, many)
    assert torch.equal(counts.cpu(), want.to(torch.bfloat16)[:, None].expand(32, H))      # whole numbers, rounded once
    del out, counts
    torch.cuda.empty_cache()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("tq,tk", [(257, 257), (96, 200)])
def test_through_the_attention(causal, tq, tk):
    """The module's bias in FlashAttention: output, and the gradient that reaches the weights, in 64 bits."""
    from oracle import oracle as O
    g = gen(7)
    B, H, d = 2, 3, 64
    m = ops.RelativePositionBias(32, H, bidirectional=not causal).cuda()
    q, k, v, do = (randn(g, B, t, H, d, dtype=torch.bfloat16) for t in (tq, tk, tk, tq))
    ins = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    bias = m(tq, tk, dtype=torch.bfloat16)
    o = ops.FlashAttention()(*ins, bias=bias, causal=causal)
    grads = torch.autograd.grad(o, [*ins, m.weight], do.cuda())
    w = m.weight.detach().cpu()
    full, which = P.relbias(w, tq, tk, not causal, 128, 0)

    def ref(t):
        b = full.to(torch.bfloat16).to(t).requires_grad_(True)
        qq, kk, vv = (x.to(t).requires_grad_(True) for x in (q, k, v))
        s = torch.einsum("bqhd,bkhd->bhqk", qq, kk) * d ** -0.5 + b
        if causal:
            s = s.masked_fill(torch.arange(tk)[None, :] > torch.arange(tq)[:, None], -torch.inf)
        out = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s, -1), vv)
        return out, torch.autograd.grad(out, [qq, kk, vv, b], do.to(t))
    exact, egrads = ref(torch.float64)
    low, lgrads = ref(torch.bfloat16)
    assert_attn(o, exact, low, "o", floor=5e-4)
    for a, b, c, what in zip(grads[:3], egrads, lgrads, ("dq", "dk", "dv")):
        assert_attn(a, b, c, what, factor=3.0, floor=2e-3)
    # dweight sums the bf16 gradients of each batch's bias (half a step each) and their sum (another), in fp32
    want = P.relbias_grad(egrads[3], which, 32)
    size = P.relbias_grad(egrads[3].abs(), which, 32)
    spread = (lgrads[3].double() - egrads[3]).abs()
    slack = 4 * P.relbias_grad(spread, which, 32) + 2.0 ** -7 * size + 1e-3
    assert ((grads[3].cpu().double() - want).abs() <= slack).all()


def test_graph_capture_streams_and_eager_graph_alive():
    """Forward and backward replayed from a captured graph on new weights, while an eager graph of the same leaf lives."""
    g = gen(8)
    w = randn(g, 32, 4).cuda().requires_grad_(True)
    dy = randn(g, 1, 4, 100, 100).cuda()
    call = lambda x: torch.autograd.grad(F_.relative_position_bias_fn(x, 100, 100), x, dy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            call(w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    static = w.detach().clone()
    with torch.cuda.graph(graph):
        leaf = static.detach().requires_grad_(True)
        out = F_.relative_position_bias_fn(leaf, 100, 100)
        dw, = torch.autograd.grad(out, leaf, dy)
    new = randn(g, 32, 4).cuda()
    static.copy_(new)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, F_.relative_position_bias_fn(new, 100, 100)) and torch.equal(dw, call(w))


def test_refusals_on_the_gpu():
    w = torch.zeros(32, 4, device="cuda")
    bad = [lambda: F_.relative_position_bias_fn(w[0], 4, 4), lambda: F_.relative_position_bias_fn(w[:31], 4, 4, True),
           lambda: F_.relative_position_bias_fn(w, 4, 4, True, 8), lambda: F_.relative_position_bias_fn(w, -1, 4),
           lambda: F_.relative_position_bias_fn(w.long(), 4, 4), lambda: F_.relative_position_bias_fn(w, 4, 4, dtype=torch.int32),
           lambda: F_.relative_position_bias_fn(w, 4, 4, offset=1 << 30)]
    for call in bad:
        with pytest.raises(AssertionError):
            call()
    assert F_.relative_position_bias_fn(w, 4, 4).shape == (1, 4, 4, 4)
