"""Paged cache and position bias through the native host path, the Python functions, torch.compile and autograd's corners:
the same launches, the same results."""
import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.utils.checkpoint import checkpoint

from rgd_triton_b200 import functional as F_, ops
from tests._util import gen, randn, rotary_table

pytestmark = pytest.mark.gpu


class _Declines:
    """A host path that covers nothing."""

    def __getattr__(self, name):
        return lambda *args: None


def _python(call):
    F_._bind_host(torch.empty(1, device="cuda"))
    host, F_._HOST = F_._HOST, _Declines()
    try:
        return call()
    finally:
        F_._HOST = host


class _Counts:
    """The native host path, counting what it took."""

    def __init__(self, host):
        self.host, self.taken = host, {}

    def __getattr__(self, name):
        def call(*args):
            out = getattr(self.host, name)(*args)
            self.taken[name] = self.taken.get(name, 0) + (out is not None)
            return out
        return call


def _step(dtype=torch.bfloat16, d=64, layout="tokens", bias=True):
    g = gen(d)
    B, N, Hq, Hk, page = 3, 5, 8, 2, 16
    table = torch.randperm(B * 6, generator=g).to(torch.int32).view(B, 6).cuda()
    shape = (B * 6, page, Hk, d) if layout == "tokens" else (B * 6, Hk, page, d)
    kc, vc = (randn(g, *shape, dtype=dtype).cuda() for _ in range(2))
    if layout != "tokens":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    new = [randn(g, B, N, h, d, dtype=dtype).cuda() for h in (Hk, Hk, Hq)]
    lengths = torch.tensor([0, 30, 77], dtype=torch.int32).cuda()
    counts = torch.tensor([5, 2, 0], dtype=torch.int32).cuda()
    pos = rotary_table(100, d, torch.float32).cuda()
    w = randn(g, 32, Hq).cuda() if bias else None
    return new, kc, vc, table, lengths, counts, pos, w


def _run(new, kc, vc, table, lengths, counts, pos, w):
    kc, vc = kc.clone(), vc.clone()
    q = F_.paged_cache_append_fn(new[0], new[1], kc, vc, table, lengths, pos, new[2], counts)
    o, lse = F_.paged_attention_func(q[:, :1], kc, vc, table, lengths + counts, rel_weight=w, return_lse=True)
    nothing = F_.paged_cache_append_fn(new[0], new[1], kc, vc, table, lengths)
    assert nothing is None
    return q, kc, vc, o, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,layout", [(64, "tokens"), (128, "heads"), (40, "tokens"), (17, "tokens")])
def test_native_and_python_functions_agree(dtype, d, layout):
    args = _step(dtype, d if d != 17 else 18, layout)
    want = _python(lambda: _run(*args))
    host = F_._HOST
    F_._HOST = counts = _Counts(host)
    try:
        got = _run(*args)
    finally:
        F_._HOST = host
    assert counts.taken["paged_append"] == 2 and counts.taken["paged_attn"] == 1
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("both", [True, False])
def test_native_and_python_position_bias_agree(dtype, both):
    w = randn(gen(1), 32, 5, dtype=torch.float16).cuda().requires_grad_(True)

    def call():
        out = F_.relative_position_bias_fn(w, 70, 91, both, 100, 3, dtype)
        return out, torch.autograd.grad(out, w, torch.ones_like(out) * 0.5)[0]
    want = _python(call)
    host = F_._HOST
    F_._HOST = counts = _Counts(host)
    try:
        got = call()
    finally:
        F_._HOST = host
    assert counts.taken["relbias"] == 1
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0].stride() == want[0].stride()
    assert got[0].grad_fn.name() == "RelativePositionBiasBackward"


def test_what_is_wrong_raises_through_the_native_path_too():
    (k, v, q), kc, vc, table, lengths, counts, pos, w = _step()
    before = kc.clone(), vc.clone()
    for call in (lambda: F_.paged_cache_append_fn(k, v[:, :2], kc, vc, table, lengths),
                 lambda: F_.paged_cache_append_fn(k, v, kc, vc, table.long(), lengths),
                 lambda: F_.paged_cache_append_fn(k, v, kc, vc, table.cpu(), lengths),
                 lambda: F_.paged_cache_append_fn(k, v, kc, vc, table, lengths, query=q),
                 lambda: F_.paged_cache_append_fn(k.float(), v.float(), kc, vc, table, lengths),
                 lambda: F_.paged_cache_append_fn(k.clone().requires_grad_(True), v, kc, vc, table, lengths),
                 lambda: F_.paged_attention_func(q, kc, vc, table, lengths), lambda: F_.paged_attention_func(q[:, :1, :7], kc, vc, table, lengths),
                 lambda: F_.paged_attention_func(q[:, :1], kc, vc, table, lengths, rel_weight=w[:, :4]),
                 lambda: F_.paged_attention_func(q[:, :1], kc, vc, table, lengths, rel_weight=w, max_distance=10),
                 lambda: F_.paged_attention_func(q[:, :1], kc, vc, table, lengths, rel_weight=w.cpu()),
                 lambda: F_.paged_attention_func(q[:, :1].clone().requires_grad_(True), kc, vc, table, lengths)):
        with pytest.raises(AssertionError):
            call()
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])


def test_no_derivative_is_dropped_silently():
    (k, v, q), kc, vc, table, lengths, counts, pos, w = _step()
    with fw.dual_level():
        with pytest.raises(AssertionError):
            F_.paged_attention_func(fw.make_dual(q[:, :1], torch.ones_like(q[:, :1])), kc, vc, table, lengths)
        with pytest.raises(AssertionError):
            F_.paged_cache_append_fn(fw.make_dual(k, torch.ones_like(k)), v, kc, vc, table, lengths)
    leaf = w.clone().requires_grad_(True)
    out = F_.relative_position_bias_fn(leaf, 20, 20)
    up = torch.ones_like(out).requires_grad_(True)
    with pytest.raises(RuntimeError):
        dw, = torch.autograd.grad(out, leaf, up, create_graph=True)
        torch.autograd.grad(dw.sum(), up)
    # ordinary corners of the engine: nothing upstream, two uses of one leaf, recomputation
    a, b = F_.relative_position_bias_fn(leaf, 20, 20), F_.relative_position_bias_fn(leaf, 20, 33, offset=2)
    (a.sum() + 2 * b.sum()).backward()
    assert torch.allclose(leaf.grad.sum(), torch.tensor(8 * (400 + 2 * 660.0), device="cuda"))
    again = w.clone().requires_grad_(True)
    checkpoint(lambda x: F_.relative_position_bias_fn(x, 20, 20).square().sum(), again, use_reentrant=False).backward()
    plain = w.clone().requires_grad_(True)
    F_.relative_position_bias_fn(plain, 20, 20).square().sum().backward()
    assert torch.equal(again.grad, plain.grad)


def test_caches_know_that_they_were_written():
    (k, v, q), kc, vc, table, lengths, *_ = _step()
    x = kc.clone().requires_grad_(True)
    y = (x * kc).sum()          # saves kc for x's gradient
    F_.paged_cache_append_fn(k, v, kc, vc, table, lengths)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_compiled_functions_equal_eager_ones():
    (k, v, q), kc, vc, table, lengths, counts, pos, w = _step()
    append, attend = ops.PagedCacheAppend(), ops.PagedAttention()
    rel = ops.RelativePositionBias(32, 8, bidirectional=False).cuda()

    def step(kc, vc):
        qr = append(k, v, kc, vc, table, lengths, pos, q, counts)
        append(k, v, kc, vc, table, lengths)
        return qr, attend(qr[:, :1], kc, vc, table, lengths + counts, rel_bias=rel)
    outs = []
    with torch.no_grad():
        for fn in (step, torch.compile(step, fullgraph=True, backend="aot_eager")):
            a, b = kc.clone(), vc.clone()
            outs.append((*fn(a, b), a, b))
    assert all(torch.equal(x, y) for x, y in zip(*outs))

    both = ops.RelativePositionBias(32, 3).cuda()
    qkv = [randn(gen(2), 1, 50, 3, 64, dtype=torch.bfloat16).cuda() for _ in range(3)]

    def train(q, k, v):
        return ops.FlashAttention()(q, k, v, bias=both(50, 50, dtype=torch.bfloat16))
    res = []
    for fn in (train, torch.compile(train, fullgraph=True, backend="aot_eager")):
        ins = [t.clone().requires_grad_(True) for t in qkv]
        o = fn(*ins)
        res.append([o.detach(), *torch.autograd.grad(o, [*ins, both.weight], torch.ones_like(o))])
    for x, y in zip(*res):
        assert torch.equal(x, y)


def test_compiled_autograd_traces_the_backward():
    w = randn(gen(3), 32, 4).cuda().requires_grad_(True)
    dy = randn(gen(4), 1, 4, 40, 61).cuda()
    want = torch.autograd.grad(F_.relative_position_bias_fn(w, 40, 61), w, dy)[0]
    out = F_.relative_position_bias_fn(w, 40, 61)
    with torch._dynamo.compiled_autograd._enable(torch.compile(backend="aot_eager")):
        out.backward(dy)
    assert torch.equal(w.grad, want)


def test_one_tensor_for_both_caches_is_refused_and_left_alone():
    (k, v, _), kc, _, table, lengths, *_ = _step()
    before = kc.clone()
    with pytest.raises(AssertionError, match="share memory"):
        F_.paged_cache_append_fn(k, v, kc, kc, table, lengths)
    assert torch.equal(kc, before)


def test_a_tangent_of_the_bias_weights_is_the_bias_of_the_tangent():
    """With and without a gradient beside it."""
    w, t = (randn(gen(i), 32, 5, dtype=torch.bfloat16).cuda() for i in (5, 6))
    want = F_.relative_position_bias_fn(t, 40, 61, dtype=torch.float32)
    for wants_grad in (False, True):
        for grad_mode in (False, True):
            with fw.dual_level(), torch.set_grad_enabled(grad_mode):
                leaf = w.clone().requires_grad_(wants_grad)
                out = F_.relative_position_bias_fn(fw.make_dual(leaf, t), 40, 61, dtype=torch.float32)
                value, tangent = fw.unpack_dual(out)
                assert torch.equal(value, F_.relative_position_bias_fn(w, 40, 61, dtype=torch.float32)) and torch.equal(tangent, want)
            if wants_grad and grad_mode:
                dw, = torch.autograd.grad(out, leaf, torch.ones_like(value))
                assert torch.equal(dw, torch.autograd.grad(F_.relative_position_bias_fn(leaf, 40, 61, dtype=torch.float32), leaf, torch.ones_like(value))[0])


@pytest.mark.parametrize("op", ["l2", "rms", "headln", "rope", "lnrope", "attn"])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_a_tangent_of_an_input_without_gradient_is_refused(op, grad_mode):
    x = randn(gen(7), 2, 9, 64).cuda()
    q, k = (randn(gen(i), 2, 24, 3, 64, dtype=torch.float16).cuda() for i in (8, 9))
    pos = rotary_table(64, 32, torch.float16).cuda()
    call, t = {"l2": (ops.L2Normalize(), x), "rms": (ops.FusedRMSNorm(64).cuda(), x), "headln": (lambda a: ops.FusedHeadLayerNorm()(a, k, False), q),
               "rope": (lambda a: ops.RoPE()(a, k, pos, 20, False), q), "lnrope": (lambda a: ops.FusedLNRoPE()(a, k, pos, (20, 24), False), q),
               "attn": (lambda a: ops.FlashAttention()(a, k, k), q)}[op]
    with fw.dual_level(), torch.set_grad_enabled(grad_mode):
        call(t)
        with pytest.raises(RuntimeError):
            call(fw.make_dual(t, torch.ones_like(t)))
