"""Forward-mode derivatives without a GPU: the launches replaced by a stub, what autograd makes of the calls."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from rgd_triton_b200 import functional as F_


def _bias(weight, seqlen_q, seqlen_k, bidirectional, max_distance, offset, dtype):
    """Linear in weight, with the layout of the launch's result; like a launch it sees values alone."""
    weight = fw.unpack_dual(weight).primal.detach()
    out = F_._bias_rows(seqlen_q, seqlen_k, weight.shape[1], dtype, weight.device)
    out.copy_(weight.sum(0)[None, :, None, None].expand(out.shape))
    return out


@pytest.mark.parametrize("wants_grad", [False, True])
@pytest.mark.parametrize("grad_mode", [False, True])
@pytest.mark.parametrize("dtype", [None, torch.float16])
def test_a_tangent_of_the_bias_weights_is_carried_on(monkeypatch, wants_grad, grad_mode, dtype):
    monkeypatch.setattr(F_, "_relbias_forward", _bias)
    monkeypatch.setattr(F_, "_HOST", None)
    w, t = torch.randn(8, 3), torch.randn(8, 3)
    with fw.dual_level(), torch.set_grad_enabled(grad_mode):
        out = F_.relative_position_bias_fn(fw.make_dual(w.clone().requires_grad_(wants_grad), t), 5, 9, dtype=dtype)
        value, tangent = fw.unpack_dual(out)
        assert out.requires_grad == (wants_grad and grad_mode)
        want = lambda x: _bias(x, 5, 9, True, 128, 0, dtype or x.dtype)
        assert torch.equal(value, want(w)) and torch.equal(tangent, want(t)) and tangent.dtype == value.dtype
        assert fw.unpack_dual(F_.relative_position_bias_fn(w, 5, 9)).tangent is None


def _value(x):
    return fw.unpack_dual(x).primal.detach().clone()


def _rows(xs, *args):
    return [_value(x) for x in xs], [_value(x) for x in xs]


CALLS = {
    "l2": (lambda x: F_.triton_norm_func_fn(x), "_l2_forward", _rows),
    "headln": (lambda x: F_.triton_fused_ln_func_fn(x, x.clone(), heads_second=False), "_ln_forward",
               lambda q, k, *args: (q, k, _value(q), _value(k))),
}


@pytest.mark.parametrize("grad_mode", [False, True])
@pytest.mark.parametrize("name", list(CALLS))
def test_a_tangent_is_refused_where_there_is_no_rule(monkeypatch, name, grad_mode):
    """Also of an input that wants no gradient."""
    call, launch, stub = CALLS[name]
    monkeypatch.setattr(F_, launch, stub)
    monkeypatch.setattr(F_, "_HOST", None)
    x = torch.randn(2, 5, 3, 8)
    call(x)
    with fw.dual_level(), torch.set_grad_enabled(grad_mode):
        call(x)
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(fw.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("op", ["append", "attention"])
def test_the_paged_operators_refuse_a_tangent(op):
    bf = torch.bfloat16
    x, cache = torch.zeros(2, 1, 4, 64, dtype=bf), [torch.zeros(5, 16, 4, 64, dtype=bf) for _ in range(2)]
    table, lengths = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with fw.dual_level(), torch.no_grad():
        dual = fw.make_dual(x, torch.ones_like(x))
        with pytest.raises(AssertionError, match="forward-mode"):
            if op == "append":
                F_.paged_cache_append_fn(dual, x, *cache, table, lengths)
            else:
                F_.paged_attention_func(dual, *cache, table, lengths)
