"""Calls of the experts' training pass that have to be refused, reported or answered at the ends of their ranges."""

import pytest
import torch

pytestmark = pytest.mark.gpu

OPERATORS = ["sort", "unsort", "linear", "glu", "mlp"]


def _operator(name):
    """A call of one input, and that input."""
    import nki_library_b200 as m
    gen = torch.Generator(device="cuda").manual_seed(4)
    T, K, E, H, I = 40, 2, 4, 64, 32
    idx = torch.randint(0, E, (T, K), device="cuda", generator=gen, dtype=torch.int32)
    hidden = torch.randn((T, H), device="cuda", generator=gen).bfloat16()
    aff = torch.rand((T, K), device="cuda", generator=gen)
    w1 = torch.randn((E, H, 2 * I), device="cuda", generator=gen).bfloat16()
    w2 = torch.randn((E, I, H), device="cuda", generator=gen).bfloat16()
    rows, plan = m.moe_sort_tokens(hidden, idx, E)
    return {
        "sort": (lambda x: m.moe_sort_tokens(x, idx, E)[0], hidden),
        "unsort": (lambda x: m.moe_unsort_tokens(x, aff, plan), rows),
        "linear": (lambda x: m.expert_linear(x, w1, plan.expert_offsets), rows),
        "glu": (m.moe_glu, rows),
        "mlp": (lambda x: m.moe_expert_mlp(x, w1, w2, plan.expert_offsets), rows),
    }[name]


@pytest.mark.parametrize("op", OPERATORS)
def test_forward_mode_is_refused(op):
    """In the operator and, forward over reverse, in its backward pass."""
    import torch.autograd.forward_ad as forward
    call, x = _operator(op)
    leaf = x.clone().requires_grad_()
    out = call(leaf)
    with forward.dual_level():
        with pytest.raises(AssertionError, match="forward-mode"):
            call(forward.make_dual(x, torch.ones_like(x)))
        with pytest.raises(AssertionError, match="forward-mode"):
            torch.autograd.grad(out, leaf, forward.make_dual(torch.ones_like(out), torch.ones_like(out)), retain_graph=True)
    with pytest.raises(Exception):
        torch.func.jvp(call, (x,), (torch.ones_like(x),))
    assert torch.autograd.grad(out, leaf, torch.ones_like(out))[0].shape == x.shape


@pytest.mark.parametrize("op", OPERATORS)
def test_tracing_is_refused(op):
    """In the operator and in its backward pass; outside, both go on as before."""
    from torch.fx.experimental.proxy_tensor import make_fx
    call, x = _operator(op)
    leaf = x.clone().requires_grad_()
    out = call(leaf)
    for trace in (lambda f, y: torch.jit.trace(f, y), lambda f, y: make_fx(f)(y)):
        with pytest.raises(AssertionError, match="cannot be traced"):
            trace(lambda y: call(y), x)
    with pytest.raises(AssertionError, match="cannot be traced"):
        make_fx(lambda d: torch.autograd.grad(out, leaf, d, retain_graph=True)[0])(torch.ones_like(out))
    assert torch.equal(call(x), out) and torch.autograd.grad(out, leaf, torch.ones_like(out))[0].shape == x.shape
