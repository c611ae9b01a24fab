"""Refusals of the training pass's C entry points and Python calls that need no device."""

import pytest
import torch

P = 1 << 20  # a pointer-like value, aligned; every call below is refused before anything is launched


def _refused(name, *args):
    from nki_library_b200 import _lib
    lib = _lib.load_library()
    rc = getattr(lib, name)(*args)
    return rc, lib.b200moe_last_error().decode()


@pytest.mark.parametrize("name,args,code,message", [
    ("b200moe_sort_pairs", (None, 4, 4, 2, 8, P, P, None, 0, None), -1, "null pointer"),
    ("b200moe_sort_pairs", (P, 2, 4, 2, 8, P, P, None, 0, None), -1, "4 or 8 bytes"),
    ("b200moe_sort_pairs", (P, 4, 0, 2, 8, P, P, None, 0, None), -1, "T, K > 0"),
    ("b200moe_sort_pairs", (P, 4, 1 << 30, 4, 8, P, P, None, 0, None), -1, "pairs"),
    ("b200moe_sort_pairs", (P, 4, 4, 2, 1025, P, P, None, 0, None), -1, "experts"),
    ("b200moe_sort_pairs", (P, 4, 4096, 2, 8, P, P, None, 0, None), -3, "workspace"),
    ("b200moe_sort_tokens", (P, 2, 64, P, 4, 4, 2, 64, 8, P, P, P, None, 0, None), -1, "fp32 or bf16"),
    ("b200moe_sort_tokens", (P, 1, 64, P, 3, 4, 2, 64, 8, P, P, P, None, 0, None), -1, "4 or 8 bytes"),
    ("b200moe_sort_rows", (P, 2, 64, 4, 2, 64, 8, P, P, P, None), -1, "fp32 or bf16"),
    ("b200moe_sort_rows", (P, 1, 64, 4, 2, 0, 8, P, P, P, None), -1, "H > 0"),
    ("b200moe_sort_rows", (P, 1, 64, 4, 2, 64, 0, P, P, P, None), -1, "experts"),
    ("b200moe_unsort_rows", (P, 1, -1, 4, 2, 64, P, None, 0, P, None), -1, "pitch"),
    ("b200moe_unsort_rows", (P, 1, 64, 4, 2, 64, P, P, 2, P, None), -1, "affinities"),
    ("b200moe_unsort_rows_backward", (P, 64, P, 64, 1, 4, 2, 64, 8, P, P, P, 0, None, None, None), -1, "null pointer"),
    ("b200moe_unsort_rows_backward", (P, 64, None, 64, 1, 4, 2, 64, 8, P, P, P, 0, None, P, None), -1, "needs rows"),
    ("b200moe_expert_product", (P, 64, P, 64, 4096, 0, P, 8, 2, 64, 64, P, None, 0, None, None), -1, "null pointer"),
    ("b200moe_expert_product", (P, 64, P, 64, 4096, 0, P, 0, 2, 64, 64, P, None, 0, P, None), -1, "one row"),
    ("b200moe_expert_product", (P, 64, P, 64, 4096, 0, P, 8, 1025, 64, 64, P, None, 0, P, None), -1, "experts"),
    ("b200moe_expert_product", (P, 64, P, 68, 4096, 0, P, 8, 2, 64, 68, P, None, 0, P, None), -1, "multiples of 8"),
    ("b200moe_expert_product", (P, 56, P, 64, 4096, 0, P, 8, 2, 64, 64, P, None, 0, P, None), -1, "16-byte boundaries"),
    ("b200moe_expert_product", (P, 64, P + 8, 64, 4096, 0, P, 8, 2, 64, 64, P, None, 0, P, None), -1, "16-byte boundaries"),
    ("b200moe_expert_product", (P, 64, P, 64, 4100, 0, P, 8, 2, 64, 64, P, None, 0, P, None), -1, "16-byte boundaries"),
    ("b200moe_expert_product", (P, 64, P, 64, 4096, 0, P, 8, 2, 64, 64, P + 2, None, 0, P, None), -1, "16-byte aligned"),
    ("b200moe_expert_product", (P, 8192, P, 64, 1 << 19, 0, P, 8, 2, 8192, 64, P, None, 0, P, None), -3, "workspace"),
    ("b200moe_expert_weight_grad", (P, 64, P, 64, P, 1 << 16, 2, 64, 64, P, None, 0, P, None), -3, "workspace"),
    ("b200moe_expert_weight_grad", (P, 64, None, 64, P, 8, 2, 64, 64, P, None, 0, P, None), -1, "null pointer"),
    ("b200moe_expert_weight_grad", (P, 64, P, 64, P, 8, 2, 64, 60, P, None, 0, P, None), -1, "multiples of 8"),
    ("b200moe_expert_weight_grad", (P, 64, P, 60, P, 8, 2, 64, 64, P, None, 0, P, None), -1, "16-byte boundaries"),
    ("b200moe_expert_weight_grad", (P, 64, P, 64, P, 8, 2, 64, 64, P + 8, None, 0, P, None), -1, "16-byte aligned"),
    ("b200moe_glu", (P, 64, 4, 32, 0, None, None, None, None), -1, "null pointer"),
    ("b200moe_glu", (P, 64, 4, 32, 0, P, P, None, None), -1, "null pointer"),
    ("b200moe_glu", (P, 64, 4, 28, 0, P, None, None, None), -1, "multiple of 8"),
    ("b200moe_glu", (P, 64, 4, 32, 4, P, None, None, None), -1, "activation"),
    ("b200moe_glu", (P, 32, 4, 32, 0, P, None, None, None), -1, "16-byte boundaries"),
    ("b200moe_glu", (P, 64, 4, 32, 0, P + 4, None, None, None), -1, "16-byte aligned"),
    ("b200moe_glu_backward", (None, 32, P, P, 4, 32, 0, P, None, None), -1, "null pointer"),
    ("b200moe_glu_backward", (P, 32, P, P, 4, 32, 0, None, None, None), -1, "null pointer"),
    ("b200moe_glu_backward", (P, 36, P, P, 4, 32, 0, P, None, None), -1, "16-byte boundaries"),
])
def test_entry_points_refuse(name, args, code, message):
    rc, text = _refused(name, *args)
    assert rc == code and message in text, (rc, text)


@pytest.mark.parametrize("name,args,message", [
    ("b200moe_sort_tokens", (P, 1, 8, P, 4, 4, 2, (1 << 30) + 8, 8, P, P, P, None, 0, None), "2^30 columns"),
    ("b200moe_unsort_rows", (P, 1, 8, 4, 2, (1 << 30) + 8, P, None, 0, P, None), "2^30 columns"),
    ("b200moe_sort_rows", (P + 1, 1, 8, 4, 2, 8, 8, P, P, P, None), "element's boundary"),
    ("b200moe_sort_tokens", (P, 0, 8, P, 4, 4, 2, 8, 8, P, P, P + 2, None, 0, None), "element's boundary"),
    ("b200moe_unsort_rows", (P, 1, 8, 4, 2, 8, P, None, 0, P + 1, None), "element's boundary"),
    ("b200moe_unsort_rows_backward", (P, 8, P, 8, 0, 4, 2, 8, 8, P, P, P, 0, P + 6, P, None), "element's boundary"),
    ("b200moe_expert_product", (P, 64, P, 64, 4096, 0, P, (1 << 30) + 1, 2, 64, 64, P, None, 0, P, None), "2^30"),
    ("b200moe_expert_product", (P, 1 << 28, P, 64, 1 << 35, 0, P, 8, 2, 1 << 28, 64, P, None, 0, P, None), "2^27"),
    ("b200moe_expert_product", (P, 64, P, 1 << 28, 1 << 35, 0, P, 8, 2, 64, 1 << 28, P, None, 0, P, None), "2^27"),
    ("b200moe_expert_weight_grad", (P, 64, P, 64, P, (1 << 30) + 1, 2, 64, 64, P, None, 0, P, None), "2^30"),
    ("b200moe_expert_weight_grad", (P, 1 << 28, P, 64, P, 8, 2, 1 << 28, 64, P, None, 0, P, None), "2^27"),
])
def test_sizes_and_addresses_without_an_index_are_refused(name, args, message):
    rc, text = _refused(name, *args)
    assert rc == -1 and message in text, (rc, text)


def test_cpu_tensors_are_refused():
    import nki_library_b200 as m
    x, idx = torch.zeros(4, 64), torch.zeros(4, 2, dtype=torch.int32)
    plan = m.SortedTokens(torch.zeros(9, dtype=torch.int32), idx, 8)
    w = torch.zeros(8, 64, 64, dtype=torch.bfloat16)
    for call in (lambda: m.moe_sort_plan(idx, 8), lambda: m.moe_sort_tokens(x, idx, 8),
                 lambda: m.moe_unsort_tokens(torch.zeros(8, 64), None, plan),
                 lambda: m.expert_linear(x.bfloat16(), w, plan.expert_offsets), lambda: m.moe_glu(x.bfloat16()),
                 lambda: m.moe_expert_mlp(x.bfloat16(), w, w, plan.expert_offsets),
                 lambda: m.moe_experts_train(x.bfloat16(), torch.zeros(4, 2), idx, w, w)):
        with pytest.raises(AssertionError, match="CUDA device"):
            call()


def test_workspaces():
    from nki_library_b200 import _lib
    lib = _lib.load_library()
    # few tiles of a long contraction are cut into parts, many or short ones are not
    assert lib.b200moe_expert_product_workspace_bytes(0, 8, 2, 8192, 64) % (8 * 64 * 4) == 0
    assert lib.b200moe_expert_product_workspace_bytes(0, 8, 2, 8192, 64) >= 2 * 8 * 64 * 4
    assert lib.b200moe_expert_product_workspace_bytes(1, 8, 2, 64, 8192) >= 2 * 8 * 64 * 4
    assert lib.b200moe_expert_product_workspace_bytes(0, 8, 2, 49 * 64 - 64, 64) == 0
    assert lib.b200moe_expert_product_workspace_bytes(0, 64, 1, 4096, 4096) == 0
    assert lib.b200moe_expert_product_workspace_bytes(0, 8192, 8, 4096, 28672) == 0
    assert lib.b200moe_expert_weight_grad_workspace_bytes(1 << 16, 2, 64, 64) >= 2 * 2 * 64 * 64 * 4
    assert lib.b200moe_expert_weight_grad_workspace_bytes(49 * 128 - 128, 2, 64, 64) == 0
    assert lib.b200moe_sort_workspace_bytes(1, 256) == 0
    assert lib.b200moe_sort_workspace_bytes(32768 * 8, 128) >= 128 * 4


@pytest.mark.parametrize("I", [8, 33, 64])
def test_the_tests_rounding_agrees_with_the_types(I):
    """The reference's hand-written rounding against torch's e4m3 cast."""
    import train_reference as ref
    gen = torch.Generator().manual_seed(I)
    v = torch.randn(40, I, generator=gen) * torch.exp2(torch.randint(-40, 40, (40, 1), generator=gen).float())
    v[0] = 0
    v[1, 0], v[2, 0], v[3, -1] = 448.0, 449.0, float("inf")
    e, value = ref.kept(v)
    s = torch.exp2(e.float()).repeat_interleave(32, 1)[:, :I]
    finite = v.isfinite()
    cast = (v / s).to(torch.float8_e4m3fn).float() * s
    assert torch.equal(value.float()[finite], cast[finite]) and value[~finite].isnan().all()
    assert (torch.where(finite, (v / s).abs(), 0.0) <= 448).all()


def test_native_part_is_built():
    """Loads without a device, against the same library as everything else."""
    from nki_library_b200.core.moe.moe_train.launch import native
    part = native()
    assert part.__file__.endswith("_autograd.so")
    with pytest.raises(TypeError):
        part.glu(None, 0)


def _native_calls():
    """The five operators on tensors, of the inputs that have a derivative: name -> (call, inputs)."""
    from nki_library_b200.core.moe.moe_train.launch import native
    op = native()
    rows, weight = torch.zeros((8, 64), dtype=torch.bfloat16), torch.zeros((2, 64, 64), dtype=torch.bfloat16)
    down = torch.zeros((2, 32, 64), dtype=torch.bfloat16)
    idx, off = torch.zeros((4, 2), dtype=torch.int32), torch.tensor([0, 4, 8], dtype=torch.int32)
    return {
        "sort": (lambda x: op.sort(x, idx, 2), [rows[:4]]),
        "unsort": (lambda x, a: op.unsort(x, a, idx, off), [rows, torch.zeros(4, 2)]),
        "linear": (lambda x, w: op.linear(x, w, off, False), [rows, weight]),
        "glu": (lambda x: op.glu(x, 0), [rows]),
        "mlp": (lambda x, w, v: op.mlp(x, w, v, off, 0, False), [rows, weight, down]),
    }


OPERATORS = ["sort", "unsort", "linear", "glu", "mlp"]


@pytest.mark.parametrize("op", OPERATORS)
def test_dual_tensors_are_refused(op):
    """A forward-mode tangent, on a tensor that asks for a gradient and on one that does not, of every input."""
    import torch.autograd.forward_ad as forward
    call, inputs = _native_calls()[op]
    for i, x in enumerate(inputs):
        for asks in (False, True):
            with forward.dual_level():
                dual = forward.make_dual(x.detach().requires_grad_(asks), torch.ones_like(x))
                with pytest.raises(AssertionError, match="forward-mode"):
                    call(*inputs[:i], dual, *inputs[i + 1:])


@pytest.mark.parametrize("op", OPERATORS)
def test_tracing_is_refused(op):
    """A recorded call would hold the allocation of its result and no launch, and replay memory that nothing has filled."""
    from torch.fx.experimental.proxy_tensor import make_fx
    call, inputs = _native_calls()[op]
    with pytest.raises(AssertionError, match="cannot be traced"):
        torch.jit.trace(call, tuple(inputs))
    with pytest.raises(AssertionError, match="cannot be traced"):
        make_fx(call)(*inputs)
