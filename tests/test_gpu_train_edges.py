"""Calls of the experts' training pass that have to be refused, reported or answered at the ends of their ranges."""

import contextlib

import math

import pytest
import torch

import train_reference as ref

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


def test_the_most_tokens():
    """2^31 - 1 tokens of one column: sorted, summed and back through both gradients."""
    import nki_library_b200 as m
    T = 2 ** 31 - 1
    hidden = torch.ones((1, 1), dtype=torch.bfloat16, device="cuda").expand(T, 1).contiguous()
    hidden[-1] = 2
    idx = torch.zeros((T, 1), dtype=torch.int32, device="cuda")
    idx[0], idx[-2] = -1, 1
    rows, plan = m.moe_sort_tokens(hidden, idx, 2)
    assert plan.expert_offsets.tolist() == [0, T - 2, T - 1]
    row = plan.row_of_pair.view(-1)
    ends = {0: -1, 1: 0, T // 2: T // 2 - 1, T - 3: T - 4, T - 2: T - 2, T - 1: T - 3}  # token: its row
    assert [int(row[t]) for t in ends] == list(ends.values())
    step = 1 << 28
    for lo in range(1, T - 2, step):
        hi = min(lo + step, T - 2)
        assert torch.equal(row[lo:hi], torch.arange(lo - 1, hi - 1, dtype=torch.int32, device="cuda"))
    assert rows[T - 3] == 2 and rows[T - 1] == 0 and int((rows == 1).sum()) == T - 2
    del idx
    rows.requires_grad_()
    out = m.moe_unsort_tokens(rows, None, plan)
    assert out[0] == 0 and out[-1] == 2 and int((out == 1).sum()) == T - 2
    d_rows, = torch.autograd.grad(out, rows, hidden)
    assert d_rows[T - 3] == 2 and d_rows[T - 1] == 0 and int((d_rows == 1).sum()) == T - 2


def test_the_widest_rows():
    """2^30 columns of bf16, 4 bytes off a 16-byte boundary: copied as fp32 rows of half the width."""
    from nki_library_b200 import _lib
    H = 2 ** 30
    flat = torch.arange(2 ** 15, dtype=torch.int32, device="cuda").to(torch.int16).repeat(H // 2 ** 15 + 1).view(torch.bfloat16)
    hidden, out = flat[2:2 + H], torch.zeros(H + 8, dtype=torch.bfloat16, device="cuda")
    idx = torch.zeros(1, dtype=torch.int32, device="cuda")
    offsets, row = torch.empty(2, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    _lib.call("b200moe_sort_tokens", hidden.data_ptr(), _lib.BF16, H, idx.data_ptr(), 4, 1, 1, H, 1, offsets.data_ptr(), row.data_ptr(),
              out[2:].data_ptr(), None, 0, _lib.stream_ptr())
    assert torch.equal(out[2:2 + H].view(torch.int16), hidden.view(torch.int16)) and not out[:2].any() and not out[2 + H:].any()
    assert offsets.tolist() == [0, 1] and row.tolist() == [0]


# ------------------------------------------------------------------ waits that run out
@contextlib.contextmanager
def _wait_cycles(cycles):
    """Products launched inside give up a wait after `cycles` clocks; below zero at the first look that finds it unfinished."""
    from nki_library_b200 import _lib
    lib = _lib.load_library()
    before = lib.b200moe_expert_wait_cycles(cycles)
    try:
        yield
    finally:
        assert lib.b200moe_expert_wait_cycles(before) == cycles


class _Product:
    """A product or a weight gradient through the C entry points."""

    def __init__(self, counts, K, N, weight_grad=False, behind=0):
        gen = torch.Generator(device="cuda").manual_seed(K + N)
        self.E, self.R, self.K, self.N, self.weight_grad = len(counts), sum(counts) + behind, K, N, weight_grad
        self.offsets = torch.tensor([0] + counts).cumsum(0).int().cuda()

        def small(*shape):
            return torch.randint(-2, 3, shape, device="cuda", generator=gen, dtype=torch.int8).bfloat16()

        self.x, self.w = small(self.R, K), small(self.R, N) if weight_grad else small(self.E, K, N)

    def run(self):
        """(output, status)"""
        from nki_library_b200 import _lib
        lib = _lib.load_library()
        E, R, K, N = self.E, self.R, self.K, self.N
        out = torch.zeros((E, K, N) if self.weight_grad else (R, N), dtype=torch.bfloat16, device="cuda")
        status = torch.full((2,), -1, dtype=torch.int32, device="cuda")
        if self.weight_grad:
            size = lib.b200moe_expert_weight_grad_workspace_bytes(R, E, K, N)
            ws = torch.empty(size, dtype=torch.uint8, device="cuda")
            _lib.call("b200moe_expert_weight_grad", self.x.data_ptr(), K, self.w.data_ptr(), N, self.offsets.data_ptr(), R, E, K, N,
                      out.data_ptr(), ws.data_ptr(), size, status.data_ptr(), _lib.stream_ptr())
        else:
            size = lib.b200moe_expert_product_workspace_bytes(0, R, E, K, N)
            ws = torch.empty(size, dtype=torch.uint8, device="cuda")
            _lib.call("b200moe_expert_product", self.x.data_ptr(), K, self.w.data_ptr(), N, K * N, 0, self.offsets.data_ptr(), R, E, K, N,
                      out.data_ptr(), ws.data_ptr(), size, status.data_ptr(), _lib.stream_ptr())
        torch.cuda.synchronize()
        return out, int(status[0])


# Contractions of 1024 slabs and more in one tile each, which an accumulator's readers wait for longer than one look lasts (20 us): one
# tile per pair, tiles handed out, a weight gradient with ragged ends, parts of a contraction, parts of a weight gradient.
LONG = [([3] * 40, 65536, 8, False, 0), ([8192], 65536, 8192, False, 3), ([70001] + [1] * 39, 8, 8, True, 0), ([5, 2], 2 ** 21, 16, False, 1),
        ([2 ** 21 + 5], 8, 16, True, 0)]


# Contractions that take far longer than 400000 clocks (0.2 ms): one tile per pair; tiles handed out; a weight gradient; one whose
# ragged ends are asked for behind tiles that have none.
LONGER = [([3] * 40, 2 ** 19, 8, False, 0), ([8192], 2 ** 17, 2560, False, 3), ([2 ** 20 + 1] + [1] * 39, 8, 8, True, 0),
          ([2 ** 18, 17], 2304, 2304, True, 0)]


@pytest.mark.parametrize("case", range(len(LONGER)))
def test_a_wait_lasts_as_long_as_the_contraction_moves_on(case):
    """The limit is on a standstill: a contraction of 2^30 rows takes longer than any limit, and is right all the same."""
    job = _Product(*LONGER[case])
    want, status = job.run()
    assert status == 0
    with _wait_cycles(400000):
        got, status = job.run()
    assert status == 0 and torch.equal(got, want)


@pytest.mark.parametrize("case", range(len(LONG)))
def test_a_wait_that_runs_out_is_reported(case):
    """The launch gives up, says so and leaves everything usable."""
    job = _Product(*LONG[case])
    want, status = job.run()
    assert status == 0 and want.any()
    with _wait_cycles(-1):
        for _ in range(3):
            got, status = job.run()
            assert 41 <= status <= 49
            # nothing is taken for a result that is none
            assert got.isnan().any() and (got.isnan() | (got == want)).all()
    again, status = job.run()
    assert status == 0 and torch.equal(again, want)


def _long_layer():
    import nki_library_b200 as m
    gen = torch.Generator(device="cuda").manual_seed(8)
    E, R, H, I = 40, 120, 65536, 8
    offsets = (torch.arange(E + 1, device="cuda") * (R // E)).int()
    idx = (torch.arange(R, device="cuda") // (R // E)).int()[:, None]
    rows = torch.randn((R, H), device="cuda", generator=gen).bfloat16().requires_grad_()
    w1 = (torch.randn((E, H, 2 * I), device="cuda", generator=gen) * 0.01).bfloat16().requires_grad_()
    w2 = torch.randn((E, I, H), device="cuda", generator=gen).bfloat16().requires_grad_()
    ones = torch.ones((R, 1), device="cuda")
    return {
        "linear": (lambda check: m.expert_linear(rows, w1, offsets, _check_status=check), (rows, w1)),
        "mlp": (lambda check: m.moe_expert_mlp(rows, w1, w2, offsets, _check_status=check), (rows, w1, w2)),
        "layer": (lambda check: m.moe_experts_train(rows, ones, idx, w1, w2, _check_status=check), (rows, w1, w2)),
    }


@pytest.mark.parametrize("call", ["linear", "mlp", "layer"])
def test_a_wait_that_runs_out_raises_or_leaves_nan(call):
    """Asked for, in the forward pass and in the backward pass; else the results are NaN where nothing was written."""
    fn, leaves = _long_layer()[call]
    want = fn(False)
    d = torch.ones_like(want)
    for check in (False, True):
        out = fn(check)
        assert torch.equal(out, want)
        grads = torch.autograd.grad(out, leaves, d, retain_graph=True)
        if call == "linear":  # what has a long contraction here is the forward product; a layer's backward pass has one, too
            continue
        with _wait_cycles(-1):
            if check:
                with pytest.raises(AssertionError, match="wait expired"):
                    torch.autograd.grad(out, leaves, d)
            else:
                got = torch.autograd.grad(out, leaves, d)
                assert got[0].isnan().any() and got[1].isnan().any()
                assert all(g.shape == w.shape for g, w in zip(got, grads))
    with _wait_cycles(-1):
        with pytest.raises(AssertionError, match="wait expired"):
            fn(True)
        with torch.no_grad(), pytest.raises(AssertionError, match="wait expired"):
            fn(True)
        assert fn(False).isnan().any()
    assert torch.equal(fn(True), want)


def test_a_gradient_whose_wait_runs_out_raises():
    """Of the weights: 65537 rows of one expert."""
    import nki_library_b200 as m
    R, E = 65537 + 39, 40
    offsets = torch.tensor([0] + [65537 + e for e in range(E)], dtype=torch.int32, device="cuda")
    x = torch.ones((R, 8), dtype=torch.bfloat16, device="cuda")
    w = torch.ones((E, 8, 8), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    out = m.expert_linear(x, w, offsets, _check_status=True)
    with _wait_cycles(-1), pytest.raises(AssertionError, match="wait expired"):
        torch.autograd.grad(out, w, torch.ones_like(out), retain_graph=True)
    dw, = torch.autograd.grad(out, w, torch.ones_like(out))
    assert (dw[0] == 65536).all() and (dw[1:] == 1).all()  # 65537 rounded to bf16


OWN_CONTEXT = """
import ctypes, sys
import numpy as np
from nki_library_b200 import _lib
cuda = ctypes.CDLL("libcuda.so.1")
def ok(rc): assert rc == 0, rc
context, now = ctypes.c_void_p(), ctypes.c_void_p()
ok(cuda.cuInit(0))
ok(cuda.cuCtxCreate_v2(ctypes.byref(context), 0, 0))
def device(array):
    p = ctypes.c_uint64()
    ok(cuda.cuMemAlloc_v2(ctypes.byref(p), ctypes.c_size_t(array.nbytes)))
    ok(cuda.cuMemcpyHtoD_v2(p, ctypes.c_void_p(array.ctypes.data), ctypes.c_size_t(array.nbytes)))
    return p.value
one = 0x3f80  # bf16 1
x, w = (device(np.full(n, one, np.uint16)) for n in (64 * 128, 128 * 64))
out, status = device(np.zeros(64 * 64, np.uint16)), device(np.full(2, -1, np.int32))
offsets = device(np.array([0, 60], np.int32))
lib = _lib.load_library()
rc = lib.b200moe_expert_product(x, 128, w, 64, 128 * 64, 0, offsets, 64, 1, 128, 64, out, None, 0, status, None)
assert rc == 0, lib.b200moe_last_error()
ok(cuda.cuCtxGetCurrent(ctypes.byref(now)))
assert now.value == context.value
ok(cuda.cuCtxSynchronize())
got = np.empty(64 * 64, np.uint16)
ok(cuda.cuMemcpyDtoH_v2(ctypes.c_void_p(got.ctypes.data), ctypes.c_uint64(out), ctypes.c_size_t(got.nbytes)))
assert (got.reshape(64, 64)[:60] == 0x4300).all() and not got.reshape(64, 64)[60:].any()  # 128
"""


def test_a_context_of_the_callers_own_stays_current():
    """A C host with a context of the driver API: the first call of a thread makes a context current only where there is none."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", OWN_CONTEXT], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


# ------------------------------------------------------------------ products of whole numbers
MANY = [(7 * e) % 23 for e in range(300)]
EXACT = [
    # counts, K, N, rows behind the last expert
    ([40001], 136, 8, 0), ([40001], 8, 136, 3), ([9000, 70, 0, 5003], 64, 72, 2), ([2 ** 20 + 17], 16, 8, 0),  # a weight gradient in parts
    ([5, 0, 9], 4096, 72, 3), ([300], 8200, 520, 0), ([1], 2048, 8, 0), ([40, 700, 3], 64, 12000, 5),  # a product in parts
    ([12000, 0, 3000, 1, 5199], 72, 14008, 40), ([12000, 0, 3000, 1, 5199], 1032, 13000, 0),  # tiles handed out
    ([0, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, 255, 256, 257, 0], 328, 120, 300), ([700, 5, 1030], 1000, 776, 1), (MANY, 136, 304, 5),
]


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("case", range(len(EXACT)))
def test_products_of_whole_numbers_are_exact(case, transposed):
    """Operands of -1 and 1: every partial sum is a whole number below 2^24, exact in fp32 in any order, so a result is the exact sum
    rounded once.  A row or a step of the contraction that is missing or counted twice changes every sum by one, which shows in the
    sums up to 256, whole numbers of bf16; the sums of n terms are of size sqrt(n)."""
    import nki_library_b200 as m
    counts, K, N, behind = EXACT[case]
    gen = torch.Generator(device="cuda").manual_seed(case)

    def signs(*shape):
        return (torch.randint(0, 2, shape, device="cuda", generator=gen, dtype=torch.int8) * 2 - 1).bfloat16()

    E, used = len(counts), sum(counts)
    offsets = torch.tensor([0] + counts).cumsum(0).int().cuda()
    x, dy = signs(used + behind, K), signs(used + behind, N)
    w = signs(E, N, K).transpose(1, 2) if transposed else signs(E, K, N)
    x[used:], dy[used:] = math.nan, math.inf
    x.requires_grad_(), w.requires_grad_()
    y = m.expert_linear(x, w, offsets, _check_status=True)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    y, x, w = y.detach(), x.detach(), w.detach()
    at = 0
    for e, n in enumerate(counts):
        part = slice(at, at + n)
        at += n
        xe, we, de = x[part].double(), w[e].double(), dy[part].double()
        for got, want in ((y[part], xe @ we), (dx[part], de @ we.t()), (dw[e], xe.t() @ de)):
            assert torch.equal(got, want.bfloat16()), e
            if n * want.numel() > 0:
                assert (want.abs() <= 256).any()
    assert not y[at:].any() and not dx[at:].any()


# ------------------------------------------------------------------ gradients of the activation far out
FAR = [1e-30, 1e-3, 0.3, 1.0, 1.25, 2.0, 3.0, 4.0, 5.0, 6.0, 7.0, 8.0, 9.0, 10.0, 11.0, 12.0, 13.0, 14.0, 20.0, 40.0, 52.0, 60.0, 87.0, 90.0,
       100.0, 300.0, 1e4, 1e10, 1e20, 1e30, 3e38, 3.38e38]


@pytest.mark.parametrize("act", ["SiLU", "GELU", "GELU_Tanh_Approx", "Swish"])
def test_gradient_of_far_gates(act):
    """A row for each magnitude, so that its gates are kept at their size: both gradients of every column against the formula at the
    kept values.

    Bounds.  The kernel's exponentials have arguments of up to 127 powers of two, rounded up to five times to 2^-24: 127 * 5 * 2^-24 *
    ln 2 = 2^-15.2, the approximations and products that follow add 2^-20 at most, GELU's fit 1.2e-6: 2^-15 of each of the slope's two
    terms.  Where sigma is near one, 1 - sigma is off by 2^-22 and becomes zero from 24 powers of two on; times |g z'|, at most 35
    there (the tanh form at 5): 2^-16.  What is flushed: sigma below 2^-126, times |g| <= 87.4 and |g z'| <= 232 (the tanh form at
    -10.1): 2.8e-36 of the slope and 1.03e-36 of the activation."""
    import nki_library_b200 as m
    I = 32
    base = torch.tensor([s * v for v in FAR for s in (-1, 1)], dtype=torch.float64)
    gates = base[:, None] * (1 - torch.arange(I) / (2.0 * I))
    gen = torch.Generator().manual_seed(2)
    ups = torch.randint(0, 2, gates.shape, generator=gen) * 2 - 1
    x = torch.cat([gates, ups], 1).bfloat16().cuda().requires_grad_()
    d = ((torch.randint(0, 2, gates.shape, generator=gen) * 2 - 1) * 0.5).bfloat16().cuda()
    grad, = torch.autograd.grad(m.moe_glu(x, m.ActFnType[act]), x, d)
    _, g = ref.kept(x.detach()[:, :I])
    _, u = ref.kept(x.detach()[:, I:])
    assert torch.equal(u, x.detach()[:, I:].double()) and ((g.abs() / x.detach()[:, :I].double().abs() - 1).abs() <= 2.0 ** -4).all()
    value, slope = ref.act_and_slope(g, act)
    cdf = value / g  # sigma, or GELU's distribution function: the slope's first term
    terms = cdf + (slope - cdf).abs()
    want = torch.cat([d.double() * u * slope, d.double() * value], 1)
    assert want.isfinite().all()
    half = want.abs() * 2.0 ** -8 * (1 + 2.0 ** -8)
    slack = torch.cat([terms * 2.0 ** -15 + (g > 0) * 2.0 ** -16 + 2.8e-36, value.abs() * 2.0 ** -15 + 1.03e-36], 1) * 0.5
    off = (grad.double() - want).abs()
    assert grad.isfinite().all()
    worst = ((off - half - slack) / slack).amax(1)
    assert (off <= half + slack).all(), [(float(base[i]), float(worst[i])) for i in (worst > 0).nonzero()[:, 0]]
