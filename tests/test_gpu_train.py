"""The experts' training pass on the GPU against plain 64-bit forms.

Tolerances.  A result rounded to bf16 (fp32) is off by at most 2^-8 (2^-24) of itself, and an fp32 sum of n terms by at most
n 2^-23 of the sum of their magnitudes (each addition rounds or truncates a partial sum that is no larger).
"""

import pytest
import torch

import train_reference as ref

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _close(got, want, magnitude, terms, extra=0.0):
    """|got - want| <= half a step of want + terms 2^-23 of the terms' magnitudes."""
    bound = want.abs() * HALF[got.dtype] * (1 + 2.0 ** -8) + magnitude * (terms * 2.0 ** -23) + extra + 1e-37
    off = (got.double() - want).abs()
    assert got.isfinite().all() and (off <= bound).all(), f"off by {((off - bound).max()).item():.3e} more than allowed"


def _ids(T, K, E, seed, dropped=0.0, repeat=False, dtype=torch.int32):
    gen = _gen(seed)
    if repeat:
        idx = torch.randint(0, E, (T, K), device="cuda", generator=gen)
    else:
        idx = torch.rand((T, E), device="cuda", generator=gen).topk(K, 1).indices
    if dropped:
        idx[torch.rand((T, K), device="cuda", generator=gen) < dropped] = -1
    return idx.to(dtype)


# ------------------------------------------------------------------ order
@pytest.mark.parametrize("T,K,E,dropped,repeat,dtype", [
    (1, 1, 1, 0.0, False, torch.int32), (1, 8, 256, 0.0, False, torch.int32), (3, 2, 5, 0.5, False, torch.int64),
    (256, 8, 128, 0.0, False, torch.int32), (257, 8, 128, 0.1, False, torch.int32), (2048, 1, 3, 0.0, True, torch.int32),
    (2049, 1, 1024, 0.0, True, torch.int64), (1000, 12, 700, 0.2, True, torch.int32), (20000, 4, 64, 0.0, False, torch.int32),
    (333, 3, 4, 1.1, False, torch.int32), (700, 16, 1, 0.0, True, torch.int32),
])
def test_order(T, K, E, dropped, repeat, dtype):
    import nki_library_b200 as m
    idx = _ids(T, K, E, T + K, dropped, repeat, dtype)
    if T > 2:
        idx[1, 0], idx[2, 0] = E, 2 ** 31 - 1  # no expert either
    plan = m.moe_sort_plan(idx, E)
    offsets, row = ref.sorted_rows(idx, E)
    assert torch.equal(plan.expert_offsets.cpu(), offsets)
    assert torch.equal(plan.row_of_pair.cpu(), row)
    assert plan.num_experts == E


@pytest.mark.parametrize("T,K,E", [(8192, 8, 1024), (8449, 8, 1024), (70000, 8, 120), (524288, 4, 3), (700001, 3, 9), (1 << 20, 8, 33)])
def test_order_of_many_pairs(T, K, E):
    """Either side of the size from which the counts are added up in a launch of their own."""
    import nki_library_b200 as m
    idx = torch.randint(-1, E + 1, (T, K), device="cuda", generator=_gen(T), dtype=torch.int32)
    plan = m.moe_sort_plan(idx, E)
    flat = idx.flatten().long()
    none = (flat < 0) | (flat >= E)
    order = torch.sort(torch.where(none, E, flat), stable=True).indices
    row = torch.empty_like(order)
    row[order] = torch.arange(T * K, device="cuda")
    row[none] = -1
    assert torch.equal(plan.row_of_pair.flatten().long(), row)
    counts = torch.bincount(flat[~none], minlength=E)
    assert plan.expert_offsets.tolist() == [0] + counts.cumsum(0).tolist()


def test_order_of_unsigned_strided_and_no_ids():
    import nki_library_b200 as m
    idx = _ids(50, 4, 16, 1)
    want = m.moe_sort_plan(idx, 16)
    wide = torch.full((50, 8), -1, dtype=torch.int32, device="cuda")
    wide[:, ::2] = idx
    for other in (idx.view(torch.uint32), wide[:, ::2], idx.t().contiguous().t()):
        got = m.moe_sort_plan(other, 16)
        assert all(torch.equal(a, b) for a, b in zip(got[:2], want[:2]))
    for shape in ((0, 4), (4, 0)):
        rows, plan = m.moe_sort_tokens(torch.ones(shape[0], 8, device="cuda"), idx[:shape[0], :shape[1]], 16)
        assert rows.shape == (0, 8) and plan.expert_offsets.tolist() == [0] * 17
        out = m.moe_unsort_tokens(rows, None, plan)
        assert out.shape == (shape[0], 8) and not out.any()


# ------------------------------------------------------------------ rows there and back
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,K,E,H,dropped,repeat", [
    (1, 1, 1, 1, 0.0, False), (1, 8, 256, 7168, 0.0, False), (5, 2, 4, 61, 0.3, False), (17, 8, 16, 512, 0.0, False),
    (64, 12, 32, 1032, 0.2, True), (1300, 3, 8, 264, 0.1, False), (2531, 4, 64, 2044, 0.0, False), (9, 2, 4, 8, 1.1, False),
])
def test_rows_there_and_back(T, K, E, H, dropped, repeat, dtype):
    import nki_library_b200 as m
    gen = _gen(T + H)
    idx = _ids(T, K, E, H, dropped, repeat)
    hidden = torch.randn((T, H), device="cuda", generator=gen).to(dtype).requires_grad_()
    rows, plan = m.moe_sort_tokens(hidden, idx, E)
    row = plan.row_of_pair.long()
    live, at = row >= 0, row.clamp(min=0)
    n = int(live.sum())
    t_of = torch.arange(T, device="cuda")[:, None].expand(T, K)
    want = torch.zeros((T * K, H), dtype=dtype, device="cuda")
    want[row[live]] = hidden.detach()[t_of[live]]
    assert torch.equal(rows.detach(), want)
    d_rows = torch.randn((T * K, H), device="cuda", generator=gen).to(dtype)
    d_rows[n:] = float("nan")  # rows without a pair have no say
    d_hidden, = torch.autograd.grad(rows, hidden, d_rows)
    picked = torch.where(live[:, :, None], d_rows[at].double(), 0.0)
    _close(d_hidden, picked.sum(1), picked.abs().sum(1), K)

    aff_dtype = torch.float32 if K % 2 == 0 else torch.bfloat16
    y = torch.randn((T * K, H), device="cuda", generator=gen).to(dtype)
    y[n:] = float("nan")
    a = torch.rand((T, K), device="cuda", generator=gen).to(aff_dtype)
    a[~live] = float("nan")
    y.requires_grad_(), a.requires_grad_()
    out = m.moe_unsort_tokens(y, a, plan)
    terms = torch.where(live[:, :, None], a.detach().double()[:, :, None] * y.detach()[at].double(), 0.0)
    _close(out.detach(), terms.sum(1), terms.abs().sum(1), 2 * K)
    d_out = torch.randn((T, H), device="cuda", generator=gen).to(dtype)
    d_y, d_a = torch.autograd.grad(out, (y, a), d_out)
    want = torch.zeros((T * K, H), dtype=torch.float64, device="cuda")
    want[row[live]] = (torch.where(live, a.detach(), 0.0).double()[:, :, None] * d_out.double()[:, None])[live]
    _close(d_y, want, want.abs(), 1)
    assert not d_y[n:].any()
    terms = torch.where(live[:, :, None], d_out.double()[:, None] * y.detach()[at].double(), 0.0)
    _close(d_a, terms.sum(2), terms.abs().sum(2), H + 1)
    # each gradient alone, and no weights
    for leaf, whole in ((y, d_y), (a, d_a)):
        yy, aa = (t if t is leaf else t.detach() for t in (y, a))
        alone, = torch.autograd.grad(m.moe_unsort_tokens(yy, aa, plan), leaf, d_out)
        assert torch.equal(alone, whole)
    plain = m.moe_unsort_tokens(y, None, plan)
    picked = torch.where(live[:, :, None], y.detach()[at].double(), 0.0)
    _close(plain.detach(), picked.sum(1), picked.abs().sum(1), K)
    ones, = torch.autograd.grad(plain, y, d_out)
    want = torch.zeros_like(d_rows)
    want[row[live]] = d_out[t_of[live]]
    assert torch.equal(ones, want)


@pytest.mark.parametrize("T,K,E", [(1, 1, 1), (1, 1, 1024), (16, 8, 128), (128, 16, 1024), (127, 16, 3), (129, 8, 256), (128, 17, 64),
                                   (40, 51, 7), (100, 20, 9)])
@pytest.mark.parametrize("H", [8, 4096, 4097, 9002])
def test_rows_of_few_tokens(T, K, E, H):
    """Order and rows of a few tokens come from one launch, which agrees with the two that more tokens take."""
    import nki_library_b200 as m
    idx = _ids(T, K, E, T + K + E, 0.2, True)
    hidden = torch.randn((T, H), device="cuda", generator=_gen(T)).bfloat16()
    rows, plan = m.moe_sort_tokens(hidden, idx, E)
    offsets, row = ref.sorted_rows(idx, E)
    assert torch.equal(plan.expert_offsets.cpu(), offsets) and torch.equal(plan.row_of_pair.cpu(), row)
    alone = m.moe_sort_plan(idx, E)
    assert all(torch.equal(a, b) for a, b in zip(alone[:2], plan[:2]))
    want = torch.zeros((T * K, H), dtype=torch.bfloat16, device="cuda")
    live = row >= 0
    want[row[live].long().cuda()] = hidden[torch.arange(T)[:, None].expand(T, K)[live].cuda()]
    assert torch.equal(rows, want)


def test_rows_with_other_strides():
    import nki_library_b200 as m
    gen = _gen(3)
    T, K, E, H = 40, 4, 8, 264
    idx = _ids(T, K, E, 5)
    base = torch.randn((T, H + 9), device="cuda", generator=gen)
    for hidden in (base[:, :H], base[:, 1:H + 1], base[:, 9:], base.t().contiguous().t()[:, :H],
                   base[:1, :H].expand(T, H), base[:, :1].expand(T, H)):
        for dtype in (torch.float32, torch.bfloat16):
            x = hidden if dtype == torch.float32 else hidden.to(dtype)
            rows, plan = m.moe_sort_tokens(x, idx, E)
            assert torch.equal(rows, m.moe_sort_tokens(x.contiguous(), idx, E)[0])
    y = torch.randn((T * K, 2 * H + 3), device="cuda", generator=gen)[:, 3::2][:, :H].requires_grad_()
    a = torch.rand((K, T), device="cuda", generator=gen).t().requires_grad_()
    out = m.moe_unsort_tokens(y, a, plan)
    again = m.moe_unsort_tokens(y.detach().contiguous(), a.detach().contiguous(), plan)
    assert torch.equal(out, again)
    # a broadcast gradient, as a sum's backward passes it on
    got = torch.autograd.grad(out.sum(), (y, a), retain_graph=True)
    want = torch.autograd.grad(out, (y, a), torch.ones(T, H, device="cuda"))
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,K,E", [(1, 1, 1), (2, 2, 3), (9, 3, 4), (200, 5, 8), (1300, 2, 8)])
@pytest.mark.parametrize("H", [1, 2, 3, 5, 8, 9, 15, 17, 31, 130, 257, 1001])
def test_rows_at_any_address(T, K, E, H, dtype):
    """Matrices anywhere between elements that are not theirs: NaN around every row that is read reaches no result, and what
    surrounds the rows that are written stays as it was."""
    from nki_library_b200 import _lib
    import nki_library_b200 as m
    gen = _gen(T + H)

    def launch(_device, name, *args):
        _lib.call(name, *args, _lib.stream_ptr())

    idx = _ids(T, K, E, H, 0.1)
    plan = m.moe_sort_plan(idx, E)
    row, used = plan.row_of_pair, int(plan.expert_offsets[-1])
    device, code = row.device, _lib.BF16 if dtype == torch.bfloat16 else _lib.F32
    MARK = -77.0

    def surrounded(rows, offset, gap, fill):
        flat = torch.full((offset + rows * (H + gap) + 40,), fill, dtype=dtype, device=device)
        return flat, flat[offset:].as_strided((rows, H), (H + gap, 1))

    def untouched(flat, view):
        view.fill_(MARK)
        return bool((flat == MARK).all())

    a = torch.rand((T, K), device=device, generator=gen)
    live = (row >= 0).flatten()
    token = (torch.arange(T * K, device=device) // K)[live]
    to = row.flatten()[live].long()
    for offset, gap in ((0, 0), (1, 0), (3, 2), (6, 0), (7, 9), (8, 16)):
        _, hidden = surrounded(T, offset, gap, float("nan"))
        _, y = surrounded(T * K, offset + 1, gap, float("nan"))
        hidden.copy_(torch.randn((T, H), device=device, generator=gen))
        y.copy_(torch.randn((T * K, H), device=device, generator=gen))
        y[used:] = float("nan")  # rows of no expert
        flat, rows = surrounded(T * K, 8 - offset, 0, MARK)
        launch(device, "b200moe_sort_rows", hidden.data_ptr(), code, H + gap, T, K, H, E, row.data_ptr(),
               plan.expert_offsets.data_ptr(), rows.data_ptr())
        want = torch.zeros((T * K, H), dtype=dtype, device=device)
        want[to] = hidden[token]
        assert torch.equal(rows, want) and untouched(flat, rows)
        if T <= 128:
            off, row2 = torch.empty_like(plan.expert_offsets), torch.empty_like(row)
            launch(device, "b200moe_sort_tokens", hidden.data_ptr(), code, H + gap, idx.data_ptr(), 4, T, K, H, E, off.data_ptr(),
                   row2.data_ptr(), rows.data_ptr(), None, 0)
            assert torch.equal(rows, want) and torch.equal(row2, row) and untouched(flat, rows)
        flat, out = surrounded(T, offset, 0, MARK)
        launch(device, "b200moe_unsort_rows", y.data_ptr(), code, H + gap, T, K, H, row.data_ptr(), a.data_ptr(), _lib.F32,
               out.data_ptr())
        terms = y.double()[to] * a.double().flatten()[live][:, None]
        zero = torch.zeros((T, H), dtype=torch.float64, device=device)
        _close(out, zero.index_add(0, token, terms), zero.index_add(0, token, terms.abs()), K)
        assert untouched(flat, out)
        for lie in (offset + 1, offset):  # like the rows that are read, and not
            flat, d_rows = surrounded(T * K, lie, 0, MARK)
            d_a = torch.empty_like(a)
            launch(device, "b200moe_unsort_rows_backward", hidden.data_ptr(), H + gap, y.data_ptr(), H + gap, code, T, K, H, E,
                   row.data_ptr(), plan.expert_offsets.data_ptr(), a.data_ptr(), _lib.F32, d_rows.data_ptr(), d_a.data_ptr())
            want = torch.zeros((T * K, H), dtype=torch.float64, device=device)
            want[to] = hidden.double()[token] * a.double().flatten()[live][:, None]
            _close(d_rows, want, want.abs(), 1)
            assert untouched(flat, d_rows)
            products = hidden.double()[token] * y.double()[to]
            want = torch.zeros(T * K, dtype=torch.float64, device=device)
            size = want.clone()
            want[live], size[live] = products.sum(1), products.abs().sum(1)
            _close(d_a.flatten(), want, size, H)


def test_sums_and_their_gradients_agree_with_differences():
    """Both directions are linear in their rows and affinities: fp32 differences against the gradients."""
    import nki_library_b200 as m
    gen = _gen(11)
    T, K, E, H = 23, 3, 6, 70
    idx = _ids(T, K, E, 2, 0.2)
    hidden, step = (torch.randn((T, H), device="cuda", generator=gen) for _ in range(2))
    rows, plan = m.moe_sort_tokens(hidden.requires_grad_(), idx, E)
    d = torch.randn(rows.shape, device="cuda", generator=gen)
    grad, = torch.autograd.grad(rows, hidden, d)
    moved = m.moe_sort_tokens(hidden.detach() + step, idx, E)[0].double() - rows.detach().double()
    # hidden + step is rounded to 2^-24 of magnitudes below 16, times |d| below 8, over T K H terms
    assert abs((moved * d).sum() - (grad.double() * step).sum()) < T * K * H * 2.0 ** -24 * 16 * 8
    a, turn = (torch.rand((T, K), device="cuda", generator=gen) for _ in range(2))
    y = torch.randn((T * K, H), device="cuda", generator=gen)
    out = m.moe_unsort_tokens(y, a.requires_grad_(), plan)
    d = torch.randn(out.shape, device="cuda", generator=gen)
    grad, = torch.autograd.grad(out, a, d)
    moved = m.moe_unsort_tokens(y, a.detach() + turn, plan).double() - out.detach().double()
    assert abs((moved * d).sum() - (grad.double() * turn).sum()) < T * K * H * 2.0 ** -24 * 16 * 16


# ------------------------------------------------------------------ products
COUNTS = {
    "one row": [1], "few": [3, 0, 1, 16, 2], "edges": [0, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, 255, 256, 257, 0],
    "long": [700, 5, 1030], "many": [(7 * e) % 23 for e in range(300)], "none": [0, 0, 0],
}


def _product_case(counts, K, N, behind, seed, transposed=False):
    gen = _gen(seed)
    E, R = len(counts), sum(counts) + behind
    offsets = torch.tensor([0] + counts).cumsum(0).int().cuda()
    x = torch.randn((R, K), device="cuda", generator=gen).bfloat16()
    dy = torch.randn((R, N), device="cuda", generator=gen).bfloat16()
    shape = (E, N, K) if transposed else (E, K, N)
    w = (torch.randn(shape, device="cuda", generator=gen) * 0.1).bfloat16()
    if behind:
        x[sum(counts):], dy[sum(counts):] = float("nan"), float("inf")
    return offsets, x, w.transpose(1, 2) if transposed else w, dy


def _check_product(counts, K, N, behind, seed, transposed):
    import nki_library_b200 as m
    offsets, x, w, dy = _product_case(counts, K, N, behind, seed, transposed)
    x.requires_grad_(), w.requires_grad_()
    y = m.expert_linear(x, w, offsets, _check_status=True)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert dw.shape == w.shape and dx.shape == x.shape
    y, x, w = y.detach(), x.detach(), w.detach()
    at = 0
    for e, n in enumerate(counts):
        part = slice(at, at + n)
        at += n
        xe, we, de = x[part].double(), w[e].double(), dy[part].double()
        _close(y[part], xe @ we, xe.abs() @ we.abs(), K)
        _close(dx[part], de @ we.t(), de.abs() @ we.t().abs(), N)
        _close(dw[e], xe.t() @ de, xe.t().abs() @ de.abs(), max(n, 1))
    assert not y[at:].any() and not dx[at:].any()


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("counts,K,N,behind", [
    ("one row", 8, 8, 0), ("one row", 64, 256, 3), ("few", 72, 40, 0), ("few", 520, 264, 37), ("edges", 256, 512, 0),
    ("edges", 328, 120, 300), ("long", 1000, 776, 1), ("long", 64, 64, 0), ("many", 136, 304, 5), ("none", 32, 48, 9),
    ("none", 32, 48, 1),
])
def test_products(counts, K, N, behind, transposed):
    _check_product(COUNTS[counts], K, N, behind, K + N, transposed)


def test_products_of_the_most_experts():
    _check_product([(5 * e) % 3 for e in range(1024)], 40, 72, 0, 3, False)


@pytest.mark.parametrize("K,N", [(72, 14008), (1032, 13000)])
def test_products_whose_tiles_are_handed_out(K, N):
    """Rows per expert, bytes and tiles enough for the pairs to draw their tiles from one counter."""
    _check_product([12000, 0, 3000, 1, 5199], K, N, 40, K, False)
    _check_product([12000, 0, 3000, 1, 5199], N, K, 0, N, True)


@pytest.mark.parametrize("counts,K,N,behind", [([5, 0, 9], 4096, 72, 3), ([300], 8200, 520, 0), ([1], 2048, 8, 0), ([40, 700, 3], 64, 12000, 5),
                                              ([9000, 70, 0, 5003], 64, 72, 2), ([40001], 136, 8, 0)])
def test_long_contractions_of_few_tiles(counts, K, N, behind):
    """Contractions that are cut into parts and joined: along a weight's columns, its rows, and an expert's rows."""
    _check_product(counts, K, N, behind, K + N, False)
    _check_product(counts, K, N, behind, K + N, True)


@pytest.mark.parametrize("rest", range(0, 64, 3))
def test_weight_gradient_ends_anywhere_in_a_slab(rest):
    """The next expert's rows are inf: none of them may reach this expert's sums."""
    import nki_library_b200 as m
    n = 64 + rest
    offsets, x, w, dy = _product_case([n, 64], 128, 384, 0, rest)
    x[n:], dy[n:] = float("inf"), float("nan")
    w.requires_grad_()
    dw, = torch.autograd.grad(m.expert_linear(x, w, offsets), w, dy)
    xe, de = x[:n].double(), dy[:n].double()
    _close(dw[0], xe.t() @ de, xe.t().abs() @ de.abs(), n)


def test_products_of_other_layouts_and_orders():
    import nki_library_b200 as m
    offsets, x, w, dy = _product_case([40, 0, 90], 96, 160, 0, 7)
    want = m.expert_linear(x, w, offsets)
    wide = torch.zeros((130, 200), dtype=torch.bfloat16, device="cuda")
    wide[:, 8:104] = x
    odd = torch.zeros((130, 99), dtype=torch.bfloat16, device="cuda")
    odd[:, 1:97] = x
    for rows in (wide[:, 8:104], odd[:, 1:97], x.t().contiguous().t()):
        assert torch.equal(m.expert_linear(rows, w, offsets), want)
    strided = torch.zeros((3, 96, 2, 168), dtype=torch.bfloat16, device="cuda")
    strided[:, :, 1, 4:164] = w
    padded = torch.zeros((3, 100, 176), dtype=torch.bfloat16, device="cuda")
    padded[:, :96, 8:168] = w
    for weight in (strided[:, :, 1, 4:164], padded[:, :96, 8:168], w.permute(1, 2, 0).contiguous().permute(2, 0, 1),
                   w.transpose(0, 1).contiguous().transpose(0, 1), w.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        leaf = weight.detach().requires_grad_()
        got = m.expert_linear(x, leaf, offsets)
        assert torch.equal(got, want)
        grad, = torch.autograd.grad(got, leaf, dy)
        assert torch.equal(grad, _weight_grad(m, x, w, offsets, dy))
    # one matrix for all experts: the gradients of its copies add up outside
    shared = w[:1].clone().requires_grad_()
    got = m.expert_linear(x, shared.expand(3, -1, -1), offsets)
    each = _weight_grad(m, x, w[:1].expand(3, -1, -1).contiguous(), offsets, dy)
    grad, = torch.autograd.grad(got, shared, dy)
    _close(grad, each.double().sum(0, keepdim=True), each.double().abs().sum(0, keepdim=True), 3)
    # gate and up in the reference's shape
    four = w.view(3, 96, 2, 80).detach().clone().requires_grad_()
    got = m.expert_linear(x, four, offsets)
    assert torch.equal(got, want) and torch.autograd.grad(got, four, dy)[0].shape == four.shape
    # a broadcast gradient
    leaf = x.detach().requires_grad_()
    got = torch.autograd.grad(m.expert_linear(leaf, w, offsets).sum(), leaf)[0]
    assert torch.equal(got, torch.autograd.grad(m.expert_linear(leaf, w, offsets), leaf, torch.ones_like(want))[0])


def _weight_grad(m, x, w, offsets, dy):
    leaf = w.detach().clone().requires_grad_()
    return torch.autograd.grad(m.expert_linear(x, leaf, offsets), leaf, dy)[0]


def test_no_rows_at_all():
    import nki_library_b200 as m
    w = torch.randn(3, 32, 48, device="cuda").bfloat16().requires_grad_()
    x = torch.zeros(0, 32, device="cuda", dtype=torch.bfloat16).requires_grad_()
    y = m.expert_linear(x, w, torch.zeros(4, dtype=torch.int32, device="cuda"))
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == (0, 48) and dx.shape == (0, 32) and not dw.any() and dw.shape == w.shape
    g = torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16).requires_grad_()
    out = m.moe_glu(g)
    assert out.shape == (0, 32) and torch.autograd.grad(out, g, torch.zeros_like(out))[0].shape == (0, 64)


def test_offsets_that_are_wrong_stay_inside():
    """Descending, negative and too large offsets are brought into [0, R] and ascending order: nothing leaves the buffers."""
    import nki_library_b200 as m
    _, x, w, dy = _product_case([50, 50, 50], 64, 128, 0, 3)
    got = m.expert_linear(x, w, torch.tensor([-5, 70, 20, 10 ** 9], dtype=torch.int32, device="cuda"))
    want = m.expert_linear(x, w, torch.tensor([0, 70, 70, 150], dtype=torch.int32, device="cuda"))
    assert torch.equal(got, want)
    got = m.expert_linear(x, w, torch.tensor([20, 40, 60, 80], dtype=torch.int32, device="cuda"))
    assert not got[:20].any() and not got[80:].any() and got[20:80].any(1).all()


def test_products_and_gradients_are_adjoint():
    """<dy, x W> = <dx, x> = <dW, W>: the three products are one trilinear form.  Each side's bf16 results are off by 2^-8 of
    themselves at most, so the sums by 2^-8 of the sums of magnitudes."""
    import nki_library_b200 as m
    offsets, x, w, dy = _product_case([33, 0, 150, 77], 200, 136, 4, 9)
    dy[260:] = 0
    x[260:] = 0
    x.requires_grad_(), w.requires_grad_()
    y = m.expert_linear(x, w, offsets)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    sides = [(a.detach().double() * b.detach().double()) for a, b in ((dy, y), (dx, x), (dw, w))]
    for a in sides[1:]:
        assert abs(a.sum() - sides[0].sum()) <= 2.0 ** -8 * (a.abs().sum() + sides[0].abs().sum())


# ------------------------------------------------------------------ activation and checkpoint
ACTS = ["SiLU", "GELU", "GELU_Tanh_Approx", "Swish"]


def _gate_up(R, I, seed, spread=1.5):
    return (torch.randn((R, 2 * I), device="cuda", generator=_gen(seed)) * spread).bfloat16()


def _kept_reference(gate_up):
    I = gate_up.shape[1] // 2
    (eg, g), (eu, u) = ref.kept(gate_up[:, :I]), ref.kept(gate_up[:, I:])
    return torch.stack([eg, eu], 1), g, u


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("R,I", [(1, 8), (3, 24), (7, 32), (130, 40), (33, 1000), (512, 1024)])
def test_activation_and_gradient(R, I, act):
    import nki_library_b200 as m
    gate_up = _gate_up(R, I, R + I).requires_grad_()
    out = m.moe_glu(gate_up, m.ActFnType[act])
    x = gate_up.detach()
    with torch.no_grad():
        assert torch.equal(m.moe_glu(x.view(R, 2, I), m.ActFnType[act]), out)
    a, _ = ref.act_and_slope(x[:, :I], act)
    # exp is good to 2^-21 + |z| 2^-23 (|z| below 64 here: 2^-17), which passes to act at most as it is; the tail of a value
    # that vanishes in fp32 is below 1e-37
    want = a * x[:, I:].double()
    _close(out.detach(), want, want.abs(), 1, want.abs() * 2.0 ** -16)
    d = (torch.randn((R, I), device="cuda", generator=_gen(I))).bfloat16()
    got, = torch.autograd.grad(out, gate_up, d)
    _, g, u = _kept_reference(x)
    a, slope = ref.act_and_slope(g, act)
    want = torch.cat([d.double() * u * slope, d.double() * a], 1)
    # act' = sigma + g sigma (1 - sigma) z' adds terms of up to 1 + |z'| (|z| below 2^-17 as above): 2^-15 of |d u| covers
    # their cancellation
    extra = torch.cat([(d.double() * u).abs() * 2.0 ** -15, want[:, I:].abs() * 2.0 ** -16], 1)
    _close(got, want, want.abs(), 2, extra)


@pytest.mark.parametrize("I", [8, 32, 104, 2048])
def test_checkpoint_is_exact(I):
    """Codes and scales bit for bit: magnitudes from the smallest to the largest, ties, blocks of zeros, NaN and infinity."""
    from nki_library_b200.core.moe.moe_train.moe_glu import glu_backward, glu_forward
    R = 96
    gen = _gen(I)
    x = torch.randn((R, 2 * I), device="cuda", generator=gen) * torch.exp2(
        torch.randint(-126, 120, (R, 1), device="cuda", generator=gen).float())
    x[:8] = torch.randint(-512, 513, (8, 2 * I), device="cuda", generator=gen) / 32.0  # ties of the rounding
    x[8] = 0
    x[9], x[9, 0] = 0, 448.0
    x[10], x[10, 0] = 1.0, 450.0
    x[11, 1], x[11, 5], x[12, 3] = float("inf"), float("-inf"), float("nan")
    x[13] = float("nan")
    x[14], x[14, 2] = 2.0 ** -133, 3.3e38
    x[15] = 2.0 ** -133
    x = x.bfloat16()
    _, checkpoint = glu_forward(x, 0, True)
    codes, scales = checkpoint[:R * 2 * I].view(R, 2 * I), checkpoint[R * 2 * I:].view(R, 2, (I + 31) // 32)
    e, g, u = _kept_reference(x)
    assert torch.equal(scales.long() - 127, e)
    s = ref.power_of_two(e).repeat_interleave(32, 2)[:, :, :I].reshape(R, 2 * I)
    got = codes.view(torch.float8_e4m3fn).double() * s
    want = torch.cat([g, u], 1)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    # and what the backward pass makes of it: m from the kept values
    with torch.no_grad():
        _, again = glu_backward(None, checkpoint, R, I, 0, want_m=True)
    a, _ = ref.act_and_slope(g, "SiLU")
    want = a * u
    rows = want.abs().amax(1) < 1e30  # also drops rows with NaN
    assert rows.sum() > 20
    # 1 / (1 + exp(-g)) is flushed to zero below 2^-126, for g below -87.33, where act(g) is smaller than 87.34 * 2^-126 =
    # 1.03e-36
    _close(again[rows], want[rows], want[rows].abs(), 1, want[rows].abs() * 2.0 ** -16 + 1.03e-36 * u[rows].abs())
    bad = g.isnan() | u.isnan()
    assert torch.equal(again.isnan() & bad, bad)


@pytest.mark.parametrize("act", ACTS)
def test_activation_far_out(act):
    """Gates far from zero: no overflow on the way to a finite result, tails keep their relative precision."""
    import nki_library_b200 as m
    g = torch.tensor([-300., -100., -88., -60., -20., -10., -5., -3., 0., 3., 5., 10., 20., 100., 300., 3e38], device="cuda")
    x = torch.cat([g, torch.ones(16, device="cuda")])[None].bfloat16().requires_grad_()
    out = m.moe_glu(x, m.ActFnType[act])
    want, _ = ref.act_and_slope(x.detach()[:, :16], act)
    if act == "GELU_Tanh_Approx":  # g^3 overflows at 3e38: the sigmoid is 1 there
        want[0, -1] = x.detach()[0, 15].double()
    near = want.abs() > 1e-30
    rel = ((out.detach().double() - want).abs() / want.abs())[near]
    # z is rounded to 2^-23 of itself and of up to 150 in the exponential's argument: 2^-15
    assert (rel <= 2.0 ** -8 * (1 + 2.0 ** -6)).all() and (out.detach()[~near].abs() < 1e-29).all()
    grad, = torch.autograd.grad(out, x, torch.ones_like(out))
    assert grad[:, :15].isfinite().all()


def test_gradient_of_the_activation_agrees_with_differences():
    import nki_library_b200 as m
    for act in ACTS:
        x = _gate_up(4, 64, 3).requires_grad_()
        got, = torch.autograd.grad(m.moe_glu(x, m.ActFnType[act]), x, torch.ones((4, 64), device="cuda").bfloat16())
        _, g, u = _kept_reference(x.detach())
        h = 1e-5
        plus, minus = (ref.act_and_slope(g + s * h, act)[0] * u for s in (1, -1))
        want = torch.cat([(plus - minus) / (2 * h), ref.act_and_slope(g, act)[0]], 1)
        # the difference quotient is good to h^2 and 2^-52 / h, both below 1e-9 of values of a few units
        _close(got, want, want.abs(), 2, torch.cat([u.abs() * 2.0 ** -15, want[:, 64:].abs() * 2.0 ** -16], 1) + 1e-8)


# ------------------------------------------------------------------ together
def _layer(seed, T=70, K=2, E=4, H=128, I=96, dropped=0.1):
    gen = _gen(seed)
    idx = _ids(T, K, E, seed, dropped)
    hidden = torch.randn((T, H), device="cuda", generator=gen).bfloat16()
    aff = torch.rand((T, K), device="cuda", generator=gen)
    w1 = (torch.randn((E, H, 2, I), device="cuda", generator=gen) * H ** -0.5).bfloat16()
    w2 = (torch.randn((E, I, H), device="cuda", generator=gen) * I ** -0.5).bfloat16()
    return idx, [hidden, aff, w1, w2], torch.randn((T, H), device="cuda", generator=gen).bfloat16()


@pytest.mark.parametrize("T,K,E,H,I,dropped", [(1, 1, 1, 8, 8, 0.0), (70, 2, 4, 128, 96, 0.1), (300, 4, 16, 256, 520, 0.0),
                                               (33, 2, 8, 64, 64, 1.1)])
def test_layer_is_its_operators(T, K, E, H, I, dropped):
    """Sort, product, activation, product, sum: the layer's output and gradients are those of the operators in a row, bit for
    bit but for the down weight's gradient, which is taken at the kept activations."""
    import nki_library_b200 as m
    from nki_library_b200.core.moe.moe_train.expert_linear import weight_grad
    from nki_library_b200.core.moe.moe_train.moe_glu import glu_backward, glu_forward
    idx, leaves, d = _layer(T, T, K, E, H, I, dropped)
    leaves = [t.requires_grad_() for t in leaves]
    hidden, aff, w1, w2 = leaves
    out = m.moe_experts_train(hidden, aff, idx, w1, w2)
    grads = torch.autograd.grad(out, leaves, d)
    rows, plan = m.moe_sort_tokens(hidden, idx, E)
    gate_up = m.expert_linear(rows, w1, plan.expert_offsets)
    act = m.moe_glu(gate_up)
    y = m.expert_linear(act, w2, plan.expert_offsets)
    one_by_one = m.moe_unsort_tokens(y, aff, plan)
    assert torch.equal(out, one_by_one)
    d_y, = torch.autograd.grad(one_by_one, y, d, retain_graph=True)
    want = torch.autograd.grad(one_by_one, (hidden, aff, w1), d)
    for g, w in zip(grads, want):
        assert torch.equal(g, w)
    with torch.no_grad():
        _, checkpoint = glu_forward(gate_up, 0, True)
        _, m_kept = glu_backward(None, checkpoint, *act.shape, 0, want_m=True)
        assert torch.equal(grads[3], weight_grad(m_kept, d_y, w2, plan.expert_offsets))
        assert torch.equal(m.moe_experts_train(*(t.detach() if t.is_floating_point() else t for t in (hidden, aff)), idx,
                                               w1.detach(), w2.detach()), out)
    # the definition in 64 bits: two bf16 roundings between the products and one at the end move single values by 2^-8 each,
    # sums of independent ones by less: three of them, 2^-8 of the norm each
    x64, a64, w164, w264 = (t.detach().double() for t in leaves)
    live = plan.row_of_pair >= 0
    total = torch.zeros((T, H), dtype=torch.float64, device="cuda")
    for e in range(E):
        for k in range(K):
            mine = (idx[:, k] == e) & live[:, k]
            gate, up = (x64[mine] @ w164[e, :, j] for j in (0, 1))
            total[mine] += a64[mine, k, None] * ((gate * torch.sigmoid(gate) * up) @ w264[e])
    assert (out.detach().double() - total).norm() <= 3 * 2.0 ** -8 * total.norm()


def test_what_the_layer_keeps():
    """Between the passes live the sorted rows and 8.25 bits per gate and up value, not their 16 and the activation."""
    import nki_library_b200 as m
    E, H, I, R = 2, 64, 4096, 4096
    w1 = torch.randn((E, H, 2 * I), device="cuda").bfloat16().requires_grad_()
    w2 = torch.randn((E, I, H), device="cuda").bfloat16().requires_grad_()
    rows = torch.randn((R, H), device="cuda").bfloat16().requires_grad_()
    offsets = torch.tensor([0, R // 2, R], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = m.moe_expert_mlp(rows, w1, w2, offsets)
    held = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert 2 * R * I <= held <= 2 * R * I * 33 / 32 + (1 << 20)


def test_frozen_parts_get_no_gradient():
    import nki_library_b200 as m
    idx, (hidden, aff, w1, w2), d = _layer(5)
    full = [t.clone().requires_grad_() for t in (hidden, aff, w1, w2)]
    want = torch.autograd.grad(m.moe_experts_train(full[0], full[1], idx, full[2], full[3]), full, d)
    for i in range(4):
        args = [t.clone().requires_grad_(i == j) for j, t in enumerate((hidden, aff, w1, w2))]
        got, = torch.autograd.grad(m.moe_experts_train(args[0], args[1], idx, args[2], args[3]), args[i], d)
        assert torch.equal(got, want[i])


def test_runs_repeat_bit_for_bit_and_on_other_streams():
    import nki_library_b200 as m
    idx, leaves, d = _layer(6, T=500, K=4, E=8, H=256, I=264)
    leaves = [t.requires_grad_() for t in leaves]

    def step():
        out = m.moe_experts_train(leaves[0], leaves[1], idx, leaves[2], leaves[3])
        return (out.detach(), *torch.autograd.grad(out, leaves, d))

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in streams:  # two steps in flight at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            results.append(step())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# handed-out tiles, parts that are joined, and the fixed walk: counts, K, N
FORMS = [([12000, 5000, 3240], 128, 14000), ([40, 24], 4096, 64), ([9000, 70, 5003], 64, 72), ([100, 28], 256, 520)]


@pytest.mark.parametrize("counts,K,N", FORMS)
def test_every_form_of_the_products_is_captured_and_runs_beside_another(counts, K, N):
    """Two graphs of the same product and gradients, replayed in turn and on two streams at once, between eager calls."""
    import nki_library_b200 as m
    offsets, x, w, dy = _product_case(counts, K, N, 2, K)
    x[sum(counts):], dy[sum(counts):] = 0, 0
    x.requires_grad_(), w.requires_grad_()

    def step():
        y = m.expert_linear(x, w, offsets)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    want = step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = step()
        graphs.append((graph, results))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for (graph, results), stream in zip(graphs, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                for r in results:
                    r.fill_(7)
                graph.replay()
        eager = step()
        torch.cuda.synchronize()
        for got in (eager, *(r for _, r in graphs)):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_first_call_of_a_thread():
    """A host thread that has made no CUDA call yet, such as the one a backward pass gets, has no context of its own."""
    import threading

    import nki_library_b200 as m
    offsets, x, w, _ = _product_case([40, 24], 64, 128, 0, 1)
    want = m.expert_linear(x, w, offsets)
    del want
    got = []
    worker = threading.Thread(target=lambda: got.append(m.expert_linear(x, w, offsets)))
    worker.start()
    worker.join()
    assert len(got) == 1 and torch.equal(got[0], m.expert_linear(x, w, offsets))


def test_second_derivatives_are_refused():
    """The passes are recorded as they are called, not differentiated again."""
    import nki_library_b200 as m
    idx, leaves, d = _layer(3)
    leaves = [t.requires_grad_() for t in leaves]
    out = m.moe_experts_train(leaves[0], leaves[1], idx, leaves[2], leaves[3])
    first = torch.autograd.grad(out, leaves, d, create_graph=True)
    plain = torch.autograd.grad(m.moe_experts_train(leaves[0], leaves[1], idx, leaves[2], leaves[3]), leaves, d)
    assert all(torch.equal(a, b) for a, b in zip(first, plain))
    d.requires_grad_()
    out = m.moe_experts_train(leaves[0], leaves[1], idx, leaves[2], leaves[3])
    first = torch.autograd.grad(out, leaves, d, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first[0].float().sum().backward()


@pytest.mark.parametrize("op", ["sort", "unsort", "linear", "glu", "mlp"])
def test_losses_of_gradients_are_refused(op):
    """A loss that holds an output and its gradient: what the gradient adds to the derivative would be missing, so it raises."""
    import nki_library_b200 as m
    idx, (hidden, aff, w1, w2), _ = _layer(2)
    rows, plan = m.moe_sort_tokens(hidden, idx, w1.shape[0])
    call, x = {
        "sort": (lambda x: m.moe_sort_tokens(x, idx, w1.shape[0])[0], hidden),
        "unsort": (lambda x: m.moe_unsort_tokens(x, aff, plan), rows),
        "linear": (lambda x: m.expert_linear(x, w1, plan.expert_offsets), rows),
        "glu": (lambda x: m.moe_glu(x), rows),
        "mlp": (lambda x: m.moe_expert_mlp(x, w1, w2, plan.expert_offsets), rows),
    }[op]
    x = x.detach().requires_grad_()
    out = call(x)
    grad, = torch.autograd.grad(out.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (out.float().sum() + grad.float().square().sum()).backward()


def test_errors_of_native_calls():
    """What does not fit is torch's own error, and a refusal of an entry point is a refusal as everywhere; both leave all usable."""
    import nki_library_b200 as m
    from nki_library_b200.core.moe.moe_train.launch import native
    one = torch.zeros(1, dtype=torch.bfloat16, device="cuda")
    idx = torch.zeros((2 ** 20, 1), dtype=torch.int32, device="cuda")
    with pytest.raises(torch.OutOfMemoryError):
        m.moe_sort_tokens(one.expand(2 ** 20, 2 ** 20), idx, 1)
    x = torch.zeros((4, 32), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(AssertionError, match="unknown activation"):
        native().glu(x, 7)
    assert not m.moe_glu(x).any()


def test_captured_step_replays_on_new_inputs():
    """Forward and backward in one graph, two graphs alive, eager steps in between."""
    import nki_library_b200 as m

    def step(idx, leaves, d):
        out = m.moe_experts_train(leaves[0], leaves[1], idx, leaves[2], leaves[3])
        return (out.detach(), *torch.autograd.grad(out, leaves, d))

    idx, leaves, d = _layer(7)
    leaves = [t.requires_grad_() for t in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(idx, leaves, d)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = step(idx, leaves, d)
        graphs.append((graph, results))
    for seed in (8, 9):
        new_idx, new, new_d = _layer(seed)
        with torch.no_grad():
            for a, b in zip((idx, d, *leaves), (new_idx, new_d, *new)):
                a.copy_(b)
        for graph, _ in graphs:
            graph.replay()
        want = step(idx, leaves, d)
        for _, got in graphs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_more_than_two_to_the_31_elements():
    """Rows whose element offsets pass 32 bits: the last ones against the same rows alone."""
    import nki_library_b200 as m
    R, I = 131200, 8192
    gate_up = torch.empty((R, 2 * I), dtype=torch.bfloat16, device="cuda")
    gate_up[:-64] = 0.5
    gate_up[-64:] = _gate_up(64, I, 1)
    assert gate_up.numel() > 2 ** 31
    gate_up.requires_grad_()
    out = m.moe_glu(gate_up)
    d = torch.ones_like(out)
    grad, = torch.autograd.grad(out, gate_up, d)
    last = gate_up.detach()[-64:].clone().requires_grad_()
    alone = m.moe_glu(last)
    assert torch.equal(out[-64:], alone)
    assert torch.equal(grad[-64:], torch.autograd.grad(alone, last, d[-64:])[0])
    del out, grad, d
    # the same buffer as sorted rows: the last token's
    T, K, E = R // 8, 8, 64
    idx = torch.arange(T * K, device="cuda").view(K, T).t().contiguous() // (T * K // E)
    rows = gate_up.detach()
    plan = m.moe_sort_plan(idx, E)
    summed = m.moe_unsort_tokens(rows, None, plan)
    row = plan.row_of_pair[-1].long()
    assert int(row.max()) == R - 1
    _close(summed[-1], rows[row].double().sum(0), rows[row].double().abs().sum(0), K)
    back, _ = m.moe_sort_tokens(summed, idx, E)
    assert torch.equal(back[-1], summed[-1])
    # and as the operand and the result of a product
    w = torch.randn((2, 2 * I, 16), device="cuda", generator=_gen(1)).bfloat16() * 0.01
    offsets = torch.tensor([0, R - 100, R], dtype=torch.int32, device="cuda")
    y = m.expert_linear(rows, w, offsets)
    x = rows[-64:].double()
    _close(y[-64:], x @ w[1].double(), x.abs() @ w[1].double().abs(), 2 * I)
    del back, summed
    thin = torch.randn((R, 16), device="cuda", generator=_gen(2)).bfloat16()
    wide = m.expert_linear(thin, w.transpose(1, 2).contiguous(), offsets)
    x = thin[-64:].double()
    _close(wide[-64:], x @ w[1].double().t(), x.abs() @ w[1].double().t().abs(), 16)


@pytest.mark.parametrize("call", ["index dtype", "index rank", "experts", "rows", "affinities", "dtype", "plan", "columns",
                                  "multiple", "offsets", "weight", "glu", "glu columns", "act", "down"])
def test_refusals(call):
    import nki_library_b200 as m
    idx, (hidden, aff, w1, w2), _ = _layer(1)
    plan = m.moe_sort_plan(idx, 4)
    rows = torch.zeros((140, 128), dtype=torch.bfloat16, device="cuda")
    off = plan.expert_offsets
    calls = {
        "index dtype": (lambda: m.moe_sort_plan(idx.float(), 4), "int32, uint32 or int64"),
        "index rank": (lambda: m.moe_sort_tokens(hidden, idx[0], 4), r"\[T, K\]"),
        "experts": (lambda: m.moe_sort_plan(idx, 1025), "num_experts"),
        "rows": (lambda: m.moe_unsort_tokens(rows[:-1], aff, plan), "T \\* K"),
        "affinities": (lambda: m.moe_unsort_tokens(rows, aff[:, :1], plan), "affinities must be"),
        "dtype": (lambda: m.moe_sort_tokens(hidden.half(), idx, 4), "bfloat16 or float32"),
        "plan": (lambda: m.moe_unsort_tokens(rows, aff, plan._replace(expert_offsets=off[:-1])), "plan must be"),
        "columns": (lambda: m.expert_linear(rows[:, :64], w1, off), "contracts 128"),
        "multiple": (lambda: m.expert_linear(rows[:, :12], w1[:, :12, 0, :8], off), "multiples of 8"),
        "offsets": (lambda: m.expert_linear(rows, w1, off.long()), "expert_offsets"),
        "weight": (lambda: m.expert_linear(rows, w1.float(), off), "weight must be bfloat16"),
        "glu": (lambda: m.moe_glu(rows.float()), "bfloat16"),
        "glu columns": (lambda: m.moe_glu(rows[:, :24]), "multiple of 8"),
        "act": (lambda: m.moe_glu(rows, 0), "ActFnType"),
        "down": (lambda: m.moe_expert_mlp(rows, w1, w2[:, :88], off), "down_proj_weight"),
    }
    fn, message = calls[call]
    with pytest.raises(AssertionError, match=message):
        fn()


@pytest.mark.parametrize("call", ["sort columns", "unsort columns", "rows", "contraction", "columns", "glu rows", "glu columns",
                                  "four sizes"])
def test_sizes_that_no_index_holds_are_refused(call):
    """Sizes beyond the kernels' 32-bit indices, as views of one element: nothing of that size is allocated."""
    import nki_library_b200 as m
    one = torch.zeros(1, dtype=torch.bfloat16, device="cuda")
    idx = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    plan = m.moe_sort_plan(idx, 1)
    off = plan.expert_offsets
    many, few = 2 ** 32 + 8, torch.zeros((1, 8, 8), dtype=torch.bfloat16, device="cuda")
    rows = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    calls = {
        "sort columns": (lambda: m.moe_sort_tokens(one.expand(1, many), idx, 1), "columns"),
        "unsort columns": (lambda: m.moe_unsort_tokens(one.expand(1, many), None, plan), "columns"),
        "rows": (lambda: m.expert_linear(one.expand(2 ** 30 + 1, 8), few, off), "2\\^30 rows"),
        "contraction": (lambda: m.expert_linear(one.expand(1, many), one.expand(1, many, 8), off), "2\\^27"),
        "columns": (lambda: m.expert_linear(one.expand(1, 8), one.expand(1, 8, many), off), "2\\^27"),
        "glu rows": (lambda: m.moe_glu(one.expand(2 ** 30 + 1, 16)), "2\\^30 rows"),
        "glu columns": (lambda: m.moe_glu(one.expand(1, 2 * many)), "2\\^27 columns"),
        "four sizes": (lambda: m.moe_expert_mlp(rows, torch.zeros((1, 64, 4, 8), dtype=torch.bfloat16, device="cuda"),
                                                torch.zeros((1, 16, 64), dtype=torch.bfloat16, device="cuda"), off), "H, 2, I"),
    }
    fn, message = calls[call]
    with pytest.raises(AssertionError, match=message):
        fn()
