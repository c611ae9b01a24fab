"""The operators of the experts' training pass: what is timed of them, in a plain form and through the package.

A case is a dict of plain values.  ``kind`` names the operator:

* ``sort``    token rows sorted by expert: ``moe_sort_tokens``
* ``unsort``  the experts' rows back at their tokens, weighted by the routing affinities: ``moe_unsort_tokens``
* ``linear``  one product per expert on sorted rows: ``expert_linear``
* ``glu``     act(gate) * up, whose inputs are kept for the backward pass as 8-bit codes with a power of two per 32
              columns: ``moe_glu``

With ``train`` a pass is the operator and its gradients, without it the operator alone, as serving calls it.

Definitions.  Pairs (token t, choice k) are ordered by (expert, t, k); pair (t, k) owns row ``row_of_pair[t, k]`` of R = T K
rows, -1 if its expert id is outside [0, E); expert e owns rows ``expert_offsets[e]`` to ``expert_offsets[e + 1]``, and rows
behind the last expert are zero in every result.

* sort: rows[row_of_pair[t, k]] = hidden[t]; d hidden[t] = sum over k of d rows[row_of_pair[t, k]].
* unsort: out[t] = sum over k of a[t, k] rows[row_of_pair[t, k]]; d rows[r] = a[t, k] d out[t];
  d a[t, k] = <d out[t], rows[r]>.
* linear: y[r] = rows[r] W[e]; d rows[r] = d y[r] W[e]^T; d W[e] = sum over its rows of rows[r]^T d y[r].
* glu: m = act(g) u.  Of g and u, e4m3(v / s) is kept, rounded to the nearest even code, with s the smallest power of two of
  at least 2^-127 for which no finite value of the block exceeds 448 s (a value that is not finite is kept as NaN).  With the
  kept values g^ and u^: d g = d m u^ act'(g^), d u = d m act(g^).
"""

import math

import torch

own = False

ACTS = ("SiLU", "GELU", "GELU_Tanh_Approx", "Swish")
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _case(kind, train=True, dtype="bf16", T=0, E=1, K=1, H=0, N=0, zipf=0.0, dropped=0.0, transposed=False, act="SiLU"):
    return dict(kind=kind, train=train, dtype=dtype, T=T, E=E, K=K, H=H, N=N, zipf=zipf, dropped=dropped,
                transposed=transposed, act=act)


def listed():
    cases = {
        # a decode batch of 16 sequences over many experts: launches
        "sort-few": _case("sort", False, T=16, E=128, K=8, H=4096),
        # the largest batch, top-8, both directions
        "sort-train": _case("sort", T=32768, E=128, K=8, H=4096),
        # a single token's eight rows
        "unsort-token": _case("unsort", False, T=1, E=256, K=8, H=7168),
        # a ragged prompt in fp32, a tenth of whose pairs were dropped
        "unsort-ragged": _case("unsort", dtype="f32", T=2531, E=64, K=4, H=2048, dropped=0.1),
        # half of the largest batch, both directions
        "unsort-train": _case("unsort", T=16384, E=128, K=8, H=4096),
        # the smallest layer of the tests and the smoke run (gate and up): launches and host work
        "linear-tiny": _case("linear", T=256, E=4, K=2, H=512, N=2048),
        # gate and up of 64 decoding sequences: the weights' stream
        "linear-few": _case("linear", False, T=64, E=8, K=2, H=4096, N=28672),
        # gate and up of the benchmark's layer, all three products
        "linear-prefill": _case("linear", T=4096, E=8, K=2, H=4096, N=28672),
        # many experts with a skewed load
        "linear-skewed": _case("linear", T=8192, E=64, K=8, H=7168, N=4096, zipf=1.2),
        # the smallest layer again
        "glu-tiny": _case("glu", T=512, N=1024),
        # a ragged prompt, a width that ends inside a block
        "glu-ragged": _case("glu", T=10124, N=1000, act="GELU"),
        # 65536 rows of 4096 intermediates
        "glu-train": _case("glu", T=65536, N=4096),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges: tokens and widths over their logarithm, up to the cost of the largest listed case of
    the kind."""
    limit = {"sort": (5e9, 1e13), "unsort": (4.4e9, 1e13), "linear": (1.1e10, 1.2e13), "glu": (5.5e9, 1e13)}
    while True:
        kind = rng.choice(["sort", "unsort", "linear", "linear", "glu"])
        train = rng.random() < 0.75
        E = _log_int(rng, 2, 256)
        K = min(rng.randint(1, 8), E)
        T = _log_int(rng, 1, 32768)
        case = _case(kind, train, T=T, E=E, K=K, H=8 * _log_int(rng, 16, 896), zipf=rng.choice([0.0, 0.0, 1.2]),
                     dropped=rng.choice([0.0, 0.0, 0.05, 0.3]))
        if kind in ("sort", "unsort"):
            case["dtype"] = rng.choice(["bf16", "bf16", "f32"])
            if rng.random() < 0.3:
                case["H"] -= rng.randint(1, 7)  # rows that are no multiple of 16 bytes
        elif kind == "linear":
            case["N"] = 8 * _log_int(rng, 16, 3584)
            case["transposed"] = rng.random() < 0.3
        else:
            case.update(T=_log_int(rng, 1, 131072), E=1, K=1, H=0, zipf=0.0, dropped=0.0, N=8 * _log_int(rng, 1, 1792),
                        act=rng.choice(ACTS))
        cost = work(case)
        if cost["bytes"] <= limit[kind][0] and cost["flops"] <= limit[kind][1] and \
                (kind != "linear" or case["E"] * case["H"] * case["N"] <= 2 ** 31):
            return case


# ------------------------------------------------------------------ what a program has in hand before the call
def _routing(case, gen):
    """Expert ids as a router picks them: the K largest of E noisy scores, some experts more popular with ``zipf``; a
    ``dropped`` share of the pairs carries the id -1."""
    T, E, K = case["T"], case["E"], case["K"]
    score = -torch.log(-torch.log(torch.rand((T, E), device="cuda", generator=gen).clamp(1e-9, 1 - 1e-7)))
    if case["zipf"]:
        rank = torch.randperm(E, device="cuda", generator=gen).float() + 1.0
        score -= case["zipf"] * torch.log(rank)
    idx = score.topk(K, dim=1).indices.to(torch.int32)
    if case["dropped"]:
        idx[torch.rand((T, K), device="cuda", generator=gen) < case["dropped"]] = -1
    return idx


def _plain_plan(idx, E):
    """Offsets and rows of the pairs, by a stable sort of their expert ids."""
    T, K = idx.shape
    flat = idx.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.sort(key, stable=True).indices
    row = torch.empty_like(order)
    row[order] = torch.arange(T * K, device=idx.device)
    row[key == E] = -1
    experts = torch.arange(E, device=idx.device)
    offsets = torch.zeros(E + 1, dtype=torch.int64, device=idx.device)
    offsets[1:] = (key[:, None] == experts).sum(0).cumsum(0) if T * K * E < 1 << 28 else torch.stack(
        [(key == e).sum() for e in range(E)]).cumsum(0)
    return offsets.to(torch.int32), row.view(T, K).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, T, E, K, H, N = (case[k] for k in ("kind", "T", "E", "K", "H", "N"))
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, to=dtype):
        out = torch.empty(shape, dtype=to, device="cuda")
        step = max(1, (1 << 28) // max(1, out[:1].numel()))
        for i in range(0, shape[0], step):
            n = min(step, shape[0] - i)
            out[i:i + n] = torch.randn((n, *shape[1:]), device="cuda", generator=gen) * scale
        return out

    state = dict(case=case)
    if kind == "glu":
        state["gate_up"] = randn(T, 2 * N, scale=1.5)
        if case["train"]:
            state["d_out"] = randn(T, N, scale=0.01)
            state["gate_up"].requires_grad_(own)
        return state
    state["index"] = _routing(case, gen)
    R = T * K
    if kind == "sort":
        state["hidden"] = randn(T, H)
        if case["train"]:
            state["d_out"] = randn(R, H, scale=0.01)
            state["hidden"].requires_grad_(own)
        return state
    # the sorted order belongs to the layer's forward pass, which has been there before
    if own:
        import nki_library_b200 as moe
        state["plan"] = moe.moe_sort_plan(state["index"], E)
    else:
        offsets, rows = _plain_plan(state["index"], E)
        state["row_of_pair"], state["bounds"] = rows, offsets.tolist()
    state["rows"] = randn(R, H)
    if kind == "unsort":
        aff = torch.rand((T, K), device="cuda", generator=gen)
        state["affinities"] = aff / aff.sum(1, keepdim=True)
        leaves = ("rows", "affinities")
    else:
        w = randn(E, N, H, scale=0.02).transpose(1, 2) if case["transposed"] else randn(E, H, N, scale=0.02)
        state["weight"] = w
        leaves = ("rows", "weight")
    if case["train"]:
        state["d_out"] = randn(T if kind == "unsort" else R, H if kind == "unsort" else N, scale=0.01)
        for name in leaves:
            state[name].requires_grad_(own)
    return state


# ------------------------------------------------------------------ one pass, through the package
def _run_own(s):
    import nki_library_b200 as moe
    case = s["case"]
    kind = case["kind"]
    if kind == "sort":
        rows, plan = moe.moe_sort_tokens(s["hidden"], s["index"], case["E"])
        out = {"out": rows, "offsets": plan.expert_offsets, "row_of_pair": plan.row_of_pair}
        leaves = {"d_hidden": s["hidden"]}
    elif kind == "unsort":
        out = {"out": moe.moe_unsort_tokens(s["rows"], s["affinities"], s["plan"])}
        leaves = {"d_rows": s["rows"], "d_affinities": s["affinities"]}
    elif kind == "linear":
        out = {"out": moe.expert_linear(s["rows"], s["weight"], s["plan"].expert_offsets)}
        leaves = {"d_rows": s["rows"], "d_weight": s["weight"]}
    else:
        out = {"out": moe.moe_glu(s["gate_up"], moe.ActFnType[case["act"]])}
        leaves = {"d_gate_up": s["gate_up"]}
    if case["train"]:
        grads = torch.autograd.grad(out["out"], list(leaves.values()), s["d_out"])
        out["out"] = out["out"].detach()
        out.update(zip(leaves, grads))
    return out


# ------------------------------------------------------------------ one pass, plainly
def _act(g, act):
    """act(g) and act'(g)."""
    if act in ("SiLU", "Swish"):
        c = 1.0 if act == "SiLU" else 1.702
        sig = 1.0 / (1.0 + torch.exp(-c * g))
        return g * sig, sig * (1.0 + c * g * (1.0 - sig))
    if act == "GELU":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * g * g)


def _power_of_two(e):
    """2^e of whole numbers e in [-1022, 1023], exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _kept(v):
    """What the 8-bit checkpoint stands for, v [R, I] in fp32."""
    R, I = v.shape
    x = torch.nn.functional.pad(v, (0, -I % 32)).view(R, -1, 32)
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(2, keepdim=True)
    fraction, exponent = torch.frexp(top)
    e = (exponent - torch.where(fraction <= 0.875, 9, 8)).clamp(min=-127)
    e = torch.where(top == 0, -127, e)
    code = (x.double() * _power_of_two(-e)).float().to(torch.float8_e4m3fn)
    kept = (code.double() * _power_of_two(e)).float()
    return torch.where(torch.isfinite(x), kept, float("nan")).view(R, -1)[:, :I]


def _run_plain(s):
    case = s["case"]
    kind, dtype, train = case["kind"], DTYPES[case["dtype"]], case["train"]
    if kind == "glu":
        out, d = [], []
        for lo in range(0, case["T"], 16384):
            gu = s["gate_up"][lo:lo + 16384].float()
            g, u = gu.chunk(2, 1)
            out.append((_act(g, case["act"])[0] * u).to(dtype))
            if train:
                g, u = _kept(g), _kept(u)
                dm = s["d_out"][lo:lo + 16384].float()
                a, da = _act(g, case["act"])
                d.append(torch.cat([dm * u * da, dm * a], 1).to(dtype))
        return {"out": torch.cat(out), "d_gate_up": torch.cat(d)} if train else {"out": torch.cat(out)}
    if kind == "sort":
        T, K = s["index"].shape
        offsets, row = _plain_plan(s["index"], case["E"])
        live = row >= 0
        rows = torch.zeros((T * K, case["H"]), dtype=dtype, device="cuda")
        for k in range(K):
            rows[row[live[:, k], k].long()] = s["hidden"][live[:, k]]
        result = {"out": rows, "offsets": offsets, "row_of_pair": row}
        if train:
            total = torch.zeros((T, case["H"]), device="cuda")
            for k in range(K):
                total += torch.where(live[:, k, None], s["d_out"][row[:, k].clamp(min=0).long()].float(), 0.0)
            result["d_hidden"] = total.to(dtype)
        return result
    if kind == "unsort":
        row, rows, a = s["row_of_pair"], s["rows"], s["affinities"]
        T, K = row.shape
        live = row >= 0
        total = torch.zeros((T, case["H"]), device="cuda")
        d_rows, d_a = torch.zeros_like(rows), torch.zeros_like(a)
        for k in range(K):
            picked = rows[row[:, k].clamp(min=0).long()].float()
            total += torch.where(live[:, k, None], a[:, k, None] * picked, 0.0)
            if train:
                d = s["d_out"].float()
                d_rows[row[live[:, k], k].long()] = (a[:, k, None] * d)[live[:, k]].to(dtype)
                d_a[:, k] = torch.where(live[:, k], (d * picked).sum(1), 0.0)
        result = {"out": total.to(dtype)}
        if train:
            result.update(d_rows=d_rows, d_affinities=d_a)
        return result
    x, w, bounds = s["rows"], s["weight"], s["bounds"]
    y = torch.zeros((x.shape[0], case["N"]), dtype=dtype, device="cuda")
    if train:
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for e in range(case["E"]):
        part = slice(bounds[e], bounds[e + 1])
        if part.start == part.stop:
            continue
        xe, we = x[part].float(), w[e].float()
        y[part] = (xe @ we).to(dtype)
        if train:
            de = s["d_out"][part].float()
            dx[part] = (de @ we.t()).to(dtype)
            dw[e] = (xe.t() @ de).to(dtype)
    return {"out": y, "d_rows": dx, "d_weight": dw} if train else {"out": y}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_order(idx, E):
    """Rows of the pairs, counted: those of smaller experts, then those of the same expert that come earlier."""
    T, K = idx.shape
    flat = idx.reshape(-1).long()
    row = torch.full_like(flat, -1)
    offsets, start = [0], 0
    for e in range(E):
        mine = (flat == e).nonzero()[:, 0]
        row[mine] = start + torch.arange(mine.numel(), device=flat.device)
        start += mine.numel()
        offsets.append(start)
    return offsets, row.view(T, K)


def _exact_kept(v):
    """v [R, I] in 64 bits, rounded by hand: step 2^-3 of the value's own power of two, but no finer than 2^-9."""
    R, I = v.shape
    out = torch.empty_like(v)
    for c in range(0, I, 32):
        x = v[:, c:c + 32]
        finite = x.isfinite()
        top = torch.where(finite, x.abs(), 0.0).max(1, keepdim=True).values
        e = torch.full_like(top, -127.0)
        live = top > 448.0 * 2.0 ** -127
        guess = torch.floor(torch.log2(torch.where(live, top, 1.0) / 448.0))
        for step in (-1, 0, 1, 2):  # the smallest power of two that is large enough, whatever log2 rounds to
            tried = guess + step
            fits = top <= 448.0 * _power_of_two(tried)
            e = torch.where(live & fits & (e == -127.0), tried, e)
        scaled = x / _power_of_two(e)
        own_power = torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** -6)))
        own_power = torch.where(_power_of_two(own_power) > scaled.abs().clamp(min=2.0 ** -6), own_power - 1, own_power)
        quantum = _power_of_two(own_power.nan_to_num(0.0, 0.0, 0.0) - 3)
        out[:, c:c + 32] = torch.where(finite, torch.round(scaled / quantum) * quantum * _power_of_two(e), float("nan"))
    return out


def _exact_act(g, act):
    if act == "GELU":
        return 0.5 * g * torch.special.erfc(-g / math.sqrt(2.0)), \
            0.5 * torch.special.erfc(-g / math.sqrt(2.0)) + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if act == "GELU_Tanh_Approx":  # (1 + tanh z) / 2 = sigmoid(2 z)
        z = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
        dz = 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g ** 2)
    else:
        z = g * (1.702 if act == "Swish" else 1.0)
        dz = torch.full_like(g, 1.702 if act == "Swish" else 1.0)
    s = torch.sigmoid(z)
    return g * s, s + g * s * torch.sigmoid(-z) * dz


def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    kind, train, E, H, N = case["kind"], case["train"], case["E"], case["H"], case["N"]
    f64 = dict(dtype=torch.float64, device="cuda")
    if kind == "glu":
        out = torch.empty((case["T"], N), **f64)
        d = torch.empty((case["T"], 2 * N), **f64) if train else None
        for lo in range(0, case["T"], 8192):
            part = slice(lo, lo + 8192)
            g, u = s["gate_up"][part, :N].double(), s["gate_up"][part, N:].double()
            out[part] = _exact_act(g, case["act"])[0] * u
            if train:
                g, u, dm = _exact_kept(g), _exact_kept(u), s["d_out"][part].double()
                a, slope = _exact_act(g, case["act"])
                d[part, :N] = dm * u * slope
                d[part, N:] = dm * a
        return {"out": out, "d_gate_up": d} if train else {"out": out}
    offsets, row = _exact_order(s["index"], E)
    T, K = row.shape
    if kind == "linear":
        R = T * K
        y = torch.zeros((R, N), **f64)
        dx = torch.zeros((R, H), **f64) if train else None
        dw = torch.zeros((E, H, N), dtype=torch.float32, device="cuda") if train else None  # 64-bit sums, kept in 32
        for e in range(E):
            lo, hi = offsets[e], offsets[e + 1]
            if lo == hi:
                continue
            xe, we = s["rows"][lo:hi].double(), s["weight"][e].double()
            y[lo:hi] = torch.mm(xe, we)
            if train:
                de = s["d_out"][lo:hi].double()
                dx[lo:hi] = torch.mm(de, we.T)
                dw[e] = torch.mm(xe.T, de).float()
        return {"out": y, "d_rows": dx, "d_weight": dw} if train else {"out": y}
    pair = (row >= 0).nonzero()  # (t, k) of the live pairs
    where = row[pair[:, 0], pair[:, 1]]
    if kind == "sort":
        out = torch.zeros((T * K, H), dtype=DTYPES[case["dtype"]], device="cuda")
        out[where] = s["hidden"][pair[:, 0]]
        result = {"out": out, "offsets": torch.tensor(offsets, dtype=torch.int32, device="cuda"),
                  "row_of_pair": row.to(torch.int32)}
        if train:
            d = torch.zeros((T, H), **f64)
            for lo in range(0, T, 2048):
                mine = (pair[:, 0] >= lo) & (pair[:, 0] < lo + 2048)
                d.index_add_(0, pair[mine, 0], s["d_out"][where[mine]].double())
            result["d_hidden"] = d
        return result
    out = torch.zeros((T, H), **f64)
    d_rows = torch.zeros((T * K, H), dtype=torch.float32, device="cuda") if train else None
    d_aff = torch.zeros((T, K), **f64) if train else None
    for lo in range(0, T, 2048):
        mine = (pair[:, 0] >= lo) & (pair[:, 0] < lo + 2048)
        t, k, r = pair[mine, 0], pair[mine, 1], where[mine]
        y, a = s["rows"][r].double(), s["affinities"][t, k].double()
        out.index_add_(0, t, y * a[:, None])
        if train:
            d = s["d_out"][t].double()
            d_rows[r] = (d * a[:, None]).float()
            d_aff[t, k] = torch.einsum("rh,rh->r", d, y)
    return {"out": out, "d_rows": d_rows, "d_affinities": d_aff} if train else {"out": out}


# ------------------------------------------------------------------ what it cannot do without
def work(case):
    kind, T, E, K, H, N, train = (case[k] for k in ("kind", "T", "E", "K", "H", "N", "train"))
    size = 4 if case["dtype"] == "f32" else 2
    if kind == "glu":
        # gate, up and output; the gradients; the 8-bit checkpoint, written by one pass and read by the other
        kept = 2 * T * N + 2 * T * -(-N // 32)
        return {"bytes": 3 * T * N * size + (3 * T * N * size + 2 * kept if train else 0), "flops": (30 if train else 10) * T * N}
    live = T * K * (1.0 - case["dropped"])
    if kind == "sort":
        one = (T + T * K) * H * size + T * K * 8 + E * 4
        return {"bytes": one * (2 if train else 1), "flops": T * K * H if train else 0}
    if kind == "unsort":
        # rows and the gradient's rows, output and its gradient, affinities and theirs
        one = (live + T) * H * size + T * K * 8
        back = (T * K + T) * H * size + T * K * 8
        return {"bytes": one + (back if train else 0), "flops": (5 if train else 2) * live * H}
    active = E * (1.0 - (1.0 - min(1.0, K * (1.0 - case["dropped"]) / E)) ** T)
    weights = H * N * size
    ways = 3 if train else 1
    return {"bytes": active * weights + (T * K) * (H + N) * size * (2 if train else 1) + (E * weights if train else 0),
            "flops": 2.0 * ways * live * H * N}
