"""Plain 64-bit forms of the training pass's operators, for the tests."""

import math

import torch


def sorted_rows(index, E):
    """(offsets, row_of_pair) of ids [T, K], on the CPU."""
    T, K = index.shape
    flat = index.reshape(-1).long().cpu()
    per_expert = [(flat == e).nonzero()[:, 0] for e in range(E)]
    order = torch.cat(per_expert) if E else flat[:0]
    offsets = torch.tensor([0] + [p.numel() for p in per_expert]).cumsum(0)
    row = torch.full((T * K,), -1)
    row[order] = torch.arange(order.numel())
    return offsets.int(), row.view(T, K).int()


def power_of_two(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def kept(v):
    """(exponents [R, blocks], kept values) of v [R, I] in 64 bits."""
    R, I = v.shape
    x = torch.nn.functional.pad(v.double(), (0, -I % 32)).view(R, -1, 32)
    finite = x.isfinite()
    top = torch.where(finite, x.abs(), 0.0).amax(2)
    fraction, exponent = torch.frexp(top)  # top = fraction * 2^exponent, fraction in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(top > 0, exponent - torch.where(fraction <= 0.875, 9, 8), -127).clamp(min=-127)
    s = power_of_two(e)[:, :, None]
    scaled = torch.where(finite, x / s, 0.0)
    _, own = torch.frexp(scaled.abs().clamp(min=2.0 ** -6))
    quantum = power_of_two(own - 1 - 3)  # three bits behind the leading one; 2^-9 below 2^-6
    value = torch.where(finite, torch.round(scaled / quantum) * quantum * s, math.nan)
    return e, value.view(R, -1)[:, :I]


def act_and_slope(g, name):
    g = g.double()
    if name == "GELU":
        cdf = 0.5 * torch.special.erfc(-g / math.sqrt(2.0))
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if name == "GELU_Tanh_Approx":
        c = math.sqrt(2 / math.pi)
        z, dz = 2 * c * (g + 0.044715 * g ** 3), 2 * c * (1 + 3 * 0.044715 * g ** 2)
    else:
        a = 1.702 if name == "Swish" else 1.0
        z, dz = a * g, torch.full_like(g, a)
    s = torch.sigmoid(z)
    return g * s, s + g * s * torch.sigmoid(-z) * dz
