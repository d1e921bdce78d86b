"""Microscaled numbers and what is computed with them, in 64 bits and one after the other."""
import torch

FOUR = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
EIGHT = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:-1]
BLOCK = 32


def nearest(x, numbers):
    """x [n, k] as blocks of 32 numbers of a type (those that are not negative are listed, every second one is even), times powers of two."""
    x = x.double().cpu()
    most = numbers[-1]
    table = torch.tensor(numbers, dtype=torch.float64)
    middles = (table[1:] + table[:-1]) / 2
    out = torch.empty_like(x)
    for at in range(0, x.shape[1], BLOCK):
        part = x[:, at:at + BLOCK]
        top = part.abs().amax(dim=1, keepdim=True)
        fine = torch.isfinite(part).all(dim=1, keepdim=True)
        part = torch.where(fine, part, 0.0)
        top = torch.where(fine, top, 0.0)
        e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0) / most)) - 1
        for _ in range(3):
            e = torch.where(top > most * torch.exp2(e), e + 1, e)
        e = torch.where(top > 0, e, -127.0).clamp(min=-127)
        a = part.abs() * torch.exp2(-e)
        low, high = torch.bucketize(a, middles), torch.bucketize(a, middles, right=True)
        q = table[torch.where(low % 2 == 0, low, high)] * torch.exp2(e)
        out[:, at:at + BLOCK] = torch.where(fine, torch.copysign(q, part), torch.nan)
    return out


def rmsnorm(x, branch, weight, eps):
    """total in float32 (one rounding) and its norm in 64 bits."""
    total = x.float().cpu() if branch is None else (x.double().cpu() + branch.double().cpu()).float()
    t = total.double()
    return total, t / torch.sqrt((t * t).mean(dim=1, keepdim=True) + eps) * weight.double().cpu()


def gate(g, u, form=None):
    alpha, limit, shift, cubic, mult = (1.0, float("inf"), 0.0, 0.0, 1.0) if form is None else [float(v) for v in form]
    g = g.clamp(max=limit)
    u = u.clamp(-limit, limit) + shift
    return g * torch.sigmoid(alpha * g * (1 + cubic * g * g)) * u * mult


def codes_of(values, k):
    """Codes [n, ceil(k / 2)] and exponents [n, ceil(k / 32)] of numbers that `nearest(., FOUR)` gave (as the library's rule chooses them)."""
    n = values.shape[0]
    blocks = -(-k // BLOCK)
    wide = torch.zeros(n, blocks * BLOCK, dtype=torch.float64)
    wide[:, :k] = values
    b = wide.view(n, blocks, BLOCK)
    top = b.abs().amax(dim=2)
    e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0) / 6.0)) - 1
    for _ in range(3):
        e = torch.where(top > 6.0 * torch.exp2(e), e + 1, e)
    e = torch.where(top > 0, e, -127.0).clamp(min=-127)
    y = b * torch.exp2(-e)[:, :, None]
    place = torch.bucketize(y.abs(), torch.tensor(FOUR, dtype=torch.float64)) + 8 * torch.signbit(b)
    place = place.to(torch.uint8).flatten(1)
    return (place[:, 0::2] | place[:, 1::2] << 4)[:, :-(-k // 2)].contiguous(), (e + 127).to(torch.uint8)
