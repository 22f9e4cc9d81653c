"""AdamW and the 8-bit form of its moments in 64 bits, written from their definition."""
import torch

BLOCK = 256
#: values of the codes without their sign: 3 bits of fraction (first moment), 4 (second), under 4 bits of exponent
FIRST = torch.tensor([(f + 8 * (e > 0)) * 2.0 ** (max(e, 1) - 10) for e in range(16) for f in range(8)], dtype=torch.float64)
SECOND = torch.tensor([(f + 16 * (e > 0)) * 2.0 ** (max(e, 1) - 11) for e in range(16) for f in range(16)], dtype=torch.float64)


def step(p, g, m, v, t, lr, b1, b2, eps, wd):
    """(p, m, v) after step t, in 64 bits."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p * (1 - lr * wd) - lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps), m, v


def spread(scale, n):
    """A block's value at each of its elements."""
    return scale.double().repeat_interleave(BLOCK)[:n]


def read(m, v, scales):
    n = m.numel()
    m, v, s = m.flatten().cpu().long(), v.flatten().cpu().long(), scales.cpu()
    first = FIRST[m & 127]
    return torch.where(m > 127, -first, first) * spread(s[0], n), SECOND[v] * spread(s[1], n)


def mix(x):
    x ^= x >> 16
    x = x * 0x7FEB352D & 0xFFFFFFFF
    x ^= x >> 15
    x = x * 0x846CA68B & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_bits(seed, t, k, n):
    key = mix(mix(mix(seed) + t & 0xFFFFFFFF) + k & 0xFFFFFFFF)
    x = (torch.arange(n) * 0x9E3779B9 + key) & 0xFFFFFFFF
    return mix(x)


def tops(x):
    """Largest magnitude of each block."""
    n = x.numel()
    full = torch.zeros((n + BLOCK - 1) // BLOCK * BLOCK, dtype=torch.float64)
    full[:n] = x.abs()
    return full.view(-1, BLOCK).amax(1)


def codes(x, scale, table, u, slack):
    """(lowest, highest) code that rounding x / scale with the random number u may give, where x / scale is known to within `slack`."""
    y = x.abs() / torch.where(scale > 0, scale, torch.ones_like(scale))
    out = []
    for z in (y * (1 - slack), y * (1 + slack)):
        z = z.clamp(max=float(table[-1]))
        k = (torch.searchsorted(table, z, right=True) - 1).clamp(0, len(table) - 2)
        out.append(k + ((z - table[k]) / (table[k + 1] - table[k]) + u >= 1).long())
    return out
