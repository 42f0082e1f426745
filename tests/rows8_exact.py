"""Rows whose products, norms and distances float32 holds exactly, and how far a tensor core's sum of others may be off.

Whole numbers of -7 .. 7 times 1 or 2 (one power a block) are e4m3 codes with their scale; terms are at most 196 in
magnitude and whole, so every sum of up to 2^24 / 196 / 2 of them, half a norm among them, is exact in any order."""
import torch

BLOCK, STEP = 128, 32


def whole_rows(n, dim, seed, powers=False):
    """float32 [n, dim] on the device.  ``powers``: rows times powers of two of their own (products stay exact, distances
    do not)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(-7, 8, (n, dim), generator=g, device="cuda").float()
    power = torch.randint(0, 2, (n, -(-dim // BLOCK)), generator=g, device="cuda").repeat_interleave(BLOCK, 1)[:, :dim]
    if powers:
        power = power + torch.randint(-6, 7, (n, 1), generator=g, device="cuda")
    return x * torch.exp2(power.float())


def products(a, b):
    return a.double() @ b.double().T


def distances(a, c):
    """float64 [n]: squared distance of every row of ``a`` to the nearest of ``c``."""
    a, c = a.double(), c.double()
    nc = (c * c).sum(1)
    return torch.cat([((r * r).sum(1)[:, None] + nc - 2 * (r @ c.T)).amin(1) for r in a.split(8192)])


def sum_error(a, c, first=0.0):
    """float64 [n, k]: how far the tensor core's a . c may be off, after a first step that held ``first`` [k].

    A step takes 32 terms and the running sum, aligns them to the largest of all, cuts each off at 2^-25 of that one's
    power of two, and cuts their sum off (toward zero) to 24 bits.  So a step is off by at most
      2^-23 of its sum, 2^-25 of the largest for the running sum, and as much for each term with bits down there: terms have
      8 significant bits, so those under 2^-17 of the largest.
    Sum and largest are bounded by the sum of all magnitudes."""
    a, c = a.double(), c.double()
    mags = a.abs() @ c.abs().T + first
    steps = -(-a.shape[1] // STEP) + 1
    small = torch.zeros_like(mags)
    for d in range(0, a.shape[1], 8):
        t = (a[:, None, d : d + 8] * c[None, :, d : d + 8]).abs()
        small += ((t > 0) & (t < (2.0 ** -17 * mags)[:, :, None])).sum(2)
    return 2.0 ** -23 * mags * (1.25 * steps + small / 4)


def product_range(a, b, dtype):
    """(the products, how far those of ``dtype`` may be off): the sum, then one rounding of half a step (or of half the
    type's smallest step, below its normal range)."""
    want, f = products(a, b), torch.finfo(dtype)
    off = sum_error(a, b)
    return want, off + torch.clamp((want.abs() + off) * f.eps / 2, min=f.smallest_normal * f.eps / 2)


def distance_range(a, c):
    """(lowest, highest) float64 [n] that a coverage of the rows ``a`` by ``c`` may give.

    Norms are sums of float32: 16 additions and one a block, half a step each.  The product's sum starts with half the centre's norm
    (more than 64 centres) or has it added to it; it counts twice.  Three roundings join the three."""
    a, c, u = a.double(), c.double(), 2.0 ** -24
    na, nc = (a * a).sum(1)[:, None], (c * c).sum(1)[None]
    d = na + nc - 2 * (a @ c.T)
    mags = a.abs() @ c.abs().T
    off = (na + nc) * (16 + -(-a.shape[1] // BLOCK)) * u + 2 * sum_error(a, c, nc / 2) + (na + nc + 2 * mags) * 3 * u
    near, j = d.min(1)
    return (d - off).clamp_min(0).amin(1), near + off.gather(1, j[:, None])[:, 0]
