"""Microscaled numbers in 64 bits: what the kernels of `mx4_*` are held to.  E2M1 (4 bits) for matrices, E2M3 (6 bits) for rows; blocks
of 32 neighbouring values of a row share the smallest power of two, from 2^-127 on, with which the block's largest magnitude is at most 7 or 7.5."""
import torch

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
E2M3 = tuple(i / 8 for i in range(16)) + tuple(2 + i / 4 for i in range(8)) + tuple(4 + i / 2 for i in range(8))
MOST = {E2M1: 7.0, E2M3: 7.5}


def power_of_two(e):
    """2^e exactly (torch.ldexp forms it in 32 bits, and not exactly on the GPU)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def blocks(x):
    k = x.shape[-1]
    return torch.nn.functional.pad(x.double(), (0, -k % 32)).unflatten(-1, (-1, 32))


def nearest(x, levels):
    """(codes, exponents) of x `[.., k]`: `[.., blocks, 32]` with the sign as the bit above the magnitude's, and `[.., blocks]`, 128 where the block is NaN."""
    b = blocks(x)
    amax = b.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    mantissa, exponent = torch.frexp(torch.where(bad, torch.ones_like(amax), amax))
    e = (exponent - 3 + (8 * mantissa > MOST[levels]).to(exponent.dtype)).clamp(min=-127)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    v = torch.where(bad[..., None], torch.zeros_like(b), b) * power_of_two(-e)[..., None]
    table = torch.tensor(levels, dtype=torch.float64, device=x.device)
    middle = (table[1:] + table[:-1]) / 2
    at = (v.abs()[..., None] > middle).sum(-1)                             # (on a middle: the lower one)
    tie = (v.abs()[..., None] == middle).any(-1)
    at = at + (tie & (at % 2 == 1)).to(at.dtype)
    sign = torch.signbit(v) & ~bad[..., None]
    return at + sign.to(at.dtype) * len(levels), torch.where(bad, torch.full_like(e, 128), e)


def values(codes, e, levels, k):
    table = torch.tensor(levels + tuple(-v for v in levels), dtype=torch.float64, device=codes.device)
    v = table[codes] * power_of_two(e.clamp(max=127))[..., None]
    return torch.where((e == 128)[..., None], torch.full_like(v, float("nan")), v).flatten(-2)[..., :k]


def rows6(x):
    return values(*nearest(x, E2M3), E2M3, x.shape[-1])


def stored(w):
    """The bytes that hold `w` `[rows][k]`, place by place: codes `[tiles][k / 128][64][16]`, powers `[tiles][k / 512][64][4]`."""
    code, e = nearest(w.cpu(), E2M1)
    rows, n_blocks = e.shape
    tiles, steps, groups = -(-rows // 16), -(-n_blocks // 4), -(-n_blocks // 16)
    codes = torch.zeros((tiles, steps, 64, 16), dtype=torch.uint8)
    powers = torch.zeros((tiles, groups, 64, 4), dtype=torch.uint8)
    both = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)
    for r in range(rows):
        for b in range(n_blocks):
            codes[r // 16, b // 4, 16 * (b % 4) + r % 16] = both[r, b]
            powers[r // 16, b // 16, 16 * (b % 4) + r % 16, b // 4 % 4] = int(e[r, b]) + 127
    return codes, powers


def read(codes, powers, rows, k):
    """The values, in 64 bits, that the stored form holds (leading dimensions stay)."""
    n_blocks = -(-k // 32)
    r, b = torch.arange(rows, device=codes.device)[:, None], torch.arange(n_blocks, device=codes.device)[None, :]
    byte = codes[..., r // 16, b // 4, 16 * (b % 4) + r % 16, :]
    e = powers[..., r // 16, b // 16, 16 * (b % 4) + r % 16, b // 4 % 4].int() - 127
    return values(torch.stack([byte & 15, byte >> 4], -1).flatten(-2).long(), e, E2M1, k)


def product(x, w):
    """(x' w^T, sum of the magnitudes of its terms) for rows x `[m][k]` and a matrix w that is in its microscaled values already."""
    x = rows6(x)
    return x @ w.T, x.abs() @ w.abs().T


def sum_error(k, size):
    """How far a 32-bit sum of k products and what is joined to it (up to 64 partial sums and a bias) may be off: every addition by a step of
    2^-23 of at most the sum of the magnitudes (the matrix cores round to nearest or cut off)."""
    return (k + 64) * 2.0 ** -23 * size


def silu(z):
    return z * torch.sigmoid(z)


def act(g, u, limit, kind):
    if kind == 1:
        return silu(g) * u
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g * torch.sigmoid(1.702 * g) * (u + 1)
