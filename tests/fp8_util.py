"""Plain restatements of the 8-bit operators for the tests, in torch on the CPU."""
import torch

BLOCK, TOP, TINY = 128, 448.0, 2.0 ** -126
F8 = torch.float8_e4m3fn
RECIP = torch.tensor(1.0 / 448.0, dtype=torch.float32)


def scale_of(amax):
    """float32, every operation rounded: max(amax * (1/448), 2^-126); NaN stays."""
    s = amax.float() * RECIP
    return torch.where(s < TINY, torch.full_like(s, TINY), s)


def to_codes(x, inv):
    """x * inv rounded to the format; past its largest value the largest."""
    y = x.float() * inv
    return torch.where(y.isnan(), y, y.clamp(-TOP, TOP)).to(F8)


def amax_of(x, dim):
    """Largest magnitude, NaN if there is one."""
    return x.abs().amax(dim)


def rows(x):
    """codes [R, K], scales [R, ceil(K/128)] of x on the CPU."""
    x = x.float()
    r, k = x.shape
    kb = -(-k // BLOCK)
    p = torch.zeros(r, kb * BLOCK)
    p[:, :k] = x
    p = p.view(r, kb, BLOCK)
    s = scale_of(amax_of(p, 2))
    return to_codes(p, (1.0 / s)[:, :, None]).view(r, -1)[:, :k], s


def square(w):
    w = w.float()
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    p = torch.zeros(nb * BLOCK, kb * BLOCK)
    p[:n, :k] = w
    p = p.view(nb, BLOCK, kb, BLOCK)
    s = scale_of(amax_of(amax_of(p, 3), 1))
    return to_codes(p, (1.0 / s)[:, None, :, None]).reshape(nb * BLOCK, -1)[:n, :k], s


def values(codes, scales):
    """float64 values of codes with row or square scales."""
    r, k = codes.shape
    s = scales.double().repeat_interleave(BLOCK, 1)[:, :k]
    if s.shape[0] != r:
        s = s.repeat_interleave(BLOCK, 0)[:r]
    return codes.double() * s


def same_bits(a, b):
    """Equal codes; NaN equals NaN."""
    a, b = a.cpu().float(), b.cpu().float()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def rel_l2(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    n = float(b.norm())
    return float((a - b).norm()) / n if n else float((a - b).norm())


def noise(index, seed, step, salt):
    """32 bits for each element (int64 tensor of indices)."""
    m = 0xFFFFFFFF
    key = (seed + 0x9E3779B1 * step + salt) & m
    h = ((index ^ key) & m) * 0x9E3779B1 & m
    h = (h ^ (h >> 15)) * 0x6A09E667 & m
    return h ^ (h >> 16)


def dither(y, r16):
    """y in [0, 448] up or down to the format by a 16-bit number."""
    low = (y < 2.0 ** -6).float() * 2.0 ** -6
    b = (y + low).view(torch.int32) + (r16.int() << 4)
    return (b & ~0xFFFFF).view(torch.float32) - low


def hold(x, r16, least):
    """8-bit form of a flat state whose length is a multiple of 128."""
    b = x.view(-1, BLOCK)
    s = scale_of(b.abs().amax(1))
    y = (b.abs() * (1.0 / s)[:, None]).clamp_max(TOP).reshape(-1)
    c = dither(y, r16)
    if least:
        c = torch.where((y > 0) & (c == 0), torch.full_like(c, 2.0 ** -9), c)
    return (c * x.sign()).to(F8), s
