"""Plain 64-bit references of the row operators, and the 8-bit state's arithmetic in torch operations (fp32, operation by operation)."""
import math

import torch

BLOCK = 128


def norm64(x, w, b, eps, dy=None):
    """-> y, or (y, dx, dw, db), and the quantities that error bounds are made of, all float64 on the CPU."""
    x = x.detach().double().cpu()
    c = x.shape[-1]
    w = torch.ones(c, dtype=torch.float64) if w is None else w.detach().double().cpu()
    b = torch.zeros(c, dtype=torch.float64) if b is None else b.detach().double().cpu()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    q = {"xh": xh, "rstd": rstd, "w": w, "b": b, "top": x.abs().amax(1, keepdim=True) if x.numel() else x.new_zeros(x.shape[0], 1)}
    if dy is None:
        return xh * w + b, q
    dy = dy.detach().double().cpu()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    q.update(g=g, dy=dy)
    return (xh * w + b, dx, (dy * xh).sum(0), dy.sum(0)), q


def grouped64(x, w, ends, b, dy=None):
    x, w = x.detach().double().cpu(), w.detach().double().cpu()
    b = None if b is None else b.detach().double().cpu()
    n, (groups, out, inner) = x.shape[0], w.shape
    y, size = torch.zeros(n, out, dtype=torch.float64), torch.zeros(n, out, dtype=torch.float64)
    spans = []
    at = 0
    for g in range(groups):                      # the offsets as a rising sequence within [0, n]
        lo = max(min(max(ends[g], 0), n), at)
        hi = max(min(max(ends[g + 1], 0), n), lo)
        spans.append((lo, hi))
        at = hi
    for g, (i, j) in enumerate(spans):
        y[i:j] = x[i:j] @ w[g].T + (0 if b is None else b[g])
        size[i:j] = x[i:j].abs() @ w[g].abs().T + (0 if b is None else b[g].abs())
    if dy is None:
        return (y,), (size,)
    dy = dy.detach().double().cpu()
    dx, sx = torch.zeros_like(x), torch.zeros_like(x)
    dw, sw, db, sb = torch.zeros_like(w), torch.zeros_like(w), torch.zeros(groups, out, dtype=torch.float64), torch.zeros(groups, out, dtype=torch.float64)
    for g, (i, j) in enumerate(spans):
        dx[i:j], sx[i:j] = dy[i:j] @ w[g], dy[i:j].abs() @ w[g].abs()
        dw[g], sw[g] = dy[i:j].T @ x[i:j], dy[i:j].abs().T @ x[i:j].abs()
        db[g], sb[g] = dy[i:j].sum(0), dy[i:j].abs().sum(0)
    return (y, dx, dw, db), (size, sx, sw, sb)


def half_step(t):
    """How far rounding to t is off at most, relative to the value (gradual underflow of fp16 apart, see `floor_step`)."""
    return torch.finfo(t).eps / 2


def floor_step(t):
    """Half the distance of t's smallest values."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


# ---------------------------------------------------------------------------------------------------------------- 8-bit states
def mix32(x):
    """MurmurHash3's finalizer on Python numbers or int64 tensors in [0, 2^32)."""
    x = x ^ (x >> 16)
    x = (x * 0x85EBCA6B) & 0xFFFFFFFF
    x = x ^ (x >> 13)
    x = (x * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def power(k):
    return ((k.to(torch.int32) + 127) << 23).view(torch.float32)


def encode_blocks(x, bits16):
    """(blocks, 128) fp32 -> e4m3 codes and the blocks' exponents; bits16: the random bits."""
    finite = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    e = torch.clamp(((finite.amax(1).view(torch.int32) >> 23) - 127), min=-119)
    y = x.abs() * power(7 - e)[:, None]
    # above 2^-6: the 20 bits behind e4m3's three mantissa bits, carried into them; below, where the values are 2^-9 apart: the exact sum
    z = ((y.view(torch.int32) + (bits16 << 4).to(torch.int32)) & -(1 << 20)).view(torch.float32)
    z = torch.where(y < 2.0 ** -6, (torch.floor(y.double() * 512 + bits16.double() / 65536) / 512).float(), z)
    z = torch.where(y < 256, z, torch.full_like(z, math.nan))
    return torch.copysign(z, x).to(torch.float8_e4m3fn), e.to(torch.int8)


def decode_blocks(codes, e):
    return codes.float() * power(e.int() - 7)[:, None]


class Adam8:
    """One parameter's step with 8-bit states in fp32 operations on the CPU: what the kernel is defined as, bit for bit."""

    def __init__(self, p, key, seed):
        self.p, self.key, self.seed, self.n = p.detach().cpu().clone().reshape(-1), key, seed, p.numel()
        nb = -(-self.n // BLOCK)
        self.m = torch.zeros(nb, BLOCK).to(torch.float8_e4m3fn)
        self.r = self.m.clone()
        self.e = torch.zeros(nb, 2, dtype=torch.int8)
        self.step_ = 0

    def step(self, g, lr, betas, eps, wd):
        self.step_ += 1
        b1, b2 = betas
        pad = lambda t: torch.nn.functional.pad(t.detach().cpu().reshape(-1).float(), (0, -self.n % BLOCK)).view(-1, BLOCK)  # noqa: E731
        p, g = pad(self.p), pad(g)
        m, r = decode_blocks(self.m, self.e[:, 0]), decode_blocks(self.r, self.e[:, 1])
        m = m * b1 + g * (1.0 - b1)
        v = r * r * b2 + g * g * (1.0 - b2)
        r = v.double().sqrt().float()      # correctly rounded (the CPU's fp32 root is not); 53 bits are enough for that
        scale = 1.0 / math.sqrt(1.0 - b2 ** self.step_)
        p = p * (1.0 - lr * wd) - lr / (1.0 - b1 ** self.step_) * (m / (r * scale + eps))
        self.ratio = (m / (r * scale + eps)).reshape(-1)[:self.n].double()
        self.p = p.reshape(-1)[:self.n].to(self.p.dtype)
        key = mix32((mix32((mix32(self.seed) + self.step_) & 0xFFFFFFFF) + self.key) & 0xFFFFFFFF)
        bits = mix32(torch.arange(m.numel()).view(-1, BLOCK) ^ key)
        self.m, em = encode_blocks(m, bits & 0xFFFF)
        self.r, er = encode_blocks(r, bits >> 16)
        self.e = torch.stack((em, er), 1)
