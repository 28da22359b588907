"""Plain 64-bit forms of the rotary positions, the 8-bit cache and the sampler, written from their definitions."""
import math

import torch

MIN_EXP = -60


def rotate(x, positions, inv_freq, interleaved=False, scale=1.0):
    """x[..., heads, Dh] at positions[...], float64."""
    x = x.double().clone()
    R = 2 * inv_freq.numel()
    ang = positions.double()[..., None, None] * inv_freq.double()
    c, s = scale * torch.cos(ang), scale * torch.sin(ang)
    first = torch.arange(R // 2) * (2 if interleaved else 1)
    second = first + (1 if interleaved else R // 2)
    a, b = x[..., first].clone(), x[..., second].clone()
    x[..., first] = a * c - b * s
    x[..., second] = b * c + a * s
    return x


def to_bf16(x):
    return x.float().to(torch.bfloat16)


def e4m3(y):
    """float64 -> the nearest e4m3 number (ties to even, below 2^-6 in steps of 2^-9), as float64."""
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), torch.clamp(e - 1, min=-6) - 3)
    return torch.round(y / step) * step


def exponent(amax: float) -> int:
    """The smallest e >= -60 with amax <= 448 * 2^e."""
    e = MIN_EXP
    while amax > math.ldexp(448.0, e):
        e += 1
    return e


class Cache:
    """Values and scale exponents, one number at a time where it matters."""

    def __init__(self, B, Hk, S, Dh, block):
        self.val = torch.zeros(B, Hk, S, Dh, dtype=torch.float64)
        self.exp = torch.zeros(B, Hk, -(-S // block), dtype=torch.int64)
        self.block, self.S = block, S

    def append(self, x, start, count):
        """x [B, L, Hk, Dh] bf16 behind start[b] tokens; returns True where tokens were dropped."""
        dropped = False
        for b in range(x.shape[0]):
            end = min(start[b] + count[b], self.S)
            dropped |= start[b] + count[b] > self.S
            for t0 in range(start[b] // self.block * self.block, end, self.block):
                lo, hi = max(start[b], t0), min(end, t0 + self.block)
                if lo >= hi:
                    continue
                for h in range(x.shape[2]):
                    new = x[b, lo - start[b]:hi - start[b], h].double()
                    fine = torch.isfinite(new)
                    e = exponent(float(torch.where(fine, new.abs(), 0.0).max()))
                    j = t0 // self.block
                    if t0 < start[b]:
                        e = max(e, int(self.exp[b, h, j]))
                        if e > int(self.exp[b, h, j]):
                            old = self.val[b, h, t0:lo]
                            self.val[b, h, t0:lo] = e4m3(old * 2.0 ** -e) * 2.0 ** e
                    self.exp[b, h, j] = e
                    code = e4m3(torch.where(fine, new, 0.0) * 2.0 ** -e)
                    if e == 120:   # 256 * 2^120 is no 32-bit number
                        code = code.clamp(-240.0, 240.0)
                    self.val[b, h, lo:hi] = torch.where(fine, code * 2.0 ** e, math.nan)
        return dropped


def attend(q, k, v, lens, scale):
    """q [B, H, Dh], k / v [B, Hk, S, Dh] float64 values."""
    B, H, Dh = q.shape
    G = H // k.shape[1]
    out = torch.zeros(B, H, Dh, dtype=torch.float64)
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        for h in range(H):
            s = (k[b, h // G, :n] @ q[b, h].double()) * scale
            out[b, h] = torch.softmax(s, 0) @ v[b, h // G, :n]
    return out


def sample_row(x, u, T, k, p, m):
    """(token, share) of one row of float64 logits."""
    V = x.numel()
    x = torch.where(torch.isnan(x), -math.inf, x)
    best = float(x.max())
    if best == -math.inf:
        return 0, 0.0
    if not T > 0 or k == 1:
        return int((x == best).nonzero()[0]), 1.0
    T = min(T, float(torch.finfo(torch.float32).max))
    order = sorted(range(V), key=lambda i: (-float(x[i]), i))
    w = [1.0 if float(x[i]) == best else math.exp((float(x[i]) - best) / T) for i in order]
    n = V if k <= 0 else min(k, V)
    total, before, kept = math.fsum(w[:n]), 0.0, []
    for i, wi in zip(order[:n], w[:n]):
        if p < 1.0 and before > max(p, 0.0) * total:
            break
        if m > 0 and wi < min(m, 1.0):
            break
        kept.append((i, wi))
        before += wi
    kept.sort()
    z, run = math.fsum(wi for _, wi in kept), 0.0
    for i, wi in kept:
        run += wi
        if run > u * z:
            return i, wi / z
    i, wi = [t for t in kept if t[1] > 0][-1]
    return i, wi / z
