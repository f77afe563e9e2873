"""NumPy restatement of the many-tensor AdamW: one step in float64 from the formula, and the 8-bit block format of the
moments in float32 / integer arithmetic, whose codes the kernel has to give bit for bit."""
from __future__ import annotations

import numpy as np

BLOCK = 256
RATE = {True: 0xC13FA9A9, False: 0x91E10DA5}  # 2^32 / r and 2^32 / r^2 (r^3 = r + 1), per step: first, second moment
TURN = 0x9E3779B9                             # 2^32 / golden ratio, per element


def top_of(signed: bool) -> int:
    return 127 if signed else 255


def decode(codes: np.ndarray, exponents: np.ndarray, signed: bool) -> np.ndarray:
    """float32 values of a tensor's codes (flat) and block exponents."""
    top = top_of(signed)
    e = np.repeat(exponents.astype(np.int64), BLOCK)[:codes.size]
    q = codes.astype(np.int64) & top
    k = q + 8 * (e + 1) - top
    bits = np.where((q > 0) & (k > 0), k << 20, 0)
    bits = np.where(e == 255, 0x7FC00000, bits).astype(np.uint32)
    x = bits.view(np.float32).copy()
    if signed:
        x = np.where(codes >= 128, -x, x)
    return x


def thresholds(n: int, step: int, signed: bool) -> np.ndarray:
    i = np.arange(n, dtype=np.uint64)
    return ((i * np.uint64(TURN) + np.uint64(step * RATE[signed] & 0xFFFFFFFF)) & np.uint64(0xFFFFFFFF)).astype(np.int64)


def encode(x: np.ndarray, step: int, signed: bool) -> tuple[np.ndarray, np.ndarray]:
    """Codes and block exponents of flat float32 values after update number `step`."""
    top = top_of(signed)
    x = np.asarray(x, np.float32)
    n = x.size
    blocks = (n + BLOCK - 1) // BLOCK
    bits = (x.view(np.uint32) & 0x7FFFFFFF).astype(np.int64)
    exponents = (np.pad(bits, (0, blocks * BLOCK - n)).reshape(blocks, BLOCK).max(1, initial=0) >> 23) if n else np.zeros(0, np.int64)
    base = 8 * (np.repeat(exponents, BLOCK)[:n] + 1) - top
    floor = np.maximum(base, 0)
    least = (floor + 1) << 20
    u = thresholds(n, step, signed)
    q = ((bits + (u >> 12)) >> 20) - base
    if signed:
        share = least.astype(np.uint32).view(np.float32) * np.float32(2.0 ** -24)
        keep = bits.astype(np.uint32).view(np.float32) > (u >> 8).astype(np.float32) * share
    else:
        keep = bits > 0
    q = np.where(bits < least, np.where(keep, floor + 1 - base, 0), q)
    q = np.minimum(q, np.minimum(top, 0x7F7 - base))
    q = q & 255
    if signed:
        q = (q & 127) | np.where(x < 0, 128, 0)
    return q.astype(np.uint8), exponents.astype(np.uint8)


def moments32(m, v, g, betas, clip=1.0) -> tuple[np.ndarray, np.ndarray]:
    """The new moments in float32, products and sums rounded one by one in the kernel's order."""
    f = np.float32
    with np.errstate(all='ignore'):
        gc = f(clip) * np.asarray(g, f)
        m = f(betas[0]) * m + f(1.0 - betas[0]) * gc
        v = f(betas[1]) * v + f(1.0 - betas[1]) * gc * gc
    return m, v


def step64(p, m, v, g, t: int, lr, betas, eps: float, weight_decay: float, clip: float = 1.0):
    """One AdamW step in float64 (lr: a number or a list cycled over the elements); returns (p, m, v)."""
    p, m, v, g = (np.asarray(a, np.float64) for a in (p, m, v, g))
    lrs = np.asarray(lr if isinstance(lr, (list, tuple)) else [lr], np.float64)
    lr = lrs[np.arange(p.size) % lrs.size]
    with np.errstate(all='ignore'):
        g = clip * g
        m = betas[0] * m + (1 - betas[0]) * g
        v = betas[1] * v + (1 - betas[1]) * g * g
        u = (m / (1 - betas[0] ** t)) / (np.sqrt(v / (1 - betas[1] ** t)) + eps)
    return p * (1 - lr * weight_decay) - lr * u, m, v


def bounds(p, m, v, g, t: int, lr, betas, eps: float, weight_decay: float, clipped: bool):
    """How far float32 arithmetic may be from step64, counted in roundings (e = 2^-24 each, relative to its result).
    Clipped gradients: the norm's squares are summed 32 at a time in float32 (33 e on the sum, 17 e on its root), then
    the norm's and the factor's own conversion and the product: 20 e on g.
    m: each product has a rounded factor and its own rounding, and g's error; the sum's one: (3 + 20) e (|b1 m| + |(1 - b1) g|).
    v: factor, two products, sum, and twice g's error: (4 + 40) e v (all terms are positive).
    update u = lr' (m / (sqrt(v) r + eps)): half of v's (2 + 20), the root within 2^-23 (2), r (1), the fused sum (1), the
    quotient within 2 ulp (4), lr' (1): (11 + 20) e |u|, and m's error through it. p: factor, product and the final fused
    difference: 3 e (|p| + |u|), which covers the difference's result."""
    e = 2.0 ** -24
    cg = 20 if clipped else 0
    lrs = np.asarray(lr if isinstance(lr, (list, tuple)) else [lr], np.float64)
    lr = lrs[np.arange(np.size(p)) % lrs.size]
    p, m, v, g = (np.asarray(a, np.float64) for a in (p, m, v, g))
    new_m, new_v = betas[0] * m + (1 - betas[0]) * g, betas[1] * v + (1 - betas[1]) * g * g
    dm = (3 + cg) * e * (np.abs(betas[0] * m) + np.abs((1 - betas[0]) * g))
    dv = (4 + 2 * cg) * e * new_v
    slope = lr / (1 - betas[0] ** t) / (np.sqrt(new_v / (1 - betas[1] ** t)) + eps)
    u = np.abs(slope * new_m)
    dp = slope * dm + (11 + cg) * e * u + 3 * e * (np.abs(p) + u)
    tiny = 2.0 ** -148  # results among the subnormals: two roundings of half their spacing
    return 1.01 * dp + tiny, 1.01 * dm + tiny, 1.01 * dv + tiny
