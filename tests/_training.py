"""Plain 64-bit forms of the training operators, and how far a kernel's results may be from them."""
from __future__ import annotations

import numpy as np
import torch

U32 = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def smallest(dtype) -> float:
    """Half a step of numbers next to 0."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rounded(want, dtype, error=0.0):
    """Bound of a result with an error before it is rounded once to dtype."""
    return error + half_step(dtype) * (want.abs() + error) + smallest(dtype)


def assert_within(got, want, bound, what=""):
    got = got.detach().double().cpu()
    off = (got - want).abs() - bound
    bad = ~(off <= 0)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, by {float(off[bad].max()):.3e} beyond the bound at most"


def philox(c0, c1, c2, c3, k0, k1, rounds=10):
    """Philox4x32 of numpy uint64 arrays (or numbers) below 2^32: four words."""
    u = np.uint64
    low = u(0xFFFFFFFF)
    c0, c1, c2, c3 = (np.asarray(c, dtype=u) for c in (c0, c1, c2, c3))
    k0, k1 = int(k0), int(k1)
    for _ in range(rounds):
        a, b = c0 * u(0xD2511F53), c2 * u(0xCD9E8D57)
        c0, c1, c2, c3 = (b >> u(32)) ^ c1 ^ u(k0), b & low, (a >> u(32)) ^ c3 ^ u(k1), a & low
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return c0, c1, c2, c3


def threshold(p):
    return int(p * 65536.0 + 0.5)


def keep_mask(rows, cols, p, seed, offset):
    """Which elements dropout keeps, [rows, cols]."""
    blocks = (cols + 7) // 8
    row, block = np.meshgrid(np.arange(rows, dtype=np.uint64), np.arange(blocks, dtype=np.uint64), indexing="ij")
    seed, offset = seed % 2 ** 64, offset % 2 ** 64
    words = philox(row, block, offset % 2 ** 32, offset >> 32, seed % 2 ** 32, seed >> 32)
    bits = np.empty((rows, blocks, 8), dtype=np.uint32)
    for j, w in enumerate(words):
        bits[:, :, 2 * j], bits[:, :, 2 * j + 1] = w & np.uint64(0xFFFF), w >> np.uint64(16)
    return torch.from_numpy(bits.reshape(rows, blocks * 8)[:, :cols] >= threshold(p))


def dropped(x, p, seed, offset):
    """Dropout of x [rows, cols] in 64 bits."""
    t = threshold(p)
    if t == 65536:
        return torch.zeros_like(x, dtype=torch.float64)
    keep = keep_mask(*x.shape, p, seed, offset)
    return torch.where(keep, x.double() * (65536.0 / (65536 - t)), torch.zeros((), dtype=torch.float64))


def table_gradient(grad, ids, rows, scale=1.0, padding=None, weights=None):
    """(gradient [rows, dim], sum of the absolute contributions, contributions a row) in 64 bits; ids already clamped."""
    g = grad.double().cpu()
    if weights is not None:
        g = g * weights[:, None]
    ids = ids.cpu().long()
    if padding is not None:
        g, ids = g[ids != padding], ids[ids != padding]
    zeros = torch.zeros(rows, g.shape[1], dtype=torch.float64)
    count = torch.zeros(rows, dtype=torch.float64).index_add_(0, ids, torch.ones(ids.numel(), dtype=torch.float64))
    return zeros.index_add(0, ids, g) * scale, zeros.index_add(0, ids, g.abs()) * abs(scale), count


def gradient_bound(want, absolute, count, dtype, mean=False):
    """k terms are added with at most k roundings in any order, scaled with one; a mean's terms have two more each."""
    return rounded(want, dtype, (count[:, None] + (4 if mean else 2)) * U32 * absolute)


class Norm64:
    """The norm of stored rows h, forward and backward, in 64 bits, with first-order bounds of fp32 arithmetic.

    `depth`: additions on the way of an element into a sum over its row."""

    def __init__(self, h, gamma, beta, eps, depth):
        self.h, self.gamma, self.beta = h.double(), gamma.double(), beta.double()
        n = h.shape[1]
        self.mean = self.h.sum(1, keepdim=True) / n
        dev = self.h - self.mean
        var = (dev * dev).sum(1, keepdim=True) / n
        self.rstd = 1 / torch.sqrt(var + eps)
        self.z = dev * self.rstd
        self.y = self.z * self.gamma + self.beta
        self.depth = depth
        self.e_mean = (depth + 2) * U32 * self.h.abs().mean(1, keepdim=True)
        # the variance: squares of rounded deviations, their sum; a wrong mean adds its square. rstd: half of that, square root
        # and quotient within two steps each
        self.r_rstd = 0.5 * ((depth + 6) * U32 + (self.e_mean * self.rstd) ** 2) + 6 * U32
        self.e_z = self.rstd * (self.e_mean + U32 * dev.abs()) + self.z.abs() * (self.r_rstd + 2 * U32)
        self.e_y = self.gamma.abs() * self.e_z + 4 * U32 * ((self.z * self.gamma).abs() + self.beta.abs())

    def backward(self, grad, grad_h=None):
        g = grad.double()
        a = g * self.gamma
        m0, m1 = a.mean(1, keepdim=True), (a * self.z).mean(1, keepdim=True)
        d = self.depth + 3
        e_m0 = d * U32 * a.abs().mean(1, keepdim=True)
        e_m1 = d * U32 * (a * self.z).abs().mean(1, keepdim=True) + (a.abs() * self.e_z).mean(1, keepdim=True)
        inner = a - m0 - self.z * m1
        parts = a.abs() + m0.abs() + (self.z * m1).abs()
        e_inner = e_m0 + self.z.abs() * e_m1 + self.e_z * m1.abs() + 5 * U32 * parts
        self.dh = self.rstd * inner
        self.e_dh = self.rstd * e_inner + self.dh.abs() * (self.r_rstd + 2 * U32)
        if grad_h is not None:
            self.dh = self.dh + grad_h.double()
            self.e_dh = self.e_dh + U32 * (self.dh.abs() + self.e_dh)
        rows = g.shape[0]
        self.dgamma, self.dbeta = (g * self.z).sum(0), g.sum(0)
        self.e_dgamma = (g.abs() * self.e_z).sum(0) + (rows + 3) * U32 * (g * self.z).abs().sum(0)
        self.e_dbeta = (rows + 2) * U32 * g.abs().sum(0)
        return self
