"""Definitions in 64 bits of the cross entropy from hidden rows and of the
counter-based dropout, with bounds that count the roundings of the kernels."""

import numpy as np
import torch

H32 = 2.0 ** -24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def subnormal(dtype):
    """Half the distance of the smallest numbers of a type."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------ Philox-4x32, 10 rounds
def philox(counter, key):
    """The 4 words for counters [..., 4] and a key of two words (uint64 arrays of 32-bit numbers)."""
    u, mask, sh = np.uint64, np.uint64(0xFFFFFFFF), np.uint64(32)
    a, b, c, d = (np.asarray(counter, dtype=u)[..., i] for i in range(4))
    k0, k1 = int(key[0]), int(key[1])
    for _ in range(10):
        pa, pc = a * u(0xD2511F53), c * u(0xCD9E8D57)
        a, b, c, d = (pc >> sh) ^ b ^ u(k0), pc & mask, (pa >> sh) ^ d ^ u(k1), pa & mask
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return np.stack([a, b, c, d], axis=-1)


def dropout_keep(rows, cols, p, seed, offset):
    """keep [rows, cols] (bool) and the scale 65536 / (65536 - T)."""
    groups = -(-cols // 8)
    ctr = np.zeros((rows, groups, 4), np.uint64)
    ctr[..., 0] = np.arange(groups)[None, :]
    ctr[..., 1] = np.arange(rows)[:, None]
    ctr[..., 2] = offset % 2 ** 32
    ctr[..., 3] = offset // 2 ** 32
    words = philox(ctr, (seed % 2 ** 32, seed // 2 ** 32))
    fields = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], axis=-1).reshape(rows, groups * 8)[:, :cols]
    cut = round(p * 65536)
    return torch.from_numpy(fields.astype(np.int64) >= cut), (65536 / (65536 - cut) if cut < 65536 else 0.0)


# ------------------------------------------------------------------ cross entropy
def _counts(labels, ignore):
    return torch.ones_like(labels, dtype=torch.bool) if ignore is None else labels != ignore


def xent(x, w, labels, ignore=None):
    """(loss, lse, bound) in 64 bits on x's device.  The bound of both: a logit is a sum of
    width products, each addition a rounding of at most the sum of the products' sizes; an
    exponent takes two roundings and the exponential two steps; a tile's sum 40 additions, and a
    row's tiles are joined one after the other, 16 runs of them, each joint two exponentials."""
    x, w, labels = x.double(), w.double(), labels.long()
    vocab = w.shape[0]
    z = x @ w.t()
    lse = torch.logsumexp(z, dim=1)
    inside = (labels >= 0) & (labels < vocab)
    t = z.gather(1, torch.where(inside, labels, 0)[:, None])[:, 0]
    loss = torch.where(_counts(labels, ignore), lse - torch.where(inside, t, 0.0), 0.0)
    dz = ((x.shape[1] + 1) * H32 * (x.abs() @ w.abs().t())).amax(dim=1)
    span = z.amax(dim=1) - z.amin(dim=1) + 1
    joints = vocab / 128 / 16 + 4
    bound = 2 * dz + H32 * ((3 * span + 4) * joints + 40 + joints + 3 * lse.abs() + 4 * z.abs().amax(dim=1))
    return loss, lse, bound


def xent_grad(x, w, labels, lse, scale=1.0, row_grad=None, ignore=None, dw_dtype=None, twice=False):
    """(dx, dw, bound of dx, bound of dw): g is rounded once to x's type (fp16: of a power of two
    times it, so that what is lost below its normal numbers is 2^-40 of the largest), sums are
    fp32 additions in any order, results are rounded once.  twice: what g's rounding leaves is
    rounded to a second number of the type."""
    dtype, dw_dtype = x.dtype, dw_dtype or w.dtype
    used = _counts(labels.long(), ignore)
    x = torch.where(used[:, None], x.double(), 0.0)  # whatever an ignored row holds
    w, labels = w.double(), labels.long()
    z = x @ w.t()
    p = torch.exp(z - lse.double()[:, None])
    inside = (labels >= 0) & (labels < w.shape[0])
    hot = torch.zeros_like(p).scatter_(1, torch.where(inside, labels, 0)[:, None], inside.double()[:, None])
    r = used.double() * (1.0 if row_grad is None else row_grad.double())
    g = (p - hot) * r[:, None]
    # of g: its rounding, and the exponential's error
    dz = (x.shape[1] + 1) * H32 * (x.abs() @ w.abs().t())
    e = dz + H32 * (3 * (z - lse.double()[:, None]).abs() + 4)
    dg = half_step(dtype) ** (2 if twice else 1) * g.abs() + (p * e + 2 * H32 * (p + hot)) * r.abs()[:, None]
    if dtype == torch.float16:
        dg = dg + 2.0 ** -40 * r.abs().max()
    dx, dw = g @ w * scale, g.t() @ x * scale
    s = abs(scale)

    def bound(d, size, n, out, t):
        return 1.01 * s * (d + (n + 2) * H32 * size) + (half_step(t) + 2 * H32) * out.abs() + subnormal(t)

    return (dx, dw, bound(dg @ w.abs(), g.abs() @ w.abs(), w.shape[0], dx, dtype),
            bound(dg.t() @ x.abs(), g.abs().t() @ x.abs(), x.shape[0], dw, dw_dtype))
