"""Two operators of a training step, as cases that can be timed and checked:
softmax cross entropy over a large vocabulary from hidden rows and the
embedding (the logits are never kept), its gradient, and dropout from a
counter-based generator (the mask is never kept) with the bias and residual
around it, and its gradient.

Where `own` is false run() computes them from elementary torch operations;
where it is true it calls mi355x_pjrt.kernels.  exact() is their definition
in 64 bits, on its own.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for _p in (_ROOT, os.path.join(_ROOT, "mccl-jax_amd")):
    if _p not in sys.path:
        sys.path.insert(0, _p)

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
IGNORE = -100


def listed():
    return [
        # The last tokens of 16 sequences scored against GPT-2-small's embedding: the weights are the traffic.
        {"name": "loss_few", "kind": "loss", "rows": 16, "width": 768, "vocab": 50257, "dtype": "bf16",
         "ignore": False},
        # The training step of GPT-2-small: 8 sequences of 1024 tokens.
        {"name": "loss_batch", "kind": "loss", "rows": 8192, "width": 768, "vocab": 50257, "dtype": "bf16",
         "ignore": False},
        # A padded batch of odd size, fp16, a tenth of its labels ignored.
        {"name": "loss_odd", "kind": "loss", "rows": 3001, "width": 2048, "vocab": 32003, "dtype": "f16",
         "ignore": True},
        # The gradient of a small last batch: latency, and one pass over the weights and their gradient.
        {"name": "grad_few", "kind": "grad", "rows": 100, "width": 768, "vocab": 50257, "dtype": "bf16",
         "ignore": False, "row_grad": False},
        # The gradient in the training step of GPT-2-small.
        {"name": "grad_batch", "kind": "grad", "rows": 8192, "width": 768, "vocab": 50257, "dtype": "bf16",
         "ignore": False, "row_grad": False},
        # A padded batch of odd sizes throughout, a weight for each token's loss.
        {"name": "grad_odd", "kind": "grad", "rows": 1777, "width": 1001, "vocab": 30011, "dtype": "f16",
         "ignore": True, "row_grad": True},
        # A wide model with a large vocabulary: matrix rate.
        {"name": "grad_wide", "kind": "grad", "rows": 8192, "width": 4096, "vocab": 65536, "dtype": "bf16",
         "ignore": True, "row_grad": False},
        # A projection's output of 64 tokens into the residual stream of GPT-2-small.  Latency.
        {"name": "drop_few", "kind": "drop", "rows": 64, "cols": 768, "dtype": "bf16", "p": 0.1, "bias": True,
         "residual": True},
        # The same in the training step: twice for every block.
        {"name": "drop_batch", "kind": "drop", "rows": 8192, "cols": 768, "dtype": "bf16", "p": 0.1, "bias": True,
         "residual": True},
        # Plain dropout of fp32 rows of an odd width, past the caches.
        {"name": "drop_odd", "kind": "drop", "rows": 20011, "cols": 4097, "dtype": "f32", "p": 0.25, "bias": False,
         "residual": False},
        # The gradient through a projection's dropout in the training step, and of the projection's bias.
        {"name": "dropgrad_batch", "kind": "dropgrad", "rows": 8192, "cols": 768, "dtype": "bf16", "p": 0.1,
         "bias": True},
        # fp16 rows of an odd width: a small batch.
        {"name": "dropgrad_odd", "kind": "dropgrad", "rows": 333, "cols": 1001, "dtype": "f16", "p": 0.5,
         "bias": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["loss", "loss", "grad", "grad", "grad", "drop", "drop", "dropgrad"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
    if kind in ("loss", "grad"):
        width, vocab = _log(rng, 64, 4096), _log(rng, 1000, 131072)
        # most widths are multiples of 16, as a model's are; the rest are whatever they are
        if rng.random() < 0.8:
            width = width // 16 * 16
        work = 1 << (35 if dtype == "f32" else 41)
        rows = min(_log(rng, 1, 16384), (1 << 29) // vocab, max(1, work // (width * vocab)))
        case = {"kind": kind, "rows": rows, "width": width, "vocab": vocab, "dtype": dtype,
                "ignore": rng.random() < 0.4}
        if kind == "grad":
            case["row_grad"] = rng.random() < 0.4
        return case
    cols = _log(rng, 64, 16384)
    if rng.random() < 0.7:
        cols = cols // 16 * 16
    rows = min(_log(rng, 1, 65536), max(1, (1 << 26) // cols))
    case = {"kind": kind, "rows": rows, "cols": cols, "dtype": dtype, "p": rng.choice([0.05, 0.1, 0.1, 0.25, 0.5]),
            "bias": rng.random() < 0.6}
    if kind == "drop":
        case["residual"] = rng.random() < 0.6
    return case


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def prepare(case, seed):
    g, kind, dt = _gen(seed), case["kind"], DT[case["dtype"]]
    if kind in ("loss", "grad"):
        N, D, V = case["rows"], case["width"], case["vocab"]
        # logits of a deviation of about 2, and rows that lean to their label by up to 10
        std = 2 / math.sqrt(D)
        w = _normal(g, (V, D), dt, std)
        labels = torch.randint(V, (N,), generator=g, device=DEV)
        lean = torch.rand((N, 1), generator=g, device=DEV) * 10
        x = (_normal(g, (N, D)) + lean * w[labels].float() / (D * std * std)).to(dt)
        if case["ignore"]:
            drop = torch.rand((N,), generator=g, device=DEV) < 0.1
            labels = torch.where(drop, torch.full_like(labels, IGNORE), labels)
        s = {"case": case, "x": x, "w": w, "labels": labels.to(torch.int32)}
        if kind == "grad":
            # what the forward pass left: the log-sum-exp of each row
            s["lse"] = torch.cat([torch.logsumexp(x[i:i + 1024].float() @ w.float().t(), dim=1)
                                  for i in range(0, N, 1024)])
            s["row_grad"] = torch.rand((N,), generator=g, device=DEV) if case["row_grad"] else None
            # the mean's gradient; fp16 gradients are scaled up, as a program that trains in fp16 scales its loss
            s["scale"] = min(65536.0 / N, 256.0) if dt == torch.float16 else 1.0 / N
        return s
    shape = (case["rows"], case["cols"])
    s = {"case": case, "seed": seed * 0x9E3779B97F4A7C15 % (1 << 63), "offset": 1000 + seed % 1000}
    if kind == "drop":
        s["x"] = _normal(g, shape, dt)
        s["bias"] = _normal(g, shape[1:], dt, 0.1) if case["bias"] else None
        s["residual"] = _normal(g, shape, dt, 3.0) if case["residual"] else None
    else:
        s["dy"] = _normal(g, shape, dt, 1e-2)
    return s


# ---------------------------------------------------------------- plain forms
def _plain_softmax_terms(s):
    x, w, labels = s["x"].float(), s["w"].float(), s["labels"].long()
    logits = x @ w.t()
    at = labels.clamp(0, w.shape[0] - 1)[:, None]
    return x, w, logits, at, labels != IGNORE


def _plain_loss(s):
    _, _, logits, at, counts = _plain_softmax_terms(s)
    top = logits.amax(dim=1)
    lse = top + torch.log(torch.exp(logits - top[:, None]).sum(dim=1))
    loss = torch.where(counts, lse - logits.gather(1, at)[:, 0], torch.zeros_like(lse))
    return {"loss": loss, "lse": lse}


def _plain_grad(s):
    x, w, logits, at, counts = _plain_softmax_terms(s)
    g = torch.exp(logits - s["lse"][:, None])
    g.scatter_add_(1, at, torch.full_like(s["lse"], -1.0)[:, None])
    scale = torch.full_like(s["lse"], s["scale"]) if s["row_grad"] is None else s["row_grad"] * s["scale"]
    g = g * (scale * counts)[:, None]
    return {"dx": (g @ w).to(s["x"].dtype), "dw": (g.t() @ x).to(s["w"].dtype)}


def _plain_keep(s):
    """The elements that are kept: 16 bits each from Philox-4x32-10, products of 32 bits in halves of 16."""
    rows, cols = s["case"]["rows"], s["case"]["cols"]
    low = 0xFFFFFFFF
    blocks = (cols + 7) // 8
    shape = (rows, blocks)
    c = [torch.arange(blocks, device=DEV).expand(shape), torch.arange(rows, device=DEV)[:, None].expand(shape),
         torch.full(shape, s["offset"] & low, device=DEV), torch.full(shape, s["offset"] >> 32, device=DEV)]
    k0, k1 = s["seed"] & low, s["seed"] >> 32
    for _ in range(10):
        hi = [(m * (v >> 16) + ((m * (v & 0xFFFF)) >> 16)) >> 16 for m, v in ((0xD2511F53, c[0]), (0xCD9E8D57, c[2]))]
        lo = [(m * v) & low for m, v in ((0xD2511F53, c[0]), (0xCD9E8D57, c[2]))]
        c = [hi[1] ^ c[1] ^ k0, lo[1], hi[0] ^ c[3] ^ k1, lo[0]]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    fields = torch.stack([f for v in c for f in (v & 0xFFFF, v >> 16)], dim=2)
    return fields.reshape(rows, blocks * 8)[:, :cols] >= round(s["case"]["p"] * 65536)


def _plain_drop(s):
    keep, cut = _plain_keep(s), round(s["case"]["p"] * 65536)
    if s["case"]["kind"] == "dropgrad":
        y = torch.where(keep, s["dy"].float(), 0.0) * (65536 / (65536 - cut))
        out = {"dx": y.to(s["dy"].dtype)}
        if s["case"]["bias"]:
            out["dbias"] = y.double().sum(dim=0).float()
        return out
    y = s["x"].float()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = torch.where(keep, y, 0.0) * (65536 / (65536 - cut))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


# ---------------------------------------------------------------- the framework's operators
def _own_run(s):
    from mi355x_pjrt import kernels as K

    case, kind = s["case"], s["case"]["kind"]
    if kind == "loss":
        loss, lse = K.linear_xent(s["x"], s["w"], s["labels"], ignore_index=IGNORE if case["ignore"] else None)
        return {"loss": loss, "lse": lse}
    if kind == "grad":
        dx, dw = K.linear_xent_bwd(s["x"], s["w"], s["labels"], s["lse"], grad_scale=s["scale"],
                                   row_grad=s["row_grad"], ignore_index=IGNORE if case["ignore"] else None)
        return {"dx": dx, "dw": dw}
    if kind == "drop":
        return K.dropout_add(s["x"], case["p"], s["seed"], offset=s["offset"], bias=s["bias"],
                             residual=s["residual"])
    dx, dbias = K.dropout_add_bwd(s["dy"], case["p"], s["seed"], offset=s["offset"], want_colsum=case["bias"])
    return {"dx": dx, "dbias": dbias} if case["bias"] else {"dx": dx}


def run(state):
    if own:
        return _own_run(state)
    return {"loss": _plain_loss, "grad": _plain_grad, "drop": _plain_drop,
            "dropgrad": _plain_drop}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- work
def work(case):
    kind, esz = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind in ("loss", "grad"):
        N, D, V = case["rows"], case["width"], case["vocab"]
        if kind == "loss":
            return {"bytes": (N + V) * D * esz + 12 * N, "flops": 2 * N * V * D}
        # the logits again, and the products that carry their gradient to x and to w
        return {"bytes": 2 * (N + V) * D * esz + (12 if case["row_grad"] else 8) * N, "flops": 6 * N * V * D}
    n = case["rows"] * case["cols"]
    passes = 3 if kind == "drop" and case["residual"] else 2
    extra = case["cols"] * (esz if kind == "drop" else 4) if case["bias"] else 0
    return {"bytes": n * passes * esz + extra, "flops": 3 * n}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_fields(s):
    """The generator's 16-bit fields [rows, cols], from unsigned products of 64 bits on the host."""
    rows, cols = s["case"]["rows"], s["case"]["cols"]
    u, mask, sh = np.uint64, np.uint64(0xFFFFFFFF), np.uint64(32)
    n = -(-cols // 8)
    a = np.tile(np.arange(n, dtype=u), rows)
    b = np.repeat(np.arange(rows, dtype=u), n)
    c, d = np.full(rows * n, s["offset"] % 2 ** 32, u), np.full(rows * n, s["offset"] // 2 ** 32, u)
    for r in range(10):
        key = [u((s["seed"] % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32), u((s["seed"] // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32)]
        pa, pc = a * u(0xD2511F53), c * u(0xCD9E8D57)
        a, b, c, d = (pc >> sh) ^ b ^ key[0], pc & mask, (pa >> sh) ^ d ^ key[1], pa & mask
    words = np.stack([a, b, c, d], axis=1).astype("<u4")
    return torch.from_numpy(words.view("<u2").reshape(rows, n * 8)[:, :cols].astype(np.int32)).to(DEV)


def _exact_drop(s):
    cut = round(s["case"]["p"] * 65536)
    weight = (_exact_fields(s) >= cut).double() / (1 - cut / 65536)
    if s["case"]["kind"] == "dropgrad":
        dx = s["dy"].double() * weight
        return {"dx": dx, "dbias": dx.sum(dim=0)} if s["case"]["bias"] else {"dx": dx}
    branch = s["x"].double() if s["bias"] is None else s["x"].double() + s["bias"].double()
    return branch * weight if s["residual"] is None else s["residual"].double() + branch * weight


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("drop", "dropgrad"):
        return _exact_drop(s)
    x, w, labels = s["x"].double(), s["w"].double(), s["labels"].long()
    if case["kind"] == "loss":
        lse, loss = [], []
        for i in range(0, case["rows"], 512):
            z = x[i:i + 512] @ w.t()
            lse.append(torch.logsumexp(z, dim=1))
            t = labels[i:i + 512]
            got = lse[-1] - z[torch.arange(t.numel(), device=DEV), torch.where(t < 0, 0, t)]
            loss.append(torch.where(t < 0, 0.0, got))
        return {"loss": torch.cat(loss), "lse": torch.cat(lse)}
    dx, dw = torch.empty_like(x), torch.zeros_like(w)
    for i in range(0, case["rows"], 512):
        xi, t = x[i:i + 512], labels[i:i + 512]
        p = torch.exp(xi @ w.t() - s["lse"][i:i + 512].double()[:, None])
        used = torch.nonzero(t >= 0)[:, 0]
        p[used, t[used]] -= 1
        weight = s["scale"] * (t >= 0).double()
        if s["row_grad"] is not None:
            weight = weight * s["row_grad"][i:i + 512].double()
        p *= weight[:, None]
        dx[i:i + 512] = p @ w
        dw += p.t() @ xi
    return {"dx": dx, "dw": dw}
