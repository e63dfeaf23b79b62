"""The operators of eight-bit serving, as cases that can be timed and checked:
the residual add and RMS norm with an int8 result, rows of activations or
weights taken to int8 with a scale each, the int8 matrix product with scales
for each token and channel, and the choice of the next token from logits.

Where `own` is false run() computes them from elementary torch operations;
where it is true it calls mi355x_pjrt.kernels.  exact() is their definition
in 64 bits, on its own.
"""

from __future__ import annotations

import math
import os
import sys

import torch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for _p in (_ROOT, os.path.join(_ROOT, "mccl-jax_amd")):
    if _p not in sys.path:
        sys.path.insert(0, _p)

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # One new token of GPT-2-small: the residual stream into the next block's norm.  Latency alone.
        {"name": "norm_token", "kind": "norm", "rows": 1, "cols": 768, "dtype": "bf16", "residual": True},
        # A prompt of a model of width 4096: every block does this twice.
        {"name": "norm_prompt", "kind": "norm", "rows": 8192, "cols": 4096, "dtype": "bf16", "residual": True},
        # fp32 rows of an odd width without a residual branch: the first norm of an fp32 stream.
        {"name": "norm_odd_f32", "kind": "norm", "rows": 1023, "cols": 1001, "dtype": "f32", "residual": False},
        # The MLP's hidden rows of 16 running sequences: activation and rounding ahead of the second product.
        {"name": "quantize_tokens", "kind": "quantize", "rows": 16, "cols": 16384, "dtype": "bf16", "gelu": True},
        # An embedding table of 50257 rows taken to eight bits, a scale for each output channel of the head.
        {"name": "quantize_weights", "kind": "quantize", "rows": 50257, "cols": 768, "dtype": "f32", "gelu": False},
        # One token through GPT-2-small's fused QKV projection: the smallest product.
        {"name": "product_one", "kind": "product", "rows": 1, "inner": 768, "cols": 2304, "out": "bf16", "bias": True},
        # 16 running sequences through the wide MLP's first product: the weights are the traffic.
        {"name": "product_tokens", "kind": "product", "rows": 16, "inner": 4096, "cols": 16384, "out": "bf16",
         "bias": True},
        # A prompt of 8192 tokens through the same product: matrix rate.
        {"name": "product_prompt", "kind": "product", "rows": 8192, "inner": 4096, "cols": 16384, "out": "bf16",
         "bias": True},
        # A batch of odd size through the vocabulary head: fp32 logits in rows of 50257.
        {"name": "product_head_odd", "kind": "product", "rows": 333, "inner": 768, "cols": 50257, "out": "f32",
         "bias": False},
        # The next token of one sequence: top-k and top-p.  Latency.
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 50257, "dtype": "bf16", "limits": "all"},
        # The next tokens of 32 sequences, each with its own temperature and limits.
        {"name": "sample_batch", "kind": "sample", "rows": 32, "vocab": 50257, "dtype": "bf16", "limits": "all"},
        # 256 sequences on fp32 logits with a nucleus alone: no top-k bounds the rows that count.
        {"name": "sample_nucleus", "kind": "sample", "rows": 256, "vocab": 50257, "dtype": "f32", "limits": "top_p"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "quantize", "product", "product", "product", "sample", "sample"])
    if kind == "norm":
        cols = _log(rng, 64, 16384)
        return {"kind": kind, "rows": min(_log(rng, 1, 32768), max(1, (1 << 25) // cols)), "cols": cols,
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "residual": rng.random() < 0.75}
    if kind == "quantize":
        cols = _log(rng, 64, 16384)
        return {"kind": kind, "rows": min(_log(rng, 1, 50257), max(1, (1 << 25) // cols)), "cols": cols,
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "gelu": rng.random() < 0.5}
    if kind == "product":
        # most widths are multiples of 16, as a model's are; the rest are whatever they are
        inner, cols = _log(rng, 64, 16384), _log(rng, 64, 50257)
        if rng.random() < 0.8:
            inner = inner // 16 * 16
        if rng.random() < 0.7:
            cols = cols // 16 * 16
        inner = min(inner, (1 << 28) // cols)
        rows = min(_log(rng, 1, 8192), max(1, (1 << 39) // (inner * cols)))
        return {"kind": kind, "rows": rows, "inner": inner, "cols": cols,
                "out": rng.choice(["bf16", "bf16", "f16", "f32"]), "bias": rng.random() < 0.5}
    vocab = _log(rng, 500, 160000)
    return {"kind": kind, "rows": min(_log(rng, 1, 512), max(1, (1 << 24) // vocab)), "vocab": vocab,
            "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
            "limits": rng.choice(["all", "all", "top_p", "top_k", "none"])}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dtype)


def _choice(g, rows, values, dtype):
    at = torch.randint(len(values), (rows,), generator=g, device=DEV)
    return torch.tensor(values, device=DEV, dtype=dtype)[at]


def _int8(g, rows, cols, std):
    """Rows as a program that serves in eight bits holds them: values and one scale each."""
    w = _normal(g, (rows, cols), std=std)
    scale = w.abs().amax(dim=1) / 127
    return torch.round(w / scale[:, None]).to(torch.int8), scale


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "norm":
        shape, dt = (case["rows"], case["cols"]), DT[case["dtype"]]
        # the residual stream grows with depth, and a few of its channels stand out
        x = _normal(g, shape) * torch.exp(_normal(g, (1, case["cols"]), std=0.5)) * 2.0
        return {"case": case, "x": x.to(dt), "r": _normal(g, shape, dt) if case["residual"] else None,
                "gamma": _normal(g, (case["cols"],), dt, 0.1, 1.0)}
    if kind == "quantize":
        return {"case": case, "x": _normal(g, (case["rows"], case["cols"]), DT[case["dtype"]],
                                           1.0 if case["gelu"] else 0.02)}
    if kind == "product":
        # the weights are stored by output channel, k contiguous, and multiplied as their transposed view
        a, sa = _int8(g, case["rows"], case["inner"], 1.0)
        w, sw = _int8(g, case["cols"], case["inner"], 1 / math.sqrt(case["inner"]))
        return {"case": case, "a": a, "sa": sa, "b": w.t(), "sb": sw,
                "bias": _normal(g, (case["cols"],), DT[case["out"]], 0.1) if case["bias"] else None}
    rows, limits = case["rows"], case["limits"]
    s = {"case": case, "x": _normal(g, (rows, case["vocab"]), DT[case["dtype"]], 3.0),
         "u": torch.rand((rows,), generator=g, device=DEV),
         # requests differ: greedy ones among them
         "temperature": _choice(g, rows, [0.0, 0.5, 0.7, 1.0, 1.0, 1.3], torch.float32),
         "top_k": None, "top_p": None, "min_p": None}
    if limits in ("all", "top_k"):
        s["top_k"] = _choice(g, rows, [0, 1, 20, 50, 400], torch.int32)
    if limits in ("all", "top_p"):
        s["top_p"] = _choice(g, rows, [0.6, 0.9, 0.95, 1.0], torch.float32)
    if limits == "all":
        s["min_p"] = _choice(g, rows, [0.0, 0.0, 0.02, 0.1], torch.float32)
    return s


# ---------------------------------------------------------------- plain forms
def _plain_rows(y, dtype):
    """The values that eight-bit rows of y stand for."""
    scale = y.abs().amax(dim=1, keepdim=True) / 127
    q = torch.round(y / torch.where(scale > 0, scale, torch.ones_like(scale)))
    return (q * scale).to(dtype), scale[:, 0]


def _plain_norm(s):
    x = s["x"]
    t = x.float() if s["r"] is None else (x.float() + s["r"].float()).to(x.dtype).float()
    y = t * torch.rsqrt(t.square().mean(dim=1, keepdim=True) + 1e-6) * s["gamma"].float()
    values, scale = _plain_rows(y, torch.bfloat16)
    out = {"values": values, "scale": scale}
    if s["r"] is not None:
        out["sum"] = t.to(x.dtype)
    return out


def _plain_quantize(s):
    y = s["x"].float()
    if s["case"]["gelu"]:
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    values, scale = _plain_rows(y, torch.bfloat16)
    return {"values": values, "scale": scale}


def _plain_product(s):
    c = (s["a"].float() @ s["b"].float()) * s["sa"][:, None] * s["sb"]
    if s["bias"] is not None:
        c = c + s["bias"].float()
    return c.to(DT[s["case"]["out"]])


def _plain_sample(s):
    """Weights and masses in 64 bits: a mass next to a limit decides which token it is."""
    x, V = s["x"], s["x"].shape[1]
    greedy = s["temperature"] == 0
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None]
    ranked, at = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((ranked.double() - ranked[:, :1].double()) / t)
    rank = torch.arange(V, device=DEV)
    k = torch.full_like(greedy, V, dtype=torch.int32) if s["top_k"] is None else s["top_k"]
    k = torch.where(k <= 0, V, k)
    keep = rank < torch.where(greedy, 1, k)[:, None]
    if s["top_p"] is not None:
        w = w * keep
        before = torch.cumsum(w, dim=1) - w
        keep = keep & ((before < s["top_p"].double()[:, None] * w.sum(dim=1, keepdim=True)) | (rank == 0)
                       | (s["top_p"] >= 1)[:, None])
    if s["min_p"] is not None:
        keep = keep & (w >= s["min_p"].double()[:, None])
    w = torch.zeros_like(w).scatter_(1, at, w * keep)  # back in the order of the vocabulary
    mass = torch.cumsum(w, dim=1)
    total = mass[:, -1:]
    token = torch.argmax((mass > s["u"].double()[:, None] * total).to(torch.int8), dim=1)
    logprob = torch.log(w.gather(1, token[:, None]) / total)[:, 0]
    return {"token": token.to(torch.int32), "logprob": logprob.float()}


# ---------------------------------------------------------------- the framework's operators
def _own_run(s):
    from mi355x_pjrt import kernels as K

    case, kind = s["case"], s["case"]["kind"]
    if kind == "norm":
        q, scale, total = K.add_rmsnorm_int8(s["x"], s["r"], s["gamma"], eps=1e-6)
        out = {"values": K.dequantize_rows(q, scale, torch.bfloat16), "scale": scale}
        if s["r"] is not None:
            out["sum"] = total
        return out
    if kind == "quantize":
        q, scale = K.quantize_rows(s["x"], gelu=case["gelu"])
        return {"values": K.dequantize_rows(q, scale, torch.bfloat16), "scale": scale}
    if kind == "product":
        return K.gemm_int8(s["a"], s["sa"], s["b"], s["sb"], out_dtype=DT[case["out"]], bias=s["bias"])
    token, logprob = K.sample_rows(s["x"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                   min_p=s["min_p"])
    return {"token": token, "logprob": logprob}


def run(state):
    if own:
        return _own_run(state)
    return {"norm": _plain_norm, "quantize": _plain_quantize, "product": _plain_product,
            "sample": _plain_sample}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind in ("norm", "quantize"):
        n, esz = case["rows"] * case["cols"], 4 if case["dtype"] == "f32" else 2
        # the values come back through their eight bits: one byte written and read, two written
        passes = 3 if kind == "norm" and case["residual"] else 1
        return {"bytes": n * (passes * esz + 4) + 4 * case["rows"], "flops": n * (12 if kind == "norm" else 6)}
    if kind == "product":
        M, K, N = case["rows"], case["inner"], case["cols"]
        return {"bytes": M * K + K * N + M * N * (4 if case["out"] == "f32" else 2) + 4 * (M + N),
                "flops": 2 * M * N * K}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + 24 * case["rows"], "flops": 8 * n}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_int8(y):
    top = y.abs().max(dim=1).values
    step = top / 127
    unit = torch.where(step > 0, 1 / step, 0.0)
    return torch.round(y * unit[:, None]) * step[:, None], step


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "norm":
        t = s["x"].double()
        if s["r"] is not None:
            t = (t + s["r"].double()).to(s["x"].dtype).double()  # the stream is kept in its own type
        y = t * s["gamma"].double() / torch.sqrt((t ** 2).sum(dim=1, keepdim=True) / case["cols"] + 1e-6)
        values, step = _exact_int8(y)
        return {"values": values, "scale": step, **({"sum": t} if s["r"] is not None else {})}
    if kind == "quantize":
        y = s["x"].double()
        if case["gelu"]:
            y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        values, step = _exact_int8(y)
        return {"values": values, "scale": step}
    if kind == "product":
        c = s["a"].double().mul(s["sa"].double()[:, None]) @ s["b"].double().mul(s["sb"].double()[None, :])
        return c if s["bias"] is None else c + s["bias"].double()
    return {"token": None, "logprob": _exact_logprob(s)}


def _exact_logprob(s):
    """Row by row, as the definition reads: rank, cut, and walk the vocabulary."""
    got = []
    for r in range(s["x"].shape[0]):
        x, t = s["x"][r].double(), float(s["temperature"][r])
        V = x.numel()
        order = torch.argsort(x, descending=True, stable=True)
        k = V if s["top_k"] is None or int(s["top_k"][r]) <= 0 else min(V, int(s["top_k"][r]))
        k, t = (1, 1.0) if t == 0 else (k, t)
        p = torch.softmax(x[order[:k]] / t, dim=0)
        if s["top_p"] is not None and float(s["top_p"][r]) < 1:
            before = torch.cat([p.new_zeros(1), torch.cumsum(p, dim=0)[:-1]])
            p = p[:max(1, int((before < float(s["top_p"][r])).sum()))]
        if s["min_p"] is not None:
            p = p[:int((p >= float(s["min_p"][r]) * p[0]).sum())]
        ids, by_id = torch.sort(order[:p.numel()])
        mass = torch.cumsum(p[by_id] / p.sum(), dim=0)
        at = min(int((mass <= float(s["u"][r])).sum()), p.numel() - 1)
        got.append(torch.log(p[by_id][at] / p.sum()))
    return torch.stack(got)
