"""Eight-bit serving on the MI355X: add_rmsnorm_int8, quantize_rows,
dequantize_rows, gemm_int8 and sample_rows against their definitions in 64 bits
on the host.

Bounds count roundings: one is off by at most half a step, eps / 2 relative
(2^-24 in fp32).  Whole numbers (sums of the product, tokens) are exact.
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

H32 = 2.0 ** -24  # half a step of fp32
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def K(cuda):
    from mi355x_pjrt import kernels

    kernels.lib()
    return kernels


def _f64(t):
    return t.detach().cpu().double()


def _normal(seed, shape, dtype=torch.float32, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std + mean).to(dtype).cuda()


def _rows_view(t, pitch, off=0):
    """t's rows `pitch` elements apart, `off` past an aligned start, in a sea of 77s."""
    sea = torch.full((t.shape[0] * pitch + off + 64,), 77, dtype=t.dtype, device=t.device)
    v = sea[off:off + t.shape[0] * pitch].view(t.shape[0], pitch)[:, :t.shape[1]]
    v.copy_(t)
    return sea, v


def _check_rows(q, scale, y, rel):
    """q and scale against the exact rows y (64 bits, host).  y carries a relative
    error of at most `rel` in the kernel; the step 127 / max two roundings more,
    of a number of up to 127 steps."""
    q, scale = _f64(q), _f64(scale)
    want = y.abs().amax(dim=1) / 127
    assert torch.all((scale - want).abs() <= (rel + 2 * H32) * want)
    off = (q - y / torch.where(want > 0, want, 1.0)[:, None]).abs()
    assert float(off.max()) <= 0.5 + 127 * (2 * rel + 2 * H32)
    assert float(q.abs().max()) <= 127


# ------------------------------------------------------------------ rows to eight bits
# one element, odd ends, the limits of each team and of the registers, past them
COLS = [1, 3, 7, 8, 9, 64, 100, 511, 512, 513, 768, 1001, 2050, 4096, 4104, 8200, 16384, 32768, 32769, 40007]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", COLS)
def test_add_rmsnorm_int8(K, dtype, cols):
    for rows in (1, 5, 600, 2500) if cols <= 4104 else (1, 3):
        print(f"case: add_rmsnorm_int8 {rows} x {cols} {dtype}", flush=True)
        x, r = _normal(cols, (rows, cols), dtype, 3.0), _normal(cols + 1, (rows, cols), dtype)
        gamma = _normal(cols + 2, (cols,), dtype, 0.1, 1.0)
        q, scale, total = K.add_rmsnorm_int8(x, r, gamma, eps=1e-5)
        assert torch.equal(total.cpu(), (x.cpu().float() + r.cpu().float()).to(dtype))
        s = _f64(total)
        # s gamma is rounded once
        _check_rows(q, scale, s / torch.sqrt((s * s).mean(dim=1, keepdim=True) + np.float64(np.float32(1e-5))) *
                    _f64(gamma), H32)
        q, scale, total = K.add_rmsnorm_int8(x, eps=1e-5)
        assert total is x
        s = _f64(x)
        _check_rows(q, scale, s / torch.sqrt((s * s).mean(dim=1, keepdim=True) + np.float64(np.float32(1e-5))), H32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", COLS)
def test_quantize_rows_and_back(K, dtype, cols):
    for rows in (1, 600, 2500) if cols <= 4104 else (2,):
        print(f"case: quantize_rows {rows} x {cols} {dtype}", flush=True)
        x = _normal(cols, (rows, cols), dtype, 2.0)
        q, scale = K.quantize_rows(x)
        _check_rows(q, scale, _f64(x), 0.0)
        for out in TYPES:
            back = K.dequantize_rows(q, scale, out)
            want = _f64(q) * _f64(scale)[:, None]  # one product, then one rounding
            tiny = torch.finfo(out).smallest_normal * torch.finfo(out).eps
            assert torch.all((_f64(back) - want).abs() <= (torch.finfo(out).eps / 2 + H32) * want.abs() + tiny)
        x[:, 0] = 1.5  # the bound below is relative to a maximum of at least 1
        q, scale = K.quantize_rows(x, gelu=True)
        v = _f64(x)
        u = math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
        # relative to the maximum: x / (1 + e) with e's exponent off by 3 roundings of
        # itself, times |y| / max <= 1 / 2 for the exponents that matter, and the
        # exponential, the reciprocal and the product within 1, 1 and 1 / 2 steps
        _check_rows(q, scale, v / (1 + torch.exp(-2 * u)), 16 * H32)


def test_rows_of_any_pitch_and_in_place(K):
    """Odd pitches, unaligned starts, the sum over x or the residual; nothing is written past a row's end."""
    for dtype in TYPES:
        for cols, pitch, off in ((257, 301, 1), (768, 768, 3), (1030, 1033, 5), (4104, 4109, 1), (40007, 40009, 1)):
            x, r = _normal(1, (9, cols), dtype), _normal(2, (9, cols), dtype)
            gamma = _normal(3, (cols + 1,), dtype, 0.1, 1.0)[1:]
            q0, s0, t0 = K.add_rmsnorm_int8(x, r, gamma.clone())
            sea_x, xv = _rows_view(x, pitch, off)
            sea_r, rv = _rows_view(r, pitch + 2, off)
            sea_q, qv = _rows_view(torch.zeros(9, cols, dtype=torch.int8, device="cuda"), pitch, off)
            for target, sea in ((xv, sea_x), (rv, sea_r)):
                xv.copy_(x)
                rv.copy_(r)
                kept = sea.clone()
                q, s, t = K.add_rmsnorm_int8(xv, rv, gamma, sum_out=target, q=qv)
                assert t is target and q is qv
                assert torch.equal(q, q0) and torch.equal(s, s0) and torch.equal(t, t0)
                target.copy_(x if target is xv else r)
                assert torch.equal(sea, kept)
            qv.zero_()
            assert int((sea_q == 77).sum()) == sea_q.numel() - 9 * cols
            y = torch.full((9, pitch), 7, dtype=dtype, device="cuda")
            K.dequantize_rows(q0, s0, dtype, out=y[:, :cols])
            assert torch.equal(y[:, :cols], K.dequantize_rows(q0, s0, dtype)) and bool((y[:, cols:] == 7).all())
            # the same row again and again (pitch 0)
            q, s, t = K.add_rmsnorm_int8(x[:1].expand(4, cols), r[:1].expand(4, cols), gamma)
            assert torch.equal(q, q0[:1].expand(4, cols)) and torch.equal(s, s0[:1].expand(4))


@pytest.mark.parametrize("cols", [5, 768, 4104, 33000])
def test_rows_with_zeros_nan_infinities_and_huge_values(K, cols):
    x = _normal(4, (9, cols))
    x[0] = 0
    x[1, cols // 2] = math.nan
    x[2, cols - 1] = math.inf
    x[3, 0] = -math.inf
    x[4] *= 1e30        # squares past fp32's range
    x[5] = 1e-38        # below the least scale: taken as zeros
    x[6, 0] = torch.tensor(0x7F800001, dtype=torch.int32).view(torch.float32).item()
    for norm in (False, True):
        q, scale = K.add_rmsnorm_int8(x, eps=1e-6)[:2] if norm else K.quantize_rows(x)
        for r in (0, 5):
            assert float(scale[r]) == 0 and not bool(q[r].any())
        for r in (1, 2, 3, 6):
            assert math.isnan(float(scale[r])) and not bool(q[r].any())
        keep = [4, 7, 8]
        s = _f64(x[keep])
        y = s / torch.sqrt((s * s).mean(dim=1, keepdim=True) + np.float64(np.float32(1e-6))) if norm else s
        _check_rows(q[keep], scale[keep], y, H32)
    # a NaN in gamma, and an infinity of x on a zero of gamma
    gamma = torch.ones(cols, device="cuda")
    gamma[cols - 1] = 0
    _, scale, _ = K.add_rmsnorm_int8(x, None, gamma)
    assert math.isnan(float(scale[2])) and not math.isnan(float(scale[7]))
    gamma[0] = math.nan
    assert bool(torch.isnan(K.add_rmsnorm_int8(x, None, gamma)[1]).all())
    # no rows
    q, scale, total = K.add_rmsnorm_int8(x[:0], x[:0])
    assert q.shape == (0, cols) and scale.shape == (0,) and total.shape == (0, cols)


# ------------------------------------------------------------------ the product
def _check_product(got, a, sa, b, sb, bias, relu):
    """The sum is exact; its conversion, the two scales and the bias are a rounding
    each, and the result is rounded to its type once more."""
    total = a.cpu().double() @ b.cpu().double()
    want = total * _f64(sa)[:, None] * _f64(sb)
    far = 3 * H32 * want.abs()
    if bias is not None:
        want = want + _f64(bias)
        far = far + H32 * (want.abs() + far)
    if relu:
        want = want.clamp(min=0)
    info = torch.finfo(got.dtype)
    far = far + info.eps / 2 * (want.abs() + far) + info.smallest_normal * info.eps
    assert torch.all((_f64(got) - want).abs() <= far)


def _int8(seed, shape):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int8).cuda()


def _scales(seed, n):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand((n,), generator=g) * 0.02 + 1e-4).cuda()


SHAPES = [
    # one token to many, odd and even, every side one at a time small
    (1, 1, 1), (1, 64, 16), (1, 768, 2304), (2, 1000, 33), (7, 17, 50), (16, 4096, 128), (16, 4097, 129),
    (17, 128, 1000), (33, 640, 96), (48, 48, 48), (64, 2048, 257), (65, 2048, 256), (100, 130, 515), (127, 64, 128),
    (128, 128, 128), (129, 192, 130), (200, 1024, 4100), (255, 272, 384), (256, 256, 256), (257, 1040, 640),
    (300, 31, 300), (333, 768, 1003), (512, 2064, 512), (1000, 100, 1000), (1024, 1008, 2048), (2048, 4096, 768),
    (1, 16, 70001), (3, 131071, 5), (70, 131071, 70), (2500, 16, 64), (128, 512, 4096), (2048, 768, 2304),
    (40, 768, 20011), (64, 272, 9000), (300, 1001, 2000), (130, 4097, 3001),
]


@pytest.mark.parametrize("M,Kd,N", SHAPES)
def test_gemm_int8(K, M, Kd, N):
    print(f"case: gemm_int8 {M} x {Kd} x {N}", flush=True)
    a, w = _int8(M, (M, Kd)), _int8(N + 1, (N, Kd))
    sa, sb = _scales(1, M), _scales(2, N)
    for dtype, bias, relu in ((torch.bfloat16, torch.bfloat16, False), (torch.float32, None, False),
                              (torch.float16, torch.float32, True), (torch.float32, torch.float32, True)):
        # f16: sums of up to 2^14 K, scaled to its range
        f = 1e-5 if dtype == torch.float16 else 1.0
        bv = None if bias is None else _normal(3, (N,), bias)
        got = K.gemm_int8(a, sa * f, w.t(), sb, out_dtype=dtype, bias=bv, relu=relu)
        _check_product(got, a, sa * f, w.t(), sb, bv, relu)


def test_gemm_int8_largest_sums(K):
    """-128 times -128, 131071 times: 16384 below 2^31, on every kernel."""
    for M, N in ((1, 3), (64, 64), (128, 256), (300, 600)):
        a = torch.full((M, 131071), -128, dtype=torch.int8, device="cuda")
        w = torch.full((N, 131071), -128, dtype=torch.int8, device="cuda")
        w[1:2] = 127
        one = torch.ones(max(M, N), device="cuda")
        c = K.gemm_int8(a, one[:M], w.t(), one[:N], out_dtype=torch.float32)
        want = torch.full((N,), 131071 * 16384, dtype=torch.int64)
        want[1:2] = -131071 * 16256
        assert torch.equal(c.cpu(), want.float().expand(M, N))


@pytest.mark.parametrize("M", [1, 16, 40, 64, 65, 130, 300, 513])
def test_gemm_int8_pitches(K, M):
    """Aligned and unaligned rows whose ends hold other values, C rows of any pitch: nothing past N or M is written."""
    for Kd, N in ((100, 70), (512, 256), (1000, 515), (1040, 384)):
        a, w = _int8(5, (M, Kd)), _int8(6, (N, Kd))
        sa, sb = _scales(1, M), _scales(2, N)
        want = {t: K.gemm_int8(a.clone(), sa, w.clone().t(), sb, out_dtype=t) for t in (torch.bfloat16, torch.float32)}
        pad = (Kd + 15) // 16 * 16
        for pa, oa, pb, ob in ((pad, 0, pad + 16, 0), (pad + 16, 16, pad, 32), (Kd + 3, 1, Kd + 1, 2), (pad, 0, Kd, 7)):
            print(f"case: gemm_int8 pitches {M} x {Kd} x {N}: {pa} + {oa}, {pb} + {ob}", flush=True)
            _, av = _rows_view(a, pa, oa)
            _, wv = _rows_view(w, pb, ob)
            for t in want:
                for pc, oc in ((N, 0), (N + 1, 1), ((N + 7) // 8 * 8 + 8, 8)):
                    sea, c = _rows_view(torch.zeros(M, N, dtype=t, device="cuda"), pc, oc)
                    got = K.gemm_int8(av, sa, wv.t(), sb, out_dtype=t, out=c)
                    assert got is c and torch.equal(c, want[t])
                    c.fill_(77)
                    assert bool((sea == 77).all())


def test_gemm_int8_empty_and_special_scales(K):
    a, w = _int8(1, (5, 64)), _int8(2, (9, 64))
    sa, sb = _scales(1, 5), _scales(2, 9)
    bias = _normal(3, (9,))
    c = K.gemm_int8(a[:, :0], sa, w[:, :0].t(), sb, out_dtype=torch.float32, bias=bias)
    assert torch.equal(c, bias.expand(5, 9))
    assert K.gemm_int8(a[:0], sa[:0], w.t(), sb).shape == (0, 9)
    assert K.gemm_int8(a, sa, w[:0].t(), sb[:0]).shape == (5, 0)
    sa[2] = math.nan
    sb[4] = 0
    c = K.gemm_int8(a, sa, w.t(), sb, out_dtype=torch.float32)
    assert bool(torch.isnan(c[2]).all()) and not bool(torch.isnan(c[[0, 1, 3, 4]]).any())
    assert not bool(c[[0, 1, 3, 4], 4].any())


# ------------------------------------------------------------------ sampling
def _want(x, u, t, k, p, m):
    """(token, logprob) of one row by the definition, in 64 bits."""
    x = np.asarray(x, np.float64)
    V = x.size
    if np.isnan(x).any() or np.isposinf(x).any() or not (x > -np.inf).any() or any(
            math.isnan(v) for v in (u, t, p, m)) or t < 0 or math.isinf(t):
        return -1, math.nan
    if t == 0:
        return int(np.argmax(x)), 0.0
    order = np.argsort(-x, kind="stable")
    w = np.exp((x[order] - x.max()) / t)
    keep = np.arange(V) < (k if k > 0 else V)
    w = np.where(keep, w, 0)
    if p < 1:
        before = np.cumsum(w) - w
        keep &= (before < p * w.sum()) | (np.arange(V) == 0)
    keep &= w >= min(m, 1.0)
    full = np.zeros(V)
    full[order] = w * keep
    mass = np.cumsum(full)
    at = np.flatnonzero(mass > u * mass[-1])
    i = int(at[0]) if at.size else int(np.flatnonzero(full)[-1])
    return i, math.log(full[i] / mass[-1])


def _check_sample(K, x, u, t=1.0, k=0, p=1.0, m=0.0, index_dtype=torch.int32):
    rows = x.shape[0]
    as_list = lambda v: v.tolist() if isinstance(v, torch.Tensor) else [float(np.float32(v))] * rows  # noqa: E731
    token, logprob = K.sample_rows(x, u, temperature=t, top_k=k, top_p=p, min_p=m, index_dtype=index_dtype)
    assert token.dtype == index_dtype
    host = _f64(x).numpy()
    want = [_want(host[r], *v) for r, v in enumerate(zip(u.tolist(), *(as_list(v) for v in (t, k, p, m))))]
    assert token.tolist() == [w[0] for w in want]
    lp = np.array([w[1] for w in want])
    # one rounding to fp32; weights are rounded to 2^-41 or finer of the largest, V of them
    far = H32 * np.abs(lp) + x.shape[1] * 2.0 ** -42 + 1e-12
    got = logprob.cpu().double().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(lp)) and np.all((np.abs(got - lp) <= far) | np.isnan(lp))
    return token, logprob


def _u(seed, n):
    return torch.rand((n,), generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 100, 511, 512, 513, 5000, 8192, 8193, 50257, 151001])
def test_sample_rows(K, dtype, vocab):
    rows = 24 if vocab < 60000 else 5
    for limits in ("none", "k", "p", "m", "all"):
        print(f"case: sample_rows {rows} x {vocab} {dtype} {limits}", flush=True)
        g = np.random.default_rng(vocab)
        x = _normal(vocab, (rows, vocab), dtype, 2.5)
        pick = lambda vs, dt: torch.tensor(g.choice(vs, rows), dtype=dt, device="cuda")  # noqa: E731
        on = lambda c: limits in (c, "all")  # noqa: E731
        _check_sample(K, x, _u(vocab, rows), pick([0.0, 0.3, 0.7, 1.0, 1.7], torch.float32),
                      pick([0, 1, 2, 40, 1000, vocab, 10 ** 6], torch.int32) if on("k") else 0,
                      pick([0.0, 0.05, 0.5, 0.9, 0.999, 1.0], torch.float32) if on("p") else 1.0,
                      pick([0.0, 0.01, 0.3, 1.0, 2.0], torch.float32) if on("m") else 0.0,
                      torch.int64 if vocab % 2 else torch.int32)


def test_sample_rows_exact_borders(K):
    """Weights whose sums are exact: a border belongs to the token after it, and ties are kept from the lowest index."""
    x = torch.zeros(1, 8, device="cuda")
    for n in range(9):
        u = torch.tensor([n / 8], device="cuda")
        assert K.sample_rows(x, u)[0].item() == min(n, 7)
        # p: before < p total, so 0.5 keeps ranks 0 .. 3; k keeps the first of equals
        assert K.sample_rows(x, u, top_p=0.5)[0].item() == min(n // 2, 3)
        assert K.sample_rows(x, u, top_k=4)[0].item() == min(n // 2, 3)
        assert K.sample_rows(x, u, top_k=4, top_p=0.5)[0].item() == min(n // 4, 1)
        assert K.sample_rows(x, u, min_p=1.0)[0].item() == min(n, 7)
    # ties across chunks of the row, with larger ones between
    x = torch.full((1, 3000), -1.0, device="cuda")
    x[0, [700, 1400, 2900]] = 0.0
    for k in (3, 4, 600, 1500, 2998):
        _check_sample(K, x.expand(64, 3000), _u(k, 64), 1.0, k)
        _check_sample(K, x.expand(64, 3000), _u(k, 64), 1.0, k, 0.83)
    x = torch.tensor([[-0.0, 0.0, -0.0, -1.0]], device="cuda")  # -0 and 0 are equal
    assert K.sample_rows(x, torch.zeros(1, device="cuda"), temperature=0.0)[0].item() == 0
    assert K.sample_rows(x, torch.full((1,), 0.6, device="cuda"), top_k=2)[0].item() == 1


def test_sample_rows_masks_and_invalid_rows(K):
    for dtype in TYPES:
        low = torch.finfo(dtype).min
        x = _normal(7, (14, 1000), dtype, 2.0)
        x[0, :] = -math.inf
        x[1, 500] = math.nan
        x[2, 3] = math.inf
        x[3, 1:] = -math.inf
        x[4, ::2] = -math.inf
        x[5, 100:] = low
        x[6, :] = low           # masked by the lowest value throughout: all alike
        x[7, :] = -math.inf
        x[7, 999] = low
        u = _u(8, 14)
        t = torch.ones(14, device="cuda")
        p, m = torch.full((14,), 0.9, device="cuda"), torch.zeros(14, device="cuda")
        t[8], t[9], p[10], m[11] = -1.0, math.inf, math.nan, math.nan
        u[12], u[13] = math.nan, 1.0
        for k in (0, 5, 700):
            _check_sample(K, x, u, t, k, p, m)
        _check_sample(K, x, u, 0.0)
        _check_sample(K, x[:8], u[:8], 1e-30)
        _check_sample(K, x[:8], u[:8], 1e30)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 7.0, -3.0], device="cuda")
    x = _normal(9, (5, 513), torch.float32, 2.0)
    x[:, [0, 512]] = -math.inf  # never drawn, at either end
    token = K.sample_rows(x, u)[0].tolist()
    assert token == [1, 511, 511, 511, 1]


def test_sample_rows_views_and_agreement(K):
    x = _normal(10, (6, 50257), torch.bfloat16, 3.0)
    u = _u(10, 6)
    want = K.sample_rows(x, u, 0.8, 50, 0.9, 0.01)
    for pitch, off in ((50264, 0), (50259, 1), (60000, 7)):
        _, v = _rows_view(x, pitch, off)
        got = K.sample_rows(v, u, 0.8, 50, 0.9, 0.01)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(K.sample_rows(x, u, 0.0)[0], K.row_argmax(x)[0])
    assert torch.equal(K.sample_rows(x, u, top_k=1)[0], K.row_argmax(x)[0])
    assert K.sample_rows(x, u, with_logprob=False)[1] is None
    got = K.sample_rows(x, u, np.float32(0.8), np.int64(50), np.float64(0.9), np.float32(0.01))
    assert torch.equal(got[0], want[0])
    assert K.sample_rows(x[:0], u[:0])[0].shape == (0,)


def test_sample_rows_longest(K):
    x = _normal(11, (2, 2097152), torch.float32, 2.0)
    _check_sample(K, x, _u(11, 2), 1.0, 0, 0.9)
    _check_sample(K, x, _u(12, 2), 0.9, 100000)


def test_sample_rows_frequencies(K):
    """20000 draws over 6 tokens: each share within 5 standard deviations."""
    x = torch.tensor([0.3, -1.0, 2.0, 0.0, 1.1, -4.0])
    n = 20000
    token = K.sample_rows(x.cuda().expand(n, 6), _u(13, n), temperature=1.3)[0]
    share = torch.bincount(token.long().cpu(), minlength=6).double() / n
    p = torch.softmax(x.double() / 1.3, 0)
    assert torch.all((share - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n))


# ------------------------------------------------------------------ as they are used
class _Block:
    """The MLP of a pre-norm block in eight bits, the head, and the next tokens."""

    def __init__(self, K, rows, d, ff, vocab):
        self.K, self.rows = K, rows
        self.gamma = _normal(1, (d,), torch.bfloat16, 0.1, 1.0)
        w1, w2, wte = (_normal(s, shape, torch.bfloat16, 1 / math.sqrt(shape[1])) for s, shape in
                       ((2, (ff, d)), (3, (d, ff)), (4, (vocab, d))))
        self.w1, self.w2, self.wte = (K.quantize_rows(w) for w in (w1, w2, wte))
        self.b1, self.b2 = _normal(5, (ff,), torch.bfloat16, 0.1), _normal(6, (d,), torch.bfloat16, 0.1)

    def __call__(self, x, r, u, stream=None):
        K, kw = self.K, {"stream": stream}
        q, s, x = K.add_rmsnorm_int8(x, r, self.gamma, **kw)
        h = K.gemm_int8(q, s, self.w1[0].t(), self.w1[1], bias=self.b1, **kw)
        g, gs = K.quantize_rows(h, gelu=True, **kw)
        y = K.gemm_int8(g, gs, self.w2[0].t(), self.w2[1], bias=self.b2, **kw)
        f, fs, x2 = K.add_rmsnorm_int8(x, y, self.gamma, **kw)
        logits = K.gemm_int8(f, fs, self.wte[0].t(), self.wte[1], out_dtype=torch.float32, **kw)
        token, logprob = K.sample_rows(logits, u, 0.8, 50, 0.95, 0.01, **kw)
        return {"q": q, "s": s, "x": x, "h": h, "g": g, "gs": gs, "y": y, "f": f, "fs": fs, "x2": x2,
                "logits": logits, "token": token, "logprob": logprob}


@pytest.mark.parametrize("rows,d,ff,vocab", [(1, 768, 2048, 5003), (19, 250, 1001, 777), (300, 512, 2048, 4096)])
def test_the_operators_together(K, rows, d, ff, vocab):
    """Each step against 64 bits on the step before's outputs; then the same bits on another stream and from a graph."""
    print(f"case: eight-bit block, {rows} rows of {d}, {ff}, {vocab}", flush=True)
    block = _Block(K, rows, d, ff, vocab)
    x, r, u = _normal(7, (rows, d), torch.bfloat16), _normal(8, (rows, d), torch.bfloat16), _u(9, rows)
    o = block(x, r, u)
    s = _f64(o["x"])
    y = s / torch.sqrt((s * s).mean(dim=1, keepdim=True) + np.float64(np.float32(1e-6))) * _f64(block.gamma)
    _check_rows(o["q"], o["s"], y, H32)
    _check_product(o["h"], o["q"], o["s"], block.w1[0].t(), block.w1[1], block.b1, False)
    _check_product(o["y"], o["g"], o["gs"], block.w2[0].t(), block.w2[1], block.b2, False)
    _check_product(o["logits"], o["f"], o["fs"], block.wte[0].t(), block.wte[1], None, False)
    host = _f64(o["logits"]).numpy()
    p32 = [float(np.float32(v)) for v in (0.8, 0.95, 0.01)]
    assert o["token"].tolist() == [_want(host[i], float(u[i]), p32[0], 50, p32[1], p32[2])[0] for i in range(rows)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    on_side = block(x, r, u, stream=side)
    side.synchronize()
    for n in o:
        assert torch.equal(on_side[n], o[n]), n

    # two graphs of the same block, replayed in turn on new inputs, eager work between
    ins = [[t.clone() for t in (x, r, u)] for _ in range(2)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(block(*ins[i]))
    for step in range(3):
        fresh = [[_normal(20 + 2 * step + i, (rows, d), torch.bfloat16), r, _u(30 + 2 * step + i, rows)] for i in range(2)]
        for i in range(2):
            for t, v in zip(ins[i], fresh[i]):
                t.copy_(v)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            eager = block(*fresh[i])
            for n in eager:
                assert torch.equal(outs[i][n], eager[n]), (step, i, n)


def test_sample_rows_where_a_step_ends_at_zero(K):
    """The largest value a whole number of 64ths of a power of two above the others, which lie at and around 0: the
    step they are in ends there to within roundings.  On the list (5000 tokens), past it (20000), one step's 400."""
    tiny = torch.tensor([0.0, 1e-30, -1e-30, 1e-45, -1e-45, -0.0])
    for vocab in (400, 5000, 20000):
        g = torch.Generator().manual_seed(vocab)
        x = tiny[torch.randint(0, 6, (24, vocab), generator=g)]
        t = torch.tensor([1.0, 0.7, 3.0, 1e-3])[torch.arange(24) % 4]
        steps = torch.tensor([1, 2, 64, 65, 100, 128])[torch.arange(24) // 4]
        x[torch.arange(24), torch.randint(0, vocab, (24,), generator=g)] = (steps / 64 * math.log(2.0) * t.double()).float()
        print(f"case: sample_rows, steps ending at 0, {vocab}", flush=True)
        for p in (0.31, 0.9):
            _check_sample(K, x.cuda(), _u(vocab, 24), t.cuda(), 0, p)
            _check_sample(K, x.cuda(), _u(vocab, 24), t.cuda(), 0, p, 0.2)


def test_sample_rows_flat_rows(K):
    """All tokens alike, more than a list holds; far from 0; at the largest temperatures, masked with -inf or the lowest value."""
    x = torch.full((6, 160001), 3.0, dtype=torch.bfloat16, device="cuda")
    for k, p, m in ((50001, 1.0, 0.0), (0, 0.31, 0.0), (50001, 0.31, 0.5), (0, 1.0, 1.0), (0, 1.0, 1e-30), (3, 1.0, 0.0)):
        print(f"case: sample_rows, flat, {k} {p} {m}", flush=True)
        _check_sample(K, x, _u(k, 6), 1.0, k, p, m)
    x = _normal(31, (16, 9001)) + 1e6
    for p, m in ((0.9, 0.0), (1.0, 1e-30), (1.0, 0.37), (0.5, 0.2)):
        _check_sample(K, x, _u(32, 16), 0.8, 0, p, m)
    low = torch.finfo(torch.float32).min
    x = torch.tensor([0.0, low, -math.inf, -low])[torch.randint(0, 4, (16, 3001), generator=torch.Generator().manual_seed(5))]
    for k, p, m in ((0, 0.97, 0.0), (0, 1.0, 1e-45), (2900, 0.97, 1e-45), (0, 0.1, 0.3)):
        _check_sample(K, x.cuda(), _u(33, 16), -low, k, p, m)


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_rows_where_the_list_overflows(K, dtype):
    """More kept than a list holds: the cut's step alone on it, of few tokens (spread), of many (16-bit values, narrow) and past it too."""
    for vocab, std in ((130001, 3.0), (130001, 1.0), (40000, 0.05), (150000, 0.003)):
        print(f"case: sample_rows, long lists, {vocab} {std} {dtype}", flush=True)
        x = _normal(vocab, (6, vocab), dtype, std)
        for p, m in ((0.95, 0.0), (0.5, 0.0), (0.9, 0.3)):
            _check_sample(K, x, _u(41, 6), torch.tensor([1.0, 1.0, 0.8, 1.3, 1.0, 2.0], device="cuda"), 0, p, m)


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_rows_of_mostly_masked_tokens(K, dtype):
    """Fewer tokens left than top_k, more, and more than a list holds; masked with -inf, the lowest value, 60 below."""
    for vocab, left in ((50257, 1), (50257, 10), (50257, 400), (50257, 20000), (3000, 7), (9, 3)):
        print(f"case: sample_rows, {left} of {vocab} left, {dtype}", flush=True)
        x = _normal(left, (6, vocab), dtype, 2.0)
        at = torch.rand((6, vocab), generator=torch.Generator().manual_seed(left)).argsort(dim=1) >= left
        for mask in (-math.inf, torch.finfo(dtype).min, -60.0):
            y = x.masked_fill(at.cuda(), mask)
            for k, p, m in ((50, 1.0, 0.0), (50, 0.9, 0.0), (1000, 0.9, 0.0), (30000, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.1)):
                _check_sample(K, y, _u(51, 6), 0.7, k, p, m)


def test_rows_far_apart(K):
    """Rows whose offsets pass 2^31 bytes and 2^31 elements, of every operand."""
    def far(t, pitch):
        v = torch.empty((t.shape[0] - 1) * pitch + t.shape[1] + 64, dtype=t.dtype, device="cuda")
        v = v.as_strided(t.shape, (pitch, 1))
        return v.copy_(t)

    for Kd, off in ((256, 0), (250, 1)):
        for M, N in ((20, 70), (70, 200)):
            a, w, sa, sb = _int8(1, (M, Kd)), _int8(2, (N, Kd)), _scales(1, M), _scales(2, N)
            want = K.gemm_int8(a, sa, w.t(), sb)
            print(f"case: gemm_int8 far apart {M} x {Kd} x {N}", flush=True)
            assert torch.equal(K.gemm_int8(far(a, (1 << 27) + off), sa, w.t(), sb), want)
            assert torch.equal(K.gemm_int8(a, sa, far(w, (1 << 25) + off).t(), sb), want)
            out = far(want, (1 << 26) + off)
            K.gemm_int8(a, sa, w.t(), sb, out=out.zero_())
            assert torch.equal(out, want)
    x, u = _normal(3, (5, 1001), torch.bfloat16), _u(4, 5)
    v = far(x, (1 << 29) + 1)
    assert all(torch.equal(i, j) for i, j in zip(K.sample_rows(v, u, 0.8, 50, 0.9), K.sample_rows(x, u, 0.8, 50, 0.9)))
    q, scale, total = K.add_rmsnorm_int8(x, x)
    s = far(x, (1 << 29) + 1)
    got = K.add_rmsnorm_int8(v, v, q=far(q, (1 << 30) + 1), sum_out=s)
    assert got[2] is s and all(torch.equal(i, j) for i, j in zip(got, (q, scale, total)))
    assert torch.equal(K.dequantize_rows(got[0], scale), K.dequantize_rows(q, scale))


def test_one_row_of_weights_for_every_column(K):
    a, w, sa, sb = _int8(1, (100, 768)), _int8(2, (1, 768)), _scales(1, 100), _scales(2, 600)
    want = K.gemm_int8(a, sa, w.expand(600, 768).contiguous().t(), sb)
    assert torch.equal(K.gemm_int8(a, sa, w.expand(600, 768).t(), sb), want)
    want = K.gemm_int8(a[:1].expand(100, 768).contiguous(), sa, w.expand(600, 768).contiguous().t(), sb)
    assert torch.equal(K.gemm_int8(a[:1].expand(100, 768), sa, w.expand(600, 768).t(), sb), want)
    # a single row, whose pitch says nothing
    for Kd in (768, 750):
        v = _int8(3, (600, Kd))
        row = a[:1, :Kd].contiguous()
        want = K.gemm_int8(row, sa[:1], v.t(), sb)
        assert torch.equal(K.gemm_int8(row.as_strided((1, Kd), (1, 1)), sa[:1], v.t(), sb), want)
        want = K.gemm_int8(v, sb, row.t(), sa[:1])
        assert torch.equal(K.gemm_int8(v, sb, row.as_strided((1, Kd), (1, 1)).t(), sa[:1]), want)


def test_two_streams_at_once(K):
    """Nothing is shared between calls: the same results with every call in flight on two streams."""
    blocks = [_Block(K, rows, 512, 1024, 5003) for rows in (40, 300)]
    ins = [(_normal(i, (b.rows, 512), torch.bfloat16), _normal(i + 9, (b.rows, 512), torch.bfloat16), _u(i, b.rows))
           for i, b in enumerate(blocks)]
    want = [b(*v) for b, v in zip(blocks, ins)]
    streams = [torch.cuda.Stream() for _ in blocks]
    torch.cuda.synchronize()
    got = []
    for _ in range(6):
        got.append([b(*v, stream=s) for b, v, s in zip(blocks, ins, streams)])
    torch.cuda.synchronize()
    for both in got:
        for o, w in zip(both, want):
            for n in w:
                assert torch.equal(o[n], w[n]), n


def test_refusals(K):
    x = _normal(1, (4, 64))
    q, s = K.quantize_rows(x)
    u = _u(1, 4)
    bad = [
        lambda: K.quantize_rows(x.double()), lambda: K.quantize_rows(x[0]), lambda: K.quantize_rows(x.t()),
        lambda: K.quantize_rows(x, q=q[:, :32]), lambda: K.quantize_rows(x, scale=s.double()),
        lambda: K.quantize_rows(x, q=q[:1].expand(4, 64)),
        lambda: K.add_rmsnorm_int8(x, x.half()), lambda: K.add_rmsnorm_int8(x, x[:2]),
        lambda: K.add_rmsnorm_int8(x, gamma=x[0, :32]), lambda: K.add_rmsnorm_int8(x, sum_out=x),
        lambda: K.add_rmsnorm_int8(x, x.cpu()),
        lambda: K.dequantize_rows(q, s, torch.float64), lambda: K.dequantize_rows(q, s[:2]),
        lambda: K.gemm_int8(q, s, q, s), lambda: K.gemm_int8(q, s, q.t().contiguous(), s),
        lambda: K.gemm_int8(q, s, q.t(), s, out_dtype=torch.int32), lambda: K.gemm_int8(q, s[:3], q.t(), s),
        lambda: K.gemm_int8(q, s, q.t(), s, bias=s.double()), lambda: K.gemm_int8(q, s, q.t(), s, relu=True),
        lambda: K.gemm_int8(q, s, q.t(), s, bias=s[:1]), lambda: K.gemm_int8(x, s, q.t(), s),
        lambda: K.gemm_int8(q, s, q.t(), s, out=torch.empty(4, device="cuda").bfloat16().expand(4, 4)),
        lambda: K.sample_rows(x, u[:2]), lambda: K.sample_rows(x, u.double()), lambda: K.sample_rows(x.t(), u),
        lambda: K.sample_rows(x, u, top_k=u), lambda: K.sample_rows(x, u, index_dtype=torch.int16),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    from mi355x_pjrt._lib import KernelError

    for f in (lambda: K.add_rmsnorm_int8(x, eps=-1.0), lambda: K.add_rmsnorm_int8(x, eps=math.nan),
              lambda: K.sample_rows(x, u, temperature=-1.0), lambda: K.sample_rows(x, u, temperature=math.inf),
              lambda: K.sample_rows(x, u, top_p=math.nan), lambda: K.quantize_rows(x[:, :0])):
        with pytest.raises(KernelError):
            f()
