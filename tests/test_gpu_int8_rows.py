"""Rows to eight bits on the MI355X, where the rounding itself is at stake:
every quotient of two 16-bit numbers that is an exact half, and rows of each
type with NaN, infinities, zeros and the ends of the type's range."""

import math

import numpy as np
import pytest
import torch

from test_gpu_int8 import _check_rows, _f64, _normal

pytestmark = pytest.mark.gpu

HALF_TYPES = [torch.bfloat16, torch.float16]
BITS = {torch.bfloat16: 8, torch.float16: 11}  # of a significand


@pytest.fixture(scope="module")
def K(cuda):
    from mi355x_pjrt import kernels

    kernels.lib()
    return kernels


def _nearest(v, top):
    """127 v / top as the nearest whole number, halves to even: whole numbers v and top (numpy int64)."""
    n, rest = np.divmod(127 * v, top)
    up = (2 * rest > top) | ((2 * rest == top) & (n % 2 == 1))
    return n + up


def _every_quotient(dtype):
    """(x, q): a row for each significand `top` of the type, which it starts with, then
    every smaller value down to top's 2^-8 that the type holds; and its rounded quotients."""
    one = 1 << (BITS[dtype] - 1)
    tops = np.arange(one, 2 * one, dtype=np.int64)
    v = np.concatenate([np.arange(one, 2 * one, dtype=np.int64) << e for e in range(9)])  # over 2^8
    v, tops = v[None, :], tops[:, None] << 8
    v = np.where(v <= tops, v, 0)
    v[:, 1::2] *= -1
    v = np.concatenate([tops, v], axis=1)
    q = np.sign(v) * _nearest(np.abs(v), tops)
    return torch.from_numpy(v * 2.0 ** -8 / one).to(dtype), torch.from_numpy(q).to(torch.int8)


# elements a row takes at most: short rows, the registers' teams, rows that are read twice
@pytest.mark.parametrize("cols", [5, 100, 900, 2000, 40000])
@pytest.mark.parametrize("dtype", HALF_TYPES)
def test_halves_go_to_the_even_number(K, dtype, cols):
    """Exact: the quotient of two significands of 11 bits is a half or 2^-12 and more away
    from one, further than its rounding to fp32 (2^-18 below 128) takes it, and a half is
    a number of fp32."""
    x, q = _every_quotient(dtype)
    halves = (q.double() - 127 * x.double() / x[:, :1].double()).abs() == 0.5
    assert int(halves.sum()) > 100
    # the values of a row over rows of `cols`, each of them behind the row's largest
    n = x.shape[1] - 1
    if cols > n:
        reps = -(-(cols - 1) // n)
        x, q = (torch.cat([t[:, :1], t[:, 1:].repeat(1, reps)[:, :cols - 1]], dim=1) for t in (x, q))
    else:
        parts = -(-n // (cols - 1))
        pad = parts * (cols - 1) - n

        def cut(t):
            body = torch.cat([t[:, 1:], t.new_zeros(t.shape[0], pad)], dim=1).reshape(-1, cols - 1)
            return torch.cat([t[:, :1].repeat_interleave(parts, dim=0), body], dim=1)

        x, q = cut(x), cut(q)
    print(f"case: halves, {tuple(x.shape)} {dtype}", flush=True)
    x = x.cuda()
    scale = (x[:, 0].float().cpu().numpy() / np.float32(127)).astype(np.float32)
    got, s = K.quantize_rows(x)
    assert torch.equal(got.cpu(), q)
    assert np.array_equal(s.cpu().numpy(), scale)
    assert torch.equal(K.quantize_rows(-x)[0].cpu(), -q)
    assert torch.equal(K.add_rmsnorm_int8(x)[0].cpu(), q)
    # a power of two in gamma and another in the residual's share: the same quotients
    gamma = torch.full((x.shape[1],), 0.5, dtype=dtype, device="cuda")
    assert torch.equal(K.add_rmsnorm_int8(x, x, gamma)[0].cpu(), q)
    # at the type's largest and least normal exponents
    for f in (2.0 ** 14, 2.0 ** -5) if dtype == torch.float16 else (2.0 ** 126, 2.0 ** -117):
        assert torch.equal(K.quantize_rows(x * f)[0].cpu(), q)


@pytest.mark.parametrize("cols", [5, 768, 4104, 33000])
@pytest.mark.parametrize("dtype", HALF_TYPES + [torch.float32])
def test_zeros_nan_infinities_and_the_ends_of_the_range(K, dtype, cols):
    """Of every type, plain, normed and through GELU, whose value at -inf is NaN (-inf times 0) and at the
    lowest number -0."""
    info = torch.finfo(dtype)
    x = _normal(1, (11, cols), dtype)
    x[0] = 0
    x[1, cols // 2] = math.nan
    x[2, cols - 1] = math.inf
    x[3, 0] = -math.inf
    x[4] = info.max
    x[5] = info.smallest_normal * info.eps  # the least number there is
    x[6] = -0.0
    x[7] = info.min
    x[8, 0] = info.max  # the others are a fraction of a step
    for mode in ("plain", "norm", "gelu"):
        print(f"case: {mode}, special values, {cols} {dtype}", flush=True)
        q, scale = K.add_rmsnorm_int8(x, eps=1e-6)[:2] if mode == "norm" else K.quantize_rows(x, gelu=mode == "gelu")
        zeros = {0, 6} | ({7} if mode == "gelu" else set()) | (set() if dtype == torch.float16 else {5})
        for r in zeros:
            assert float(scale[r]) == 0 and not bool(q[r].any()), r
        for r in (1, 2, 3):
            assert math.isnan(float(scale[r])) and not bool(q[r].any()), r
            assert bool(torch.isnan(K.dequantize_rows(q, scale, dtype)[r]).all())
        keep = [r for r in range(11) if r not in zeros | {1, 2, 3}]
        v = _f64(x)[keep]
        if mode == "norm":
            v = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + np.float64(np.float32(1e-6)))
        elif mode == "gelu":
            v = v / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
        # GELU: half a step of the exponent's rounding at each of 3, the exponential, the
        # reciprocal and the product, of the row's largest value (a positive one)
        _check_rows(q[keep], scale[keep], v, 16 * 2.0 ** -24 if mode == "gelu" else 2.0 ** -24)
        for r in (4, 5):
            assert r in zeros or bool((q[r] == 127).all())
        assert mode == "gelu" or bool((q[7] == -127).all())
