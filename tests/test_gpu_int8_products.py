"""Every kernel of the eight-bit product on the MI355X, on the products of
int8_products.py (test_int8_products.py holds that each runs on the kernel it is
listed for): operands whose rows end before their pitch, with other values there, and
results inside a larger buffer.

The sum is exact; its conversion, the two scales and the bias are a rounding each, and
the result is rounded to its type once more (half a step each, eps / 2)."""

import pytest
import torch

from int8_products import BF16, DEEP, F32, FEW, STREAMED, TILED, lines, pitch

pytestmark = pytest.mark.gpu

H32 = 2.0 ** -24  # half a step of fp32
TYPES = {BF16: torch.bfloat16, F32: torch.float32}


@pytest.fixture(scope="module")
def K(cuda):
    from mi355x_pjrt import kernels

    kernels.lib()
    return kernels


def _rows(seed, rows, cols, ld):
    """Rows of all 256 values, and others between a row's end and its pitch."""
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, (rows, ld), generator=g, dtype=torch.int8).cuda()[:, :cols]


def _floats(seed, n, low, high):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand((n,), generator=g) * (high - low) + low).cuda()


def _sums(a, w):
    """a w^T in 64 bits: whole numbers below 2^31 are exact in every order."""
    return torch.mm(a.double(), w.double().t().contiguous())


def _check(got, sums, sa, sb, bias=None, relu=False):
    want = sums * sa.double()[:, None] * sb.double()
    far = 3 * H32 * want.abs()
    if bias is not None:
        want = want + bias.double()
        far = far + H32 * (want.abs() + far)
    if relu:
        want = want.clamp(min=0)
    info = torch.finfo(got.dtype)
    far = far + info.eps / 2 * (want.abs() + far) + info.smallest_normal * info.eps
    assert bool(((got.double() - want).abs() <= far).all())


def _run(K, m, k, n, ld):
    a, w = _rows(m, m, k, ld), _rows(n, n, k, ld)
    sa, sb = _floats(1, m, 1e-4, 0.02), _floats(2, n, 1e-4, 0.02)
    sums = _sums(a, w)
    # f16: sums of up to 2^14 k, scaled to its range
    for dtype, bias, relu, f in ((torch.bfloat16, torch.bfloat16, False, 1.0), (torch.float32, None, False, 1.0),
                                 (torch.float16, torch.float32, True, 1e-4)):
        b = None if bias is None else _floats(3, n, -1.0, 1.0).to(bias)
        sea = torch.full((m + 2, n + 5), 77.0, dtype=dtype, device="cuda")
        out = sea[1:m + 1, 2:n + 2]
        assert K.gemm_int8(a, sa * f, w.t(), sb, out_dtype=dtype, bias=b, relu=relu, out=out) is out
        _check(out, sums, sa * f, sb, b, relu)
        out.fill_(77.0)
        assert bool((sea == 77.0).all())


@pytest.mark.parametrize("name,m,n,ks,on_grid", TILED)
def test_tiles(K, name, m, n, ks, on_grid):
    for k in ks:
        print(f"case: gemm_int8 {name}: {m} x {k} x {n}", flush=True)
        _run(K, m, k, n, pitch(k, on_grid))


@pytest.mark.parametrize("name,m,n,ks,on_grid", FEW)
def test_few_rows(K, name, m, n, ks, on_grid):
    for k in ks:
        print(f"case: gemm_int8 {name}: {m} x {k} x {n}", flush=True)
        _run(K, m, k, n, pitch(k, on_grid))


@pytest.mark.parametrize("name,m,n", DEEP)
def test_largest_sums_on_each_tile(K, name, m, n):
    """-128 times -128, 131071 times, 16384 below 2^31, with a column of the other sign;
    what lies behind a row's end would take the sum past it."""
    print(f"case: gemm_int8 {name}: {m} x 131071 x {n}", flush=True)
    a = torch.full((m, 131072), -128, dtype=torch.int8, device="cuda")[:, :131071]
    w = torch.full((n, 131072), -128, dtype=torch.int8, device="cuda")[:, :131071]
    w[1] = 127
    one = torch.ones(max(m, n), device="cuda")
    c = K.gemm_int8(a, one[:m], w.t(), one[:n], out_dtype=torch.float32)
    want = torch.full((n,), 131071 * 16384, dtype=torch.int64)
    want[1] = -131071 * 16256
    assert bool((c == want.float().cuda()).all())


@pytest.mark.parametrize("name,ct,m,n,k", STREAMED)
def test_results_past_the_caches(K, name, ct, m, n, k):
    """All of C, in parts; the columns behind the last one stay as they were."""
    print(f"case: gemm_int8 {name}: {m} x {k} x {n} past the caches", flush=True)
    ld = (k + 15) // 16 * 16 if "true" in name else k
    a, w, sa, sb = _rows(1, m, k, ld), _rows(2, n, k, ld), _floats(1, m, 1e-4, 0.02), _floats(2, n, 1e-4, 0.02)
    buffer = torch.full((m, lines(n)), 77.0, dtype=TYPES[ct], device="cuda")
    assert buffer.data_ptr() % 128 == 0 and lines(n) > n
    c = K.gemm_int8(a, sa, w.t(), sb, out_dtype=TYPES[ct], out=buffer[:, :n])
    for r in range(0, m, 2048):
        _check(c[r:r + 2048], _sums(a[r:r + 2048], w), sa[r:r + 2048], sb)
    assert bool((buffer[:, n:] == 77.0).all())


def _far(t, ld):
    """t's rows ld elements apart."""
    v = torch.empty((t.shape[0] - 1) * ld + t.shape[1] + 64, dtype=t.dtype, device="cuda")
    return v.as_strided(t.shape, (ld, 1)).copy_(t)


@pytest.mark.parametrize("m,n", [(1500, 4101), (201, 2101)])
def test_tiles_of_rows_far_apart(K, m, n):
    """Operands and results whose offsets pass 2^32 bytes, on the tiles; operands on the
    16-byte grid up to the last byte that goes to LDS directly, below 2^31."""
    k = 515
    a, w, sa, sb = _rows(1, m, k, k), _rows(2, n, k, k), _floats(1, m, 1e-4, 0.02), _floats(2, n, 1e-4, 0.02)
    want = K.gemm_int8(a, sa, w.t(), sb)
    _check(want, _sums(a, w), sa, sb)
    print(f"case: gemm_int8 far apart: {m} x {k} x {n}", flush=True)
    past = lambda rows: (1 << 32) // (rows - 1) + 1 | 1  # noqa: E731
    assert torch.equal(K.gemm_int8(_far(a, past(m)), sa, w.t(), sb), want)
    assert torch.equal(K.gemm_int8(a, sa, _far(w, past(n)).t(), sb), want)
    below = lambda rows: ((1 << 31) - 17 - k) // (rows - 1) // 16 * 16  # noqa: E731
    near = [_far(t, below(t.shape[0])) for t in (a, w)]
    assert torch.equal(K.gemm_int8(near[0], sa, near[1].t(), sb), want)
    for on_grid in (False, True):
        x, y = (_rows(s, r, k, pitch(k, on_grid)).copy_(t) for s, r, t in ((1, m, a), (2, n, w)))
        out = _far(want, past(m)).zero_()
        K.gemm_int8(x, sa, y.t(), sb, out=out)
        assert torch.equal(out, want)
