"""Refusals of the eight-bit entry points at the C-ABI, before anything is
launched: run on a host without a GPU, on pointers that are never followed."""

import math

import pytest

from mi355x_pjrt import _lib

BF16, F16, F32, F64, S32, S64 = 13, 10, 11, 12, 4, 5
P, Q = 1 << 20, 1 << 21  # stand for aligned device memory


@pytest.fixture(scope="module")
def lib():
    return _lib.load_kernels()


def _refused(lib, code, word, rc):
    assert rc == code
    assert word in lib.mk_last_error().decode()


def test_rows(lib):
    def norm(t=BF16, rows=4, cols=64, x=P, ldx=64, r=P, ldr=64, g=P, eps=1e-6, s=Q, lds=64, q=Q, ldq=64, sc=Q):
        return lib.mk_add_rmsnorm_int8(None, t, rows, cols, x, ldx, r, ldr, g, eps, s, lds, q, ldq, sc)

    _refused(lib, 2, "type", norm(t=F64))
    _refused(lib, 1, "rows", norm(rows=-1))
    _refused(lib, 1, "cols", norm(cols=0))
    _refused(lib, 1, "eps", norm(eps=-1.0))
    _refused(lib, 1, "eps", norm(eps=math.nan))
    for name in ("x", "s", "q", "sc"):
        _refused(lib, 1, "null", norm(**{name: None}))
    _refused(lib, 1, "aligned", norm(x=P + 1))
    _refused(lib, 1, "aligned", norm(g=P + 1))
    _refused(lib, 1, "aligned", norm(sc=Q + 2))
    _refused(lib, 1, "pitch", norm(ldx=-64))
    _refused(lib, 1, "pitch", norm(lds=63))
    _refused(lib, 1, "pitch", norm(ldq=63))
    assert norm(rows=0, x=None) == 0
    _refused(lib, 2, "type", lib.mk_quantize_rows(None, S32, 4, 64, P, 64, 0, Q, 64, Q))
    _refused(lib, 1, "null x", lib.mk_quantize_rows(None, F32, 4, 64, None, 64, 0, Q, 64, Q))
    _refused(lib, 1, "pitch", lib.mk_quantize_rows(None, F32, 4, 64, P, 64, 0, Q, 32, Q))
    _refused(lib, 2, "type", lib.mk_dequantize_rows(None, F64, 4, 64, P, 64, P, Q, 64))
    _refused(lib, 1, "pitch", lib.mk_dequantize_rows(None, F16, 4, 64, P, 64, P, Q, 60))
    _refused(lib, 1, "aligned", lib.mk_dequantize_rows(None, F16, 4, 64, P, 64, P, Q + 1, 64))


def test_product(lib):
    def gemm(t=BF16, M=4, N=8, Kd=64, a=P, lda=64, sa=P, b=P, ldb=64, sb=P, c=Q, ldc=8, bias=None, epi=0):
        return lib.mk_gemm_int8(None, t, M, N, Kd, a, lda, sa, b, ldb, sb, c, ldc, bias, epi)

    _refused(lib, 2, "c_type", gemm(t=S32))
    _refused(lib, 1, "negative", gemm(M=-1))
    _refused(lib, 2, "131071", gemm(Kd=131072))
    _refused(lib, 2, "tiles", gemm(M=1 << 40, N=1 << 40, ldc=1 << 41))
    for epi in (-1, 3, 4, 7):
        _refused(lib, 1, "epilogue", gemm(epi=epi, bias=P))
    _refused(lib, 1, "null", gemm(epi=1))
    for name in ("a", "b", "sa", "sb", "c"):
        _refused(lib, 1, "null", gemm(**{name: None}))
    _refused(lib, 1, "stride", gemm(ldc=7))
    _refused(lib, 1, "stride", gemm(lda=-64))
    _refused(lib, 1, "aligned", gemm(c=Q + 1))
    _refused(lib, 1, "aligned", gemm(sa=P + 2))
    _refused(lib, 1, "aligned", gemm(epi=5, bias=P + 2))
    assert gemm(M=0, a=None) == 0 and gemm(N=0, b=None) == 0


def test_sampling(lib):
    def sample(t=BF16, rows=4, vocab=100, x=P, ld=100, u=P, temp=None, t_all=1.0, k=None, p=None, p_all=1.0, m=None,
               m_all=0.0, it=S32, tok=Q, lp=Q):
        return lib.mk_sample_rows(None, t, rows, vocab, x, ld, u, temp, t_all, k, 0, p, p_all, m, m_all, it, tok, lp)

    _refused(lib, 2, "io_type", sample(t=F64))
    _refused(lib, 2, "index_type", sample(it=F32))
    _refused(lib, 1, "vocab", sample(vocab=0))
    _refused(lib, 1, "rows", sample(rows=-1))
    _refused(lib, 2, "2097152", sample(vocab=2097153))
    _refused(lib, 2, "rows", sample(rows=1 << 22))
    for v in (-1.0, math.inf, math.nan):
        _refused(lib, 1, "temperature", sample(t_all=v))
    _refused(lib, 1, "top_p", sample(p_all=math.nan))
    _refused(lib, 1, "min_p", sample(m_all=math.nan))
    for name in ("x", "u", "tok"):
        _refused(lib, 1, "null", sample(**{name: None}))
    _refused(lib, 1, "pitch", sample(ld=-1))
    for name in ("x", "u", "temp", "k", "p", "m", "tok", "lp"):
        _refused(lib, 1, "aligned", sample(**{name: P + 1}))
    assert sample(rows=0, x=None) == 0


def test_wrappers_take_device_tensors():
    import torch

    from mi355x_pjrt import kernels as K

    x, q, s = torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)
    for f in (lambda: K.quantize_rows(x), lambda: K.add_rmsnorm_int8(x), lambda: K.dequantize_rows(q, s),
              lambda: K.gemm_int8(q, s, q.t(), s), lambda: K.sample_rows(x, s)):
        with pytest.raises(ValueError, match="device"):
            f()
