"""Every kernel of linear_xent, linear_xent_bwd, dropout_add and dropout_add_bwd on
the MI355X against the definitions in 64 bits, at sizes where tiles follow
each other in a workgroup, operands are copied in pieces, or weights lie past 2^31
bytes (tests/xent_cases.py)."""

import pytest
import torch

from test_gpu_dropout import _check_bwd, _check_out
from test_gpu_linear_xent_labels import _reference
from xent_cases import DROP_GRADS, DROPS, FEW, PIECES, TILES
from xent_dropout_ref import xent, xent_grad

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def K(cuda):
    from mi355x_pjrt import kernels

    kernels.lib()
    return kernels


def _inputs(seed, rows, width, vocab, dtype, ignore):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.empty((vocab, width), dtype=dtype, device="cuda").normal_(0, 2 / width ** 0.5, generator=g)
    labels = torch.randint(vocab, (rows,), generator=g, device="cuda")
    x = torch.randn((rows, width), generator=g, device="cuda")
    # rows that lean to their label by up to 8
    x = (x + 8 * torch.rand((rows, 1), generator=g, device="cuda") * w[labels].float() / 4).to(dtype)
    labels[-1], labels[rows // 2] = vocab - 1, vocab // 256 * 256 - (vocab % 256 == 0)
    if ignore:
        labels[::5] = -100
    return x, w, labels.int(), torch.rand((rows,), generator=g, device="cuda") + 0.5


def _within(got, want, bound, what):
    assert bool(torch.isfinite(got).all()), what
    over = (got.double() - want).abs() - bound
    assert float(over.max()) <= 0, (what, float(over.max()), int((over > 0).sum()))


def _grad_reference(x, w, labels, lse, scale, row_grad, ignore, dw_dtype, rows):
    if x.dtype != torch.float32 and rows > 64:
        return _reference(x, w, labels, lse, scale, row_grad, ignore, dw_dtype)
    return xent_grad(x, w, labels, lse, scale, row_grad, ignore, dw_dtype, twice=x.dtype != torch.float32)


def _check_all(K, x, w, labels, row_grad, ignore, dw_dtype):
    """Loss, lse and both gradients; the reference by blocks of rows, each block's dw and its bound added."""
    rows, vocab = x.shape[0], w.shape[0]
    loss, lse = K.linear_xent(x, w, labels, ignore_index=ignore)
    dx, dw = K.linear_xent_bwd(x, w, labels, lse, grad_scale=0.25, row_grad=row_grad, ignore_index=ignore, dw_dtype=dw_dtype)
    block = max(1, min(rows, (1 << 28) // vocab))
    want_dw = bound_dw = 0
    # a block's own reference rounds fp16 by its largest row_grad; the whole's is the largest there is
    for i in range(0, rows, block):
        at = slice(i, i + block)
        want, want_lse, bound = xent(x[at], w, labels[at], ignore)
        _within(loss[at], want, bound, "loss")
        _within(lse[at], want_lse, bound, "lse")
        wx, ww, bx, bw = _grad_reference(x[at], w, labels[at], lse[at], 0.25, row_grad[at], ignore, dw_dtype, rows)
        _within(dx[at], wx, bx, "dx")
        want_dw, bound_dw = want_dw + ww, bound_dw + bw
        del wx, ww, bx, bw
    _within(dw, want_dw, bound_dw, "dw")
    if ignore is not None:
        assert torch.all(dx[labels == ignore] == 0) and torch.all(loss[labels == ignore] == 0)
    return loss, lse, dx, dw


@pytest.mark.parametrize("rows,width,vocab,dtype,dw_dtype,ignore", TILES + PIECES + FEW)
def test_against_the_definition(K, rows, width, vocab, dtype, dw_dtype, ignore):
    print(f"case: linear_xent {rows} x {width} x {vocab} {dtype} {dw_dtype} {ignore}", flush=True)
    x, w, labels, row_grad = _inputs(rows + vocab, rows, width, vocab, DT[dtype], ignore)
    row_grad[0] = 1.5  # the largest, in every block of rows alike
    block = max(1, min(rows, (1 << 28) // vocab))
    row_grad[::block] = 1.5
    if ignore:  # of a row that counts
        labels[::block] = vocab // 3
    _check_all(K, x, w, labels, row_grad, -100 if ignore else None, DT[dw_dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_large_tiles_in_graphs_and_on_streams(K, dtype):
    """Two calls at once, and a captured one replayed beside another, give the bits of a call alone."""
    cases = []
    for rows, width, vocab in ((2041, 776, 16379), (3001, 264, 9000)):
        print(f"case: at once {rows} x {width} x {vocab} {dtype}", flush=True)
        x, w, labels, row_grad = _inputs(rows, rows, width, vocab, DT[dtype], True)
        loss, lse = K.linear_xent(x, w, labels, ignore_index=-100)
        cases.append((x, w, labels, row_grad, loss, lse) + K.linear_xent_bwd(x, w, labels, lse, row_grad=row_grad, ignore_index=-100))

    def run(c, **kw):
        loss, lse = K.linear_xent(*c[:3], ignore_index=-100, **kw)
        return (loss, lse) + K.linear_xent_bwd(*c[:3], lse, row_grad=c[3], ignore_index=-100, **kw)

    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = [run(c, stream=s) for c, s in zip(cases, streams)]
        torch.cuda.synchronize()
        for g, c in zip(got, cases):
            assert all(torch.equal(a, b) for a, b in zip(g, c[4:]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        out = run(cases[0])
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        eager = run(cases[1], stream=streams[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, cases[0][4:]))
        assert all(torch.equal(a, b) for a, b in zip(eager, cases[1][4:]))


@pytest.mark.parametrize("rows,cols,dtype", DROPS)
def test_dropout_add(K, rows, cols, dtype):
    print(f"case: dropout_add {rows} x {cols} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x, res = (torch.randn((rows, cols), generator=g, device="cuda").to(DT[dtype]) for _ in range(2))
    bias = torch.randn((cols,), generator=g, device="cuda").to(DT[dtype])
    out = K.dropout_add(x, 0.1, 2 ** 40 + 7, offset=3, bias=bias, residual=res)
    _check_out(out, x, bias, res, 0.1, 2 ** 40 + 7, 3)
    place = res.clone()
    assert torch.equal(K.dropout_add(x, 0.1, 2 ** 40 + 7, offset=3, bias=bias, residual=place, out=place), out)
    # rows at a pitch, off the 16-byte boundaries, over themselves
    sea = torch.full((rows * (cols + 3) + 5,), 77, dtype=DT[dtype], device="cuda")
    view = sea[5:].view(rows, cols + 3)[:, :cols]
    view.copy_(x)
    assert torch.equal(K.dropout_add(view, 0.1, 2 ** 40 + 7, offset=3, bias=bias, residual=res, out=view), out)
    view.fill_(77)
    assert torch.all(sea == 77)


@pytest.mark.parametrize("rows,cols,dtype", DROP_GRADS)
def test_dropout_add_bwd(K, rows, cols, dtype):
    print(f"case: dropout_add_bwd {rows} x {cols} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    dy = torch.randn((rows, cols), generator=g, device="cuda").to(DT[dtype])
    dx, colsum = K.dropout_add_bwd(dy, 0.1, 99, offset=5, want_colsum=True)
    _check_bwd(dx, colsum, dy, 0.1, 99, 5)
    alone, _ = K.dropout_add_bwd(dy, 0.1, 99, offset=5)
    assert torch.equal(alone, dx)
