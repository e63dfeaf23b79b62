"""The gradient of linear_xent past 64 rows of 16 bits: what the rounding of the
gradient of the logits leaves of each label's element is kept, so that a class
that one token alone has as its label is off by no more than the roundings of
the small elements around it."""

import pytest
import torch

from xent_dropout_ref import H32, half_step, subnormal

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def K(cuda):
    from mi355x_pjrt import kernels

    kernels.lib()
    return kernels


def _inputs(seed, rows, width, vocab, dtype, lean=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn((vocab, width), generator=g, device="cuda") * (2 / width ** 0.5)).to(dtype)
    labels = torch.randint(vocab, (rows,), generator=g, device="cuda")
    x = torch.randn((rows, width), generator=g, device="cuda")
    # rows that lean to their label by up to `lean`
    x = x + lean * torch.rand((rows, 1), generator=g, device="cuda") * w[labels].float() / 4
    return x.to(dtype), w, labels.int(), torch.rand((rows,), generator=g, device="cuda") + 0.5


def _reference(x, w, labels, lse, scale, row_grad, ignore, dw_dtype):
    """(dx, dw, bound of dx, bound of dw) in 64 bits.  A logit's error is that of width fp32
    additions, an exponential's that of its exponent's roundings and two steps.  Of g, every element
    but the label's is rounded once to x's type; what that leaves of the label's is kept in 16 bits, so
    that it is off by the square of half a step.  fp16 is scaled by a power of two, so that what is
    lost below its normal numbers is 2^-40 of the largest row_grad.  Sums are fp32 additions in any order,
    two more for the labels' shares; results are rounded once."""
    dtype = x.dtype
    labels = labels.long()
    used = torch.ones_like(labels, dtype=torch.bool) if ignore is None else labels != ignore
    x = torch.where(used[:, None], x.double(), 0.0)
    w = w.double()
    z = x @ w.t()
    p = torch.exp(z - lse.double()[:, None])
    inside = (labels >= 0) & (labels < w.shape[0])
    hot = torch.zeros_like(p).scatter_(1, torch.where(inside, labels, 0)[:, None], inside.double()[:, None])
    r = used.double() * (1.0 if row_grad is None else row_grad.double())
    g = (p - hot) * r[:, None]
    h = half_step(dtype)
    e = (x.shape[1] + 1) * H32 * (x.abs() @ w.abs().t()) + H32 * (3 * (z - lse.double()[:, None]).abs() + 4)
    dg = torch.where(hot > 0, h * h, h) * g.abs() + (p * e + 4 * H32 * (p + hot)) * r.abs()[:, None]
    if dtype == torch.float16:
        dg = dg + 2.0 ** -40 * r.abs().max()
    s = abs(scale)

    def bound(d, size, n, out, t):
        return 1.01 * s * (d + (n + 4) * H32 * size) + (half_step(t) + 2 * H32) * out.abs() + subnormal(t)

    dx, dw = g @ w * scale, g.t() @ x * scale
    return (dx, dw, bound(dg @ w.abs(), g.abs() @ w.abs(), w.shape[0], dx, dtype),
            bound(dg.t() @ x.abs(), g.abs().t() @ x.abs(), x.shape[0], dw, dw_dtype))


def _within(got, want, bound, what):
    assert bool(torch.isfinite(got).all()), what
    over = (got.double() - want).abs() - bound
    assert float(over.max()) <= 0, (what, float(over.max()), int((over > 0).sum()), float(want.abs().max()))


def _check(K, x, w, labels, scale=1.0, row_grad=None, ignore=None):
    _, lse = K.linear_xent(x, w, labels, ignore_index=ignore)
    for dw_dtype in (torch.float32, x.dtype):
        dx, dw = K.linear_xent_bwd(x, w, labels, lse, grad_scale=scale, row_grad=row_grad, ignore_index=ignore,
                                   dw_dtype=dw_dtype)
        wx, ww, bx, bw = _reference(x, w, labels, lse, scale, row_grad, ignore, dw_dtype)
        _within(dx, wx, bx, "dx")
        _within(dw, ww, bw, "dw")
    return lse, dx, dw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,vocab", [(65, 8, 300), (100, 96, 3000), (130, 57, 2500), (300, 136, 5000),
                                              (333, 768, 20011), (129, 1001, 1000)])
def test_labels_keep_what_rounding_leaves(K, dtype, rows, width, vocab):
    print(f"case: labels {rows} x {width} x {vocab} {dtype}", flush=True)
    for lean in (0.0, 8.0):
        x, w, labels, row_grad = _inputs(1, rows, width, vocab, dtype, lean)
        labels[0], labels[-1], labels[1] = vocab - 1, 0, vocab // 256 * 256  # edges of tiles
        _check(K, x, w, labels)
        _check(K, x, w, labels, scale=1 / 3, row_grad=row_grad)
        labels[2::7] = -100
        labels[3] = vocab
        _check(K, x, w, labels, row_grad=row_grad, ignore=-100)


@pytest.mark.parametrize("dtype", TYPES)
def test_one_label_for_all_and_few_classes(K, dtype):
    """Many labels in one wave's classes: every step of a k tile has some."""
    for rows, width, vocab in ((200, 64, 2000), (1000, 136, 300), (2500, 24, 5)):
        print(f"case: one label {rows} x {width} x {vocab} {dtype}", flush=True)
        x, w, labels, row_grad = _inputs(2, rows, width, vocab, dtype)
        _check(K, x, w, labels, row_grad=row_grad)
        labels[:] = 3
        _check(K, x, w, labels, row_grad=row_grad)
        labels[::2] = 4
        _check(K, x, w, labels, row_grad=row_grad, ignore=4)


@pytest.mark.parametrize("dtype", TYPES)
def test_labels_of_every_piece_and_run(K, dtype):
    """g in pieces of the vocabulary, dw's rows in runs, 64-bit labels and rows off the 16-byte boundaries."""
    for rows, width, vocab in ((16500, 24, 33000), (4571, 64, 2148)):
        print(f"case: pieces {rows} x {width} x {vocab} {dtype}", flush=True)
        x, w, labels, _ = _inputs(3, rows, width, vocab, dtype)
        labels[5], labels[6] = vocab - 1, 0
        _check(K, x, w, labels, scale=1 / 64)
    x, w, labels, row_grad = _inputs(4, 257, 100, 4000, dtype)
    sea_x, sea_w = (torch.full((t.shape[0], 103), float("nan"), dtype=dtype, device="cuda") for t in (x, w))
    sea_x[:, 1:101], sea_w[:, 2:102] = x, w
    lse, dx, dw = _check(K, sea_x[:, 1:101], sea_w[:, 2:102], labels.long(), row_grad=row_grad)
    _, dx2, dw2 = _check(K, x, w, labels, row_grad=row_grad)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


@pytest.mark.parametrize("dtype", TYPES)
def test_labels_in_graphs_and_on_streams(K, dtype):
    x, w, labels, row_grad = _inputs(5, 400, 96, 3000, dtype)
    x2, w2, labels2, _ = _inputs(6, 400, 96, 3000, dtype)
    wants = []
    for a in ((x, w, labels), (x2, w2, labels2)):
        lse = K.linear_xent(*a)[1]
        wants.append((lse, K.linear_xent_bwd(*a, lse, row_grad=row_grad)))
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = K.linear_xent_bwd(x, w, labels, wants[0][0], row_grad=row_grad)
    for _ in range(3):
        got[0].zero_(), got[1].zero_()
        graph.replay()
        other = K.linear_xent_bwd(x2, w2, labels2, wants[1][0], row_grad=row_grad, stream=torch.cuda.Stream())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, wants[0][1]))
        assert all(torch.equal(a, b) for a, b in zip(other, wants[1][1]))
