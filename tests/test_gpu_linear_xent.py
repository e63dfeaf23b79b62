"""linear_xent and linear_xent_bwd on the MI355X against their definitions in
64 bits (tests/xent_dropout_ref.py, which derives the bounds)."""

import pytest
import torch

from xent_dropout_ref import H32, xent, xent_grad

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def K(cuda):
    from mi355x_pjrt import kernels

    kernels.lib()
    return kernels


def _inputs(seed, rows, width, vocab, dtype, label_type=torch.int32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn((vocab, width), generator=g, device="cuda") * (2 / width ** 0.5)).to(dtype)
    x = torch.randn((rows, width), generator=g, device="cuda").to(dtype)
    labels = torch.randint(vocab, (rows,), generator=g, device="cuda").to(label_type)
    return x, w, labels


def _within(got, want, bound, what):
    err = (got.double() - want).abs() - bound
    assert bool(torch.isfinite(got).all()), what
    assert float(err.max()) <= 0, (what, float(err.max()), float((got.double() - want).abs().max()))


def _check(K, x, w, labels, scale=1.0, row_grad=None, ignore=None, dw_dtype=None, **kw):
    loss, lse = K.linear_xent(x, w, labels, ignore_index=ignore)
    want, want_lse, bound = xent(x, w, labels, ignore)
    _within(lse, want_lse, bound, "lse")
    _within(loss, want, bound, "loss")
    if ignore is not None:
        assert torch.all(loss[labels == ignore] == 0)
    dx, dw = K.linear_xent_bwd(x, w, labels, lse, grad_scale=scale, row_grad=row_grad, ignore_index=ignore,
                               dw_dtype=dw_dtype, **kw)
    assert dx.dtype == x.dtype and dw.dtype == (dw_dtype or w.dtype)
    wx, ww, bx, bw = xent_grad(x, w, labels, lse, scale, row_grad, ignore, dw_dtype)
    _within(dx, wx, bx, "dx")
    _within(dw, ww, bw, "dw")
    if ignore is not None:
        assert torch.all(dx[labels == ignore] == 0)
    return loss, lse, dx, dw


# one of everything, the tiles' edges in each direction, odd sizes that are copied first
SHAPES = [(1, 1, 1), (1, 8, 2), (2, 7, 129), (3, 64, 1000), (16, 768, 5003), (100, 97, 257), (127, 128, 127),
          (128, 136, 256), (129, 1, 300), (200, 264, 1025), (255, 33, 255), (257, 768, 2049), (600, 200, 777)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,vocab", SHAPES)
def test_shapes(K, dtype, rows, width, vocab):
    print(f"case: linear_xent {rows} x {width} x {vocab} {dtype}", flush=True)
    x, w, labels = _inputs(rows + width, rows, width, vocab, dtype)
    _check(K, x, w, labels, scale=1.0 / rows)


@pytest.mark.parametrize("dtype", TYPES)
def test_ignored_rows_hold_anything(K, dtype):
    for rows, width, vocab in ((90, 64, 300), (300, 72, 600)):
        for ignore in (-100, 5):
            print(f"case: ignored rows {rows} {ignore} {dtype}", flush=True)
            x, w, labels = _inputs(1, rows, width, vocab, dtype, torch.int64)
            labels[::3] = ignore
            clean = x.clone()
            x[::6] = float("nan")
            x[3::6] = float("inf")
            loss, lse = K.linear_xent(x, w, labels, ignore_index=ignore)
            want, want_lse, bound = xent(clean, w, labels, ignore)
            kept = labels != ignore
            _within(loss[kept], want[kept], bound[kept], "loss")
            assert torch.all(loss[~kept] == 0)
            lse = torch.where(kept, lse, float("nan"))
            dx, dw = K.linear_xent_bwd(x, w, labels, lse, ignore_index=ignore)
            wx, ww, bx, bw = xent_grad(clean, w, labels, torch.where(kept, lse, 0.0), ignore=ignore)
            _within(dx, wx, bx, "dx")
            _within(dw, ww, bw, "dw")
            assert torch.all(dx[~kept] == 0)
            labels[:] = ignore  # nothing is left
            loss, lse = K.linear_xent(x, w, labels, ignore_index=ignore)
            dx, dw = K.linear_xent_bwd(x, w, labels, lse, ignore_index=ignore)
            assert torch.all(loss == 0) and torch.all(dx == 0) and torch.all(dw == 0)


@pytest.mark.parametrize("dtype", TYPES)
def test_weights_and_labels_outside(K, dtype):
    for rows in (50, 270):
        x, w, labels = _inputs(2, rows, 80, 400, dtype)
        labels[0], labels[1], labels[2] = -1, 400, 2 ** 31 - 1  # no target term
        row_grad = torch.rand(rows, device="cuda") * 4 - 1
        row_grad[5] = 0
        row_grad[6] = 1e-6
        print(f"case: row_grad {rows} {dtype}", flush=True)
        loss, lse, dx, _ = _check(K, x, w, labels, scale=0.5, row_grad=row_grad, ignore=400)
        assert torch.equal(loss[:1], lse[:1]) and torch.all(dx[5] == 0)
        zero = torch.zeros(rows, device="cuda")
        dx, dw = K.linear_xent_bwd(x, w, labels, lse, row_grad=zero)
        assert torch.all(dx == 0) and torch.all(dw == 0)


def test_large_factors_keep_fp16_in_range(K):
    x, w, labels = _inputs(3, 140, 64, 500, torch.float16)
    _, lse = K.linear_xent(x, w, labels)
    for power in (-60, -20, 0, 20, 60):
        row_grad = torch.full((140,), 1.5 * 2.0 ** power, device="cuda")
        dx, dw = K.linear_xent_bwd(x, w, labels, lse, grad_scale=2.0 ** -power, row_grad=row_grad)
        if power == -60:
            first = dx, dw
        assert torch.equal(dx, first[0]) and torch.equal(dw, first[1])  # powers of two change no bit


def test_fp16_range_of_row_gradients(K):
    """Their largest finite value sets fp16's range; an ignored row's, whatever it holds, does not."""
    x, w, labels = _inputs(13, 140, 64, 500, torch.float16)
    _, lse = K.linear_xent(x, w, labels)
    want = K.linear_xent_bwd(x, w, labels, lse, row_grad=torch.full((140,), 1.5, device="cuda"))
    for power in (-110, 110, 126):
        row_grad = torch.full((140,), 1.5 * 2.0 ** power, device="cuda")
        got = K.linear_xent_bwd(x, w, labels, lse, grad_scale=2.0 ** -power, row_grad=row_grad)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    row_grad = torch.rand(140, device="cuda") + 0.5
    labels[::5] = -100
    row_grad[::5] = 0
    want = K.linear_xent_bwd(x, w, labels, lse, row_grad=row_grad, ignore_index=-100)
    row_grad[::5] = torch.tensor([1e30, float("inf"), float("nan"), -3e38], device="cuda").repeat(7)
    got = K.linear_xent_bwd(x, w, labels, lse, row_grad=row_grad, ignore_index=-100)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_a_row_of_nan_stays_one(K, dtype):
    """A row that counts and holds a NaN spoils its own dx and all of dw, beside ignored rows and at the last
    classes alike, also with a row_grad of 0; no other row's dx."""
    x, w, labels = _inputs(14, 150, 40, 300, dtype)
    labels[::3] = -100
    row_grad = torch.ones(150, device="cuda")
    row_grad[4] = 0
    _, lse = K.linear_xent(x, w, labels, ignore_index=-100)
    want, _ = K.linear_xent_bwd(x, w, labels, lse, row_grad=row_grad, ignore_index=-100)
    x[4, 7] = lse[4] = float("nan")
    dx, dw = K.linear_xent_bwd(x, w, labels, lse, row_grad=row_grad, ignore_index=-100)
    others = torch.arange(150, device="cuda") != 4
    assert torch.equal(dx[others], want[others])
    assert torch.isnan(dx[4]).all() and torch.isnan(dw).all()


def test_no_rows_of_a_large_gradient(K):
    w = torch.zeros(1, 32768, dtype=torch.bfloat16, device="cuda").expand(140000, 32768)
    x = torch.zeros(0, 32768, dtype=torch.bfloat16, device="cuda")
    dw = torch.full((140000, 32768), 7.0, dtype=torch.bfloat16, device="cuda")
    K.linear_xent_bwd(x, w, torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, device="cuda"), dw=dw)
    assert not any(bool(dw[i:i + 20000].any()) for i in range(0, 140000, 20000))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_offsets_and_outputs(K, dtype):
    """Views of any pitch and start give the same numbers; nothing is written past a row's end."""
    esz = torch.finfo(dtype).bits // 8
    for rows, width, vocab in ((70, 48, 300), (300, 48, 700), (140, 39, 150)):
        x, w, labels = _inputs(4, rows, width, vocab, dtype)
        loss, lse = K.linear_xent(x, w, labels)
        dx, dw = K.linear_xent_bwd(x, w, labels, lse)
        for pitch, off in ((width, 1), (width + 3, 0), (64, 0), (width + 5, 3)):
            print(f"case: pitch {pitch} offset {off} of {rows} x {width} x {vocab} {dtype}", flush=True)

            def view(t, fill=77.0):
                sea = torch.full((t.shape[0] * pitch + off + 9,), fill, dtype=t.dtype, device="cuda")
                v = sea[off:off + t.shape[0] * pitch].view(t.shape[0], pitch)[:, :t.shape[1]]
                v.copy_(t)
                return sea, v

            (_, xv), (_, wv) = view(x, float("nan")), view(w, float("nan"))
            (sea_dx, dxv), (sea_dw, dwv) = view(torch.zeros_like(x)), view(torch.zeros_like(w))
            l2, z2 = K.linear_xent(xv, wv, labels)
            assert torch.equal(l2, loss) and torch.equal(z2, lse)
            K.linear_xent_bwd(xv, wv, labels, lse, dx=dxv, dw=dwv)
            assert torch.equal(dxv, dx) and torch.equal(dwv, dw)
            for sea, n in ((sea_dx, rows), (sea_dw, vocab)):
                past = torch.ones(sea.numel(), dtype=torch.bool, device="cuda")
                past[off:off + n * pitch].view(n, pitch)[:, :width] = False
                assert torch.all(sea[past] == 77)
    # every row the same row
    row = torch.randn(1, 64, device="cuda").to(dtype)
    x, w = row.expand(40, 64), torch.randn(90, 64, device="cuda").to(dtype)
    _check(K, x, w, torch.arange(40, device="cuda", dtype=torch.int32))
    assert esz in (2, 4)


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("rows,width,vocab", [(1, 64, 500), (4, 208, 5819), (33, 39, 1000), (64, 768, 5003)])
def test_few_rows_keep_what_rounding_leaves(K, dtype, rows, width, vocab):
    """Up to 64 rows hold the gradients of the logits in two numbers of 16 bits."""
    print(f"case: few rows {rows} x {width} x {vocab} {dtype}", flush=True)
    x, w, labels = _inputs(11, rows, width, vocab, dtype, torch.int64)
    labels[rows // 2] = vocab - 1
    row_grad = torch.rand(rows, device="cuda") + 0.5
    for ignore in (None, int(labels[0])) if rows > 1 else (None,):
        _, lse = K.linear_xent(x, w, labels, ignore_index=ignore)
        dx, dw = K.linear_xent_bwd(x, w, labels, lse, row_grad=row_grad, ignore_index=ignore, dw_dtype=torch.float32)
        wx, ww, bx, bw = xent_grad(x, w, labels, lse, 1.0, row_grad, ignore, torch.float32, twice=True)
        _within(dx, wx, bx, "dx")
        _within(dw, ww, bw, "dw")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 5, 31, 32, 33])
def test_up_to_32_rows(K, dtype, rows):
    """The kernels of few rows: any pitch and start, ignored rows that hold anything, streams, graphs."""
    for width, vocab in ((130, 1000), (64, 70), (520, 333)):
        print(f"case: rows {rows} x {width} x {vocab} {dtype}", flush=True)
        x, w, labels = _inputs(15, rows, width, vocab, dtype, torch.int64)
        labels[-1] = vocab - 1
        row_grad = torch.rand(rows, device="cuda") + 0.5
        if rows > 1:
            labels[0] = -100
            row_grad[0] = float("nan")
        clean = torch.where((labels != -100)[:, None], x, torch.zeros_like(x))
        x = torch.where((labels != -100)[:, None], x, torch.full_like(x, float("inf")))
        kept = labels != -100
        loss, lse = K.linear_xent(x, w, labels, ignore_index=-100)
        want, want_lse, bound = xent(clean, w, labels, -100)
        _within(loss, want, bound, "loss")
        _within(lse[kept], want_lse[kept], bound[kept], "lse")
        dx, dw = K.linear_xent_bwd(x, w, labels, lse, grad_scale=0.5, row_grad=row_grad, ignore_index=-100,
                                   dw_dtype=torch.float32)
        wx, ww, bx, bw = xent_grad(clean, w, labels, torch.where(kept, lse, 0.0), 0.5,
                                   torch.where(kept, row_grad, 0.0), -100, torch.float32, twice=dtype != torch.float32)
        _within(dx, wx, bx, "dx")
        _within(dw, ww, bw, "dw")
        assert torch.all(dx[~kept] == 0)
        for pitch, off in ((width + 1, 1), (width + 11, 3)):
            def view(t):
                sea = torch.full((t.shape[0] * pitch + off + 9,), float("nan"), dtype=t.dtype, device="cuda")
                v = sea[off:off + t.shape[0] * pitch].view(t.shape[0], pitch)[:, :width]
                v.copy_(t)
                return sea, v

            (_, xv), (_, wv) = view(x), view(w)
            (sx, dxv), (sw, dwv) = view(torch.zeros_like(x)), view(torch.zeros(vocab, width, device="cuda"))
            l2, z2 = K.linear_xent(xv, wv, labels, ignore_index=-100)
            assert torch.equal(l2, loss) and torch.equal(z2[kept], lse[kept])
            K.linear_xent_bwd(xv, wv, labels, lse, grad_scale=0.5, row_grad=row_grad, ignore_index=-100, dx=dxv, dw=dwv)
            assert torch.equal(dxv, dx) and torch.equal(dwv, dw)
            dxv.fill_(float("nan")), dwv.fill_(float("nan"))
            assert torch.isnan(sx).all() and torch.isnan(sw).all()  # nothing past the rows' ends
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            l3, z3 = K.linear_xent(x, w, labels, ignore_index=-100)
            d3 = K.linear_xent_bwd(x, w, labels, z3, grad_scale=0.5, row_grad=row_grad, ignore_index=-100,
                                   dw_dtype=torch.float32)
        for _ in range(3):
            for t in (l3, z3, *d3):
                t.zero_()
            graph.replay()
            eager = K.linear_xent(x, w, labels, ignore_index=-100, stream=torch.cuda.Stream())
            torch.cuda.synchronize()
            assert torch.equal(l3, loss) and torch.equal(eager[0], loss)
            assert torch.equal(d3[0], dx) and torch.equal(d3[1], dw)


def test_few_rows_of_more_classes_than_a_piece(K):
    rows, width, vocab = 3, 8, (1 << 20) + 77
    x, w, labels = _inputs(16, rows, width, vocab, torch.bfloat16)
    labels[0], labels[1] = vocab - 1, 1 << 20
    _check(K, x, w, labels, dw_dtype=torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_of_few_classes(K, dtype):
    """The weights' gradient has few tiles here: its rows are cut into runs."""
    for rows, width, vocab in ((4571, 64, 2148), (9001, 16, 300), (3000, 130, 2)):
        print(f"case: many rows {rows} x {width} x {vocab} {dtype}", flush=True)
        x, w, labels = _inputs(12, rows, width, vocab, dtype)
        labels[::3] = -100
        sea = torch.full((vocab * (width + 3) + 5,), 77.0, device="cuda").to(dtype)
        dw = sea[5:].view(vocab, width + 3)[:, :width]
        _, lse, dx, alone = _check(K, x, w, labels, scale=1.0 / rows, ignore=-100)
        K.linear_xent_bwd(x, w, labels, lse, grad_scale=1.0 / rows, ignore_index=-100, dw=dw)
        assert torch.equal(dw, alone)
        assert torch.all(sea[:5] == 77) and torch.all(sea[5:].view(vocab, width + 3)[:, width:] == 77)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = K.linear_xent_bwd(x, w, labels, lse, grad_scale=1.0 / rows, ignore_index=-100)
        for _ in range(2):
            got[0].zero_(), got[1].zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got[0], dx) and torch.equal(got[1], alone)
            _check(K, x[:100], w, labels[:100])


def test_one_gradient_alone_and_fp32_weights_gradient(K):
    for dtype in TYPES:
        for rows in (60, 400):
            x, w, labels = _inputs(5, rows, 128, 900, dtype)
            _, lse, dx, dw = _check(K, x, w, labels, dw_dtype=torch.float32)
            assert K.linear_xent_bwd(x, w, labels, lse, want_dw=False)[1] is None
            assert torch.equal(K.linear_xent_bwd(x, w, labels, lse, want_dw=False)[0], dx)
            assert K.linear_xent_bwd(x, w, labels, lse, want_dx=False)[0] is None
            assert torch.equal(K.linear_xent_bwd(x, w, labels, lse, want_dx=False, dw_dtype=torch.float32)[1], dw)


def test_no_rows(K):
    x, w = torch.zeros(0, 40, device="cuda"), torch.randn(30, 40, device="cuda")
    labels = torch.zeros(0, dtype=torch.int64, device="cuda")
    loss, lse = K.linear_xent(x, w, labels)
    assert loss.shape == lse.shape == (0,)
    for dtype in TYPES:
        dw = torch.full((30, 44), 77.0, device="cuda").to(dtype)
        K.linear_xent_bwd(x.to(dtype), w.to(dtype), labels, lse, dw=dw[:, :40])
        assert torch.all(dw[:, :40] == 0) and torch.all(dw[:, 40:] == 77)


def test_minus_infinity_and_nan_logits(K):
    for dtype in TYPES:
        x, w, labels = _inputs(6, 20, 16, 200, dtype)
        w[:, 0], x[:, 0] = 0, 1
        w[50:150, 0] = torch.finfo(dtype).min  # masked classes: logits of the type's lowest value
        x[3] = float("nan")
        labels[:] = 7
        loss, lse = K.linear_xent(x, w, labels)
        keep = torch.arange(20, device="cuda") != 3
        live = torch.cat([torch.arange(50), torch.arange(150, 200)]).cuda()
        want, want_lse, bound = xent(x[keep], w[live], labels[keep])
        _within(loss[keep], want, bound, "loss")
        assert torch.isnan(loss[3]) and torch.isnan(lse[3])
        dx, dw = K.linear_xent_bwd(x[keep], w, labels[keep], lse[keep])
        _, ww, _, bw = xent_grad(x[keep], w[live], labels[keep], lse[keep])
        _within(dw[live], ww, bw, "dw")
        assert torch.all(dw[50:150] == 0)


def test_pieces_of_the_vocabulary(K):
    """More of g than one piece holds, and of copied weights."""
    for rows, width, vocab in ((16384, 64, 20011), (3, 1025, 131101)):
        print(f"case: pieces {rows} x {width} x {vocab}", flush=True)
        x, w, labels = _inputs(7, rows, width, vocab, torch.bfloat16)
        labels[-1] = vocab - 1
        loss, lse = K.linear_xent(x, w, labels)
        dx, dw = K.linear_xent_bwd(x, w, labels, lse)
        want_dw = bound_dw = 0
        for i in range(0, rows, 2048):
            at = slice(i, i + 2048)
            want, want_lse, bound = xent(x[at], w, labels[at])
            _within(loss[at], want, bound, "loss")
            wx, ww, bx, bw = xent_grad(x[at], w, labels[at], lse[at])
            _within(dx[at], wx, bx, "dx")
            want_dw, bound_dw = want_dw + ww, bound_dw + bw
        _within(dw, want_dw, bound_dw, "dw")


def test_weights_past_two_gigabytes(K):
    rows, width, vocab = 2, 8456, 131072
    w = torch.empty(vocab, width, dtype=torch.bfloat16, device="cuda")
    w.normal_(0, 0.02)
    x = torch.randn(rows, width, device="cuda").bfloat16()
    labels = torch.tensor([vocab - 1, 5], dtype=torch.int32, device="cuda")
    loss, lse = K.linear_xent(x, w, labels)
    dx, dw = K.linear_xent_bwd(x, w, labels, lse)
    z = torch.cat([x.double() @ w[i:i + 16384].double().t() for i in range(0, vocab, 16384)], dim=1)
    want = torch.logsumexp(z, dim=1)
    # bounds as in xent(): width products of at most 5 * 0.1, sums of sizes below 8456 * 0.015
    assert float((lse.double() - want).abs().max()) <= 2 * (width + 1) * H32 * 130 + H32 * 1e4
    assert float((loss.double() - (want - z.gather(1, labels.long()[:, None])[:, 0])).abs().max()) <= \
        2 * (width + 1) * H32 * 130 + H32 * 1e4
    g = torch.exp(z - lse.double()[:, None])
    g[torch.arange(2), labels.long()] -= 1
    for i in (0, 65536, 131000):  # rows of dw on both sides of 2^31 bytes
        want = g[:, i:i + 72].t() @ x.double()
        bound = (2.0 ** -8 * 2.1 + 1e-3) * (g[:, i:i + 72].abs().t() @ x.double().abs())
        assert torch.all((dw[i:i + 72].double() - want).abs() <= bound)
    want = sum(g[:, i:i + 16384] @ w[i:i + 16384].double() for i in range(0, vocab, 16384))
    size = sum(g[:, i:i + 16384].abs() @ w[i:i + 16384].double().abs() for i in range(0, vocab, 16384))
    assert torch.all((dx.double() - want).abs() <= (2.0 ** -8 + 131072 * H32 + 1e-3) * size + 2.0 ** -8 * want.abs())


def test_gradient_is_the_losses_difference(K):
    x, w, labels = _inputs(8, 12, 24, 60, torch.float32)
    weight = torch.rand(12, device="cuda")
    _, lse = K.linear_xent(x, w, labels)
    dx, dw = K.linear_xent_bwd(x, w, labels, lse, row_grad=weight)
    h = 2.0 ** -6

    def total(x, w):
        return float((K.linear_xent(x, w, labels)[0].double() * weight.double()).sum())

    # the third derivative of a log-sum-exp along one coordinate is at most the range of its slopes
    # cubed; a loss's rounding is below the bound of xent(), twelve of them over 2 h
    noise = 2 * float((xent(x, w, labels)[2] * weight.double()).sum()) / (2 * h)
    for n, d in ((0, 0), (5, 7), (11, 23)):
        lo, hi = x.clone(), x.clone()
        lo[n, d] -= h
        hi[n, d] += h
        step = float(hi[n, d].double() - lo[n, d].double())
        slope = float(w[:, d].max() - w[:, d].min()) ** 3 * h * h / 6
        assert abs((total(hi, w) - total(lo, w)) / step - float(dx[n, d])) <= noise + slope + 1e-6
    for v, d in ((int(labels[0]), 0), (13, 5), (59, 23)):
        lo, hi = w.clone(), w.clone()
        lo[v, d] -= h
        hi[v, d] += h
        step = float(hi[v, d].double() - lo[v, d].double())
        slope = float((x[:, d].abs() ** 3 * weight).sum()) * h * h / 6
        assert abs((total(x, hi) - total(x, lo)) / step - float(dw[v, d])) <= noise + slope + 1e-6


def test_same_bits_on_streams_and_in_graphs(K):
    cases = []
    for dtype, rows, width, vocab in ((torch.bfloat16, 300, 256, 3000), (torch.float16, 90, 57, 2000)):
        x, w, labels = _inputs(9, rows, width, vocab, dtype)
        labels[::4] = -100
        row_grad = torch.rand(rows, device="cuda")
        loss, lse = K.linear_xent(x, w, labels, ignore_index=-100)
        dx, dw = K.linear_xent_bwd(x, w, labels, lse, row_grad=row_grad, ignore_index=-100)
        cases.append((x, w, labels, row_grad, loss, lse, dx, dw))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):  # two calls at once, each with a workspace of its stream's
        got = []
        for s, c in zip(streams, cases):
            loss, lse = K.linear_xent(*c[:3], ignore_index=-100, stream=s)
            got.append((loss, lse) + K.linear_xent_bwd(*c[:3], lse, row_grad=c[3], ignore_index=-100, stream=s))
        torch.cuda.synchronize()
        for g, c in zip(got, cases):
            assert all(torch.equal(a, b) for a, b in zip(g, c[4:]))
    graphs = []
    for s, c in zip(streams, cases):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            loss, lse = K.linear_xent(*c[:3], ignore_index=-100)
            out = (loss, lse) + K.linear_xent_bwd(*c[:3], lse, row_grad=c[3], ignore_index=-100)
        graphs.append((graph, out))
    for _ in range(3):
        for graph, out in graphs:
            for t in out:
                t.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for (_, out), c in zip(graphs, cases):
            assert all(torch.equal(a, b) for a, b in zip(out, c[4:]))
        K.linear_xent(*cases[0][:3])  # the program's own work between replays


def test_wrapper_refusals(K):
    x, w, labels = _inputs(10, 8, 16, 20, torch.bfloat16)
    lse = torch.zeros(8, device="cuda")
    for bad in (lambda: K.linear_xent(x.double(), w, labels), lambda: K.linear_xent(x, w.float(), labels),
                lambda: K.linear_xent(x, w[:, :8], labels), lambda: K.linear_xent(x, w, labels[:4]),
                lambda: K.linear_xent(x, w, labels.short()), lambda: K.linear_xent(x, w, labels, ignore_index=2 ** 63), lambda: K.linear_xent(x.t(), w, labels),
                lambda: K.linear_xent(x.cpu(), w, labels), lambda: K.linear_xent(x, w, labels.cpu()),
                lambda: K.linear_xent(x, w, labels, workspace=torch.empty(8, dtype=torch.uint8, device="cuda")),
                lambda: K.linear_xent_bwd(x, w, labels, lse[:4]), lambda: K.linear_xent_bwd(x, w, labels, lse.double()),
                lambda: K.linear_xent_bwd(x, w, labels, lse, row_grad=lse[:3]),
                lambda: K.linear_xent_bwd(x, w, labels, lse, dw_dtype=torch.float16),
                lambda: K.linear_xent_bwd(x, w, labels, lse, dx=torch.empty(8, 16, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    from mi355x_pjrt._lib import KernelError

    with pytest.raises(KernelError, match="over"):
        K.linear_xent_bwd(x, w, labels, lse, dx=x)
