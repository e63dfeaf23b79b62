"""dropout_add and dropout_add_bwd on the MI355X against their definitions in
64 bits (tests/xent_dropout_ref.py).  Which elements are dropped is exact; values
are off by the roundings of (x + bias) * scale + residual: one each, and the
scale's own."""

import pytest
import torch

from xent_dropout_ref import H32, dropout_keep, half_step, subnormal

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
COLS = [1, 7, 8, 9, 64, 100, 768, 1001, 2056, 4097]


@pytest.fixture(scope="module")
def K(cuda):
    from mi355x_pjrt import kernels

    kernels.lib()
    return kernels


def _normal(seed, shape, dtype, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda()


def _check_out(got, x, bias, residual, p, seed, offset):
    rows, cols = x.shape
    keep, scale = dropout_keep(rows, cols, p, seed, offset)
    x64, b = x.cpu().double(), 0.0 if bias is None else bias.cpu().double()
    r = torch.zeros(rows, cols, dtype=torch.float64) if residual is None else residual.cpu().double()
    branch = (x64 + b) * scale
    want = torch.where(keep, r + branch, r)
    bound = 3 * H32 * branch.abs() + (half_step(x.dtype) + H32) * want.abs() + subnormal(x.dtype)
    got = got.cpu()
    assert torch.equal(got[~keep], r[~keep].to(x.dtype))
    assert torch.all((got.double() - want).abs() <= bound)


def _check_bwd(dx, colsum, dy, p, seed, offset):
    rows, cols = dy.shape
    keep, scale = dropout_keep(rows, cols, p, seed, offset)
    want = torch.where(keep, dy.cpu().double() * scale, 0.0)
    dx = dx.cpu()
    assert torch.all(dx[~keep] == 0)
    assert torch.all((dx.double() - want).abs() <= (half_step(dy.dtype) + 2 * H32) * want.abs() + subnormal(dy.dtype))
    if colsum is not None:
        assert torch.all((colsum.cpu().double() - want.sum(0)).abs() <= (rows + 4) * H32 * want.abs().sum(0) + 1e-44)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", COLS)
def test_dropout_add(K, dtype, cols):
    for rows in (1, 3, 65, 700):
        print(f"case: dropout_add {rows} x {cols} {dtype}", flush=True)
        x, bias, res = _normal(1, (rows, cols), dtype), _normal(2, (cols,), dtype), _normal(3, (rows, cols), dtype, 3.0)
        for k, (b, r, p) in enumerate(((bias, res, 0.1), (None, res, 0.5), (bias, None, 0.25), (None, None, 0.9))):
            seed, offset = (1 << 63) + 12345 * k + cols, (7 << 32) + k
            _check_out(K.dropout_add(x, p, seed, offset=offset, bias=b, residual=r), x, b, r, p, seed, offset)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", COLS)
def test_dropout_add_bwd(K, dtype, cols):
    for rows in (1, 3, 65, 700, 5000) if cols <= 1001 else (1, 300):
        print(f"case: dropout_add_bwd {rows} x {cols} {dtype}", flush=True)
        dy = _normal(4, (rows, cols), dtype)
        dx, colsum = K.dropout_add_bwd(dy, 0.1, 99, offset=5, want_colsum=True)
        _check_bwd(dx, colsum, dy, 0.1, 99, 5)
        alone, none = K.dropout_add_bwd(dy, 0.1, 99, offset=5)
        assert none is None and torch.equal(alone, dx)


def test_probabilities_and_extremes(K):
    x = _normal(5, (200, 96), torch.float32)
    assert torch.equal(K.dropout_add(x, 0.0, 1), x)
    assert torch.all(K.dropout_add(x, 1.0, 1) == 0)
    assert torch.equal(K.dropout_add(x, 1.0, 1, residual=x), x)
    dx, colsum = K.dropout_add_bwd(x, 1.0, 1, want_colsum=True)
    assert torch.all(dx == 0) and torch.all(colsum == 0)
    for p in (2.0 ** -16, 0.3333, 1 - 2.0 ** -16):
        _check_out(K.dropout_add(x, p, 2 ** 64 - 1, offset=2 ** 64 - 1), x, None, None, p, 2 ** 64 - 1, 2 ** 64 - 1)
    # what is dropped may hold anything
    for dtype in TYPES:
        x = _normal(6, (64, 64), dtype)
        keep, _ = dropout_keep(64, 64, 0.5, 3, 4)
        bad = torch.where(keep.cuda(), x, torch.tensor(float("nan"), dtype=dtype, device="cuda"))
        bad[0] = torch.where(keep[0].cuda(), x[0], torch.tensor(float("inf"), dtype=dtype, device="cuda"))
        assert torch.equal(K.dropout_add(bad, 0.5, 3, offset=4), K.dropout_add(x, 0.5, 3, offset=4))
        for a, b in zip(K.dropout_add_bwd(bad, 0.5, 3, offset=4, want_colsum=True),
                        K.dropout_add_bwd(x, 0.5, 3, offset=4, want_colsum=True)):
            assert torch.equal(a, b)


def test_a_mask_is_its_numbers(K):
    """The same elements whatever the type, pitch and rows beside; others for another seed, offset or step."""
    ones = torch.ones(300, 200, device="cuda")
    kept = K.dropout_add(ones, 0.5, 11, offset=2) != 0
    for dtype in TYPES:
        wide = torch.ones(100, 333, dtype=dtype, device="cuda")
        assert torch.equal(K.dropout_add(wide[:, 5:205], 0.5, 11, offset=2) != 0, kept[:100])
    step = torch.tensor([1], dtype=torch.int64, device="cuda")
    assert torch.equal(K.dropout_add(ones, 0.5, 11, offset=1, step=step) != 0, kept)
    for other in (dict(seed=12, offset=2), dict(seed=11, offset=3), dict(seed=11 + 2 ** 32, offset=2),
                  dict(seed=11, offset=2 + 2 ** 32)):
        diff = ((K.dropout_add(ones, 0.5, **other) != 0) != kept).double().mean()
        assert 0.45 < float(diff) < 0.55  # 60000 draws: 24 deviations on each side
    big = torch.ones(4096, 4096, dtype=torch.bfloat16, device="cuda")
    share = float((K.dropout_add(big, 0.1, 77) == 0).double().mean())
    assert abs(share - 6554 / 65536) < 6 * (0.1 * 0.9 / 2 ** 24) ** 0.5


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_in_place_and_past_the_rows(K, dtype):
    for cols, pitch, off in ((257, 301, 1), (768, 768, 3), (1030, 1033, 5), (40, 41, 1)):
        x, res = _normal(7, (9, cols), dtype), _normal(8, (9, cols), dtype)
        want = K.dropout_add(x, 0.3, 5, residual=res)
        want_dx, want_sum = K.dropout_add_bwd(x, 0.3, 5, want_colsum=True)

        def view(t):
            sea = torch.full((9 * pitch + off + 64,), 77, dtype=dtype, device="cuda")
            v = sea[off:off + 9 * pitch].view(9, pitch)[:, :cols]
            v.copy_(t)
            return sea, v

        for target in ("x", "residual", "new"):
            (sx, xv), (sr, rv), (so, ov) = view(x), view(res), view(x)
            sea, out = {"x": (sx, xv), "residual": (sr, rv), "new": (so, ov)}[target]
            assert K.dropout_add(xv, 0.3, 5, residual=rv, out=out) is out
            assert torch.equal(out, want)
            out.fill_(77)
            assert torch.all(sea == 77)
        for place in (True, False):
            (sx, xv), (so, ov) = view(x), view(x)
            sea, out = (sx, xv) if place else (so, ov)
            dx, colsum = K.dropout_add_bwd(xv, 0.3, 5, want_colsum=True, dx=out)
            assert torch.equal(dx, want_dx) and torch.equal(colsum, want_sum)
            out.fill_(77)
            assert torch.all(sea == 77)
        row = x[:1].expand(9, cols)  # one row for all
        _check_out(K.dropout_add(row, 0.3, 5), row, None, None, 0.3, 5, 0)


def test_no_elements(K):
    assert K.dropout_add(torch.zeros(0, 8, device="cuda"), 0.1, 1).shape == (0, 8)
    assert K.dropout_add(torch.zeros(8, 0, device="cuda"), 0.1, 1).shape == (8, 0)
    dx, colsum = K.dropout_add_bwd(torch.zeros(0, 8, device="cuda"), 0.1, 1, want_colsum=True)
    assert dx.shape == (0, 8) and torch.equal(colsum, torch.zeros(8, device="cuda"))


def test_more_columns_than_a_grid_of_sums(K):
    """One row of 2^27 + 40 columns: its sums are the row itself."""
    cols = (1 << 27) + 40
    dy = torch.randn(1, cols, device="cuda").bfloat16()
    dx, colsum = K.dropout_add_bwd(dy, 0.25, 3, want_colsum=True)
    kept = dx[0] != 0
    assert abs(float(kept.double().mean()) - 0.75) < 6 * (0.1875 / cols) ** 0.5 + 2.0 ** -8  # a few values round to 0
    want = torch.where(kept, dy[0].float(), 0.0) * float(torch.tensor(65536 / (65536 - 16384), dtype=torch.float32))
    assert torch.equal(colsum, want)
    keep, _ = dropout_keep(1, 4096, 0.25, 3, 0)
    assert torch.equal(kept[:4096].cpu() | (dy[0, :4096].cpu() == 0), keep[0] | (dy[0, :4096].cpu() == 0))


def test_numbers_of_numpy(K):
    import numpy as np

    x = _normal(11, (20, 40), torch.float32)
    assert torch.equal(K.dropout_add(x, np.float64(0.5), np.int64(7), offset=np.uint64(2 ** 63)),
                       K.dropout_add(x, 0.5, 7, offset=2 ** 63))


def test_streams_and_graphs(K):
    """A captured step draws anew on every replay from its device number, forward and backward alike."""
    x, bias = _normal(9, (500, 104), torch.bfloat16), _normal(10, (104,), torch.bfloat16)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    streams, graphs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    torch.cuda.synchronize()
    for k, s in enumerate(streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = K.dropout_add(x, 0.2, 8 + k, offset=3, step=step, bias=bias, residual=x)
            dx, colsum = K.dropout_add_bwd(x, 0.2, 8 + k, offset=3, step=step, want_colsum=True)
        graphs.append((graph, out, dx, colsum))
    for n in range(4):
        step.fill_(n * 2 ** 31)
        for graph, *outs in graphs:
            for t in outs:
                t.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for k, (_, out, dx, colsum) in enumerate(graphs):
            offset = 3 + n * 2 ** 31
            _check_out(out, x, bias, x, 0.2, 8 + k, offset)
            _check_bwd(dx, colsum, x, 0.2, 8 + k, offset)
            s = streams[k]
            with torch.cuda.stream(s):
                pass
            eager = K.dropout_add(x, 0.2, 8 + k, offset=offset, bias=bias, residual=x, stream=s)
            again = K.dropout_add_bwd(x, 0.2, 8 + k, offset=offset, want_colsum=True, stream=s)
            torch.cuda.synchronize()
            assert torch.equal(eager, out) and torch.equal(again[0], dx) and torch.equal(again[1], colsum)


def test_wrapper_refusals(K):
    x = torch.zeros(4, 8, device="cuda")
    for bad in (lambda: K.dropout_add(x.double(), 0.1, 1), lambda: K.dropout_add(x.t(), 0.1, 1),
                lambda: K.dropout_add(x.cpu(), 0.1, 1), lambda: K.dropout_add(x, 0.1, -1),
                lambda: K.dropout_add(x, 0.1, 1, offset=2 ** 64), lambda: K.dropout_add(x, 0.1, 1, bias=x[0, :4]),
                lambda: K.dropout_add(x, 0.1, 1, residual=x.half()), lambda: K.dropout_add(x, 0.1, 1, residual=x[:2]),
                lambda: K.dropout_add(x, 0.1, 1, out=x[:2]), lambda: K.dropout_add(x, 0.1, 1, step=x),
                lambda: K.dropout_add_bwd(x, 0.1, 1, colsum=x[0, :4])):
        with pytest.raises(ValueError):
            bad()
    from mi355x_pjrt._lib import KernelError

    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(KernelError, match="p must be"):
            K.dropout_add(x, p, 1)


def test_the_operators_together(K):
    """The end of a training step: a projection's branch dropped into the residual
    stream, the loss against the embedding, and back, against torch's autograd in
    64 bits with the same mask; bounds are of relative size, from bf16 roundings of
    the stream (2^-8) and of the gradient's operand and results (3 of 2^-8)."""
    rows, width, vocab, p = 200, 96, 700, 0.2
    g = torch.Generator(device="cuda").manual_seed(5)

    def make(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).bfloat16()

    branch, bias, stream, w = make(rows, width), make(width), make(rows, width), make(vocab, width, std=0.2)
    labels = torch.randint(vocab, (rows,), generator=g, device="cuda").int()
    h = K.dropout_add(branch, p, 21, bias=bias, residual=stream)
    loss, lse = K.linear_xent(h, w, labels)
    dh, dw = K.linear_xent_bwd(h, w, labels, lse, grad_scale=1.0 / rows)
    db, dbias = K.dropout_add_bwd(dh, p, 21, want_colsum=True)
    keep, scale = dropout_keep(rows, width, p, 21, 0)
    leaves = [t.double().requires_grad_(True) for t in (branch, bias, stream, w)]
    exact = leaves[2] + (leaves[0] + leaves[1]) * keep.cuda() * scale
    rounded = exact + (h.double() - exact).detach()  # the stream as it is kept
    want = torch.nn.functional.cross_entropy(rounded @ leaves[3].t(), labels.long())
    want.backward()
    assert torch.all((h.double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 1e-6)
    assert abs(float(loss.double().mean()) - float(want)) <= 1e-4
    for got, leaf in ((db, leaves[0]), (dbias, leaves[1]), (dh, leaves[2]), (dw, leaves[3])):
        err = (got.double() - leaf.grad).norm() / leaf.grad.norm()
        assert float(err) <= 3 * 2.0 ** -8
