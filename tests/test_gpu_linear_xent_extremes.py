"""linear_xent and linear_xent_bwd where logits lie at the ends of fp32's range, as
classes or whole rows masked by weights of a type's lowest value have them: products
with log2(e) are beyond it, the losses and gradients are not."""

import pytest
import torch

from xent_dropout_ref import xent

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def K(cuda):
    from mi355x_pjrt import kernels

    kernels.lib()
    return kernels


def _inputs(seed, rows, width, vocab, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn((vocab, width), generator=g, device="cuda") * (2 / width ** 0.5)).to(dtype)
    x = torch.randn((rows, width), generator=g, device="cuda").to(dtype)
    w[:, 0], x[:, 0] = 0, 1
    return x, w, torch.randint(vocab, (rows,), generator=g, device="cuda").int()


def _within(got, want, bound, what):
    assert bool(torch.isfinite(got).all()), what
    assert float(((got.double() - want).abs() - bound).max()) <= 0, what


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,vocab", [(1, 16, 40), (20, 24, 700), (100, 64, 300), (300, 72, 2500), (2000, 64, 20000)])
def test_rows_whose_classes_are_all_masked(K, dtype, rows, width, vocab):
    """Every class at the lowest value: a row's logits are that value, to which the rest of the sum
    adds nothing, and so is its lse in fp32; each loss is what is left of lse, below a step of it."""
    print(f"case: lowest {rows} x {width} x {vocab} {dtype}", flush=True)
    x, w, labels = _inputs(1, rows, width, vocab, dtype)
    for value in (torch.finfo(dtype).min, torch.finfo(dtype).max, torch.finfo(dtype).min * 0.75, 45000.0, -1e4, 700.0) + \
            ((1e6, -1e10, 1e20) if dtype != torch.float16 else ()):
        w[:, 0] = value
        loss, lse = K.linear_xent(x, w, labels)
        want, want_lse, bound = xent(x, w, labels)
        _within(lse, want_lse, bound, "lse")
        _within(loss, want, bound, "loss")
        if abs(value) > 1e19:
            assert torch.all(loss == 0) and torch.all(lse == float(w[0, 0]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 40, 64, 100, 200, 256])
def test_one_class_above_all(K, dtype, rows):
    """A class at the largest value among zeros: the whole probability is its own, exactly, and the
    gradients are counts of rows, which every type here holds."""
    vocab, width, top = 1100, 8, 333
    print(f"case: largest {rows} {dtype}", flush=True)
    for value in (torch.finfo(dtype).max, torch.finfo(dtype).max / 2, torch.finfo(dtype).max * 0.7, 60000.0, 1000.0):
        x = torch.zeros(rows, width, device="cuda", dtype=dtype)
        w = torch.zeros(vocab, width, device="cuda", dtype=dtype)
        x[:, 0] = 1
        w[top, 0] = value
        value = float(w[top, 0])
        labels = torch.arange(rows, device="cuda").int() % 7 * 50
        labels[::3] = top
        loss, lse = K.linear_xent(x, w, labels)
        assert torch.all(lse == value)
        assert torch.all(loss[::3] == 0) and torch.all(loss[labels != top] == value)
        _, dw = K.linear_xent_bwd(x, w, labels, lse, want_dx=False)
        want = torch.zeros(vocab, device="cuda")
        others = labels[labels != top].long()
        want[top] = others.numel()
        want -= torch.bincount(others, minlength=vocab).float()
        assert torch.equal(dw[:, 0].float(), want.to(dtype).float())
        assert torch.all(dw[:, 1:] == 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 50, 200])
def test_all_masked_gradient(K, dtype, rows):
    """Logits that are all the lowest value equal their lse in fp32, and the gradient is formed from the
    two as they are: 1 for every class, 0 for the label's."""
    vocab, width = 90, 8
    print(f"case: masked gradient {rows} {dtype}", flush=True)
    x = torch.zeros(rows, width, device="cuda", dtype=dtype)
    w = torch.zeros(vocab, width, device="cuda", dtype=dtype)
    x[:, 0] = 1
    w[:, 0] = torch.finfo(dtype).min
    labels = torch.arange(rows, device="cuda").int() % vocab
    lse = torch.full((rows,), float(w[0, 0]), device="cuda")
    _, dw = K.linear_xent_bwd(x, w, labels, lse, want_dx=False)
    want = rows - torch.bincount(labels.long(), minlength=vocab).float()
    assert torch.equal(dw[:, 0].float(), want.to(dtype).float())


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_nan_stay(K, dtype):
    """A logit of +inf or NaN leaves its row's loss and lse NaN (inf - inf), of -inf nothing; rows beside them
    are as they were."""
    for rows in (4, 300):
        print(f"case: infinities {rows} {dtype}", flush=True)
        x, w, labels = _inputs(2, rows, 16, 500, dtype)
        labels[:] = 9
        loss, lse = K.linear_xent(x, w, labels)
        y = x.clone()
        y[1], y[2] = float("nan"), float("inf")
        got, got_lse = K.linear_xent(y, w, labels)
        others = torch.ones(rows, dtype=torch.bool, device="cuda")
        others[1:3] = False
        assert torch.equal(got[others], loss[others]) and torch.equal(got_lse[others], lse[others])
        assert torch.isnan(got_lse[1:3]).all() and torch.isnan(got[1:3]).all()
        v = w.clone()
        v[100:200, 0] = float("-inf")  # x's first column is 1
        live = torch.cat([torch.arange(100), torch.arange(200, 500)]).cuda()
        got, got_lse = K.linear_xent(x, v, labels)
        want, want_lse, bound = xent(x, w[live], labels)
        _within(got, want, bound, "loss")
        _within(got_lse, want_lse, bound, "lse")
