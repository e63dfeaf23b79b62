"""A GPT-2 training step on a stream of its own, made on another: the step starts
after the fills and copies that made its buffers, whichever stream is busy."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def G(cuda):
    from mi355x_pjrt import gpt2

    return gpt2


def test_buffers_are_filled_before_the_first_step(G):
    """The current stream is held for a tenth of a second while the step's buffers are made."""

    class Late(G.GPT2TrainStep):
        def _alloc(self):
            torch.cuda._sleep(200_000_000)
            super()._alloc()

    cfg = G.GPT2Config(n_layer=1, d_model=128, n_head=2, seq=128, batch=1, vocab=257, dropout=0.25)
    ids = np.random.default_rng(1).integers(0, cfg.vocab, (cfg.batch, cfg.seq))
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    want = G.GPT2TrainStep(cfg, dropout_seed=5)
    want.set_batch(ids, ids)
    want.forward_backward()
    torch.cuda.synchronize()
    step = Late(cfg, dropout_seed=5, stream=stream)
    with torch.cuda.stream(other):
        step.set_batch(ids, ids)  # not behind the stream that is held
    step.forward_backward()
    torch.cuda.synchronize()
    assert int(step.drop_step) == int(want.drop_step) == 1
    assert torch.equal(step.loss_sum, want.loss_sum) and torch.equal(step.grad, want.grad)
