"""The GPT-2 training step without its logits in memory (linear_xent) and with
dropout (dropout_add), against the float64 restatement with the same masks
(oracle/gpt2_ref.py), eager and as a replayed graph.

Tolerances are those of tests/test_gpu_gpt2.py for the step without them: bf16
activations, each gradient by its relative L2 error, the loss to 2e-3."""

import numpy as np
import pytest
import torch

from oracle import gpt2_ref
from test_gpu_gpt2 import _params
from xent_dropout_ref import dropout_keep

pytestmark = pytest.mark.gpu
SEED = 2 ** 63 + 77


@pytest.fixture(scope="module")
def G(cuda):
    from mi355x_pjrt import gpt2

    return gpt2


def _config(G, dropout):
    return G.GPT2Config(n_layer=2, d_model=128, n_head=2, seq=128, batch=2, vocab=257, dropout=dropout)


def _batch(cfg, seed=5):
    rng = np.random.default_rng(seed)
    return rng.integers(0, cfg.vocab, (cfg.batch, cfg.seq)), rng.integers(0, cfg.vocab, (cfg.batch, cfg.seq))


def _masks(G, cfg, step):
    """Dropout's multipliers of the step-th draw."""
    if cfg.dropout == 0:
        return None
    out = []
    for site in range(2 * cfg.n_layer + 1):
        keep, scale = dropout_keep(cfg.tokens, cfg.d_model, cfg.dropout, SEED, site * G.GPT2TrainStep.DROP_SITE + step)
        out.append(keep.double().reshape(cfg.batch, cfg.seq, cfg.d_model) * scale)
    return torch.stack(out)


def _check(step, cfg, ids, labels, masks):
    loss = step.loss_value()
    ref_loss, ref = gpt2_ref.loss_and_grads(step.params_numpy(step.param), ids, labels, cfg.n_layer, cfg.n_head, drop=masks)
    assert abs(loss - ref_loss) < 2e-3 * abs(ref_loss), (loss, ref_loss)
    bad = {}
    for n, g in step.params_numpy(step.grad).items():
        e = float(np.linalg.norm(g - ref[n]) / max(np.linalg.norm(ref[n]), 1e-30))
        if e > 3e-2:
            bad[n] = e
    assert not bad, bad


@pytest.mark.parametrize("keep_logits,dropout", [(False, 0.0), (True, 0.2), (False, 0.1)])
def test_gradients(G, keep_logits, dropout):
    cfg = _config(G, dropout)
    print(f"case: gpt2 small keep_logits {keep_logits} dropout {dropout}", flush=True)
    step = G.GPT2TrainStep(cfg, params=_params(G, cfg), keep_logits=keep_logits, dropout_seed=SEED)
    assert hasattr(step, "logits") == keep_logits
    ids, labels = _batch(cfg)
    step.set_batch(ids, labels)
    for n in (1, 2):  # another draw each time
        step.forward_backward()
        torch.cuda.synchronize()
        _check(step, cfg, ids, labels, _masks(G, cfg, n))


def test_replays_draw_anew(G):
    cfg = _config(G, 0.1)
    ids, labels = _batch(cfg, 21)
    params = _params(G, cfg, seed=4)
    eager, graphed = (G.GPT2TrainStep(cfg, params=params, lr=2e-3, stream=torch.cuda.Stream(), keep_logits=False,
                                      dropout_seed=SEED) for _ in range(2))
    for st in (eager, graphed):
        st.set_batch(ids, labels)
        st.step()
    graphed.capture()
    losses = []
    for i in range(3):
        eager.step()
        graphed.replay()
        torch.cuda.synchronize()
        junk = torch.randn(1000, device="cuda").sum()  # unrelated eager work between replays
        assert float(junk) == float(junk)
        # the same kernels in the same order: the same bits
        assert int(graphed.drop_step) == int(eager.drop_step) == i + 2
        assert torch.equal(graphed.loss_sum, eager.loss_sum) and torch.equal(graphed.master, eager.master)
        losses.append(graphed.loss_value())
    assert len(set(losses)) == 3


def test_refuses_a_dropout_of_one(G):
    with pytest.raises(ValueError, match="dropout"):
        G.GPT2TrainStep(_config(G, 1.0))
    with pytest.raises(ValueError, match="dropout_seed"):
        G.GPT2TrainStep(_config(G, 0.1), dropout_seed=-1)
