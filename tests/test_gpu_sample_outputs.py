"""sample_rows into the caller's tensors: on the current stream, on a stream named by
its bare handle (whose memory the wrapper cannot take outputs from), from a graph;
and which tensors it refuses."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cuda):
    from mi355x_pjrt import kernels

    kernels.lib()
    return kernels


class _Handle:
    """A stream that is no torch stream: its handle alone."""

    def __init__(self, stream):
        self.cuda_stream = stream.cuda_stream


def _inputs(rows, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((rows, vocab), generator=g).mul(3).cuda(), torch.rand((rows,), generator=g).cuda()


@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
def test_sample_rows_into_given_outputs(K, index_dtype):
    x, u = _inputs(9, 5003, 1)
    want = K.sample_rows(x, u, 0.8, 50, 0.9, index_dtype=index_dtype)
    token = torch.full((13,), -7, dtype=index_dtype, device="cuda")
    logprob = torch.full((13,), 7.0, device="cuda")
    # the tensor's own type counts, whatever index_dtype says
    got = K.sample_rows(x, u, 0.8, 50, 0.9, token=token[2:11], logprob=logprob[1:10])
    assert got[0].data_ptr() == token[2:11].data_ptr() and got[1].data_ptr() == logprob[1:10].data_ptr()
    assert torch.equal(token[2:11], want[0]) and torch.equal(logprob[1:10], want[1])
    assert bool((token[[0, 1, 11, 12]] == -7).all()) and bool((logprob[[0, 10, 11, 12]] == 7).all())
    got = K.sample_rows(x, u, 0.8, 50, 0.9, token=token[:9], with_logprob=False)
    assert got[1] is None and torch.equal(got[0], want[0])


def test_sample_rows_on_a_bare_handle(K):
    x, u = _inputs(33, 20011, 2)
    want = K.sample_rows(x, u, 0.7, 0, 0.9)
    side = torch.cuda.Stream()
    token, logprob = torch.zeros(33, dtype=torch.int32, device="cuda"), torch.zeros(33, device="cuda")
    torch.cuda.synchronize()
    got = K.sample_rows(x, u, 0.7, 0, 0.9, stream=_Handle(side), token=token, logprob=logprob)
    side.synchronize()
    assert got[0] is token and got[1] is logprob
    assert torch.equal(token, want[0]) and torch.equal(logprob, want[1])


def test_sample_rows_from_a_graph_into_given_outputs(K):
    x, u = _inputs(5, 3001, 3)
    token, logprob = torch.zeros(5, dtype=torch.int64, device="cuda"), torch.zeros(5, device="cuda")
    K.sample_rows(x, u, top_p=0.9, token=token, logprob=logprob)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.sample_rows(x, u, top_p=0.9, token=token, logprob=logprob)
    for seed in (4, 5, 6):
        y, v = _inputs(5, 3001, seed)
        x.copy_(y)
        u.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = K.sample_rows(y, v, top_p=0.9, index_dtype=torch.int64)
        assert torch.equal(token, want[0]) and torch.equal(logprob, want[1])


def test_refused_outputs(K):
    x, u = _inputs(4, 100, 7)
    wide = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    for kw in ({"token": wide[:, 0]}, {"token": wide[:3, 0].contiguous()}, {"token": wide[:, 0].contiguous().short()},
               {"token": torch.zeros(4, dtype=torch.int32)}, {"token": u}, {"logprob": u.half()}, {"logprob": u[:3]},
               {"logprob": u[:1].expand(4)}, {"logprob": u.cpu()}, {"logprob": u.clone(), "with_logprob": False}):
        with pytest.raises(ValueError, match="sample_rows"):
            K.sample_rows(x, u, **kw)
