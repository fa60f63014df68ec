"""stream=: the rows' operators on a stream beside the current one, while either has work queued."""
import pytest
import torch

from cogni_ml_b200 import Norm, gemm_glu, norm_residual
from test_gpu_row_block import Q4_K, Q6_K, Weight, make_norm, rows

pytestmark = pytest.mark.gpu
CYCLES = 100_000_000  # of torch.cuda._sleep: about 50 ms


def setup(cuda, oracle, m=40, n=512, k=512):
    w, u = Weight(cuda, oracle, Q4_K, n, k, 1).dev, Weight(cuda, oracle, Q4_K, n, k, 2).dev
    x = rows(cuda, m, k, 3, torch.bfloat16)
    norm = make_norm(cuda, n, "rms", 4)
    # results of one size: bf16 [m, n]
    return x, {"epilogue": lambda x, s: w.gemm_epilogue(x, out_dtype=torch.bfloat16, stream=s),
               "glu": lambda x, s: gemm_glu(w, u, x, stream=s),
               "norm": lambda x, s: norm_residual(x, norm=norm, stream=s)[1],
               "hidden": lambda x, s: norm_residual(x, x, norm=norm, stream=s)[0]}


OPS = ["epilogue", "glu", "norm", "hidden"]


@pytest.mark.parametrize("op", OPS)
def test_a_result_does_not_share_memory_with_queued_work(cuda, oracle, engine, op):
    """A temporary of the result's size is written by a kernel that is still queued when the temporary is freed: the result must
    not lie there."""
    x, ops = setup(cuda, oracle)
    want = ops[op](x, None)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        torch.cuda._sleep(CYCLES)
        late = torch.empty_like(want)
        late.fill_(7.0)
        del late
        y = ops[op](x, side)
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.parametrize("op", OPS)
def test_a_temporary_input_lives_until_it_is_read(cuda, oracle, engine, op):
    """The side stream comes to the call late; the caller has dropped x by then and filled a new tensor of its size."""
    x, ops = setup(cuda, oracle)
    want = ops[op](x, None)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        temporary = x.clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(CYCLES)
        y = ops[op](temporary, side)
        del temporary
        over = [torch.full_like(x, float("nan")) for _ in range(4)]
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        del over


def test_norm_vectors_and_biases_live_until_they_are_read(cuda, oracle, engine):
    m, n, k = 5, 512, 512
    w = Weight(cuda, oracle, Q6_K, n, k, 1).dev
    x, bias = rows(cuda, m, k, 3, torch.bfloat16), rows(cuda, 1, n, 4).view(-1)
    norm = make_norm(cuda, n, "layer", 5)
    want = w.gemm_epilogue(x, bias=bias), norm_residual(x, norm=norm)[1]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    vectors = [bias.clone(), norm.weight.clone(), norm.bias.clone()]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(CYCLES)
    y = w.gemm_epilogue(x, bias=vectors[0], stream=side)
    z = norm_residual(x, norm=Norm(vectors[1], norm.eps, "layer", vectors[2]), stream=side)[1]
    vectors.clear()
    over = [torch.full_like(bias, float("nan")) for _ in range(64)]
    torch.cuda.synchronize()
    assert torch.equal(y, want[0]) and torch.equal(z, want[1])
    del over


def test_side_streams_in_a_captured_graph(cuda, oracle, engine):
    """Two calls on two streams between a fork and a join, captured once and replayed on new inputs."""
    x, ops = setup(cuda, oracle)
    for op in OPS:
        ops[op](x, None)
    torch.cuda.synchronize()
    sides = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        current = torch.cuda.current_stream()
        for s in sides:
            s.wait_stream(current)
        got = [ops[op](x, s) for op, s in (("glu", sides[0]), ("epilogue", sides[1]), ("norm", sides[0]), ("hidden", sides[1]))]
        for s in sides:
            current.wait_stream(s)
    for seed in (5, 6):
        x.copy_(rows(cuda, x.shape[0], x.shape[1], seed, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        for op, y in zip(("glu", "epilogue", "norm", "hidden"), got):
            assert torch.equal(y, ops[op](x, None)), op
