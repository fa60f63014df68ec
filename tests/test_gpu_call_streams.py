"""stream=: the calls on quantised weights on a stream beside the current one, while either has work queued (the operators over
many rows: test_gpu_row_streams.py)."""
import pytest
import torch

from cogni_ml_b200 import DeviceQuantWeight, QuantWeight, gemv_many, synth

pytestmark = pytest.mark.gpu
CYCLES = 100_000_000  # of torch.cuda._sleep: about 50 ms
N, K, B = 512, 512, 4


@pytest.fixture(scope="module")
def ops(cuda):
    """name -> (call of (input, stream) -> list of results, input)."""
    def weight(t, seed):
        return DeviceQuantWeight.upload(QuantWeight(synth.make_weight(t, N, K, seed=seed, tensor_id=t), t, N, K), cuda)

    w, u = weight(synth.Q4_K, 1), weight(synth.Q4_K, 2)
    x = torch.from_numpy(synth.make_activation(B, K, seed=3)).to(cuda).view(B, K)
    ids = torch.arange(100, 100 + B, dtype=torch.int32, device=cuda)
    norm = torch.ones(K, device=cuda)
    return {"gemv": (lambda x, s: [w.gemv(x, stream=s)], x),
            "gemv_residual": (lambda x, s: [w.gemv(x, residual=x, stream=s)], x),
            "gemv_swiglu": (lambda x, s: [w.gemv_swiglu(x, x, stream=s)], x),
            "gemv_many": (lambda x, s: gemv_many([w, u], x, stream=s), x),
            "gemv_many_norm": (lambda x, s: gemv_many([w, u], x, stream=s, norm_weight=norm), x),
            "top1": (lambda x, s: list(w.gemv_top1(x, stream=s, want_keys=True)), x),
            "top2": (lambda x, s: list(w.gemv_top2(x, stream=s, want_keys=True)), x),
            "embedding": (lambda x, s: [w.embedding_lookup(x, check_range=False, stream=s)], ids),
            "embedding_checked": (lambda x, s: [w.embedding_lookup(x, stream=s)], ids),
            "gemm": (lambda x, s: [w.gemm(x, stream=s)], x.bfloat16()),
            "dequantize": (lambda x, s: [w.dequantize(stream=s)], x)}


OPS = ["gemv", "gemv_residual", "gemv_swiglu", "gemv_many", "gemv_many_norm", "top1", "top2", "embedding", "embedding_checked", "gemm",
       "dequantize"]


@pytest.mark.parametrize("op", OPS)
def test_results_do_not_share_memory_with_queued_work(ops, op):
    call, x = ops[op]
    want = call(x, None)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(CYCLES)
    late = [torch.empty_like(t) for t in want]
    for t in late:
        t.fill_(7)
    del late, t
    got = call(x, side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("op", [o for o in OPS if o != "dequantize"])
def test_a_temporary_input_lives_until_it_is_read(ops, op):
    call, x = ops[op]
    want = call(x, None)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    temporary = x.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(CYCLES)
    got = call(temporary, side)
    del temporary
    over = [torch.full_like(x, 0 if x.dtype == torch.int32 else float("nan")) for _ in range(8)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del over


def test_an_id_outside_the_table_is_seen_on_another_stream(ops, cuda):
    call, _ = ops["embedding_checked"]
    side = torch.cuda.Stream()
    bad = torch.tensor([3, N], dtype=torch.int32, device=cuda)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(CYCLES)
    with pytest.raises(IndexError, match=str(N)):
        call(bad, side)
