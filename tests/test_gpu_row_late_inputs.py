"""A kernel of the stream that lets the next one start and then takes longer than the limit of the bounded waits (one second):
the products with an epilogue wait for it outside of them, give the same results, and no wait expires."""
import pytest
import torch

from cogni_ml_b200 import gemm_glu
from test_gpu_row_block import IQ4_NL, Q4_K, Q5_K, Q6_K, Q8_0, Weight, healthy, rows

pytestmark = pytest.mark.gpu
HOLD_US = 1_300_000


# few rows, 128-token tiles two CTAs an SM and alone, in parts, CTA pairs, direct loads (Q6_K rows that are no multiple of 16 bytes)
@pytest.mark.parametrize("qtype,m,n,k", [(Q4_K, 3, 640, 1024), (Q4_K, 64, 640, 4096), (Q4_K, 128, 20000, 512), (Q5_K, 1100, 640, 768),
                                         (Q6_K, 100, 640, 2048), (Q6_K, 300, 640, 1280), (Q8_0, 100, 640, 1024),
                                         (IQ4_NL, 600, 20000, 512)])
@pytest.mark.parametrize("resident", [True, False])
def test_a_slow_kernel_before_the_product(cuda, oracle, engine, qtype, m, n, k, resident):
    gate, up = Weight(cuda, oracle, qtype, n, k, 1).dev, Weight(cuda, oracle, qtype, n, k, 2).dev
    gate.resident = up.resident = resident
    x = rows(cuda, m, k, 3, torch.bfloat16)
    calls = (lambda: gate.gemm_epilogue(x), lambda: gemm_glu(gate, up, x))
    want = [call() for call in calls]
    torch.cuda.synchronize()
    for call, w in zip(calls, want):
        assert engine.lib.cogni_qmm_diag_hold(HOLD_US, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(call(), w)
        healthy(engine)
