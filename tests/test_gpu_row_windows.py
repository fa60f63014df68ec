"""Tiles whose weights pass through windows that TMA fills again and again: two CTAs an SM and parts of K, called many
times.  A window filled before its last readers have their words gives rows of a tile another superblock's weights, now and
then; every call has to give the first one's bits, and those the definition's values."""
import pytest
import torch

from cogni_ml_b200 import gemm_glu
from test_gpu_row_block import (IQ4_NL, Q4_K, Q5_K, Q6_K, Q8_0, Weight, check, epilogue_reference, glu_reference, healthy,
                                rows)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qtype,k", [(Q4_K, 4352), (Q5_K, 4352), (Q8_0, 4352), (Q6_K, 4096), (IQ4_NL, 4352)])
@pytest.mark.parametrize("m", [33, 64, 128, 200])
def test_many_calls_on_tiles_side_by_side(cuda, oracle, engine, qtype, k, m):
    n = 4104
    gate, up = Weight(cuda, oracle, qtype, n, k, 11), Weight(cuda, oracle, qtype, n, k, 12)
    wide = Weight(cuda, oracle, qtype, 2 * n, k, 13)
    x = rows(cuda, m, k, 14, torch.bfloat16, 1.5 / (gate.rms * k ** 0.5))
    calls = (lambda: gemm_glu(gate.dev, up.dev, x), lambda: wide.dev.gemm_epilogue(x), lambda: wide.dev.gemm(x))
    first = [call() for call in calls]
    ref, tol = epilogue_reference(x, wide, None, "none", None, torch.float32)
    check(first[0], *glu_reference(x, gate.rounded, up.rounded, None, None, "silu"))
    check(first[1], ref, tol)
    check(first[2], ref, tol)
    for call, want in zip(calls, first):
        assert all(torch.equal(call(), want) for _ in range(100))
    healthy(engine)
