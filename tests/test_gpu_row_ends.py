"""Rows of outputs that end inside four, in buffers whose rows are multiples of four apart (where whole groups could be read at
once): every activation, bias, both residuals, in place and beside, on every kernel of the products with an epilogue."""
import pytest
import torch

from cogni_ml_b200 import ACTIVATIONS, gemm_glu
from test_gpu_row_block import IQ4_NL, Q4_K, Q6_K, Q8_0, Weight, check, epilogue_reference, glu_reference, healthy, inputs, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qtype", [Q4_K, Q6_K, Q8_0, IQ4_NL])
@pytest.mark.parametrize("n", [1, 3, 11, 135, 258])
@pytest.mark.parametrize("m,k", [(3, 512), (40, 256), (100, 2048), (300, 512), (773, 256), (1100, 768)])
def test_rows_that_end_inside_four_outputs(cuda, oracle, engine, qtype, n, m, k):
    w, x = inputs(cuda, oracle, qtype, m, n, k, seed=n)
    wu = Weight(cuda, oracle, qtype, n, k, seed=n + 1)
    bias = rows(cuda, 1, n, 5).view(-1)
    width = (n + 3) // 4 * 4
    for act in ACTIVATIONS:
        for dtype in (torch.float32, torch.bfloat16):
            residual = rows(cuda, m, n, 6, dtype)
            ref, tol = epilogue_reference(x, w, bias, act, residual, dtype)
            buf = torch.full((m, width), 7.0, dtype=dtype, device=cuda)
            buf[:, :n] = residual
            w.dev.gemm_epilogue(x, bias=bias, activation=act, residual=buf[:, :n], out=buf[:, :n])
            check(buf[:, :n].contiguous(), ref, tol)
            assert (buf[:, n:] == 7).all()
            apart = torch.full((m, width), 7.0, dtype=dtype, device=cuda)
            w.dev.gemm_epilogue(x, bias=bias, activation=act, residual=residual, out=apart[:, :n])
            assert torch.equal(apart, buf)
        buf = torch.full((m, width), 7.0, dtype=torch.bfloat16, device=cuda)
        gemm_glu(w.dev, wu.dev, x, activation=act, bias_gate=bias, bias_up=bias, out=buf[:, :n])
        check(buf[:, :n].contiguous(), *glu_reference(x, w.rounded, wu.rounded, bias, bias, act))
        assert (buf[:, n:] == 7).all()
    healthy(engine)
