"""gemm_glu takes a weight as bf16(dequant(W)), whatever the type and however many rows stand beside a token."""
import pytest
import torch

from cogni_ml_b200 import gemm_glu
from test_gpu_row_block import Q4_K, Q5_K, TYPES, Weight, check, glu_reference, healthy, rows
from test_gpu_row_sums import one_hot

pytestmark = pytest.mark.gpu
ROWS = (1, 3, 8, 9, 16, 17, 24, 25, 32, 33, 64, 65, 140)  # around the widths of the kernels' tiles


class Pair:
    def __init__(self, cuda, oracle, qtype, n, k):
        self.gate, self.up = Weight(cuda, oracle, qtype, n, k, 11), Weight(cuda, oracle, qtype, n, k, 12)


@pytest.fixture(scope="module", params=[(t, n, k) for t in TYPES for n, k in ((4104, 4352), (200, 768))],
                ids=lambda p: f"{p[0]}-{p[1]}x{p[2]}")
def pair(request, cuda, oracle):
    return Pair(cuda, oracle, *request.param), request.param


def test_one_hot_rows(cuda, engine, pair):
    """Both factors are then bf16 numbers (times a power of two): their product is exact in f32 and rounded once."""
    (p, (_, n, k)) = pair
    for m in ROWS:
        x, at, factor = one_hot(cuda, m, k, seed=m)
        want = (p.gate.rounded[:, at].T * p.up.rounded[:, at].T * factor[:, None] ** 2).float().bfloat16()
        y = gemm_glu(p.gate.dev, p.up.dev, x, activation="none")
        assert torch.equal(y, want), f"{m} rows: {int((y != want).sum())} of {y.numel()} differ"
    healthy(engine)


def test_a_token_among_others(cuda, engine, pair):
    (p, (_, n, k)) = pair
    x = rows(cuda, max(ROWS), k, 13, torch.bfloat16, 1.5 / (p.gate.rms * k ** 0.5))
    ref, tol = glu_reference(x, p.gate.rounded, p.up.rounded, None, None, "silu")
    for m in ROWS:
        check(gemm_glu(p.gate.dev, p.up.dev, x[:m]), ref[:m], tol[:m])


@pytest.mark.parametrize("qtype", [Q4_K, Q5_K])
@pytest.mark.parametrize("m", [1, 8, 20, 40])
def test_large_activations(cuda, oracle, engine, qtype, m):
    """x = 2^121: W x is finite for every weight below 2^6."""
    n, k = 136, 512
    gate, up = Weight(cuda, oracle, qtype, n, k, 21), Weight(cuda, oracle, qtype, n, k, 22)
    assert float(up.rounded.abs().max()) < 64 and float(gate.rounded.abs().max()) < 64
    x, at, _ = one_hot(cuda, m, k, seed=m)
    x[x != 0] = 2.0 ** 121
    g, u = gate.rounded[:, at].T * 2.0 ** 121, up.rounded[:, at].T * 2.0 ** 121
    want = (torch.sigmoid(g) * u).float().bfloat16()
    assert torch.equal(gemm_glu(gate.dev, up.dev, x, activation="sigmoid"), want)
    y, want = up.dev.gemm_epilogue(x), u
    assert torch.equal(y.double(), want)


@pytest.mark.parametrize("m", [2, 12, 20, 30, 40, 300])
def test_infinities_and_nan_stay_in_their_row(cuda, engine, pair, m):
    (p, (_, n, k)) = pair
    x = rows(cuda, m, k, 14, torch.bfloat16, 1.5 / (p.gate.rms * k ** 0.5))
    clean = p.gate.dev.gemm_epilogue(x), gemm_glu(p.gate.dev, p.up.dev, x)
    x[0, 3], x[1, 5] = float("nan"), float("inf")
    y, g = p.gate.dev.gemm_epilogue(x), gemm_glu(p.gate.dev, p.up.dev, x)
    assert y[0].isnan().all() and g[0].isnan().all() and not torch.isfinite(y[1]).any()
    assert torch.equal(y[2:], clean[0][2:]) and torch.equal(g[2:], clean[1][2:])
