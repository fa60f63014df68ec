"""The plans of 128-token tiles two CTAs an SM, each split along K, and the activations over the whole range of f32 results."""
import pytest
import torch

from cogni_ml_b200 import gemm_glu
from test_gpu_row_block import (Q4_K, Q5_K, Q8_0, Weight, check, epilogue_reference, glu_reference, healthy, inputs, rows)

pytestmark = pytest.mark.gpu


# cogni_qmm_set_kernel_choice 72: two CTAs an SM; 53 whole K, 54, 70, 59, 69: two, three, four, eight parts
@pytest.mark.parametrize("split", [53, 54, 70, 59, 69])
@pytest.mark.parametrize("qtype", [Q4_K, Q5_K, Q8_0])
@pytest.mark.parametrize("m,n,k", [(70, 200, 4352), (128, 4104, 4352), (300, 1000, 2048)])
def test_two_ctas_an_sm_with_every_split(cuda, oracle, engine, split, qtype, m, n, k):
    w, x = inputs(cuda, oracle, qtype, m, n, k, seed=17)
    wu = Weight(cuda, oracle, qtype, n, k, seed=18)
    bias, residual = rows(cuda, 1, n, 5).view(-1), rows(cuda, m, n, 6)
    calls = (lambda: w.dev.gemm_epilogue(x, bias=bias, activation="relu", residual=residual),
             lambda: gemm_glu(w.dev, wu.dev, x, bias_gate=bias))
    try:
        for c in (72, split):
            assert engine.lib.cogni_qmm_set_kernel_choice(c) == 0
        first = [call() for call in calls]
        same = [all(torch.equal(call(), want) for _ in range(40)) for call, want in zip(calls, first)]
    finally:
        for c in (71, 52):
            engine.lib.cogni_qmm_set_kernel_choice(c)
    check(first[0], *epilogue_reference(x, w, bias, "relu", residual, torch.float32))
    check(first[1], *glu_reference(x, w.rounded, wu.rounded, bias, None, "silu"))
    assert all(same)
    healthy(engine)


def tail_reference(v, act):
    """act(v) in f64 and the bound of its f32 form, in units u = 2^-23 of a relative error.  exp(a) by __expf: 2 + 1.173 |a| u; the
    sum with 1 half a u, the quotient 2 u, and where 1 + exp(a) is above 2^126 the quotient is zero.  gelu_tanh's exponent a
    comes from seven roundings, which the exponential turns into 3.5 |a| u.  erff is off by 2 u / 2, its argument by one and
    a half roundings (slope times argument below 0.5), 1 + erf by half a u: 2 u in all, times |v| / 2, and two products."""
    u = 2.0 ** -23
    if act in ("none", "relu"):
        return (v.clamp(min=0) if act == "relu" else v), torch.zeros_like(v)
    if act == "gelu":
        y = 0.5 * v * torch.special.erfc(-v * 0.5 ** 0.5)
        return y, v.abs() * u + u * y.abs()
    a = -v if act != "gelu_tanh" else -2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3)
    y = torch.exp(-torch.logaddexp(torch.zeros_like(a), a))  # 1 / (1 + exp(a))
    slope = 1.173 + (3.5 if act == "gelu_tanh" else 0.0)
    if act != "sigmoid":
        y = v * y
    return y, (5 + slope * a.abs()) * u * y.abs() + 2.0 ** -126 * (1 + v.abs())


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid"])
@pytest.mark.parametrize("m", [1, 40, 300])
def test_activations_over_their_range(cuda, oracle, engine, act, m):
    n, k = 4096, 256
    w = Weight(cuda, oracle, Q8_0, n, k, 1)
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=cuda)
    v = torch.cat([torch.linspace(-120, 40, n - 1024), torch.linspace(-6, 6, 1024)]).to(cuda)
    y = w.dev.gemm_epilogue(x, bias=v, activation=act)
    ref, tol = tail_reference(v.double(), act)
    check(y, ref.expand(m, n), (tol + 2.0 ** -24 * ref.abs()).expand(m, n))
