"""The sums of the products over many rows where their value is known exactly, and how far long f32 sums are off.

One non-zero activation, a power of two, makes every product but one a zero: no step of an accumulation rounds or
truncates anything, and the result is the bf16 weight times that power, bit for bit.
"""
import pytest
import torch

from test_gpu_row_block import Q6_K, TYPES, Weight, check, epilogue_reference, healthy, inputs, rows

pytestmark = pytest.mark.gpu


def one_hot(cuda, m, k, seed):
    """bf16 [m, k] with 2^-2 .. 2^3 at one place of every row, and that place and factor."""
    gen = torch.Generator().manual_seed(seed)
    at = torch.randint(0, k, (m,), generator=gen).to(cuda)
    factor = torch.exp2(torch.randint(-2, 4, (m,), generator=gen).double()).to(cuda)
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=cuda)
    x[torch.arange(m, device=cuda), at] = factor.bfloat16()
    return x, at, factor


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("n,k", [(130, 512), (72, 2560), (264, 12288)])
def test_one_hot_rows_give_the_weight(cuda, oracle, engine, qtype, n, k):
    w = Weight(cuda, oracle, qtype, n, k, seed=n)
    for m in (1, 9, 20, 31, 40, 60, 130, 300, 1100):
        x, at, factor = one_hot(cuda, m, k, seed=m)
        want = w.rounded[:, at].T * factor[:, None]
        y = w.dev.gemm_epilogue(x)
        assert torch.equal(y.double(), want), f"{m} rows: off by up to {((y.double() - want).abs() / want.abs()).nan_to_num().max():.2e}"
        assert torch.equal(w.dev.gemm_epilogue(x, out_dtype=torch.bfloat16).double(), want)
    healthy(engine)


def test_long_f32_sums(cuda, oracle, engine):
    """The accumulator loses at most 1.58e-8 of a sum's norm a step of sixteen products to truncation, and a part of K has at
    most 6144 of them: 6.1e-6; f32 sums in order of 12288 products are 1.4e-6 off.  1, 20 and 60 rows, 2048 as a prompt
    chunk on tiles that fill the GPU, 300 in two tiles."""
    n, k = 4096, 12288
    w, x = inputs(cuda, oracle, Q6_K, 2048, n, k, seed=3)
    want = x.double() @ w.rounded.T
    for m in (1, 20, 60, 100, 300, 2048):
        y = w.dev.gemm_epilogue(x[:m]).double()
        assert float((y - want[:m]).norm() / want[:m].norm()) < 6.1e-6 + 1.4e-6, m
    healthy(engine)


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("k", [8192, 12288, 13312])
def test_long_f32_sums_in_every_form(cuda, oracle, engine, qtype, k):
    """Bias, residuals of both types, beside y and in place, rows apart, with and without an activation: a bias or residual
    counts once, however the sum is put together."""
    m, n = 1040, 2180
    w, x = inputs(cuda, oracle, qtype, m, n, k, seed=5)
    bias = rows(cuda, 1, n, 7).view(-1)
    for act in ("none", "relu"):
        for dtype in (None, torch.float32, torch.bfloat16):
            residual = None if dtype is None else rows(cuda, m, n + 4, 8, dtype)[:, :n]
            ref, tol = epilogue_reference(x, w, bias, act, residual, torch.float32)
            check(w.dev.gemm_epilogue(x, bias=bias, activation=act, residual=residual), ref, tol)
            buf = torch.full((m, n + 9), 7.0, device=cuda)
            out = buf[:, 4:n + 4]
            if dtype is torch.float32:
                residual, _ = out, out.copy_(residual)
            w.dev.gemm_epilogue(x, bias=bias, activation=act, residual=residual, out=out)
            check(out, ref, tol)
            assert (buf[:, :4] == 7).all() and (buf[:, n + 4:] == 7).all()
    healthy(engine)


@pytest.mark.parametrize("qtype", TYPES)
def test_f32_sums_of_few_rows(cuda, oracle, engine, qtype):
    """Up to 32 rows a superblock's sixteen steps lose at most 16 x 1.58e-8 of its share, and forty-eight superblocks and eight parts
    are added in f32: the errors of 2^-25 a sum on average add up like a walk, sqrt(56) x 2^-25 x 2 / 3 of the norm."""
    n, k = 520, 12288
    w, x = inputs(cuda, oracle, qtype, 32, n, k, seed=4)
    want = x.double() @ w.rounded.T
    for m in (1, 9, 17, 32):
        y = w.dev.gemm_epilogue(x[:m]).double()
        assert float((y - want[:m]).norm() / want[:m].norm()) < 16 * 1.58e-8 + 56 ** 0.5 * 2.0 ** -25 * 2 / 3, m
    healthy(engine)
