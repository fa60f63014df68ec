"""What the operators over many rows refuse, before anything is launched: no GPU is needed."""
import pytest
import torch

GEMM = dict(w=16, w_up=0, x=16, bias=0, bias_up=0, residual=0, y=16, x_stride=512, residual_stride=0, y_stride=64,
            type=12, activation=0, residual_type=0, y_type=0, m_rows=3, n_out=64, k_in=512, resident=0)
GLU = dict(GEMM, w_up=32, y_type=1)
NORM = dict(residual=16, block=16, gate=0, h=16, y=16, residual_stride=64, block_stride=64, gate_stride=0, h_stride=64,
            y_stride=64, post_weight=0, post_bias=0, post_eps=0.0, post_kind=0, pre_weight=16, pre_bias=0, pre_eps=1e-6,
            pre_kind=0, residual_type=0, block_type=1, gate_type=0, h_type=0, y_type=1, scale=1.0, m_rows=2, n=64)
ARG, ALIGN, TYPE, LIMIT = 1002, 1003, 1001, 1006


def gemm(engine, base, **changes):
    from cogni_ml_b200.quant_matmul import _GEMM_ARGS
    fn = engine.lib.cogni_qmm_gemm_glu if base is GLU else engine.lib.cogni_qmm_gemm_epilogue
    return fn(_GEMM_ARGS.pack(*{**base, **changes}.values()), None)


def norm(engine, **changes):
    from cogni_ml_b200.norm import _NORM_ARGS
    return engine.lib.cogni_qmm_norm_residual(_NORM_ARGS.pack(*{**NORM, **changes}.values()), None)


@pytest.mark.parametrize("base", [GEMM, GLU], ids=["epilogue", "glu"])
@pytest.mark.parametrize("changes,status", [
    ({"w": 0}, ARG), ({"x": 0}, ARG), ({"y": 0}, ARG), ({"m_rows": 0}, ARG), ({"m_rows": -1}, ARG), ({"n_out": 0}, ARG),
    ({"k_in": 0}, ARG), ({"k_in": 500}, ARG), ({"k_in": 128}, ARG), ({"type": 2}, TYPE), ({"type": -1}, TYPE),
    ({"activation": 6}, ARG), ({"activation": -1}, ARG), ({"x_stride": 511}, ARG), ({"x_stride": 504}, ARG),
    ({"x_stride": 516}, ARG), ({"x_stride": 0}, ARG), ({"y_stride": 63}, ARG), ({"y_type": 2}, ARG),
    ({"m_rows": 4194305}, LIMIT), ({"w": 24}, ALIGN), ({"x": 24}, ALIGN), ({"y": 17}, ALIGN), ({"bias": 18}, ALIGN),
])
def test_products_refuse(engine, base, changes, status):
    assert gemm(engine, base, **changes) == status


def test_products_refuse_what_belongs_to_the_other(engine):
    assert gemm(engine, GEMM, w_up=32) == ARG
    assert gemm(engine, GEMM, bias_up=16) == ARG
    assert gemm(engine, GEMM, residual=16, residual_stride=63) == ARG
    assert gemm(engine, GEMM, residual=16, residual_stride=64, residual_type=3) == ARG
    assert gemm(engine, GEMM, residual=18, residual_stride=64) == ALIGN
    assert gemm(engine, GLU, w_up=0) == ARG
    assert gemm(engine, GLU, w_up=40) == ALIGN
    assert gemm(engine, GLU, residual=16, residual_stride=64) == ARG
    assert gemm(engine, GLU, y_type=0) == ARG
    assert engine.lib.cogni_qmm_gemm_epilogue(None, None) == ARG
    assert engine.lib.cogni_qmm_gemm_glu(None, None) == ARG


@pytest.mark.parametrize("changes,status", [
    ({"residual": 0}, ARG), ({"m_rows": 0}, ARG), ({"n": 0}, ARG), ({"n": 32769}, LIMIT), ({"y": 0}, ARG),
    ({"pre_weight": 0}, ARG), ({"pre_weight": 0, "y": 0, "h": 0}, ARG), ({"block": 0, "post_weight": 16}, ARG),
    ({"block": 0, "gate": 16}, ARG), ({"pre_eps": -1.0}, ARG), ({"pre_eps": float("nan")}, ARG), ({"pre_kind": 2}, ARG),
    ({"post_weight": 16, "post_kind": -1}, ARG), ({"residual_stride": 63}, ARG), ({"block_stride": 0}, ARG),
    ({"h_stride": 1}, ARG), ({"y_stride": -64}, ARG), ({"gate": 16, "gate_stride": 8}, ARG), ({"residual_type": 2}, ARG),
    ({"block_type": -1}, ARG), ({"y_type": 7}, ARG), ({"h": 18}, ALIGN), ({"y": 17}, ALIGN), ({"pre_weight": 18}, ALIGN),
    ({"pre_bias": 18}, ALIGN),
])
def test_norm_refuses(engine, changes, status):
    assert norm(engine, **changes) == status


def test_norm_refuses_nothing(engine):
    assert engine.lib.cogni_qmm_norm_residual(None, None) == ARG


def test_structs_have_the_layout_of_the_header(engine, tmp_path):
    import subprocess
    from pathlib import Path

    from cogni_ml_b200.norm import _NORM_ARGS
    from cogni_ml_b200.quant_matmul import _GEMM_ARGS
    root = Path(__file__).resolve().parent.parent
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "cogni_qmm.h"\nint main(void) { printf("%zu %zu %zu %zu %zu",'
                   " sizeof(cogni_qmm_gemm_args), offsetof(cogni_qmm_gemm_args, type), sizeof(cogni_qmm_norm_args),"
                   " offsetof(cogni_qmm_norm_args, post), offsetof(cogni_qmm_norm_args, scale)); return 0; }\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", str(root / "include"), "-o", str(exe), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [_GEMM_ARGS.size, 80, _NORM_ARGS.size, 80, 148]
    fields = list(GEMM), list(NORM)
    header = (root / "include" / "cogni_qmm.h").read_text()
    crystal = (root / "crystal" / "src" / "ml" / "cuda" / "cogni_qmm.cr").read_text()
    body = header[header.index("typedef struct cogni_qmm_gemm_args"):header.index("} cogni_qmm_gemm_args;")]
    in_c = [n.strip(" *;") for line in body.splitlines()[1:] for n in line.split(None, 1)[-1].replace("void *", "").replace("float *", "").split(",")]
    assert in_c == fields[0]
    cr = crystal[crystal.index("struct GemmArgs"):]
    assert [line.split(" : ")[0].strip() for line in cr[:cr.index("end")].splitlines()[1:] if " : " in line] == fields[0]


X, Y, OTHER = 1 << 20, 1 << 24, 1 << 28  # addresses far apart; nothing there is touched
APART = dict(x=X, y=Y)


@pytest.mark.parametrize("base", [GEMM, GLU], ids=["epilogue", "glu"])
@pytest.mark.parametrize("changes", [
    {"y": X}, {"y": X + 2 * 3 * 512 - 4}, {"y": X - 4}, {"y": X, "y_stride": 0}, {"bias": Y}, {"bias": Y + 4 * 63},
    {"m_rows": 1, "y": X + 1020}, {"x_stride": 1024, "y": X + 1020, "y_stride": 0},
])
def test_products_refuse_results_over_their_inputs(engine, base, changes):
    size = 2 if base is GLU else 4
    changes = dict(changes)
    if "y_stride" in changes:  # filled in: the same bytes between rows as x has
        changes["y_stride"] = changes.get("x_stride", 512) * 2 // size
    assert gemm(engine, base, **{**APART, **changes}) == ARG


@pytest.mark.parametrize("changes", [
    {"residual": Y + 4, "residual_stride": 64}, {"residual": Y, "residual_stride": 128}, {"residual": Y, "residual_stride": 64, "residual_type": 1},
    {"residual": Y - 256 * 2, "residual_stride": 64}, {"y_stride": 100, "residual": Y + 252, "residual_stride": 100},
    {"y_stride": 100, "residual": Y + 200, "residual_stride": 100},
])
def test_epilogue_refuses_residuals_half_over_the_result(engine, changes):
    assert gemm(engine, GEMM, **{**APART, **changes}) == ARG


NORM_APART = dict(residual=X, block=2 * X, gate=3 * X, gate_stride=64, h=4 * X, y=5 * X, pre_weight=6 * X)


@pytest.mark.parametrize("changes", [
    {"y": 4 * X}, {"y": 4 * X + 2}, {"h": X + 4}, {"h": X, "h_type": 1}, {"h": X, "h_stride": 65}, {"h": 2 * X},
    {"y": X}, {"y": 2 * X + 2}, {"y": 3 * X}, {"h": 3 * X}, {"h": 3 * X, "gate_stride": 0}, {"y": 6 * X}, {"h": 6 * X + 252},
    {"pre_bias": 4 * X}, {"post_weight": 5 * X}, {"post_weight": 7 * X, "post_bias": 4 * X + 256},
])
def test_norm_refuses_results_over_their_inputs(engine, changes):
    assert norm(engine, **{**NORM_APART, **changes}) == ARG


# ------------------------------------------------------------------------------- the Python layer
def weight(engine, device="cpu", n=8, k=256, t=12):
    return engine.DeviceQuantWeight(torch.zeros(n * k // 256 * 144, dtype=torch.uint8, device=device), t, n, k)


def test_python_refuses_host_tensors_and_wrong_types(engine):
    w = weight(engine)
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device of the weights"):
        w.gemm_epilogue(x)
    with pytest.raises(ValueError, match="bf16"):
        w.gemm_epilogue(x.float())
    with pytest.raises(ValueError, match="bf16"):
        engine.gemm_glu(w, w, x, out=torch.zeros(2, 8))
    with pytest.raises(ValueError, match="CUDA device"):
        engine.norm_residual(torch.zeros(2, 8), norm=engine.Norm(torch.ones(8)))
