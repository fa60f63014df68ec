"""The Crystal binding of the products and norms over many rows, as text (no Crystal compiler exists here)."""
import re
from pathlib import Path

from test_row_block_refusals import GEMM, NORM

ROOT = Path(__file__).resolve().parent.parent
CR = (ROOT / "crystal" / "src" / "ml" / "cuda" / "cogni_qmm.cr").read_text()
HEADER = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "cogni_qmm.h").read_text(), flags=re.S)
CRYSTAL_TYPE = {"int32_t": "Int32", "int64_t": "Int64", "float": "Float32"}


def c_fields(name):
    """(field, type as Crystal has it) of a struct of the header, in order."""
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER, re.S).group(1)
    out = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        base, names = re.match(r"(?:const )?(\w+) (.*)", decl, re.S).groups()
        for n in names.split(","):
            kind = "DevPtr" if "*" in n else "Norm" if base == "cogni_qmm_norm" else CRYSTAL_TYPE[base]
            out.append((n.strip(" *\n"), kind))
    return out


def crystal_fields(name):
    body = re.search(r"^  struct %s\n(.*?)^  end" % name, CR, re.S | re.M).group(1)
    return re.findall(r"^    (\w+) : (\w+)$", body, re.M)


def test_structs_have_the_header_fields():
    for c, cr in (("cogni_qmm_gemm_args", "GemmArgs"), ("cogni_qmm_norm", "Norm"), ("cogni_qmm_norm_args", "NormArgs")):
        assert c_fields(c) == crystal_fields(cr), cr
    assert [n for n, _ in crystal_fields("GemmArgs")] == list(GEMM)
    flat = [f"{n}_{f}" if kind == "Norm" else n for n, kind in crystal_fields("NormArgs")
            for f in (("weight", "bias", "eps", "kind") if kind == "Norm" else ("",))]
    assert flat == list(NORM)


def method(name):
    return re.search(r"^    (?:private )?def %s\(.*?^    end" % name, CR, re.S | re.M).group(0)


def test_glu_refuses_another_up_matrix():
    """The C entry point takes the gate's type and shape for both matrices, so a smaller or differently typed up
    matrix would be read past its end: the binding has to compare all three before the call."""
    body = method("gemm_glu")
    check, call = body.index("raise ArgumentError"), body.index("LibCogniQMM.cogni_qmm_gemm_glu")
    assert check < call
    for field in ("type", "out_dim", "in_dim"):
        assert re.search(r"up\.%s == @%s" % (field, field), body[:call]), field
