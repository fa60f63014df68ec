"""What cogni_qmm_diag_hold refuses, before anything is launched: no GPU is needed."""


def test_hold_refuses(engine):
    assert engine.lib.cogni_qmm_diag_hold(0, None) == 1002
    assert engine.lib.cogni_qmm_diag_hold(2_000_001, None) == 1002
