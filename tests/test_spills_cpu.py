"""No kernel of the library spills registers, as the pipeline's verify stage asks of a candidate."""
from cuda_tempiler_b200 import build
from cuda_tempiler_b200.tempo.plugins.sm100.toolchain import parse_ptxas


def test_no_kernel_spills():
    log = build.PKG / "libtempo_sm100.ptxas.log"
    build.build(force=not log.exists())
    facts = parse_ptxas(log.read_text())
    assert any("k_moe_down" in k for k in facts) and any("k_epi_swap" in k for k in facts)
    bad = {k: v for k, v in facts.items() if v["spill_st"] or v["spill_ld"]}
    assert not bad, bad
