"""The build's check of scalar spills (s2cnn_amd/csrc/build.py), on reports as the compiler writes them."""
import pytest

from s2cnn_amd.csrc import build

LINE = "attention_bwd.h:46:1: remark: %s [-Rpass-analysis=kernel-resource-usage]"


def _report(**spills):
    lines = []
    for kernel, n in spills.items():
        lines += [LINE % ("Function Name: " + kernel), "   46 | template <class T> __global__ void", LINE % "    TotalSGPRs: 106", LINE % "    VGPRs: 256",
                  LINE % "    VGPRs Spill: 300", LINE % ("    SGPRs Spill: %d" % n)]
    return "\n".join(lines)


def test_numbers_of_a_report():
    assert build.scalar_spills(_report(a=0, b=217)) == {"a": 0, "b": 217}
    assert build.scalar_spills("warning: something else: 5\n") == {}


def test_limits():
    build.check_scalar_spills("attention_f32.hip", _report(a=0, b=build.MOST_SCALAR_SPILLS))
    build.check_scalar_spills("layer_norm.hip", _report(a=build.MAX_SCALAR_SPILLS["layer_norm.hip"]))
    for src, n in (("attention_f32.hip", 217), ("so3_mm.hip", build.MOST_SCALAR_SPILLS + 1), ("layer_norm.hip", build.MAX_SCALAR_SPILLS["layer_norm.hip"] + 1)):
        with pytest.raises(RuntimeError, match="bad_kernel"):
            build.check_scalar_spills(src, _report(a=0, bad_kernel=n))


def test_a_report_without_numbers_is_refused():
    """A compiler that words it otherwise is not taken for one that spills nothing; a source without kernels has none."""
    with pytest.raises(RuntimeError, match="no scalar spills"):
        build.check_scalar_spills("attention_f32.hip", "")
    build.check_scalar_spills("attention.hip", "")


def test_limits_are_of_sources_that_exist():
    assert set(build.MAX_SCALAR_SPILLS) <= set(build.SOURCES + build.PROBE_SOURCES)
