"""CPU: the device code of nz_fp8.hip: no packed float32 forms, no scratch memory, and registers and LDS that leave room
for the workgroups that the host counts on; the rules of its inline assembly."""
import os
import re
import subprocess

import pytest

from neuzip_amd import _build

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.fixture(scope="module")
def unit(tmp_path_factory):
    """(assembly, kernel -> fields of its metadata)"""
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not installed")
    source = os.path.join(_build.CSRC, "nz_fp8.hip")
    assert source in [u[0] for u in _build.operator_units("")]
    out = tmp_path_factory.mktemp("code") / "unit.s"
    flags = [f for f in _build.HIPCC_FLAGS if f != "-fPIC"]
    res = subprocess.run([HIPCC, *flags, "--cuda-device-only", "-S", source, "-o", str(out)], cwd=_build.CSRC,
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    text, kernels = out.read_text(), {}
    for part in text.split("- .agpr_count:")[1:]:
        fields = dict(re.findall(r"^\s+(\.\w+):\s+(\S+)", part, re.M))
        kernels[fields[".symbol"].replace(".kd", "")] = fields
    return text, kernels


def test_no_packed_float32_and_no_scratch(unit):
    text, kernels = unit
    assert len(kernels) >= 60
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
    for name, f in kernels.items():
        assert int(f[".vgpr_spill_count"]) == 0 and int(f[".private_segment_fixed_size"]) == 0, name
        assert int(f[".group_segment_fixed_size"]) <= 160 * 1024, name


def test_inline_assembly_writes_no_register_that_the_compiler_does_not_know_of():
    """m0, which cannot be named among the clobbered registers, is an operand"""
    found = 0
    for name in ("nz_fp8.hip", "nz_products.h"):
        with open(os.path.join(_build.CSRC, name)) as f:
            text = f.read()
        for block in re.findall(r"\basm(?: volatile)?\s*\(((?:[^;])*)\);", text):
            found += 1
            instructions = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', block.split("::")[0]))
            assert not re.search(r"\b(m0|vcc|exec|[sv]\d+|[sv]\[\d)", instructions), block
    assert found >= 5
