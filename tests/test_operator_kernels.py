"""CPU: the device code of the operators' translation units: no packed float32 forms, no scratch memory, and registers
and LDS that leave room for the workgroups that the host counts on."""
import os
import re
import subprocess

import pytest

from neuzip_amd import _build

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
KERNELS = {"nz_mx": 30, "nz_embedding": 12}  # at least


@pytest.fixture(scope="module", params=sorted(KERNELS))
def unit(request, tmp_path_factory):
    """(stem, assembly, kernel -> fields of its metadata)"""
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not installed")
    source = os.path.join(_build.CSRC, request.param + ".hip")
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
    return request.param, text, kernels


def test_no_packed_float32_and_no_scratch(unit):
    stem, text, kernels = unit
    assert len(kernels) >= KERNELS[stem]
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
    for name, f in kernels.items():
        assert int(f[".vgpr_spill_count"]) == 0 and int(f[".private_segment_fixed_size"]) == 0, name


def test_room_for_two_workgroups_of_the_larger_tiles(unit):
    """The 128x256 and 128x128 tiles are counted as two workgroups of four wavefronts to a compute unit: a wavefront to
    each of its SIMD units from either, of whose 512 registers it may have half, and half of 160 KB."""
    stem, _, kernels = unit
    if stem != "nz_mx":
        return
    found = 0
    for name, f in kernels.items():
        if re.search(r"nz_mx_tiles_kernelILi2ELi2ELi4ELi[48]E", name):
            found += 1
            assert int(f[".group_segment_fixed_size"]) <= 80 * 1024, name
            assert int(f[".vgpr_count"]) <= 256, name  # of both kinds together
    assert found == 4
