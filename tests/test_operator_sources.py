"""CPU: rules that the operators' sources keep."""
import os
import re

from neuzip_amd import _build


def test_inline_assembly_writes_no_register_that_the_compiler_does_not_know_of():
    """m0, which cannot be named among the clobbered registers, is an operand"""
    for source, _, _ in _build.operator_units(""):
        with open(source) as f:
            text = f.read()
        blocks = re.findall(r"\basm(?: volatile)?\s*\(((?:[^;])*)\);", text)
        assert blocks or os.path.basename(source) != "nz_mx.hip"
        for block in blocks:
            instructions = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', block.split("::")[0]))
            assert not re.search(r"\b(m0|vcc|exec|[sv]\d+|[sv]\[\d)", instructions), block
