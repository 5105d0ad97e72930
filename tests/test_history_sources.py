"""What holds of the kernels' sources themselves."""

import re

from tests.conftest import ROOT

CSRC = ROOT / "mdl_amd" / "csrc"


def test_inline_assembly_leaves_m0_to_the_compiler():
    """m0 holds what the compiler may set once for several uses: assembly takes
    it as an operand and writes it nowhere by itself."""

    used = 0
    for source in sorted([*CSRC.glob("*.hip"), *CSRC.glob("*.cuh")]):
        for asm in re.findall(r"\basm\b[^;]*;", source.read_text()):
            text = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', asm.split(":", 1)[0]))
            assert not re.search(r"\bm0\b", text), (source.name, asm)
            if "load_lds" in text:
                used += 1
                assert '"{m0}"' in asm, (source.name, asm)
    assert used
