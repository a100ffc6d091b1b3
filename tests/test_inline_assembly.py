"""Inline assembly of the kernels, as it stands in the sources."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stepquant_amd", "csrc")


@pytest.mark.parametrize("name", sorted(os.listdir(CSRC)))
def test_m0_is_an_operand_of_the_assembly_that_needs_it(name):
    """The compiler, which writes M0 for instructions of its own, is not to find it changed."""
    text = open(os.path.join(CSRC, name)).read()
    for statement in re.findall(r"\basm\b[^;]*\(.*?\);", text, re.S):
        assert not re.search(r"\bm0\s*,", statement), statement
        if re.search(r"\bglobal_load_lds_|\bbuffer_load_\w+ .*\blds\b", statement):
            assert '"{m0}"(' in statement, statement
