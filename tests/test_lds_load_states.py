"""The wait states in the asm of loads into LDS cover a base out of v_readfirstlane wherever the
compiler puts that instruction: five states, s_nop 4, which cover m0's one too."""
import re

import pytest

from test_lds_loads import CSRC, FILES, LOAD


@pytest.mark.parametrize("name", FILES)
def test_five_states_before_a_load(name):
    for text in LOAD.findall((CSRC / name).read_text()):
        assert int(re.match(r"s_nop ([0-9]+)\\n", text).group(1)) >= 4, text
