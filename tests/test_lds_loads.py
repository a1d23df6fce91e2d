"""Loads into LDS that are written as inline asm carry their wait states themselves.

The compiler does not look into an asm, so it puts no wait between a write of m0 and the load
that uses it (one state), nor between v_readfirstlane and a load whose base it wrote (five).
Without them the load may take a stale m0 or half of an address.
"""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "sqwen-moe-3090_amd" / "csrc"
LOAD = re.compile(r'asm\s+volatile\(\s*"([^"]*global_load_lds[^"]*)"')
FILES = sorted(p.name for p in CSRC.iterdir() if p.suffix in (".hip", ".hpp") and LOAD.search(p.read_text()))


def test_loads_are_found():
    assert {"fa_decode.hip", "fa_prefill.hip", "out_proj.hip", "paged_attn.hpp"} <= set(FILES)


@pytest.mark.parametrize("name", FILES)
def test_load_waits(name):
    for text in LOAD.findall((CSRC / name).read_text()):
        assert re.match(r"s_nop [0-9]+\\n", text), text
