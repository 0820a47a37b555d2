"""What is read from shared memory is read before a copy may overwrite it.

A statement without an instruction (asm with an empty body) holds nothing back: the assembler never sees it, drops what only it
used, and a copy that it was meant to precede may arrive first. Such a race is not shown by running it; the source says so."""

from __future__ import annotations

import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "gdn2_tilelang_b200" / "csrc"
SOURCES = sorted(CSRC.glob("*.cu*"))


def _code(path):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_no_order_by_an_empty_statement(path):
    assert not re.search(r'\basm\s+(?:volatile\s*)?\(\s*""', _code(path))


def test_a_piece_is_read_by_every_lane_before_the_next_is_asked_for():
    """The gated gradient's epilogue: pieces of one warp share their memory. Between the loads of a piece and the copy of the
    next stand an arrival of every lane and a wait for all of them."""
    code = _code(CSRC / "ffn.cu")
    loop = code[code.index("get_kept(chunk + 2048"):]
    ask = loop.index("load_piece(i, c + 1)")
    before = loop[:ask]
    arrive, wait = before.index("arrive_read(&sh.read[ew])"), before.index("tc::mbar_wait(&sh.read[ew]")
    assert arrive < wait and "if" not in before[:arrive]
    assert re.search(r"mbar_init\(&sh\.read\[i\], 32\)", code)
