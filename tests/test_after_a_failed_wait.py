"""What the gated operators' kernels do after a bounded wait has run out: no further copy is started, and a block stays
until what is on its way to its shared memory has arrived. Read from the sources: on a device such a wait never runs out."""

from __future__ import annotations

import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "gdn2_tilelang_b200" / "csrc"


def _code(name):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", (CSRC / name).read_text(), flags=re.S)


def _body(code, at):
    """From a function's name to its closing brace."""
    i = code.index("{", code.index(")", at))
    depth, j = 0, i
    while True:
        depth += {"{": 1, "}": -1}.get(code[j], 0)
        j += 1
        if depth == 0:
            return code[i:j]


def _kernels(name):
    code = _code(name)
    return [(m.group(1), _body(code, m.end(1))) for m in re.finditer(r"\b(\w+_kernel)\s*\(const __grid_constant__", code)]


KERNELS = {n: b for f in ("recurrence.cu", "ffn.cu") for n, b in _kernels(f) if "mbar_wait" in b}


def test_the_kernels_are_found():
    assert set(KERNELS) == {"scan_forward_kernel", "scan_backward_kernel", "product_kernel", "skinny_kernel"}


@pytest.mark.parametrize("name", KERNELS)
def test_a_block_stays_after_a_failure(name):
    assert re.search(r"after_a_failure\(&sh\.abort\)", KERNELS[name])


@pytest.mark.parametrize("name", ["scan_forward_kernel", "scan_backward_kernel"])
def test_the_recurrence_asks_for_no_more_tiles(name):
    body = KERNELS[name]
    assert re.search(r"if \(tile [^;{}]*&& !\*static_cast<volatile int\*>\(&sh\.abort\)\) St::fetch\(", body) and body.count("St::fetch(") == 1
    # messages of other blocks may be on their way until every block of the cluster has come to its end
    assert body.rindex("cluster_sync()") < body.rindex("after_a_failure(&sh.abort)")
