"""Arrays that the draft and adapter kernels read in wider pieces than their elements: where they lie must not follow from what else a kernel declares."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "frisk_b200" / "csrc"


@pytest.mark.parametrize("source,name,piece", [("draft_verify.cu", "v", "uint4"), ("draft_verify.cu", "nodes", "double"), ("adapters.cuh", "v", "uint4"),
                                               ("adapters_rows.cuh", "memory", "uint4"), ("adapters_rows.cuh", "keys", "int4")])
def test_arrays_that_are_read_in_wider_pieces(source, name, piece):
    text = (CSRC / source).read_text()
    assert re.search(rf"reinterpret_cast<(const )?{piece}\*>\({name}\b", text)
    wide = [m.group(0) for m in re.finditer(rf"^.*\b(?:T|C|int|uint8_t) {name}\[.*$", text, re.M)]
    assert wide and all(re.search(r"alignas\(16\)|__align__\(16\)", d) for d in wide), wide
