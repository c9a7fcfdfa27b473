"""That the attention over 4-bit caches loads nothing past the rows of its range, on the code that the compiler makes of it. (No GPU.)

A raw buffer's range check compares a lane's offset with the buffer's size less the load's scalar offset; what happens where that is
below zero is not stated. Tiles are issued ahead of the walk, some of them past the range's end, so that every load has to carry its place
in the buffer (whose rows end at the range's end, none being left for such tiles) and 0 as its scalar offset."""
import re
import subprocess

import pytest

from uno_amd import build as B


def test_loads_into_lds_have_no_scalar_offset(tmp_path):
    try:
        hipcc = B._hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    out = tmp_path / "tree4.s"
    subprocess.run([hipcc, *B.HIPCC_FLAGS, *B.FILE_FLAGS["tree4.hip"], "-I", str(B.CSRC), "--cuda-device-only", "-S",
                    str(B.CSRC / "tree4.hip"), "-o", str(out)], check=True, capture_output=True)
    loads = re.findall(r"^\s+buffer_load_\w+ v\d+, s\[\d+:\d+\], (\S+) offen.* lds$", out.read_text(), re.M)
    assert len(loads) >= 100                             # four loads and more to a tile, 8 kernels
    assert set(loads) == {"0"}
    assert len(re.findall(r"^\s+buffer_load_\w+ .* lds\b", out.read_text(), re.M)) == len(loads)
