"""The f32 tensor-core tiles keep q's terms and the accumulators in registers: the compiler's report of the
build gives their kernels no stack frame."""
import os
import re

import pytest

from moearc_b200 import build

REPORT = os.path.join(build.BUILD, "attn_batch.o.ptxas.txt")


def frames():
    """Bytes of stack of each kernel over a tf32 tile, by the tile's (channels, keys)."""
    got, tile = {}, None
    for line in open(REPORT):
        name = re.search(r"Function properties for (\S+)", line)
        if name:
            tile = re.search(r"k_attn_batch.*tf32_tileILi(\d+)ELi(\d+)E", name.group(1))
        elif tile and "bytes stack frame" in line:
            got[int(tile.group(1)), int(tile.group(2))] = int(line.split()[0])
            tile = None
    return got


@pytest.mark.skipif(not os.path.exists(REPORT), reason="the library was not built here")
def test_f32_tiles_have_no_stack_frame():
    got = frames()
    assert {d for d, _ in got} == {64, 80, 128, 256}
    assert not any(got.values()), got
