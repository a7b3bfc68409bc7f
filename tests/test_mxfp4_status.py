"""The status words of the 4-bit products' waits: none means something else elsewhere, and the header names each."""
import os
import re

from _util import ROOT

CSRC = os.path.join(ROOT, "bf16_huffman_infer_b200", "csrc")


def _source(*names):
    return "".join(open(os.path.join(CSRC, n)).read() for n in names)


def test_codes_are_their_own_and_documented():
    others = {int(n) for n in re.findall(r"atomicExch\(&g_staged_status, (\d+)\)", _source(*sorted(os.listdir(CSRC))))}
    rows, tiles = ({int(n) for n in re.findall(r"mx_wait\(.*?, (\d+)\);", _source(f"bhi_mxfp4_{kind}.cuh"))} for kind in ("rows", "tile"))
    assert rows and tiles and not (rows | tiles) & others and not rows & tiles
    header = open(os.path.join(ROOT, "include", "bf16_huffman_b200.h")).read()
    text = header[header.index("Reads and clears the device-side status word"):header.index("int bhi_debug_status(")]
    assert rows == {11, 12} and re.search(r"\b11 X and 12\b", text)
    assert tiles == set(range(20, 26)) and "20-25" in text and all(re.search(rf"\b{n} ", text) for n in tiles)


def test_limits_begin_when_the_kernel_before_is_done():
    """Warps of a kernel with launch overlap wait for what the kernel before writes; that one may take longer than the limit by itself."""
    text = _source("bhi_mxfp4.cuh")
    wait = text[text.index("void mx_wait("):]
    wait = wait[:wait.index("\n}\n")]
    assert wait.index("pdl_wait()") < wait.index("t0 = global_ns()") < wait.index("1000000000ull")
    for name in ("bhi_mxfp4_rows.cuh", "bhi_mxfp4_tile.cuh"):    # and there are no other waits
        assert "mbar_try_wait" not in _source(name) and "mbar_wait" not in _source(name)
