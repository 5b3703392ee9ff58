"""CPU tests of which kernels of the MXFP4 operators and the block norms the library holds, and which of them calls reach.
No kernel runs."""

import re

from conftest import REPO

LIB = REPO / "comfyui-featherops_amd" / "lib" / "libfeatherops_amd.so"


def test_norm_kernels_are_reached(pkg):
    """Two vectors a thread are for rows of more than 512 vectors, which no single wave holds."""
    names = set(re.findall(rb"norm_kernelILi(\d)ELi(\d)ELb([01])ELi(\d)ELb([01])ELb([01])ELb([01])E", LIB.read_bytes()))
    assert len(names) >= 50
    for x, y, mods, vectors, one_wave, codes, tiny in names:
        assert not (vectors == b"2" and (one_wave == b"1" or tiny == b"1"))
        assert not (tiny == b"1" and one_wave == b"0")
