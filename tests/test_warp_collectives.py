"""Which lanes meet in a warp's collective instruction is the program's to say, not what happens to be running."""
import glob
import os
import re

import pytest

from foundry_b200.kernels.library import CSRC


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.cu*"))), ids=os.path.basename)
def test_no_collective_takes_the_lanes_that_are_running(path):
    """`__activemask()` is the lanes that run that instruction together. Nothing keeps them together until the next
    one, and a collective whose lanes come one after another is undefined: it may wait for good."""
    with open(path) as handle:
        code = re.sub(r"//[^\n]*", "", handle.read())
    assert "__activemask" not in code
