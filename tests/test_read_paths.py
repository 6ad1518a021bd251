"""How the kernels read what an earlier kernel of the stream may still be writing.

Every kernel here is launched as a programmatic dependent: it may be resident while its
predecessor runs, and reads that one's results after griddepcontrol.wait.  The read-only path
(ld.global.nc, which __ldg and const __restrict__ pointers select) is for data that nobody
writes while the kernel runs, and a compiler may move such a load in front of the wait."""
import glob
import os
import re

import mx_flash_attn_kernel_opt__b200 as pgqa

CSRC = os.path.join(os.path.dirname(pgqa.__file__), "csrc")


def code(path):
    """A source file without its comments."""
    with open(path) as f:
        return re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S))


def test_no_kernel_reads_through_the_read_only_path():
    files = sorted(glob.glob(os.path.join(CSRC, "*.cu*")) + glob.glob(os.path.join(CSRC, "*.h")))
    assert len(files) >= 8
    found = [(os.path.basename(f), m) for f in files
             for m in re.findall(r"__ldg|global\.nc|__restrict__|\bld_nc\w*", code(f))]
    assert not found, found
