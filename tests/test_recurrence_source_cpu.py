"""What the recurrence kernels' source has to keep to and no result shows."""
import os
import re

import pysiglib_b200

SOURCE = os.path.join(os.path.dirname(pysiglib_b200.__file__), "csrc", "recurrence_kernels.cuh")


def test_copies_of_rows_that_are_not_there_start_at_the_array():
    """A copy of 16 bytes needs a source aligned to 16 bytes even where it brings nothing but zeros.  The start of
    an array is (the plan asks for it); a thread's first channel lies 8 bytes off for every other thread of 16-bit
    rows, so it must not be that source."""
    with open(SOURCE) as f:
        calls = re.findall(r"\bf[xgd]\.issue\(stage, (.+?), (?:p[xgd]|f[xgd]\.start)", f.read())
    assert len(calls) == 7  # x and gates of the three kernels, the backward pass's derivatives
    for source in calls:
        assert re.fullmatch(r"static_cast<const [XG]\*>\((?:REVERSE \? p\.derivs : p\.x|p\.\w+)\)", source), source
