"""The operators around an expert layer's products, and dropout: what cannot be seen from results on a device without a
misuse or a fault there, read from the sources instead."""
import re

from test_dependent_launch import _functions, _source


def test_places_out_of_memory_are_bounded_before_a_store():
    """dispatch's copies store a row where a number out of memory says.  What is not below the number of slots is skipped:
    executions that share a scratchpad against the rules may make any number."""
    functions = _functions(_source("moe_dispatch.cu"))
    copy, shift = functions["dispatch_copy_kernel"], functions["dispatch_shift_kernel"]
    assert re.search(r"slots = \(uint32_t\)a\.tokens \* a\.choices;", copy)
    assert re.search(r"if \(\(uint32_t\)to\[q\]\[j\] < slots\) \*\(uint4 \*\)", copy)
    assert re.search(r"if \(\(uint32_t\)mine >= \(uint32_t\)a\.tokens \* a\.choices\) mine = -1;", shift)
    assert re.search(r"to = __shfl_sync\(0xffffffffu, mine, j\);\s*if \(to < 0\) continue;", shift)
    assert "max(kept, 0)" in functions["zero_behind"]
