"""Lists of blocks that lanes of a wave leave in LDS for each other, in the assembly that the
source compiles to: the order of their stores and reads is stated, not left to what the
compiler can tell of the addresses."""
from __future__ import annotations

import os
import re

import pytest

from test_lds_load_hazards import HIPCC
from test_lds_load_order import assembly


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
def test_lists_are_in_order(tmp_path):
    text = assembly(tmp_path, "ff_int8_list")
    kernels = re.findall(r"^(_Z\w*ff_int8_list_kernel\w*):(.*?)^\.Lfunc_end", text, re.M | re.S)
    assert len(kernels) == 18
    for name, code in kernels:
        code = [line.strip() for line in code.splitlines()]
        at = lambda what: [i for i, line in enumerate(code) if line.startswith(what)]
        order, barrier = at("; wave barrier"), at("s_barrier")[0]
        stores, reads = at("ds_write"), at("ds_read")
        # the first window's lists, ahead of the first workgroup barrier: their absent entries,
        # then what is stored, then the first reads
        first = [i for i in order if i < barrier]
        assert len(first) >= 3, name
        absent = [i for i in stores if first[0] < i < first[1]]
        stored = [i for i in stores if first[1] < i < first[2]]
        assert absent and stored and not [i for i in reads if i < first[2]], name
        # and the same again in the loop, before the sums leave through LDS
        assert len([i for i in order if i > barrier]) >= 3, name
