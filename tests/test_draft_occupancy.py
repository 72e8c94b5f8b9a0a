"""Waves a SIMD of the attention of drafted tokens, as the compiler states them for architectural and accumulation registers together."""
import os
import re

import pytest

from test_kernel_resources import HIPCC, _usage


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
def test_two_workgroups_of_four_waves_a_cu():
    out = _usage("tree_attn.hip")
    names = re.findall(r"Function Name: (\S+)", out)
    waves = [int(x) for x in re.findall(r"Occupancy \[waves/SIMD\]: (\d+)", out)]
    lds = [int(x) for x in re.findall(r"LDS Size \[bytes/block\]: (\d+)", out)]
    assert names and len(names) == len(waves) == len(lds)
    few = [(n, w, b) for n, w, b in zip(names, waves, lds) if w < 2 or 2 * b > 160 * 1024]
    assert not few
