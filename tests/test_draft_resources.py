"""Registers of the kernels of drafted tokens and of the 8-bit cache: no scratch, and the workgroups a CU that their launches count on."""
import os
import re

import pytest

from test_kernel_resources import HIPCC, _usage

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")


def _kernels(src):
    out = _usage(src)
    names = re.findall(r"Function Name: (\S+)", out)
    scratch = [int(x) for x in re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", out)]
    vgprs = [int(x) for x in re.findall(r" VGPRs: (\d+)", out)]
    lds = [int(x) for x in re.findall(r"LDS Size \[bytes/block\]: (\d+)", out)]
    assert names and len(names) == len(scratch) == len(vgprs) == len(lds)
    return list(zip(names, scratch, vgprs, lds))


@pytest.mark.parametrize("src", ["tree_attn.hip", "draft.hip", "kv8.hip"])
def test_no_scratch(src):
    assert not [(n, s) for n, s, _, _ in _kernels(src) if s]


def test_two_workgroups_a_cu():
    """256 registers a lane and 80 KB of LDS at most: the schedule fills the chip with two workgroups of four waves a CU."""
    for n, _, v, lds in _kernels("tree_attn.hip"):
        assert v <= 256 and lds <= 80 * 1024, n
