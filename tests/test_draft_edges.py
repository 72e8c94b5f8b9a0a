"""Drafted tokens and the 8-bit cache at the edges of what their calls allow: the CPU forms, and refusals that need no GPU."""
import pytest
import torch

from draft_cases import attend, step


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("what", ["no column in the tables", "no block in the pool"])
def test_no_key_at_all_gives_rows_of_zeros(eight, what):
    s = step([(5, 40), (1, 3), (0, 0)], 8, 2, 64, eight, "tree", 5, pad=3)
    if what.startswith("no column"):
        s["table"] = s["table"][:, :0].contiguous()
    else:
        for t in ("k", "v", "ks", "vs"):
            s[t] = None if s[t] is None else s[t][:0]
    out = torch.full((9, 8, 64), 7.0, dtype=torch.bfloat16)
    attend(s, out=out)
    assert not out[:6].any() and bool((out[6:] == 7.0).all())
