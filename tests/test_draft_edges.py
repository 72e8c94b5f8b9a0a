"""Drafted tokens and the 8-bit cache at the edges of what their calls allow: the CPU forms, and refusals that need no GPU."""
import ctypes

import pytest
import torch

from distributed_llm_amd import ops
from distributed_llm_amd._build import HIP_SO
from draft_cases import BS, attend, attention64, i32, step, to


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


@pytest.mark.skipif(torch.cuda.is_available(), reason="hands the launcher no real memory")
@pytest.mark.parametrize("eight,rf,wide,units", [(False, 1, 0, 128), (False, 2, 0, 128), (True, 1, 0, 256), (True, 2, 0, 128), (True, 3, 0, 128),
                                                 (False, 1, 1, 64), (False, 2, 1, 64)])
def test_the_launcher_refuses_units_that_are_not_whole_rounds(eight, rf, wide, units):
    """A piece begins whole units behind its first key and goes on in rounds of all waves' chunks: units of part of a round would leave keys out."""
    if not ops.native_available():
        pytest.skip("extension not built")
    call = ctypes.CDLL(HIP_SO).dllm_tree_attention
    P, I, L = ctypes.c_void_p, ctypes.c_int, ctypes.c_long
    call.argtypes, call.restype = [P, L, L] + [P] * 13 + [I] * 15 + [ctypes.c_float, P], I
    some, scale = 4096, 4096 if eight else None
    run = lambda u: call(some, 512, 64, some, some, scale, scale, some, some, some, some, None, some, some, some, some,  # noqa: E731
                         0, 1, 8, 8, 1, 64, 64, 64, 8, u, 1, 1, rf, wide, 16, 0.125, None)
    for u in range(-64, 513, 32):
        if u < 0 or u % units:
            assert run(u) == -3, u


def test_attention_refuses_an_output_that_overlaps_its_queries():
    s = step([(4, 20)], 8, 2, 64, False, "chain", 1)
    for rows in (0, 1, 3):
        both = torch.zeros(4 + rows, 8, 64, dtype=torch.bfloat16)
        both[rows:] = s["q"]
        for q, out in ((both[rows:], both[:4]), (both[:4], both[rows:])):
            with pytest.raises(ValueError, match="overlaps"):
                attend(dict(s, q=q), out=out)
    room = torch.zeros(8, 8, 64, dtype=torch.bfloat16)              # beside each other in one tensor
    room[:4] = s["q"]
    attend(dict(s, q=room[:4]), out=room[4:])
    assert torch.equal(room[4:], attend(s))


def test_rope_and_cache_refuses_queries_that_overlap_its_rows():
    cache, cs, at = ops.kv8.alloc(4, 2, 64), ops.rope_cos_sin(8, 64, 1e4), i32([0, 1, 2])
    room = torch.ones(3 * 8 * 64 + 3 * 4 * 64, dtype=torch.bfloat16)
    qkv = room[:3 * 8 * 64].view(3, 512)
    for start in (0, 64, 3 * 8 * 64 - 8):
        with pytest.raises(ValueError, match="overlaps"):
            ops.kv8.rope_and_cache(qkv, at, cs, at, cache, 4, 2, 64, q_out=room[start:start + 3 * 4 * 64].view(3, 4, 64))
    q = ops.kv8.rope_and_cache(qkv, at, cs, at, cache, 4, 2, 64, q_out=room[3 * 8 * 64:].view(3, 4, 64))
    assert torch.equal(q, ops.kv8.rope_and_cache(qkv, at, cs, at, cache, 4, 2, 64))
    ops.kv8.rope_and_cache(qkv, at, cs, at, cache, 0, 2, 64, q_out=room[:0].view(3, 0, 64))      # no value to overlap


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("keys", [9, 700])
def test_a_row_whose_scores_are_all_minus_infinity_is_zero(device, eight, keys):
    """A score of minus infinity weighs nothing, as a key that is not seen; of plus infinity the row is NaN.  Keys of -3e38 in 64 dims overflow."""
    s = step([(2, keys), (3, 40)], 8, 2, 64, eight, "chain", 6)
    want, bound = attention64(s)
    mine = s["table"][0, :-(-keys // BS)].long()
    if eight:
        s["ks"][mine] = 3e38 / 448
        s["k"].view(torch.uint8)[mine] = 0xFE                       # -448
    else:
        s["k"][mine] = -3e38
    s["q"][0], s["q"][1] = 2.0, -2.0
    got = attend(to(s, device)).cpu()
    assert not got[0].any() and got[1].isnan().all()
    assert bool(((got[2:].double() - want[2:]).abs() <= bound[2:]).all())


def test_tensors_of_another_device_are_refused():
    """As the kernels' checks have it; here a device without data."""
    away = lambda t: t.to("meta")  # noqa: E731
    s = step([(4, 20)], 8, 2, 64, True, "tree", 1)
    for t in ("k", "vs", "table", "qlen", "mask"):
        with pytest.raises(ValueError, match="another device"):
            attend(dict(s, **{t: away(s[t])}))
    with pytest.raises(ValueError, match="another device"):
        attend(s, out=away(s["q"]))
    p, tok, u, n = torch.full((3, 8), 0.125), i32([0, 1, 2]), torch.rand(3), i32([3])
    good = dict(target=p, tokens=tok, uniform=u, seq_qstart=i32([0]), seq_qlen=n, max_nodes=3)
    for bad in (dict(tokens=away(tok)), dict(uniform=away(u)), dict(seq_qlen=away(n)), dict(parents=away(tok)), dict(draft=away(p))):
        with pytest.raises(ValueError, match="another device"):
            ops.draft.verify(**dict(good, **bad))
    path = i32([[0, 2, 3, -1]])
    good = dict(k_cache=s["k"], v_cache=s["v"], block_tables=s["table"], seq_qlen=s["qlen"], seq_ctx=s["ctx"], path=path, accepted=i32([2]), k_scale=s["ks"],
                v_scale=s["vs"])
    for t in ("v_cache", "block_tables", "seq_ctx", "path", "accepted", "k_scale"):
        with pytest.raises(ValueError, match="another device"):
            ops.draft.keep(**dict(good, **{t: away(good[t])}))
    c, qkv, cs = ops.kv8.alloc(4, 2, 64), torch.zeros(3, 512, dtype=torch.bfloat16), ops.rope_cos_sin(8, 64, 1e4)
    for args in ((qkv, away(tok), cs, tok, c), (qkv, tok, away(cs), tok, c), (qkv, tok, cs, away(tok), c), (qkv, tok, cs, tok, c._replace(v=away(c.v)))):
        with pytest.raises(ValueError, match="another device"):
            ops.kv8.rope_and_cache(*args, 4, 2, 64)
    with pytest.raises(ValueError, match="another device"):
        ops.kv8.rope_and_cache(qkv, tok, cs, tok, c, 4, 2, 64, q_out=away(torch.zeros(3, 4, 64, dtype=torch.bfloat16)))
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    for args in ((x, away(x), tok, c), (x, x, away(tok), c)):
        with pytest.raises(ValueError, match="another device"):
            ops.kv8.write(*args)
    with pytest.raises(ValueError, match="another device"):
        ops.kv8.read(c, away(tok))
