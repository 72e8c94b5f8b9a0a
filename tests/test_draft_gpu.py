"""Kernels of drafted tokens and of the 8-bit cache against their definitions in 64 bits (tests/draft_cases.py derives the bounds)."""
import math
import random

import pytest
import torch

from distributed_llm_amd import ops
from distributed_llm_amd.ops import reference as ref
from draft_cases import BS, attend, attention64, dense, i32, step, to, tree, visible

pytestmark = pytest.mark.gpu
DEV = "cuda"
HEADS = [(8, 2, 64), (6, 2, 96), (4, 4, 128), (16, 1, 128), (5, 1, 64), (24, 2, 96)]
SINGLE = [(1, 1), (1, 16), (1, 17), (1, 255), (1, 256), (1, 257), (1, 1000)]
RAGGED = [(5, 40), (0, 7), (3, 3), (33, 700), (64, 333), (1, 1), (100, 513)]


@pytest.fixture(autouse=True, scope="module")
def _native():
    assert ops.native_available(), "HIP extension must be built for GPU tests"


def near(got, want, bound):
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"off {off.max():.3g}, {(off / bound).max():.3g} of the bound"


# ------------------------------------------------------------------------------------------------ codes
def test_codes_are_the_references():
    """Every bf16 magnitude beside a top of its own, so that quotients fall everywhere: the same bytes and scales."""
    bits = torch.arange(0, 0x7F80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = bits[torch.randperm(bits.numel(), generator=torch.Generator().manual_seed(0))][: 32512].view(-1, 4, 64)[:, :, :]
    x = torch.cat([x, -x], 0).contiguous()
    T = x.shape[0]
    slots = torch.randperm(T + 16, generator=torch.Generator().manual_seed(1))[:T].to(torch.int32)
    blocks = (T + 16 + BS - 1) // BS
    c, g = ops.kv8.alloc(blocks, 4, 64), ops.kv8.alloc(blocks, 4, 64, DEV)
    ops.kv8.write(x, x, slots, c)
    ops.kv8.write(x.to(DEV), x.to(DEV), slots.to(DEV), g)
    for a, b in zip(c, g):
        assert torch.equal(a.view(torch.uint8 if a.dtype != torch.float32 else torch.int32), b.cpu().view(torch.uint8 if a.dtype != torch.float32 else torch.int32))


@pytest.mark.parametrize("nq,nkv,d", [(32, 4, 64), (12, 4, 96), (7, 1, 128), (3, 3, 16), (4, 2, 112)])
@pytest.mark.parametrize("T", [1, 5, 37, 300])
@pytest.mark.parametrize("order", ["run", "shuffled"])
def test_rope_and_cache_writes_the_references_bytes(nq, nkv, d, T, order):
    g = torch.Generator().manual_seed(T + d)
    qkv = torch.randn(T, (nq + 2 * nkv) * d + 8, generator=g).bfloat16()[:, : (nq + 2 * nkv) * d]
    blocks = T // BS + 3
    slots = torch.arange(7, 7 + T) if order == "run" else torch.randperm(blocks * BS, generator=g)[:T]
    slots = slots.to(torch.int32)
    if T > 4:
        slots[2], slots[4] = -1, blocks * BS + 3
    pos, cs = torch.randint(0, 700, (T,), generator=g).to(torch.int32), ops.rope_cos_sin(700, d, 10000.0)
    c, h = ops.kv8.alloc(blocks, nkv, d), ops.kv8.alloc(blocks, nkv, d, DEV)
    want = ops.kv8.rope_and_cache(qkv, pos, cs, slots, c, nq, nkv, d)
    wide = torch.zeros(T, (nq + 2 * nkv) * d + 8, dtype=torch.bfloat16, device=DEV)
    wide[:, : (nq + 2 * nkv) * d] = qkv
    got = ops.kv8.rope_and_cache(wide[:, : (nq + 2 * nkv) * d], pos.to(DEV), cs.to(DEV), slots.to(DEV), h, nq, nkv, d)
    assert torch.equal(want, got.cpu())
    for a, b in zip(c, h):
        assert torch.equal(a.float(), b.cpu().float())
    k, v = ops.kv8.read(h, slots.to(DEV))
    rk, rv = ops.kv8.read(c, slots)
    assert torch.equal(k.cpu(), rk) and torch.equal(v.cpu(), rv)


def test_a_vector_that_is_not_finite_stays_its_own():
    g = ops.kv8.alloc(2, 2, 96, DEV)
    x = torch.ones(3, 2, 96, dtype=torch.bfloat16, device=DEV)
    x[0, 1, 95], x[2, 0, 0] = math.nan, -math.inf
    s = i32([3, 4, 30], DEV)
    ops.kv8.write(x, x, s, g)
    for t in ops.kv8.read(g, s):
        assert t[0, 1].isnan().all() and t[2, 0].isnan().all()
        assert bool((t[1] == 1).all()) and bool((t[0, 0] == 1).all()) and bool((t[2, 1] == 1).all())


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("nq,nkv,d", HEADS)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("known", [False, True])
def test_single_tokens(nq, nkv, d, eight, known):
    s = step(SINGLE, nq, nkv, d, eight, "chain", d + nq)
    near(attend(to(s, DEV), **(dict(max_qlen=1, max_ctx=1000) if known else {})), *attention64(s))


@pytest.mark.parametrize("nq,nkv,d", HEADS)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("mode", ["chain", "tree"])
@pytest.mark.parametrize("known", [False, True])
def test_ragged_batches(nq, nkv, d, eight, mode, known):
    s = step(RAGGED, nq, nkv, d, eight, mode, d + nq + 1)
    near(attend(to(s, DEV), **(dict(max_qlen=100, max_ctx=700) if known else {})), *attention64(s))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("seqs", [[(2, 33)], [(6, 200)] * 3, [(13, 129), (12, 90)]])
@pytest.mark.parametrize("d", [64, 128])
def test_few_rows_of_short_contexts_in_one_launch(eight, seqs, d):
    s = step(seqs, 8, 4, d, eight, "tree", 9)
    near(attend(to(s, DEV), max_qlen=max(q for q, _ in seqs), max_ctx=max(c for _, c in seqs)), *attention64(s))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("qlen", [2, 4, 5, 8, 9, 16, 17])
def test_row_blocks_of_every_form(eight, d, qlen):
    """Twelve sequences of 900 keys, eight query heads to each of three: blocks of 16, 32 and 48 rows of a wave, of 64 and 128 of four, filled and a row over."""
    s = step([(qlen, 900 + i) for i in range(11)] + [(1, 5)], 24, 3, d, eight, "tree", qlen)
    near(attend(to(s, DEV), max_qlen=qlen, max_ctx=910), *attention64(s))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("hints", [dict(max_qlen=1, max_ctx=1), dict(max_qlen=1), dict(max_ctx=16), dict(max_qlen=10 ** 6, max_ctx=10 ** 6)])
def test_hints_that_are_wrong_cost_time_alone(eight, hints):
    s = step([(40, 700), (9, 1300), (2, 2)], 8, 2, 64, eight, "tree", 15)
    near(attend(to(s, DEV), **hints), *attention64(s))


@pytest.mark.parametrize("eight", [False, True])
def test_contexts_shorter_than_their_new_tokens(eight):
    """No key at all, or fewer than new tokens: rows ahead of the first key see nothing and are zero."""
    s = step([(2, 0), (5, 3), (40, 7), (3, 50)], 4, 2, 64, eight, "chain", 16)
    want, bound = attention64(s)
    got = attend(to(s, DEV))
    near(got, want, bound)
    assert not got[:4].any() and not want[:4].any()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_other_scales(eight, scale):
    """A negative scale turns the order of scores, 0 makes the mean.  Bounds as attention64's, whose scale is 1 / 8 here: queries carry the rest exactly
    (-1.6 and 24 do not fit bf16: the expected value is computed with them in 64 bits)."""
    s = step([(9, 300), (1, 40)], 4, 2, 64, eight, "tree", 17)
    wide = dict(s, q=s["q"].double() * (8.0 * scale))
    near(attend(to(s, DEV), scale=scale), *attention64(wide))


def test_a_part_longer_than_its_window_of_pages():
    """430 sequences over the same 20000 keys: a workgroup's part passes 16384 keys of one row block, so its pages are looked up again on the way."""
    n, ctx, qlen, d = 430, 20000, 9, 64
    s = to(step([(qlen, ctx)], 4, 1, d, False, "chain", 18), DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    s["q"] = (1.5 * torch.randn(n * qlen, 4, d, device=DEV, generator=g)).bfloat16()
    s["table"] = s["table"].repeat(n, 1)
    s["qstart"], s["qlen"], s["ctx"] = i32(list(range(0, n * qlen, qlen)), DEV), i32([qlen] * n, DEV), i32([ctx] * n, DEV)
    got = attend(s)
    k, v = dense({t: None if x is None else x.cpu() for t, x in dict(s, table=s["table"][:1]).items()}, 0)
    k, v = k[0].to(DEV), v[0].to(DEV)
    see = torch.arange(ctx, device=DEV)[None] <= ctx - qlen + torch.arange(qlen, device=DEV)[:, None]
    for b in range(0, n, 43):
        x = s["q"][b * qlen:(b + 1) * qlen].double()                                        # [qlen, 4, d]
        w = torch.softmax((x.transpose(0, 1) @ k.T / 8).masked_fill(~see, -math.inf), -1)   # [4, qlen, keys]
        o, a = (w @ v).transpose(0, 1), (w @ v.abs()).transpose(0, 1)
        ds = (d + 3) * 2.0 ** -24 * (x.abs() @ k.abs().T / 8).amax(-1)[..., None]
        e = (2.0 ** -8 + 2 * ds + (2 * ctx + 16) * 2.0 ** -24) * a
        near(got[b * qlen:(b + 1) * qlen], o.cpu(), (e + 2.0 ** -8 * (o.abs() + e)).cpu())


@pytest.mark.parametrize("eight", [False, True])
def test_rows_of_a_prompt_behind_a_cached_one(eight):
    s = step([(300, 300), (129, 1001)], 8, 2, 64, eight, "chain", 5)
    near(attend(to(s, DEV)), *attention64(s))


@pytest.mark.parametrize("eight", [False, True])
def test_a_long_context_in_many_parts(eight):
    """Every unit in a part of its own, joined in order; the same bits again."""
    s = step([(3, 9000), (1, 20), (17, 4097)], 4, 1, 128, eight, "tree", 6)
    h = to(s, DEV)
    got = attend(h)
    near(got, *attention64(s))
    assert torch.equal(got, attend(h))


@pytest.mark.parametrize("eight", [False, True])
def test_many_sequences(eight):
    """More sequences than a wave has lanes, most of them without new tokens."""
    rng = random.Random(1)
    s = step([(rng.choice([0, 0, 1, 4]), rng.randrange(4, 400)) for _ in range(333)], 2, 1, 64, eight, "tree", 7)
    near(attend(to(s, DEV)), *attention64(s))


def test_scores_far_apart():
    """A key late in the context outweighs all before it by e^60, and one early: the running maximum moves once, or never again."""
    for at in (3, 690):
        s = step([(4, 700)], 4, 2, 64, False, "chain", 8)
        page, off = int(s["table"][0, at // BS]), at % BS
        s["k"][page, :, off] = 0
        s["k"][page, :, off, 0] = 300
        s["q"][:, :, 0] = 2
        near(attend(to(s, DEV)), *attention64(s))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_what_a_row_does_not_see_does_not_reach_it(eight, d):
    """Infinities and NaN: in stale keys behind the context, in drafted tokens of another branch (K and V), in pages no sequence holds."""
    s = step([(40, 190), (5, 37), (20, 20)], 8, 2, d, eight, "tree", 10)
    clean = {k: v if v is None else v.clone() for k, v in s.items()}
    want, bound = attention64(clean)
    tainted = torch.zeros(s["q"].shape[0], dtype=torch.bool)
    nan8 = torch.tensor([0x7F], dtype=torch.uint8)
    values = [math.inf, -math.inf, math.nan]
    for b, nodes in ((0, [7, 39, 20]), (1, [4]), (2, [9, 19])):
        n, c, q0 = int(s["qlen"][b]), int(s["ctx"][b]), int(s["qstart"][b])
        see = visible(s, b)
        for i, node in enumerate(nodes):
            at = c - n + node
            page, off = int(s["table"][b, at // BS]), at % BS
            if eight:
                s["v"].view(torch.uint8)[page, :, 1 + i, off] = nan8
                s["k"].view(torch.uint8)[page, :, off, 2] = nan8
                s["vs"][page, 0, off] = values[i]
            else:
                s["v"][page, :, 1 + i, off] = values[i]
                s["k"][page, :, off, 2] = values[i]
            tainted[q0:q0 + n] |= see[:, at]
        for at in range(c, -(-c // BS) * BS):                   # stale memory behind the last key
            page, off = int(s["table"][b, at // BS]), at % BS
            if eight:
                s["v"].view(torch.uint8)[page, :, :, off] = nan8
                s["k"].view(torch.uint8)[page, :, off] = nan8
                s["ks"][page, :, off], s["vs"][page, :, off] = math.nan, math.inf
            else:
                s["v"][page, :, :, off], s["k"][page, :, off] = math.nan, math.inf
    assert 0 < int(tainted.sum()) < tainted.numel()
    got = attend(to(s, DEV)).cpu()
    near(got[~tainted], want[~tainted], bound[~tainted])
    assert not torch.isfinite(got[tainted].float()).all(-1).any()


def test_an_infinity_of_v_reaches_the_rows_that_see_it():
    s = step([(12, 60)], 4, 2, 64, False, "tree", 12)
    at = 60 - 12 + 3
    page, off = int(s["table"][0, at // BS]), at % BS
    s["v"][page, :, 9, off] = -math.inf
    see = visible(s, 0)[:, at]
    got = attend(to(s, DEV)).cpu().float()
    assert bool((got[see][:, :, 9] == -math.inf).all()) and torch.isfinite(got[~see]).all()
    assert torch.isfinite(got[:, :, :9]).all() and torch.isfinite(got[:, :, 10:]).all()


@pytest.mark.parametrize("eight", [False, True])
def test_pages_outside_the_pool_are_not_seen(eight):
    s = step([(4, 150), (2, 20)], 4, 2, 64, eight, "tree", 3)
    see = [visible(s, 0), visible(s, 1)]
    see[0][:, 16:48] = False
    see[1][:, 16:] = False
    want, bound = attention64(s, see)
    s["table"][0, 1], s["table"][0, 2], s["table"][1, 1] = 10 ** 6, s["k"].shape[0], -7
    near(attend(to(s, DEV)), want, bound)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("most", [512, 513])
def test_the_longest_contexts_of_one_launch(eight, d, most):
    """Tables of 32 blocks are not cut, of 33 they are: rows of every form."""
    s = step([(64, most), (33, 511), (1, 500), (16, 480), (0, 70), (5, 5)], 8, 2, d, eight, "tree", 21)
    want, bound = attention64(s)
    near(attend(to(s, DEV)), want, bound)
    near(attend(to(s, DEV), max_qlen=64, max_ctx=most), want, bound)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_row_blocks_cut_at_different_keys(eight, d):
    """Several row blocks over the same keys, each in parts of its own: parts begin in their middle.  Pages outside the pool anywhere on the way, the last
    one of a sequence too."""
    s = step([(75, 3001), (41, 1500), (20, 777)], 8, 2, d, eight, "tree", 19)
    see = [visible(s, b) for b in range(3)]
    for b, page in ((0, 0), (0, 31), (0, 100), (0, 187), (1, 64), (1, 93), (2, 48)):
        see[b][:, page * BS:(page + 1) * BS] = False
    want, bound = attention64(s, see)
    whole = attention64(s)
    near(attend(to(s, DEV)), *whole)
    for b, page in ((0, 0), (0, 31), (0, 100), (0, 187), (1, 64), (1, 93), (2, 48)):
        s["table"][b, page] = -1 if page % 2 else s["k"].shape[0]
    near(attend(to(s, DEV)), want, bound)


def test_a_row_that_sees_nothing_is_zero():
    s = step([(6, 6), (3, 40)], 8, 2, 64, False, "tree", 4)
    s["mask"][2] = 0
    got = attend(to(s, DEV)).cpu()
    assert not got[2].any() and got[3].any() and got[6:].any()


def test_views_padding_rows_and_out():
    s = step([(9, 70), (4, 300)], 6, 3, 64, False, "tree", 13, pad=5)
    want, bound = attention64(s)
    h = to(s, DEV)
    wide = torch.zeros(18, 20, 64, dtype=torch.bfloat16, device=DEV)
    wide[:, 2:8] = h["q"]
    out = torch.full_like(h["q"], 7.0)
    got = attend(dict(h, q=wide[:, 2:8]), out=out)
    assert got is out or got.data_ptr() == out.data_ptr()
    near(got[:13], want[:13], bound[:13])
    assert bool((got[13:] == 7.0).all())


def test_offsets_past_32_bits():
    """Pages at the end of a pool of more than 2^31 values."""
    s = step([(5, 100), (2, 400)], 4, 4, 128, False, "tree", 14)
    blocks = (1 << 31) // (4 * BS * 128) + 40
    h, n = to(s, DEV), s["k"].shape[0]
    for t in ("k", "v"):
        pool = torch.empty((blocks, *s[t].shape[1:]), dtype=torch.bfloat16, device=DEV)
        pool[blocks - n:] = h[t]
        h[t] = pool
    h["table"] = h["table"] + (blocks - n)
    near(attend(h), *attention64(s))
    k5, v5 = h["k"][None], h["v"][None]
    base = [int(c) - int(q) for c, q in zip(s["ctx"], s["qlen"])]
    path = i32([[0, 3, 4, -1, -1], [0, 1, -1, -1, -1]], DEV)
    ops.draft.keep(k5, v5, h["table"], h["qlen"], h["ctx"], path, i32([2, 1], DEV))
    at = lambda b, i: (int(s["table"][b, (base[b] + i) // BS]), (base[b] + i) % BS)  # noqa: E731
    (p1, o1), (p3, o3) = at(0, 1), at(0, 3)
    assert torch.equal(h["k"][p1 + blocks - n, :, o1].cpu(), s["k"][p3, :, o3])
    assert torch.equal(h["v"][p1 + blocks - n, :, :, o1].cpu(), s["v"][p3, :, :, o3])


@pytest.mark.parametrize("eight", [False, True])
def test_a_captured_step_takes_new_trees_and_lengths(eight):
    """Mask, attention, verification and keep in one graph; other trees, lengths and tables before each replay, eager work between them."""
    nq, nkv, d, most, V = 8, 2, 64, 24, 500
    shapes = [[(24, 300), (3, 40), (9, 100)], [(1, 1), (24, 700), (11, 19)], [(12, 999), (12, 500), (12, 12)]]
    steps = [step(q, nq, nkv, d, eight, "tree", 20 + i, spare=0, pad=36 - sum(n for n, _ in q)) for i, q in enumerate(shapes)]
    pool = max(s["k"].shape[0] for s in steps)
    g = torch.Generator().manual_seed(3)
    extra = [dict(target=torch.softmax(3 * torch.randn(36, V, generator=g), -1), tokens=torch.randint(0, V, (36,), generator=g).int(),
                  uniform=torch.rand(36, generator=g) * 0.02) for _ in steps]
    for s, e in zip(steps, extra):                              # likely candidates, so that some are accepted
        seq = torch.repeat_interleave(s["qstart"], s["qlen"])
        e["tokens"][:seq.numel()] = e["target"][(seq + s["parents"][:seq.numel()].clamp_min(0)).long()].argmax(-1).int()

    def grown(s):
        wide = dict(s)
        for t in ("k", "v", "ks", "vs"):
            if s[t] is not None:
                x = torch.zeros((pool, *s[t].shape[1:]), dtype=torch.uint8 if s[t].element_size() == 1 else s[t].dtype)
                x[:s[t].shape[0]] = s[t].view(torch.uint8) if s[t].element_size() == 1 else s[t]
                wide[t] = x.view(s[t].dtype)
        wide["table"] = torch.zeros(3, 64, dtype=torch.int32)
        wide["table"][:, :s["table"].shape[1]] = s["table"]
        return wide

    def run(h, e):
        mask, depth = ops.draft.tree_mask(h["parents"], h["qstart"], h["qlen"], most)
        out = attend(dict(h, mask=mask), max_qlen=most, max_ctx=1024, out=h["out"])
        acc, nxt, path = ops.draft.verify(e["target"], e["tokens"], e["uniform"], h["qstart"], h["qlen"], most, parents=h["parents"])
        ops.draft.keep(h["k"], h["v"], h["table"], h["qlen"], h["ctx"], path, acc, k_scale=h["ks"], v_scale=h["vs"])
        return [out, acc, nxt, path, depth]

    steps = [grown(s) for s in steps]
    fixed, fe = to(dict(steps[0], out=torch.zeros_like(steps[0]["q"])), DEV), to(extra[0], DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(fixed, fe)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(fixed, fe)
    for i in (0, 1, 2, 1, 0):
        h, e = to(dict(steps[i], out=torch.zeros_like(steps[i]["q"])), DEV), to(extra[i], DEV)
        for a, b in ((fixed, h), (fe, e)):
            for t in a:
                if a[t] is not None and t != "mask":
                    a[t].view(torch.uint8).copy_(b[t].view(torch.uint8)) if a[t].element_size() == 1 else a[t].copy_(b[t])
        graph.replay()
        want = run(h, e)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for t in ("k", "v", "ks", "vs"):
            if h[t] is not None:
                assert torch.equal(h[t].view(torch.uint8), fixed[t].view(torch.uint8))
        assert int(want[1].sum()) > 0


def test_two_streams_at_once():
    """Calls on streams of their own share nothing."""
    a, b = to(step([(9, 3000)] * 4, 8, 2, 128, False, "tree", 30), DEV), to(step([(5, 5000)] * 3, 8, 2, 128, True, "tree", 31), DEV)
    want = attend(a), attend(b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(s1):
            x = attend(a)
        with torch.cuda.stream(s2):
            y = attend(b)
        got.append((x, y))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[0]) and torch.equal(y, want[1]) for x, y in got)


# ------------------------------------------------------------------------------------------------ verification
def drafts(lens, V, given, kind, seed, dtype=torch.float32):
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    T = sum(lens) + 2
    logits = 3 * torch.randn(T, V, generator=g)
    target, near_ = torch.softmax(logits, -1).to(dtype), torch.softmax(logits + 0.7 * torch.randn(T, V, generator=g), -1).to(dtype)
    s = dict(qstart=i32([sum(lens[:i]) for i in range(len(lens))]), qlen=i32(lens), target=target, uniform=torch.rand(T, generator=g), parents=None, draft=None)
    if kind == "tree":
        s["parents"] = i32(sum([tree(rng, n) for n in lens], []) + [-1, -1])
    if given:
        start = torch.repeat_interleave(s["qstart"], s["qlen"]).long()
        par = torch.arange(sum(lens)) - 1 if kind == "chain" else start + s["parents"][: sum(lens)].clamp_min(0)
        top = torch.topk(near_.float(), min(4, V), -1).indices
        tok = top[par.clamp_min(0), torch.randint(0, min(4, V), (sum(lens),), generator=g)]     # (siblings may be alike)
        s["tokens"] = torch.cat([tok, torch.zeros(2, dtype=torch.int64)]).int()
    else:
        s["draft"] = near_.roll(1, 0).contiguous()
        s["tokens"] = torch.multinomial(s["draft"].float(), 1, generator=g)[:, 0].int()
    return s


def check_verify(s, most):
    args = [s[t] for t in ("target", "tokens", "uniform", "qstart", "qlen")]
    want = ops.draft.verify(*args, most, parents=s["parents"], draft=s["draft"])
    h = to(s, DEV)
    got = ops.draft.verify(*[h[t] for t in ("target", "tokens", "uniform", "qstart", "qlen")], most, parents=h["parents"], draft=h["draft"])
    for a, b in zip(want, got):
        assert torch.equal(a, b.cpu())


@pytest.mark.parametrize("kind,given", [("chain", False), ("chain", True), ("tree", True)])
@pytest.mark.parametrize("V", [1, 5, 4099, 32000, 128256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_verification_is_the_walk(kind, given, V, dtype):
    lens = [1, 9, 0, 30, 4, 2, 70] if V < 100000 else [5, 1, 8]
    check_verify(drafts(lens, V, given, kind, V, dtype), max(lens))


@pytest.mark.parametrize("given", [False, True])
def test_many_uniform_draws(given):
    """600 sequences: flat rows too, where the token hangs on the last bits of sums; and the largest u below one."""
    lens = [2] * 600
    s = drafts(lens, 1031, given, "chain", 2)
    s["target"][::3] = 1.0 / 1031
    s["uniform"][::7] = 1.0 - 2.0 ** -24
    s["uniform"][4::7] = 0.0
    check_verify(s, 2)


def test_rows_of_a_view_and_odd_alignment():
    s = drafts([6, 3], 1001, False, "chain", 3)
    h = to(s, DEV)
    wide, wide2 = torch.zeros(11, 1005, device=DEV), torch.zeros(11, 1010, device=DEV)
    wide[:, 3:1004], wide2[:, 1:1002] = h["target"], h["draft"]
    want = ops.draft.verify(*[s[t] for t in ("target", "tokens", "uniform", "qstart", "qlen")], 6, draft=s["draft"])
    got = ops.draft.verify(wide[:, 3:1004], h["tokens"], h["uniform"], h["qstart"], h["qlen"], 6, draft=wide2[:, 1:1002])
    for a, b in zip(want, got):
        assert torch.equal(a, b.cpu())


def test_verification_at_the_ends():
    V = 4100
    s = drafts([3, 4, 2, 5, 1], V, True, "tree", 4)
    s["target"][0] = 0                                          # a row without probability
    s["target"][4] = math.nan
    s["target"][7, 5] = math.inf
    s["tokens"][1], s["tokens"][5], s["tokens"][8] = -3, V, 2 ** 30
    s["parents"][10] = 77
    s["parents"][12] = -1                                       # a node that cannot be reached
    s["uniform"][14] = 1.0
    check_verify(s, 5)
    check_verify(s, 2)                                          # sequences of more nodes than max_nodes: the first ones count
    same = drafts([2, 2], V, False, "chain", 5)
    same["draft"] = same["target"].clone()
    same["target"][1] = same["target"][0]
    same["draft"][1] = same["target"][0]
    same["uniform"][1] = 1.0                                    # refused although nothing lies above the draft
    check_verify(same, 2)


def test_the_largest_trees():
    lens = [1024, 300]
    s = drafts(lens, 300, True, "tree", 6)
    check_verify(s, 1024)
    h = to(s, DEV)
    want, got = ref.tree_mask(s["parents"], s["qstart"], s["qlen"], 1024), ops.draft.tree_mask(h["parents"], h["qstart"], h["qlen"], 1024)
    assert torch.equal(want[0], got[0].cpu()) and torch.equal(want[1], got[1].cpu())


@pytest.mark.parametrize("lens,most", [([1, 33, 0, 64, 5], 64), ([7] * 100, 7), ([31, 32], 32)])
def test_masks(lens, most):
    rng = random.Random(8)
    par = i32(sum([tree(rng, n) for n in lens], []) + [3] * 4)
    par[sum(lens) - 1] = 10 ** 6                                # a parent behind its child counts as none
    start, n = i32([sum(lens[:i]) for i in range(len(lens))]), i32(lens)
    want, got = ref.tree_mask(par, start, n, most), ops.draft.tree_mask(par.to(DEV), start.to(DEV), n.to(DEV), most)
    assert torch.equal(want[0], got[0].cpu()) and torch.equal(want[1], got[1].cpu())


def test_masks_of_many_sequences_with_rows_between():
    """700 sequences in rows of their own order, rows of none between them: more than one workgroup has of either."""
    rng = random.Random(9)
    lens = [rng.choice([0, 1, 2, 5, 9]) for _ in range(700)]
    starts, at = [], 0
    for n in lens:
        at += rng.choice([0, 0, 1, 3])
        starts.append(at)
        at += n
    par = [5] * (at + 300)
    for q0, n in zip(starts, lens):
        par[q0:q0 + n] = tree(rng, n)
    order = rng.sample(range(700), 700)
    start, n = i32([starts[i] for i in order]), i32([lens[i] for i in order])
    want, got = ref.tree_mask(i32(par), start, n, 9), ops.draft.tree_mask(i32(par, DEV), start.to(DEV), n.to(DEV), 9)
    assert torch.equal(want[0], got[0].cpu()) and torch.equal(want[1], got[1].cpu())


def test_masks_of_sequences_that_do_not_fit():
    """More nodes than max_nodes, a start outside the rows: those rows are zero."""
    par = i32([-1] + list(range(69)) + [-1, 0, 0])
    start, n = i32([0, 70, 500, -3]), i32([70, 3, 4, 2])
    want, got = ref.tree_mask(par, start, n, 40), ops.draft.tree_mask(par.to(DEV), start.to(DEV), n.to(DEV), 40)
    assert torch.equal(want[0], got[0].cpu()) and torch.equal(want[1], got[1].cpu())
    assert not got[0][64:70].any() and bool(got[0][63].any())


def test_no_sequences_and_no_rows():
    e, z = i32([], DEV), torch.zeros(0, 8, device=DEV)
    assert [t.numel() for t in ops.draft.verify(z, e, z[:, 0].contiguous(), e, e, 3)] == [0, 0, 0]
    acc, nxt, path = ops.draft.verify(z, e, z[:, 0].contiguous(), i32([0, 0], DEV), i32([0, 0], DEV), 3)
    assert acc.tolist() == [0, 0] and nxt.tolist() == [-1, -1] and bool((path == -1).all())
    assert [t.shape[0] for t in ops.draft.tree_mask(e, e, e, 3)] == [0, 0]
    c = ops.kv8.alloc(2, 1, 64, DEV)
    assert ops.kv8.read(c, e)[0].shape == (0, 1, 64)
    s = to(step([(0, 5)], 2, 1, 64, False, "chain", 1), DEV)
    assert attend(s).shape == (0, 2, 64)
    ops.draft.keep(s["k"], s["v"], s["table"], s["qlen"], s["ctx"], i32([[-1]], DEV), i32([0], DEV))


# ------------------------------------------------------------------------------------------------ keep
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("nkv,d,layers", [(2, 64, 3), (1, 96, 0), (3, 128, 2), (2, 16, 1), (1, 112, 2)])
def test_keep_is_the_references(eight, nkv, d, layers):
    """Paths within a block, over blocks, longer than a batch of moves, of one node, past what was accepted; places outside the pool and the table stay."""
    rng = random.Random(d)
    seqs = [(40, 60), (60, 61), (1, 5), (64, 300), (5, 4), (9, 50), (30, 47)]
    s = step(seqs, 1, 1, 64, False, "chain", 2)
    g, lead = torch.Generator().manual_seed(1), (layers,) if layers else ()
    pool = s["k"].shape[0]
    k = torch.randint(0, 120, (*lead, pool, nkv, BS, d * (1 if eight else 2)), generator=g).to(torch.uint8)
    v = torch.randint(0, 120, (*lead, pool, nkv, d, BS * (1 if eight else 2)), generator=g).to(torch.uint8)
    kind = torch.float8_e4m3fn if eight else torch.bfloat16
    k, v = k.view(kind), v.view(kind)
    ks, vs = (torch.rand(*lead, pool, nkv, BS, generator=g), torch.rand(*lead, pool, nkv, BS, generator=g)) if eight else (None, None)
    paths, acc = [], []
    for n, _ in seqs:
        nodes = [0] + sorted(rng.sample(range(1, n), min(n - 1, rng.randrange(0, 36) if n < 64 else 50)))
        paths.append(nodes + [-1] * (64 - len(nodes)))
        acc.append(len(nodes) - 1)
    acc[0] = max(acc[0] - 2, 0)
    acc[5] = 63                                                 # more than the path holds
    s["table"][6, 2] = pool + 9
    path, acc = i32(paths), i32(acc)
    args = (s["table"], s["qlen"], s["ctx"], path, acc)
    got = [None if t is None else t.to(DEV) for t in (k, v, ks, vs)]
    ops.draft.keep(got[0], got[1], *[t.to(DEV) for t in args], k_scale=got[2], v_scale=got[3])
    ref.keep_drafts(k, v, *args, ks, vs)
    for a, b in zip((k, v, ks, vs), got):
        if a is not None:
            assert torch.equal(a.view(torch.uint8), b.cpu().view(torch.uint8))
