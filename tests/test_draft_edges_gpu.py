"""Drafted tokens at the edges of what their calls allow: kernels against their definitions and against the CPU forms."""
import math
import random

import pytest
import torch

from distributed_llm_amd import ops
from draft_cases import BS, attend, attention64, dense, i32, step, to, visible

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True, scope="module")
def _native():
    assert ops.native_available(), "HIP extension must be built for GPU tests"


# ------------------------------------------------------------------------------------------------ verification
def verified(s, most):
    """The same from both forms of the call; what they say."""
    args = [s[t] for t in ("target", "tokens", "uniform", "qstart", "qlen")]
    kw = {t: s.get(t) for t in ("parents", "draft")}
    want = ops.draft.verify(*args, most, **kw)
    got = ops.draft.verify(*[x.to(DEV) for x in args], most, **{t: None if x is None else x.to(DEV) for t, x in kw.items()})
    for a, b in zip(want, got):
        assert torch.equal(a, b.cpu())
    return [x.tolist() for x in want]


@pytest.mark.parametrize("nodes", [3, 64, 65, 90])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_candidates_behind_a_nan_are_refused(nodes, dtype):
    """What a NaN leaves of the target is no number, so nothing compares below a later sibling's probability; the earlier ones are tried as ever.  Lanes
    hold trees of up to 64 nodes, LDS larger ones; the nodes behind the third hang on it."""
    V = 40
    for at, want in ((1, 0), (2, 1)):                           # the NaN ahead of the likely candidate, and behind it
        target = torch.full((nodes, V), 1.0 / V).to(dtype)
        target[0, 7], target[0, 9] = (math.nan, 0.25) if at == 1 else (0.95, math.nan)
        s = dict(target=target, tokens=i32([0, 7, 9] + [3] * (nodes - 3)), uniform=torch.full((nodes,), 0.9), qstart=i32([0]), qlen=i32([nodes]),
                 parents=i32([-1, 0, 0] + list(range(2, nodes - 1))))
        accepted, token, _ = verified(s, nodes)
        assert accepted == [want]
        assert want or token[0] not in (7, 9)


def test_a_part_without_weight_is_not_drawn_from():
    """Running sums of parts of 4096 tokens meet in an order of their own: here the sum up to the fifth part, which has no weight, rounds to one bit more
    than the one up to the fourth, and u times the whole lies between them.  The draw is one of the tokens with weight, the same from both forms."""
    V, e = 6 * 4096, 2.0 ** -54
    target = torch.zeros(1, V)
    for at, p in ((7, 0.5), (4096 + 5, e), (3 * 4096 + 6, e), (5 * 4096 + 8, 0.5)):
        target[0, at] = p
    _, token, _ = verified(dict(target=target, tokens=i32([0]), uniform=torch.tensor([0.5]), qstart=i32([0]), qlen=i32([1])), 1)
    assert token == [5 * 4096 + 8]


def test_the_last_tokens_of_the_largest_vocabulary():
    """0x7fff0000 tokens, the most that a call takes: the last part ends past 2^31 if it is whole."""
    V = 0x7FFF0000
    target = torch.zeros(1, V, dtype=torch.bfloat16, device=DEV)
    target[0, V - 1] = 0.75
    got = ops.draft.verify(target, i32([0], DEV), torch.tensor([0.5], device=DEV), i32([0], DEV), i32([1], DEV), 1)
    assert [t.tolist() for t in got] == [[0], [V - 1], [[0]]]


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("what", ["no column in the tables", "no block in the pool"])
def test_no_key_at_all_gives_rows_of_zeros(eight, d, what):
    """Rows of the sequences become zero, rows behind the last one stay what they were, as in the CPU form."""
    s = step([(5, 40), (1, 3), (0, 0), (70, 90)], 8, 2, d, eight, "tree", 5, pad=3)
    if what.startswith("no column"):
        s["table"] = s["table"][:, :0].contiguous()
    else:
        for t in ("k", "v", "ks", "vs"):
            s[t] = None if s[t] is None else s[t][:0]
    for mask in (s["mask"], None):
        outs = []
        for h in (dict(s, mask=mask), to(dict(s, mask=mask), DEV)):
            out = torch.full((79, 8, d), 7.0, dtype=torch.bfloat16, device=h["q"].device)
            attend(h, out=out)
            assert not attend(h)[:76].any()
            outs.append(out.cpu())
        assert torch.equal(*outs) and not outs[1][:76].any() and bool((outs[1][76:] == 7.0).all())


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("seqs", [[(40, 1190), (3, 37)], [(5, 1190), (3, 37)], [(1, 1190), (1, 37)]])
def test_an_infinity_beside_a_page_outside_the_pool(eight, d, seqs):
    """V of a committed key whose chunk lacks a page, long before the drafted ones: every row of the sequence gets it, no other row does; a NaN of a
    drafted key reaches its own branch alone."""
    s = step(seqs, 8, 2, d, eight, "tree", 23)
    n, c = seqs[0]
    see = [visible(s, b) for b in range(2)]
    see[0][:, 16 * BS:17 * BS] = False
    want, bound = attention64(s, see)
    s["table"][0, 16] = -5
    page, off = int(s["table"][0, 17]), 3                       # key 275, at dim 9
    s["v"].view(torch.uint8 if eight else torch.bfloat16)[page, :, 9, off] = 0x7F if eight else -math.inf
    got = attend(to(s, DEV)).cpu()
    hit = got[:n, :, 9].float()
    assert bool((hit.isnan() if eight else hit == -math.inf).all())
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[:n, :, 9] = False
    assert bool(((got.double() - want).abs() <= bound)[rest].all())
    if n < 2:
        return
    at = c - 1                                                  # the last node: no node is behind it
    page, off = int(s["table"][0, at // BS]), at % BS
    s["v"].view(torch.uint8 if eight else torch.bfloat16)[page, :, 20, off] = 0x7F if eight else math.nan
    got = attend(to(s, DEV)).cpu()
    assert got[n - 1, :, 20].isnan().all()
    rest[n - 1, :, 20] = False
    assert bool(((got.double() - want).abs() <= bound)[rest].all())


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("nodes", [1, 12, 40])
def test_a_nan_of_a_drafted_token_does_not_hold_up_the_batch(eight, nodes):
    """One broken sequence of 30000 keys: what is looked at again are its drafted keys, not its context (that took 40 times a call's time and more; four
    times are allowed here)."""
    s = to(step([(nodes, 30000), (nodes, 900), (nodes, 77)], 8, 2, 128, eight, "tree", 24), DEV)

    def time():
        took = []
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            attend(s, max_qlen=nodes)
            b.record()
            torch.cuda.synchronize()
            took.append(a.elapsed_time(b))
        return sorted(took)[3]
    clean = time()
    page, off = int(s["table"][0, 29999 // BS]), 29999 % BS
    s["v"].view(torch.uint8 if eight else torch.bfloat16)[page, :, :, off] = 0x7F if eight else math.nan
    broken = time()
    assert broken < 4 * clean, f"{1e3 * clean:.0f} us, with a NaN {1e3 * broken:.0f}"


def heads_at_once(s):
    """``attention64`` for many sequences: the same definition and bound, all heads of a sequence in one product."""
    T, nq, d = s["q"].shape
    out, bound = torch.zeros(T, nq, d, dtype=torch.float64), torch.zeros(T, nq, d, dtype=torch.float64)
    for b in range(s["table"].shape[0]):
        q0, n, c = int(s["qstart"][b]), int(s["qlen"][b]), int(s["ctx"][b])
        k, v = dense(s, b)
        x = s["q"][q0:q0 + n].double().transpose(0, 1).reshape(k.shape[0], -1, d)                # [nkv, G n, d]
        hidden = ~visible(s, b).repeat(nq // k.shape[0], 1)
        w = torch.softmax((x @ k.transpose(1, 2) / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
        ds = (d + 3) * 2.0 ** -24 * (x.abs() @ k.abs().transpose(1, 2) / math.sqrt(d)).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
        e = (2.0 ** -8 + 2 * ds + (2 * c + 16) * 2.0 ** -24) * (w @ v.abs())
        for to, x in ((out, w @ v), (bound, e + 2.0 ** -8 * ((w @ v).abs() + e) + 1e-30)):
            to[q0:q0 + n] = x.view(nq, n, d).transpose(0, 1)
    return out, bound


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("batch,nodes", [(75, 12), (90, 1), (90, 12)])
def test_many_short_contexts(eight, batch, nodes):
    """Below and above the number of row blocks from which contexts of up to 512 keys are cut, lengths of their own; with the longest ones given and without."""
    rng = random.Random(batch)
    s = step([(min(nodes, c), c) for c in (rng.randrange(1, 512) for _ in range(batch))], 64, 32, 64, eight, "tree", 25)
    want, bound = heads_at_once(s)
    h = to(s, DEV)
    for kw in ({}, dict(max_qlen=nodes, max_ctx=511)):
        got = attend(h, **kw)
        assert bool(((got.double().cpu() - want).abs() <= bound).all())
        assert torch.equal(got, attend(h, **kw))


@pytest.mark.parametrize("d,hint", [(64, 0), (64, 9), (128, 9), (96, 0)])
def test_every_part_longer_than_its_window_of_pages(d, hint):
    """430 sequences of 20000 keys, each with an order of pages of its own: a workgroup's part passes 16384 keys of one row block, from a context's first
    key on or from inside it, and its pages are looked up again on the way.  All rows are compared; then with two pages of every sequence outside the
    pool, most of them past a window's first 1024.  Bounds as attention64's."""
    n, ctx, qlen, blocks = 430, 20000, 9, 1250
    s = to(step([(qlen, ctx)], 4, 1, d, False, "chain", 18), DEV)
    g = torch.Generator().manual_seed(2)
    s["q"] = (1.5 * torch.randn(n * qlen, 4, d, generator=g)).bfloat16().to(DEV)
    order = torch.stack([torch.randperm(blocks, generator=g) for _ in range(n)])
    s["table"] = s["table"][0].cpu()[order].contiguous().to(DEV)
    s["qstart"], s["qlen"], s["ctx"] = i32(list(range(0, n * qlen, qlen)), DEV), i32([qlen] * n, DEV), i32([ctx] * n, DEV)
    k, v = (s["k"][:, 0].double(), s["v"][:, 0].transpose(1, 2).double())                       # [pages, 16, d]
    see = torch.arange(ctx, device=DEV)[None] <= ctx - qlen + torch.arange(qlen, device=DEV)[:, None]
    away = torch.stack([torch.randint(0, blocks, (n,), generator=g), torch.randint(1024, blocks, (n,), generator=g)], 1).to(DEV)
    holed = s["table"].scatter(1, away, torch.where(away % 2 == 0, -1, s["k"].shape[0]).int())
    for table in (s["table"], holed):
        got = attend(dict(s, table=table), max_qlen=hint).double()
        for b in range(n):
            pages = s["table"][b].long()
            kk, vv = k[pages].reshape(ctx, d), v[pages].reshape(ctx, d)
            seen = see & ((table[b] >= 0) & (table[b] < s["k"].shape[0])).repeat_interleave(BS)[None]
            x = s["q"][b * qlen:(b + 1) * qlen].double().transpose(0, 1)                        # [4, qlen, d]
            w = torch.softmax((x @ kk.T / math.sqrt(d)).masked_fill(~seen, -math.inf), -1)
            ds = (d + 3) * 2.0 ** -24 * (x.abs() @ kk.abs().T / math.sqrt(d)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            o = w @ vv
            e = (2.0 ** -8 + 2 * ds + (2 * ctx + 16) * 2.0 ** -24) * (w @ vv.abs())
            off = (got[b * qlen:(b + 1) * qlen].transpose(0, 1) - o).abs()
            assert bool((off <= e + 2.0 ** -8 * (o.abs() + e)).all()), b


# ------------------------------------------------------------------------------------------------ vocabularies past 4096 tokens a part
BIG = 4096 * 256 + 3


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_vocabularies_of_more_than_a_million(drawn, dtype):
    """Parts of 8192 tokens, 32 a thread, the last part of three: draws all over the vocabulary, of flat and of peaked rows."""
    g = torch.Generator().manual_seed(7)
    n = 6
    logits = 3 * torch.randn(2 * n, BIG, generator=g)
    target = torch.softmax(logits, -1)
    target[::4] = 1.0 / BIG
    draft = torch.softmax(logits + torch.randn(2 * n, BIG, generator=g), -1) if drawn else None
    tokens = torch.multinomial(target, 1, generator=g)[:, 0].int()
    u = torch.rand(2 * n, generator=g)
    u[::2] = (torch.arange(n) + 0.37) / n                       # the roots': the next token's
    s = dict(target=target.to(dtype), tokens=tokens, uniform=u, qstart=i32(list(range(0, 2 * n, 2))), qlen=i32([2] * n),
             draft=None if draft is None else draft.to(dtype))
    _, token, _ = verified(s, 2)
    assert len(set(token)) == n


def test_tokens_at_the_ends_of_threads_and_parts():
    """One row each with all its weight in two places, the draw of the second: the first and the last sixteen of a thread's tokens, a part's ends and the
    three tokens of the last part."""
    places = [0, 15, 16, 31, 32, 8191, 8192, 8192 + 17, 100 * 8192 + 40, BIG - 4, BIG - 3, BIG - 2, BIG - 1]
    target = torch.zeros(len(places), BIG)
    for i, at in enumerate(places):
        target[i, max(at - 3, 0)], target[i, at] = 0.25, 0.5
    n = len(places)
    _, token, _ = verified(dict(target=target, tokens=i32([0] * n), uniform=torch.full((n,), 0.75), qstart=i32(list(range(n))), qlen=i32([1] * n)), 1)
    assert token == places
