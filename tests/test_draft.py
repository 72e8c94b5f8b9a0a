"""Drafted tokens and the 8-bit cache: definitions, refusals and a whole step, on the CPU and (marked) on the GPU."""
import math
import random

import pytest
import torch

from distributed_llm_amd import ops
from distributed_llm_amd.ops import reference as ref
from draft_cases import BS, attend, attention64, i32, step, to, tree, visible

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
SEQS = [(5, 40), (0, 7), (3, 3), (1, 1), (12, 300)]


@pytest.mark.parametrize("mode", ["chain", "tree"])
@pytest.mark.parametrize("eight", [False, True])
def test_attention_is_its_definition(eight, mode):
    s = step(SEQS, 6, 2, 64, eight, mode, 1)
    want, bound = attention64(s)
    assert bool(((attend(s).double() - want).abs() <= bound).all())


def test_tree_mask_is_the_walk_up():
    rng = random.Random(0)
    lens = [1, 70, 0, 33]
    par = i32(sum([tree(rng, n) for n in lens], []) + [5, 5])
    s = {"qstart": i32([0, 1, 71, 71]), "qlen": i32(lens), "ctx": i32(lens), "parents": par}
    mask, depth = ops.draft.tree_mask(par, s["qstart"], s["qlen"], 70)
    assert mask.shape == (106, 3)
    for b, n in enumerate(lens):
        see = visible(s, b)
        q0 = int(s["qstart"][b])
        for i in range(n):
            bits = [(int(mask[q0 + i, j // 32]) >> (j % 32)) & 1 for j in range(n)]
            assert bits == see[i].int().tolist()
            assert int(depth[q0 + i]) == sum(bits) - 1
    assert not mask[104:].any() and not depth[104:].any()


def test_pages_outside_the_pool_are_not_seen():
    s = step([(4, 50), (2, 20)], 4, 2, 64, False, "tree", 3)
    s["table"][0, 1], s["table"][1, 1] = 10 ** 6, -7
    see = [visible(s, 0), visible(s, 1)]
    see[0][:, 16:32] = False
    see[1][:, 16:] = False
    got = attend(s)
    s["table"][0, 1] = s["table"][1, 1] = 0
    want, bound = attention64(s, see)
    assert bool(((got.double() - want).abs() <= bound).all())


def test_codes_are_nearest_and_even():
    """Against a table of the 127 magnitudes: 448 x / top at ties and beside them."""
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2
    x = torch.cat([codes, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20), torch.tensor([448.0])]).float()
    got, scale = ref.kv8_quantise(torch.cat([x, -x])[None])
    assert float(scale) == 1.0
    near = (x.double()[:, None] - codes).abs()
    best = near.amin(1, keepdim=True)
    want = torch.stack([c[c % 2 == 0][0] if len(c) > 1 else c[0] for c in ((row == b).nonzero()[:, 0] for row, b in zip(near, best))])
    assert torch.equal(got[0, :x.numel()].long(), want)
    value = got.view(torch.float8_e4m3fn).double()[0]
    assert torch.equal(value[:x.numel()], -value[x.numel():])


@pytest.mark.parametrize("top", [0.0, 1e-38, 2.0 ** -101, 3e38])
def test_vectors_at_the_ends_of_the_range(top):
    """A code is within half a step of it (2^-4 of the value, 2^-10 below the smallest normal) of what the scale makes it."""
    x = (torch.linspace(-1, 1, 64) * top).bfloat16().float()
    code, scale = ref.kv8_quantise(x)
    got = code.view(torch.float8_e4m3fn).double() * scale.double()
    bound = torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * scale.double()) * (1 + 2.0 ** -20)
    assert bool(((got - x.double()).abs() <= bound).all())


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_vector_that_is_not_finite_reads_back_as_nan(bad):
    cache = ops.kv8.alloc(2, 1, 16)
    k, v = torch.ones(2, 1, 16).bfloat16(), torch.ones(2, 1, 16).bfloat16()
    k[0, 0, 3] = bad
    ops.kv8.write(k, v, i32([5, 20]), cache)
    rk, rv = ops.kv8.read(cache, i32([5, 20]))
    assert rk[0].isnan().all() and torch.equal(rk[1], k[1]) and torch.equal(rv, v)


@pytest.mark.parametrize("kind", ["drawn", "given", "tree"])
def test_tokens_are_distributed_as_the_targets(kind):
    """The two tokens after a root over 40000 steps of a vocabulary of 5, against the target's joint probabilities: counts are within five of their own
    standard deviations, sqrt(n p (1 - p)), and one."""
    n, V = 40000, 5
    g = torch.Generator().manual_seed(4)
    first, second = torch.softmax(torch.randn(V, generator=g), 0), torch.softmax(1.5 * torch.randn(V, V, generator=g), -1)
    drafts = torch.softmax(torch.randn(V, generator=g), 0)
    nodes = 2 if kind != "tree" else 4
    tok = torch.zeros(n, nodes, dtype=torch.int64)
    par = None
    if kind == "tree":
        tok[:, 1:] = torch.stack([torch.randperm(V, generator=g)[:3] for _ in range(n)])
        par = i32([-1, 0, 0, 0] * n)
    elif kind == "given":
        tok[:, 1] = torch.randint(0, V, (n,), generator=g)
    else:
        tok[:, 1] = torch.multinomial(drafts.expand(n, V), 1, generator=g)[:, 0]
    target = second[tok]
    target[:, 0] = first
    q = drafts.expand(n * nodes, V).contiguous() if kind == "drawn" else None
    u = torch.rand(n, nodes, generator=g)
    acc = torch.zeros(n, dtype=torch.int32)
    nxt, path = acc.clone(), torch.zeros(n, nodes, dtype=torch.int32)
    for i in range(0, n, 20000):
        rows = slice(i * nodes, (i + 20000) * nodes)
        got = ops.draft.verify(target.view(-1, V)[rows].contiguous(), tok.view(-1)[rows].int(), u.view(-1)[rows].contiguous(),
                               i32(list(range(0, 20000 * nodes, nodes))), i32([nodes] * 20000), nodes, parents=None if par is None else par[rows],
                               draft=None if q is None else q[rows])
        acc[i:i + 20000], nxt[i:i + 20000], path[i:i + 20000] = got
    one = torch.where(acc > 0, tok.gather(1, path[:, 1].clamp_min(0).long()[:, None])[:, 0], nxt.long())
    count = torch.bincount(one, minlength=V).double()
    assert bool(((count - n * first.double()).abs() <= 5 * (n * first * (1 - first)).double().sqrt() + 1).all())
    both = torch.zeros(V, V)
    took = acc > 0
    both.index_put_((one[took], nxt[took].long()), torch.ones(int(took.sum())), accumulate=True)
    per = both.sum(1, keepdim=True).double()
    assert bool(((both - per * second).abs() <= 5 * (per * second * (1 - second)).sqrt() + 1).all())


def test_verify_at_the_ends():
    """Nothing above the draft: the target itself; no probability at all: token 0; u = 1 and infinities: the last token with weight; NaN: none."""
    V = 6
    p = torch.tensor([0.1, 0.2, 0.3, 0.4, 0.0, 0.0])
    same = ops.draft.verify(torch.stack([p, p]), i32([0, 5]), torch.tensor([0.15, 0.5]), i32([0]), i32([2]), 2, draft=torch.stack([p, p]))
    assert [x.tolist() for x in same] == [[0], [1], [[0, -1]]]            # token 5 has no probability in either; 0.1 < 0.15
    none = ops.draft.verify(torch.zeros(1, V), i32([0]), torch.tensor([0.5]), i32([0]), i32([1]), 1)
    assert none[1].tolist() == [0]
    end = ops.draft.verify(p[None].contiguous(), i32([0]), torch.tensor([1.0]), i32([0]), i32([1]), 1)
    assert end[1].tolist() == [3]
    odd = torch.tensor([[0.1, math.nan, math.inf, 0.4, math.nan, 0.0]])
    assert ops.draft.verify(odd, i32([0]), torch.tensor([0.5]), i32([0]), i32([1]), 1)[1].tolist() == [3]
    empty = ops.draft.verify(p[None].contiguous(), i32([0]), torch.tensor([0.5]), i32([0, 0]), i32([0, 1]), 3)
    assert [x.tolist() for x in empty] == [[0, 0], [-1, 2], [[-1, -1, -1], [0, -1, -1]]]


# ------------------------------------------------------------------------------------------------ a whole step
class Toy:
    """One attention layer between an embedding and a head, greedy: enough for a token to hang on every key it should see and on no other."""

    def __init__(self, device, eight, V=97, nq=4, nkv=2, d=64):
        g = torch.Generator().manual_seed(11)
        self.nq, self.nkv, self.d, self.eight, self.device = nq, nkv, d, eight, device
        self.emb = torch.randn(V, (nq + 2 * nkv) * d, generator=g).bfloat16().to(device)
        self.head = (3 * torch.randn(nq * d, V, generator=g)).to(device)
        self.table = ops.rope_cos_sin(512, d, 10000.0, device)
        self.pages = torch.randperm(40, generator=g).to(torch.int32).view(2, 20).to(device)
        if eight:
            self.cache = ops.kv8.alloc(40, nkv, d, device)
        else:
            self.cache = [torch.zeros(s, dtype=torch.bfloat16, device=device) for s in ((40, nkv, BS, d), (40, nkv, d, BS))] + [None, None]

    def run(self, tokens, depth, qlen, ctx, mask, most):
        """Probabilities [T, V] after each of the new tokens, K and V of them in the cache."""
        qstart = torch.cumsum(qlen, 0).to(torch.int32) - qlen
        seq = torch.repeat_interleave(torch.arange(len(qlen), device=self.device), qlen.long())
        at = torch.arange(tokens.numel(), device=self.device) - qstart[seq] + (ctx - qlen)[seq]
        slots = (self.pages[seq, at // BS] * BS + at % BS).to(torch.int32)
        pos = ((ctx - qlen)[seq] + depth).to(torch.int32)
        qkv = self.emb[tokens.long()]
        if self.eight:
            q = ops.kv8.rope_and_cache(qkv, pos, self.table, slots, self.cache, self.nq, self.nkv, self.d)
        else:
            q = ops.rope_and_cache(qkv, pos, self.table, slots, self.cache[0], self.cache[1], self.nq, self.nkv, self.d)
        k, v, ks, vs = self.cache
        o = ops.draft.tree_attention(q, k, v, self.pages, qstart, qlen, ctx, mask, k_scale=ks, v_scale=vs, max_qlen=most)
        return torch.softmax(o.float().flatten(1) @ self.head, -1), qstart


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("eight", [False, True])
def test_speculative_steps_give_the_tokens_of_plain_ones(device, eight):
    """Prompt, then single tokens one by one; and the same answers from drafted trees that hold right and wrong candidates, verified greedily (a target of
    ones and zeros) and kept."""
    prompts = [[5, 8, 13, 21, 34], [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17]]
    new = 24
    I = lambda v: i32(v, device)  # noqa: E731

    def prefill(m):
        lens = I([len(p) for p in prompts])
        depth = torch.cat([torch.arange(len(p), device=device) for p in prompts])
        p, start = m.run(I(sum(prompts, [])), depth, lens, lens, None, 0)
        return p[(start + lens - 1).long()].argmax(-1).tolist(), [len(p) for p in prompts]

    plain = Toy(device, eight)
    last, ctx = prefill(plain)
    answers = [[t] for t in last]
    for _ in range(new):
        ctx = [c + 1 for c in ctx]
        p, _ = plain.run(I(last), I([0, 0]), I([1, 1]), I(ctx), None, 1)
        last = p.argmax(-1).tolist()
        for a, t in zip(answers, last):
            a.append(t)

    spec, rng = Toy(device, eight), random.Random(2)
    last, ctx = prefill(spec)
    got, steps, kept = [[t] for t in last], 0, 0
    while min(len(g) for g in got) < new:
        tokens, parents, lens = [], [], []
        for b in range(2):                      # wrong candidates beside the right ones, the right branch interleaved with others
            right, tok, par, at = answers[b][len(got[b]):], [last[b]], [-1], 0
            for depth in range(rng.randrange(1, 5)):
                more = depth < len(right)
                kids = [x for x in rng.sample(range(97), rng.randrange(0, 3)) if not more or x != right[depth]]
                here = at
                tok += kids
                par += [here] * len(kids)
                if more and rng.random() < 0.85:
                    at = len(tok)
                    tok.append(right[depth])
                    par.append(here)
                if at == here:
                    break
            tokens += tok
            parents += par
            lens.append(len(tok))
        most = max(lens)
        ctx = [c + n for c, n in zip(ctx, lens)]
        qlen, dctx = I(lens), I(ctx)
        qstart = torch.cumsum(qlen, 0).to(torch.int32) - qlen
        mask, depth = ops.draft.tree_mask(I(parents), qstart, qlen, most)
        p, _ = spec.run(I(tokens), depth, qlen, dctx, mask, most)
        sure = torch.nn.functional.one_hot(p.argmax(-1), p.shape[1]).float()
        acc, nxt, path = ops.draft.verify(sure, I(tokens), torch.full((len(tokens),), 0.5, device=device), qstart, qlen, most, parents=I(parents))
        k, v, ks, vs = spec.cache
        ops.draft.keep(k, v, spec.pages, qlen, dctx, path, acc, k_scale=ks, v_scale=vs)
        for b, (a, t) in enumerate(zip(acc.tolist(), nxt.tolist())):
            got[b] += [tokens[int(qstart[b]) + i] for i in path[b, 1:a + 1].tolist()] + [t]
            ctx[b] += a + 1 - lens[b]
            last[b] = t
            kept += a
        steps += 1
    for g, a in zip(got, answers):
        n = min(len(g), len(a))
        assert g[:n] == a[:n]
    assert kept >= steps


# ------------------------------------------------------------------------------------------------ refusals
def _attention_refusals(s):
    half = s["q"].half()
    yield "type of q", dict(s, q=half)
    yield "heads", dict(s, q=s["q"][:, :5].contiguous())
    yield "head_dim", dict(s, q=torch.zeros(s["q"].shape[0], 6, 80, dtype=torch.bfloat16, device=half.device))
    yield "a cache of 32-token blocks", dict(s, k=torch.zeros(4, 2, 32, 64, dtype=torch.bfloat16, device=half.device))
    yield "a cache of another type", dict(s, k=s["k"].half(), v=s["v"].half())
    yield "one scale", dict(s, ks=torch.ones(s["k"].shape[:3], device=half.device))
    yield "scales with a bf16 cache", dict(s, ks=torch.ones(s["k"].shape[:3], device=half.device), vs=torch.ones(s["k"].shape[:3], device=half.device))
    yield "a strided cache", dict(s, k=s["k"].transpose(2, 3).contiguous().transpose(2, 3))
    yield "tables", dict(s, table=s["table"].long())
    yield "lengths", dict(s, ctx=s["ctx"][:-1].contiguous())
    yield "mask's rows", dict(s, mask=s["mask"][1:].contiguous())
    yield "mask's type", dict(s, mask=s["mask"].bool())


@pytest.mark.parametrize("device", DEVICES)
def test_attention_refuses(device):
    s = to(step([(4, 20), (2, 9)], 6, 2, 64, False, "tree", 0), device)
    attend(s)
    for what, bad in _attention_refusals(s):
        with pytest.raises(ValueError):
            attend(bad)
            pytest.fail(what)
    for kw in (dict(max_qlen=-1), dict(out=s["q"]), dict(out=torch.empty_like(s["q"]).float()), dict(out=torch.empty_like(s["q"])[:-1])):
        with pytest.raises(ValueError):
            attend(s, **kw)


@pytest.mark.parametrize("device", DEVICES)
def test_verify_refuses(device):
    p, tok, u = torch.full((3, 8), 0.125, device=device), i32([0, 1, 2], device), torch.rand(3, device=device)
    a, n = i32([0], device), i32([3], device)
    ops.draft.verify(p, tok, u, a, n, 3)
    for args, kw in [((p.half(), tok, u, a, n, 3), {}), ((p, tok.long(), u, a, n, 3), {}), ((p, tok, u.double(), a, n, 3), {}), ((p, tok, u[:2], a, n, 3), {}),
                     ((p, tok, u, a, n, 0), {}), ((p, tok, u, a, n, 1025), {}), ((p, tok, u, a, i32([3, 3], device), 3), {}),
                     ((p.t(), tok, u, a, n, 3), {}), ((p, tok, u, a, n, 3), dict(parents=i32([-1, 0], device))),
                     ((p, tok, u, a, n, 3), dict(draft=p[:2])), ((p, tok, u, a, n, 3), dict(draft=p.bfloat16())),
                     ((p, tok, u, a, n, 3), dict(parents=i32([-1, 0, 0], device), draft=p))]:
        with pytest.raises(ValueError):
            ops.draft.verify(*args, **kw)
    for args in [(tok.long(), a, n, 3), (tok, a, n, 0), (tok, a, n, 2000), (tok, a, i32([], device), 3)]:
        with pytest.raises(ValueError):
            ops.draft.tree_mask(*args)


@pytest.mark.parametrize("device", DEVICES)
def test_keep_refuses(device):
    k, v = torch.zeros(2, 6, 2, 16, 64, dtype=torch.bfloat16, device=device), torch.zeros(2, 6, 2, 64, 16, dtype=torch.bfloat16, device=device)
    good = dict(k_cache=k, v_cache=v, block_tables=i32([[0, 1]], device), seq_qlen=i32([4], device), seq_ctx=i32([9], device), path=i32([[0, 2, 3, -1]], device),
                accepted=i32([2], device))
    ops.draft.keep(**good)
    for bad in [dict(k_cache=k[0, 0]), dict(v_cache=v[0]), dict(v_cache=v[:1].contiguous()), dict(k_cache=k.float()), dict(k_scale=torch.ones(2, 6, 2, 16, device=device)),
                dict(path=i32([0, 2], device)), dict(path=i32([[0], [1]], device)), dict(accepted=i32([1, 1], device)), dict(seq_qlen=good["seq_qlen"].long())]:
        with pytest.raises(ValueError):
            ops.draft.keep(**dict(good, **bad))


@pytest.mark.parametrize("device", DEVICES)
def test_kv8_refuses(device):
    c = ops.kv8.alloc(4, 2, 64, device)
    qkv, pos, cs = torch.zeros(3, 8 * 64, dtype=torch.bfloat16, device=device), i32([0, 1, 2], device), ops.rope_cos_sin(8, 64, 1e4, device)
    ops.kv8.rope_and_cache(qkv, pos, cs, pos, c, 4, 2, 64)
    for args in [(qkv.float(), pos, cs, pos, c, 4, 2, 64), (qkv, pos.long(), cs, pos, c, 4, 2, 64), (qkv, pos, cs, pos[:2], c, 4, 2, 64),
                 (qkv, pos, cs, pos, c, 5, 2, 64), (qkv, pos, cs, pos, c, 4, 1, 64), (qkv, pos, cs[:, :32].contiguous(), pos, c, 4, 2, 64),
                 (qkv, pos, cs.bfloat16(), pos, c, 4, 2, 64), (qkv, pos, cs, pos, c._replace(k_scale=c.k_scale[:3]), 4, 2, 64),
                 (qkv, pos, cs, pos, c._replace(k=c.k.view(torch.uint8)), 4, 2, 64)]:
        with pytest.raises(ValueError):
            ops.kv8.rope_and_cache(*args)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=device)
    for args in [(k.float(), k.float(), pos, c), (k, k[:2], pos, c), (k[:, :1].contiguous(), k[:, :1].contiguous(), pos, c), (k, k, pos.long(), c)]:
        with pytest.raises(ValueError):
            ops.kv8.write(*args)
    for args in [(c, pos.long()), (c, pos[None]), (c._replace(v=c.k), pos)]:
        with pytest.raises(ValueError):
            ops.kv8.read(*args)
