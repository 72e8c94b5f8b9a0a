"""Inputs, definitions in 64 bits and bounds that the tests of drafted tokens and of the 8-bit cache share."""
import math
import random

import torch

from distributed_llm_amd import ops
from distributed_llm_amd.ops import reference as ref

BS = 16


def i32(v, device="cpu"):
    return torch.tensor(v, dtype=torch.int32, device=device)


def tree(rng, n, width=3):
    """Parents of a tree: deep branches and forks."""
    return [-1 if i == 0 else i - 1 if rng.random() < 0.4 else rng.randrange(max(0, i - 2 * width), i) for i in range(n)]


def step(seqs, nq, nkv, d, eight, mode, seed, spare=3, pad=0):
    """A batch on the CPU: ``seqs`` [(new tokens, keys)], shuffled pages, K and V everywhere (stale ones in what no sequence holds), ``pad`` rows of no
    sequence behind the last one.  ``mode``: chain or tree."""
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    nb = [-(-c // BS) for _, c in seqs]
    pool = sum(nb) + spare
    perm = torch.randperm(pool, generator=g).tolist()
    table = torch.zeros(len(seqs), max(nb + [1]), dtype=torch.int32)
    at = 0
    for s, n in enumerate(nb):
        table[s, :n] = i32(perm[at:at + n])
        at += n
    lens = [q for q, _ in seqs]
    starts = [sum(lens[:i]) for i in range(len(lens))]
    T = sum(lens) + pad
    k, v = torch.randn(pool, nkv, BS, d, generator=g), torch.randn(pool, nkv, d, BS, generator=g)
    ks = vs = None
    if eight:
        ck, ks = ref.kv8_quantise(k)
        cv, vs = ref.kv8_quantise(v.transpose(2, 3))
        k, v = ck.view(torch.float8_e4m3fn), cv.transpose(2, 3).contiguous().view(torch.float8_e4m3fn)
    else:
        k, v = k.bfloat16(), v.bfloat16()
    s = dict(q=(1.5 * torch.randn(T, nq, d, generator=g)).bfloat16(), k=k, v=v, table=table, qstart=i32(starts), qlen=i32(lens), ctx=i32([c for _, c in seqs]),
             mask=None, ks=ks, vs=vs, parents=None)
    if mode == "tree":
        s["parents"] = i32(sum([tree(rng, n) for n in lens], []) + [-1] * pad)
        s["mask"] = ref.tree_mask(s["parents"], s["qstart"], s["qlen"], max(lens + [1]))[0]
    return s


def to(s, device):
    return {k: v if v is None else v.to(device) for k, v in s.items()}


def attend(s, **kw):
    return ops.draft.tree_attention(s["q"], s["k"], s["v"], s["table"], s["qstart"], s["qlen"], s["ctx"], s["mask"], k_scale=s["ks"], v_scale=s["vs"], **kw)


def dense(s, b):
    """K and V [nkv, keys, d] of sequence ``b`` in 64 bits."""
    c = int(s["ctx"][b])
    pages = s["table"][b, :-(-c // BS)].long()
    k, v = s["k"].float().double()[pages], s["v"].float().double()[pages]
    if s["ks"] is not None:
        k, v = k * s["ks"].double()[pages][..., None], v * s["vs"].double()[pages][:, :, None]
    nkv, d = k.shape[1], k.shape[3]
    return k.permute(1, 0, 2, 3).reshape(nkv, -1, d)[:, :c], v.permute(1, 0, 3, 2).reshape(nkv, -1, d)[:, :c]


def visible(s, b):
    """[new tokens, keys] of sequence ``b``, from the parents."""
    q0, n, c = int(s["qstart"][b]), int(s["qlen"][b]), int(s["ctx"][b])
    see = torch.zeros(n, c, dtype=torch.bool)
    see[:, :max(c - n, 0)] = True
    for i in range(n):
        at = i
        while at >= 0:
            if 0 <= c - n + at < c:
                see[i, c - n + at] = True
            at = at - 1 if s["parents"] is None else int(s["parents"][q0 + at])
    return see


def attention64(s, see=None):
    """(out, bound): the definition in 64 bits, and how far a bf16 result may be off it.

    Scores are sums of d exact products in f32, scaled: off by (d + 3) 2^-24 of the sum of magnitudes.  A weight e^x is off by that (to first order), by two
    units of the exponential and by half a step of bf16, 2^-8, as it enters the second product (2^-24 more with a scale); sums over n keys in f32 add n
    2^-24 of sum w |v|, and as much for the joining of parts.  The result is rounded to bf16 once, 2^-8 of itself."""
    q = s["q"].double()
    T, nq, d = q.shape
    out, bound = torch.zeros(T, nq, d, dtype=torch.float64), torch.zeros(T, nq, d, dtype=torch.float64)
    for b in range(s["table"].shape[0]):
        q0, n, c = int(s["qstart"][b]), int(s["qlen"][b]), int(s["ctx"][b])
        if n == 0 or c == 0:
            continue
        k, v = dense(s, b)
        sees = visible(s, b) if see is None else see[b]
        G = nq // k.shape[0]
        for h in range(nq):
            x, kk, vv = q[q0:q0 + n, h], k[h // G], v[h // G]
            sc = (x @ kk.T) / math.sqrt(d)
            sc = sc.masked_fill(~sees, -math.inf)
            w = torch.softmax(sc, -1)
            w = torch.where(sees.any(-1, keepdim=True), w, 0.0)
            ds = (d + 3) * 2.0 ** -24 * ((x.abs() @ kk.abs().T) / math.sqrt(d)).masked_fill(~sees, 0.0).amax(-1, keepdim=True)
            o, a = w @ vv, w @ vv.abs()
            e = (2.0 ** -8 + 2 * ds + (2 * c + 16) * 2.0 ** -24) * a
            out[q0:q0 + n, h], bound[q0:q0 + n, h] = o, e + 2.0 ** -8 * (o.abs() + e) + 1e-30
    return out, bound
