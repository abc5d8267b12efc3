"""The operators that take a chunk of new tokens into the paged cache and attend
from it, at the sizes a serving loop calls them with: prompts in pieces, drafts
of a few tokens to be verified, single decode tokens, and mixes of these.

A case is a dict of plain values.  ``op`` says which operator one pass calls:

  rotate  norms of queries and keys for each head with the position rotation
          in the same pass (cvsa.ops.qk_norm_rope)
  append  keys (normed and rotated on the way) and values of new tokens
          written to the paged cache, the queries rotated in the same pass
          (cvsa.ops.append_chunk_kv)
  attend  attention of the new tokens over the paged cache
          (cvsa.ops.chunk_attention)

  q_heads, kv_heads, dim, block   shapes (bf16 caches)
  batch, new, context             sequences, most new tokens of one, most
                                  tokens that one held before
  ragged    new tokens and contexts spread from nothing to the most
  singles   sequences (the last ones) that bring one token, whatever `new` is
  dtype     type of the queries, keys and values before the cache
  rot, pairs, norm, split         rotated dimensions; rotation of neighbours
                                  (else of halves); norms taken; q, k, v are
                                  views of one projection's rows
  causal, lse                     attend: mask; log-sum-exps returned too
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SCORES = 1 << 30  # scores that the plain form holds at once


def _ops():
    pkg = os.path.join(os.getcwd(), "coverage-verified-sparse-attention_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from cvsa import ops
    return ops


def _case(name, op, **kw):
    c = dict(name=name, op=op, batch=1, q_heads=32, kv_heads=8, dim=128, block=16, new=1,
             context=0, ragged=False, singles=0, dtype="bf16", rot=128, pairs=False, norm=True,
             split=True, causal=True, lse=False)
    c.update(kw)
    return c


def listed():
    return [
        # One user's decode step: latency of the smallest call.
        _case("rotate_1", "rotate", context=8191),
        # A long prompt's projection, rows of a fused projection.
        _case("rotate_8191", "rotate", new=8191, q_heads=28, kv_heads=4),
        # Half the dimensions rotated as neighbouring pairs, no norms, a batch
        # of prompts held in fp16.
        _case("rotate_pairs_b4", "rotate", batch=4, new=2049, q_heads=64, dim=64, rot=32,
              pairs=True, norm=False, dtype="fp16", split=False),
        # One user's decode step.
        _case("append_b1", "append", context=8190),
        # A serving batch's decode step in the middle of its conversations.
        _case("append_b32", "append", batch=32, context=8185, ragged=True, singles=32),
        # Prompts of different lengths taken in together, 64-token pages.
        _case("append_b8_ragged", "append", batch=8, new=4093, q_heads=28, kv_heads=4, block=64,
              ragged=True),
        # A serving batch's decode step through the same entry point.
        _case("attend_b32_single", "attend", batch=32, context=8185, ragged=True, singles=32),
        # Drafts of five tokens to be verified against long documents.
        _case("attend_b8_draft", "attend", batch=8, new=5, context=32749, q_heads=28,
              kv_heads=4, split=False),
        # A chunk of a very long prompt.
        _case("attend_512_at_128k", "attend", new=512, context=130560),
        # The second half of a long prompt: the largest product.
        _case("attend_8k_at_8k", "attend", new=8192, context=8192),
        # Decode steps of most sequences with one prompt's chunk among them.
        _case("attend_mixed", "attend", batch=32, new=2041, context=8185, ragged=True,
              singles=31),
        # Prompts of different lengths, small heads, 64-token pages, log-sum-exps
        # kept for a later merge.
        _case("attend_b8_ragged", "attend", batch=8, new=4093, q_heads=64, dim=64, block=64,
              ragged=True, lse=True),
    ]


# Bounds of a drawn case: multiply-adds of its scores over all query heads
# (half of the largest listed case's), cache elements, and elements of q.
_DRAW_SCORES = 1 << 38
_DRAW_CACHE = 1 << 28
_DRAW_ROWS = 1 << 25


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["rotate", "append", "attend", "attend"])
    kv = rng.choice([1, 2, 3, 4, 8, 8, 16])
    group = rng.choice([1, 2, 4, 4, 5, 7, 8, 16])
    dim = rng.choice([32, 64, 128, 128, 128, 256])
    batch = _log_uniform(rng, 1, 32)
    heads = kv * group
    new = min(_log_uniform(rng, 1, 8192), _DRAW_ROWS // (batch * heads * dim) or 1)
    context = min(_log_uniform(rng, 1, 131072), _DRAW_CACHE // (batch * kv * dim))
    if op == "append":
        context = min(context, 8192)  # tokens before the chunk are not read
    if op == "attend":
        new = max(1, min(new, _DRAW_SCORES // (batch * heads * dim * (context + new))))
    singles = rng.randint(0, batch) if rng.random() < 0.3 else 0
    c = _case("", op, batch=batch, q_heads=heads, kv_heads=kv, dim=dim,
              block=rng.choice([8, 16, 16, 16, 32, 64, 128]), new=new, context=context,
              ragged=batch > 1 and rng.random() < 0.6, singles=singles,
              split=rng.random() < 0.5)
    if op != "attend":
        c["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c["rot"] = rng.choice([r for r in (16, 32, 64, 128, 256) if r <= dim])
        c["pairs"] = rng.random() < 0.3
        c["norm"] = rng.random() < 0.6
    else:
        c["causal"] = rng.random() < 0.8
        c["lse"] = rng.random() < 0.3
    return c


def _lengths(case):
    """(new tokens, tokens before) of each sequence."""
    B, n, ctx = case["batch"], case["new"], case["context"]
    news, before = [], []
    for i in range(B):
        f = (i * 2654435761 % 4294967296) / 4294967296  # 0 for the first
        if not case["ragged"]:
            f = 0.0
        single = i >= B - case["singles"]
        # the first sequence is the longest; the others spread down to nothing
        news.append(1 if single else n - int(n * f))
        before.append(ctx - int(ctx * f))
    return news, before


class _State:
    pass


def _inputs(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32)

    s = _State()
    s.case = case
    s.news, s.before = _lengths(case)
    T = sum(s.news)
    Hq, Hk, D, bs = case["q_heads"], case["kv_heads"], case["dim"], case["block"]
    dt = _DTYPES[case["dtype"]]
    # Projections have channels of unlike size; in attention some heads are
    # flat and some look at few keys.
    chan = torch.exp(0.4 * normal(D))
    q, k, v = normal(T, Hq, D), normal(T, Hk, D), normal(T, Hk, D)
    if case["op"] == "attend":
        q *= torch.linspace(0.5, 3.0, Hq, device=dev)[:, None]
    else:
        q *= chan
        k *= chan
    if case["split"]:
        rows = torch.cat([q, k, v], 1).to(dt)
        s.q, s.k, s.v = rows[:, :Hq], rows[:, Hq:Hq + Hk], rows[:, Hq + Hk:]
    else:
        s.q, s.k, s.v = q.to(dt), k.to(dt), v.to(dt)
    if case["op"] != "attend":
        R = case["rot"]
        P = max(b + n for b, n in zip(s.before, s.news))
        freq = 500000.0 ** (-torch.arange(0, R, 2, device=dev, dtype=torch.float64) / R)
        ang = torch.arange(P, device=dev, dtype=torch.float64)[:, None] * freq
        s.table = torch.cat([ang.cos(), ang.sin()], 1).to(torch.float32)
        s.q_weight = s.k_weight = None
        if case["norm"]:
            s.q_weight = (1 + 0.2 * normal(D)).to(torch.bfloat16)
            s.k_weight = (1 + 0.2 * normal(D)).to(torch.bfloat16)
        s.positions = torch.cat([torch.arange(b, b + n, device=dev, dtype=torch.int32)
                                 for b, n in zip(s.before, s.news)])
    if case["op"] != "rotate":
        totals = [b + n for b, n in zip(s.before, s.news)]
        pages = [-(-t // bs) for t in totals]
        blocks = sum(pages) + 3
        W = max(pages)
        perm = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
        s.block_tables = torch.zeros(len(pages), W, dtype=torch.int32, device=dev)
        at = 0
        for b, p in enumerate(pages):
            s.block_tables[b, :p] = perm[at:at + p]
            at += p
        s.context_lens = torch.tensor(totals, dtype=torch.int32, device=dev)
        # Values share a mean for each channel, so that outputs keep a size
        # when many keys are averaged.
        s.k_cache = normal(blocks, bs, Hk, D).to(torch.bfloat16)
        s.v_cache = (normal(blocks, bs, Hk, D) + normal(Hk, D)).to(torch.bfloat16)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        ops = _ops()
        if case["op"] != "attend":
            s.rotary = ops.RotaryTable(s.table, interleaved=case["pairs"])
        if case["op"] != "rotate":
            s.layout = ops.ChunkLayout(s.news, s.q.device)
    return s


def run(s):
    if not own:
        return _PLAIN[s.case["op"]](s)
    ops, case = _ops(), s.case
    if case["op"] == "rotate":
        return ops.qk_norm_rope(s.q, s.k, s.positions, s.rotary, q_weight=s.q_weight,
                                k_weight=s.k_weight, eps=EPS)
    if case["op"] == "append":
        q = ops.append_chunk_kv(s.k, s.v, s.k_cache, s.v_cache, s.block_tables, s.context_lens,
                                s.layout, case["block"], rotary=s.rotary, k_weight=s.k_weight,
                                q=s.q, q_weight=s.q_weight, eps=EPS)
        return q, s.k_cache, s.v_cache
    return ops.chunk_attention(s.q, s.k_cache, s.v_cache, s.block_tables, s.context_lens,
                               s.layout, case["kv_heads"], case["q_heads"] // case["kv_heads"],
                               case["block"], causal=case["causal"], return_lse=case["lse"])


# ------------------------------------------------------------ plain forms

def _plain_rotated(x, weight, positions, table, pairs):
    """One side's norm and rotation in 32 bits, rounded at the end."""
    y = x.to(torch.float32)
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.to(torch.float32)
    rows = table[positions.long()]
    half = rows.shape[1] // 2
    cos, sin = rows[:, None, :half], rows[:, None, half:]
    if pairs:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, y[..., 2 * half:]], -1)


def _plain_rotate(s):
    pairs = s.case["pairs"]
    return (_plain_rotated(s.q, s.q_weight, s.positions, s.table, pairs).to(s.q.dtype),
            _plain_rotated(s.k, s.k_weight, s.positions, s.table, pairs).to(s.k.dtype))


def _plain_append(s):
    bs, dev = s.case["block"], s.q.device
    news = torch.tensor(s.news, device=dev)
    seq = torch.repeat_interleave(torch.arange(len(s.news), device=dev), news)
    first = torch.cumsum(news, 0) - news
    pos = torch.arange(seq.numel(), device=dev) - first[seq] + (s.context_lens - news)[seq]
    slot = s.block_tables[seq, pos // bs].long() * bs + pos % bs
    k = _plain_rotated(s.k, s.k_weight, pos, s.table, s.case["pairs"])
    s.k_cache.view(-1, *s.k_cache.shape[2:])[slot] = k.to(torch.bfloat16)
    s.v_cache.view(-1, *s.v_cache.shape[2:])[slot] = s.v.to(torch.bfloat16)
    q = _plain_rotated(s.q, s.q_weight, pos, s.table, s.case["pairs"])
    return q.to(s.q.dtype), s.k_cache, s.v_cache


def _plain_attend(s):
    case = s.case
    Hk, D = case["kv_heads"], case["dim"]
    G = case["q_heads"] // Hk
    out = torch.empty(s.q.shape, dtype=s.q.dtype, device=s.q.device)
    lse = torch.empty(s.q.shape[:2], dtype=torch.float32, device=s.q.device)
    at = 0
    for b, (n, before) in enumerate(zip(s.news, s.before)):
        if n == 0:
            continue
        ctx = before + n
        pages = s.block_tables[b, :-(-ctx // case["block"])].long()
        k = s.k_cache[pages].flatten(0, 1)[:ctx].permute(1, 2, 0).to(torch.float32).contiguous()
        v = s.v_cache[pages].flatten(0, 1)[:ctx].permute(1, 0, 2).to(torch.float32).contiguous()
        q = s.q[at:at + n].view(n, Hk, G, D).permute(1, 0, 2, 3).reshape(Hk, n * G, D)
        q = q.to(torch.float32) * D ** -0.5
        hidden = None
        if case["causal"] and n > 1:
            row = torch.arange(n, device=q.device).repeat_interleave(G)
            hidden = torch.arange(ctx, device=q.device)[None] > (before + row)[:, None]
        step = max(1, _SCORES // (n * G * ctx))
        for h in range(0, Hk, step):
            x = q[h:h + step] @ k[h:h + step]
            if hidden is not None:
                x.masked_fill_(hidden, -math.inf)
            m = x.amax(-1, keepdim=True)
            p = torch.exp(x.sub_(m))
            l = p.sum(-1, keepdim=True)
            o = (p @ v[h:h + step]) / l
            h2 = min(h + step, Hk)
            out[at:at + n, h * G:h2 * G] = (o.view(h2 - h, n, G, D).permute(1, 0, 2, 3)
                                            .reshape(n, -1, D).to(out.dtype))
            lse[at:at + n, h * G:h2 * G] = ((m + torch.log(l)).view(h2 - h, n, G)
                                            .permute(1, 0, 2).reshape(n, -1))
        at += n
    return (out, lse) if case["lse"] else out


_PLAIN = {"rotate": _plain_rotate, "append": _plain_append, "attend": _plain_attend}


# ------------------------------------------------------------ in 64 bits

def _exact_rotated(x, weight, positions, table, pairs):
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    R = table.shape[1]
    t = table.double()[positions.long()]
    # The rotation as a product of complex numbers.
    turn = torch.complex(t[:, :R // 2], t[:, R // 2:])[:, None]
    y = x.clone()
    if pairs:
        z = torch.complex(x[..., 0:R:2].contiguous(), x[..., 1:R:2].contiguous()) * turn
        y[..., 0:R:2], y[..., 1:R:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :R // 2].contiguous(), x[..., R // 2:R].contiguous()) * turn
        y[..., :R // 2], y[..., R // 2:R] = z.real, z.imag
    return y


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] != "attend":
        q = _exact_rotated(s.q, s.q_weight, s.positions, s.table, case["pairs"])
        k = _exact_rotated(s.k, s.k_weight, s.positions, s.table, case["pairs"])
        if case["op"] == "rotate":
            return q, k
        kc, vc = s.k_cache.double(), s.v_cache.double()
        bs, at = case["block"], 0
        for b, (n, before) in enumerate(zip(s.news, s.before)):
            pos = torch.arange(before, before + n, device=q.device)
            block = s.block_tables[b].long()[pos // bs]
            kc[block, pos % bs] = k[at:at + n]
            vc[block, pos % bs] = s.v[at:at + n].double()
            at += n
        return q, kc, vc
    Hk, D, bs = case["kv_heads"], case["dim"], case["block"]
    G = case["q_heads"] // Hk
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=s.q.device)
    lse = torch.full(s.q.shape[:2], -math.inf, dtype=torch.float64, device=s.q.device)
    at = 0
    for b, (n, before) in enumerate(zip(s.news, s.before)):
        pos = torch.arange(before + n, device=s.q.device)
        block = s.block_tables[b].long()[pos // bs]
        for h in range(Hk):
            k = s.k_cache[block, pos % bs, h].double()
            v = s.v_cache[block, pos % bs, h].double()
            for i in range(0, n, 1024):
                j = min(i + 1024, n)
                q = s.q[at + i:at + j, h * G:(h + 1) * G].double().reshape(-1, D)
                x = q @ k.t() / math.sqrt(D)
                if case["causal"]:
                    own_pos = pos[before + i:before + j].repeat_interleave(G)
                    x = torch.where(pos[None] <= own_pos[:, None], x, -math.inf)
                total = torch.logsumexp(x, -1, keepdim=True)
                o = torch.exp(x - total) @ v
                out[at + i:at + j, h * G:(h + 1) * G] = o.view(j - i, G, D)
                lse[at + i:at + j, h * G:(h + 1) * G] = total.view(j - i, G)
        at += n
    return (out, lse) if case["lse"] else out


# ------------------------------------------------------------------ work

def work(case):
    news, before = _lengths(case)
    T = sum(news)
    Hq, Hk, D, bs = case["q_heads"], case["kv_heads"], case["dim"], case["block"]
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attend":
        pairs = 0
        keys = 0
        for n, b in zip(news, before):
            if n:
                keys += b + n
                pairs += n * b + (n * (n + 1) // 2 if case["causal"] else n * n)
        nbytes = 4 * T * Hq * D + 4 * keys * Hk * D + 4 * sum(-(-(b + n) // bs) for n, b in
                                                              zip(news, before) if n)
        if case["lse"]:
            nbytes += 4 * T * Hq
        # two products of D multiply-adds and an exponential for each pair
        return {"bytes": nbytes, "flops": pairs * Hq * (4 * D + 4)}
    rot_rows = max((b + n for b, n in zip(before, news)), default=0)
    rot_rows = min(rot_rows, T)  # the table's rows that the tokens use
    nbytes = 4 * case["rot"] * rot_rows + 4 * T
    nbytes += 2 * e * T * Hq * D + (e * T * Hk * D if case["op"] == "rotate" else 0)
    nbytes += e * T * Hk * D
    if case["op"] == "append":
        nbytes += e * T * Hk * D + 4 * T * Hk * D
    flops = T * (Hq + Hk) * (3 * case["rot"] + (4 * D if case["norm"] else 0))
    return {"bytes": nbytes, "flops": flops}
