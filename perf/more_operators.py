"""The operators that keep a paged cache small: 8 bits a value, and only the
tokens that attention looks at.

A case is a dict of plain values.  ``op`` says which operator one pass calls:

  append  keys (normed and rotated on the way) and values of new tokens
          written to the 8-bit paged cache, with a scale for each page and
          head, the queries rotated in the same pass (cvsa.ops.append_chunk_kv
          with k_scales and v_scales)
  attend  attention of the new tokens over the 8-bit cache
          (cvsa.ops.chunk_attention with k_scales and v_scales)
  weigh   the attention weight that the new tokens give to each key, added to
          what the keys have (cvsa.ops.add_key_weights)
  evict   tokens of little weight taken out of the cache
          (cvsa.ops.evict_tokens)

  q_heads, kv_heads, dim, block   shapes
  bits                            of a cached value: 8, or 16 (bf16; weigh, evict)
  batch, new, context             sequences, most new tokens of one, most
                                  tokens that one held before
  ragged    new tokens and contexts spread from nothing to the most
  singles   sequences (the last ones) that bring one token, whatever `new` is
  dtype     append: type of the queries, keys and values before the cache
  rot, pairs, norm                append: rotated dimensions; rotation of
                                  neighbours (else of halves); norms taken
  split                           q, k, v are views of one projection's rows
  causal, lse                     attend: mask; log-sum-exps returned too
  window                          weigh: only the last tokens of a chunk (0: all)
  keep, sinks, recent             evict: tokens kept of a sequence, first and
                                  last ones among them
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SCORES = 1 << 29       # scores that the plain forms hold at once
_LOW, _HIGH = -110, 119  # exponents of a scale
_TOP = 448.0            # the largest 8-bit value


def _ops():
    pkg = os.path.join(os.getcwd(), "coverage-verified-sparse-attention_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from cvsa import ops
    return ops


def _case(name, op, **kw):
    c = dict(name=name, op=op, batch=1, q_heads=32, kv_heads=8, dim=128, block=16, bits=8, new=1,
             context=0, ragged=False, singles=0, dtype="bf16", rot=128, pairs=False, norm=True,
             split=True, causal=True, lse=False, window=0, keep=0, sinks=0, recent=0)
    c.update(kw)
    return c


def listed():
    return [
        # One user's decode step: latency of the smallest call.
        _case("append_b1", "append", context=8190),
        # A serving batch's decode step in the middle of its conversations.
        _case("append_b32", "append", batch=32, context=8185, ragged=True, singles=32),
        # A long prompt's projection, rows of a fused projection.
        _case("append_8191", "append", new=8191, q_heads=28, kv_heads=4),
        # A serving batch's decode step.
        _case("attend_b32_single", "attend", batch=32, context=8185, ragged=True, singles=32),
        # Drafts of five tokens to be verified against long documents.
        _case("attend_b8_draft", "attend", batch=8, new=5, context=32749, q_heads=28,
              kv_heads=4, block=64, split=False),
        # A chunk of a very long prompt.
        _case("attend_512_at_128k", "attend", new=512, context=130560),
        # The second half of a long prompt, log-sum-exps kept for the weights:
        # the largest product.
        _case("attend_8k_at_8k", "attend", new=8192, context=8192, lse=True),
        # A serving batch's decode step keeps account of its keys.
        _case("weigh_b32_single", "weigh", batch=32, context=8185, ragged=True, singles=32),
        # A prompt's last tokens choose among its keys before it is cut.
        _case("weigh_window_32k", "weigh", bits=16, new=2048, context=30720, window=64),
        # Every token of a prompt counts.
        _case("weigh_4k", "weigh", new=4096),
        # A serving batch after 64 steps: back to 4096 tokens each.
        _case("evict_b32_64", "evict", batch=32, context=4160, keep=4096, sinks=4, recent=256),
        # A very long prompt cut to an eighth.
        _case("evict_128k", "evict", bits=16, context=131072, keep=16384, sinks=4, recent=1024),
    ]


# Bounds of a drawn case: multiply-adds of its scores over all query heads
# (a half of the largest listed case's), cache elements, and elements of q.
_DRAW_SCORES = 1 << 38
_DRAW_CACHE = 1 << 28
_DRAW_ROWS = 1 << 25


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "weigh", "evict"])
    kv = rng.choice([1, 2, 3, 4, 8, 8, 16])
    group = rng.choice([1, 2, 4, 4, 5, 7, 8, 16])
    dim = rng.choice([32, 64, 128, 128, 128, 256])
    batch = _log_uniform(rng, 1, 32)
    heads = kv * group
    new = min(_log_uniform(rng, 1, 8192), _DRAW_ROWS // (batch * heads * dim) or 1)
    context = min(_log_uniform(rng, 1, 131072), _DRAW_CACHE // (batch * kv * dim))
    if op == "append":
        context = min(context, 8192)  # tokens before a chunk's first page are not read
    if op == "evict":
        new = 1
        context = max(context, 64)
    if op in ("attend", "weigh"):
        new = max(1, min(new, _DRAW_SCORES // (batch * heads * dim * (context + new))))
    singles = rng.randint(0, batch) if rng.random() < 0.3 else 0
    c = _case("", op, batch=batch, q_heads=heads, kv_heads=kv, dim=dim,
              block=rng.choice([8, 16, 16, 16, 32, 64, 128]), new=new, context=context,
              ragged=batch > 1 and rng.random() < 0.6, singles=singles,
              split=rng.random() < 0.5)
    if op == "append":
        c["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c["rot"] = rng.choice([r for r in (16, 32, 64, 128, 256) if r <= dim])
        c["pairs"] = rng.random() < 0.3
        c["norm"] = rng.random() < 0.6
    elif op == "attend":
        c["causal"] = rng.random() < 0.8
        c["lse"] = rng.random() < 0.3
    else:
        c["bits"] = rng.choice([8, 8, 16])
    if op == "weigh":
        c["causal"] = rng.random() < 0.8
        if rng.random() < 0.5:
            c["window"] = _log_uniform(rng, 1, new)
    if op == "evict":
        c["keep"] = _log_uniform(rng, max(8, context // 16), context)
        c["sinks"] = rng.randint(0, min(8, c["keep"] // 4))
        c["recent"] = rng.randint(0, min(1024, c["keep"] // 2))
    return c


def _lengths(case):
    """(new tokens, tokens before) of each sequence."""
    B, n, ctx = case["batch"], case["new"], case["context"]
    if case["op"] == "evict":
        n = 0  # all of them are there already
    news, before = [], []
    for i in range(B):
        f = (i * 2654435761 % 4294967296) / 4294967296  # 0 for the first
        if not case["ragged"]:
            f = 0.0
        single = i >= B - case["singles"] and n > 0
        # the first sequence is the longest; the others spread down to nothing
        news.append(1 if single else n - int(n * f))
        before.append(ctx - int(ctx * f))
    return news, before


class _State:
    pass


def _page_exponents(top):
    """Smallest exponents e with top <= 448 * 2^e."""
    m, x = torch.frexp(top)
    e = torch.where(m <= 0.875, x - 9, x - 8)  # 448 = 0.875 * 2^9
    return torch.where(top > 0, e, _LOW).clamp(_LOW, _HIGH)


def _held_in_8_bits(x):
    """(payload, scales) of pages [blocks, block, heads, D]."""
    e = _page_exponents(x.abs().amax((1, 3)))
    y = torch.ldexp(x, -e[:, None, :, None]).to(torch.float8_e4m3fn)
    return y, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _scale(scales):
    """Scales as 32-bit numbers."""
    return torch.exp2(scales.view(torch.uint8).to(torch.float32) - 127)


def _inputs(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32)

    s = _State()
    s.case = case
    s.news, s.before = _lengths(case)
    op, T = case["op"], sum(s.news)
    Hq, Hk, D, bs = case["q_heads"], case["kv_heads"], case["dim"], case["block"]
    # Channels of unlike size, as projections have them.
    chan = torch.exp(0.4 * normal(D))
    if op != "evict":
        q, k, v = normal(T, Hq, D), normal(T, Hk, D), normal(T, Hk, D)
        if op == "append":
            q *= chan
            k *= chan
        else:
            # Some heads are flat and some look at few keys.
            q *= torch.linspace(0.5, 3.0, Hq, device=dev)[:, None] / chan
        dt = _DTYPES[case["dtype"]]
        if case["split"]:
            rows = torch.cat([q, k, v], 1).to(dt)
            s.q, s.k, s.v = rows[:, :Hq], rows[:, Hq:Hq + Hk], rows[:, Hq + Hk:]
        else:
            s.q, s.k, s.v = q.to(dt), k.to(dt), v.to(dt)
    totals = [b + n for b, n in zip(s.before, s.news)]
    if op == "append":
        R, P = case["rot"], max(totals)
        freq = 500000.0 ** (-torch.arange(0, R, 2, device=dev, dtype=torch.float64) / R)
        ang = torch.arange(P, device=dev, dtype=torch.float64)[:, None] * freq
        s.table = torch.cat([ang.cos(), ang.sin()], 1).to(torch.float32)
        s.q_weight = s.k_weight = None
        if case["norm"]:
            s.q_weight = (1 + 0.2 * normal(D)).to(torch.bfloat16)
            s.k_weight = (1 + 0.2 * normal(D)).to(torch.bfloat16)
    pages = [-(-t // bs) for t in totals]
    blocks, W = sum(pages) + 3, max(pages)
    perm = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
    s.block_tables = torch.zeros(len(pages), W, dtype=torch.int32, device=dev)
    at = 0
    for b, p in enumerate(pages):
        s.block_tables[b, :p] = perm[at:at + p]
        at += p
    s.context_lens = torch.tensor(totals, dtype=torch.int32, device=dev)
    # Keys of each page are of their own size, so that scales differ.  Values
    # share a mean for each channel, so that outputs keep a size when many keys
    # are averaged.
    k_cache = normal(blocks, bs, Hk, D) * chan * torch.exp(0.3 * normal(blocks, 1, Hk, 1))
    v_cache = normal(blocks, bs, Hk, D) + normal(Hk, D)
    s.k_scales = s.v_scales = None
    if case["bits"] == 8:
        s.k_cache, s.k_scales = _held_in_8_bits(k_cache)
        s.v_cache, s.v_scales = _held_in_8_bits(v_cache)
    else:
        s.k_cache, s.v_cache = k_cache.to(torch.bfloat16), v_cache.to(torch.bfloat16)
    if op in ("weigh", "evict"):
        # Few keys have most of the weight; none is held of tokens to come.
        S = W * bs
        s.weights = torch.exp(2 * normal(len(pages), Hk, S))
        old = torch.tensor(s.before, device=dev)
        s.weights *= torch.arange(S, device=dev) < old[:, None, None]
    if op == "weigh":
        s.lse = _plain_lse(s)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        ops = _ops()
        if case["op"] == "append":
            s.rotary = ops.RotaryTable(s.table, interleaved=case["pairs"])
        if case["op"] != "evict":
            s.layout = ops.ChunkLayout(s.news, s.context_lens.device)
    return s


def run(s):
    if not own:
        return _PLAIN[s.case["op"]](s)
    ops, case = _ops(), s.case
    heads = (case["kv_heads"], case["q_heads"] // case["kv_heads"])
    if case["op"] == "append":
        q = ops.append_chunk_kv(s.k, s.v, s.k_cache, s.v_cache, s.block_tables, s.context_lens,
                                s.layout, case["block"], rotary=s.rotary, k_weight=s.k_weight,
                                eps=EPS, q=s.q, q_weight=s.q_weight, k_scales=s.k_scales,
                                v_scales=s.v_scales)
        return q, s.k_cache, s.v_cache, s.k_scales, s.v_scales
    if case["op"] == "attend":
        return ops.chunk_attention(s.q, s.k_cache, s.v_cache, s.block_tables, s.context_lens,
                                   s.layout, *heads, case["block"], causal=case["causal"],
                                   return_lse=case["lse"], k_scales=s.k_scales,
                                   v_scales=s.v_scales)
    if case["op"] == "weigh":
        return ops.add_key_weights(s.weights, s.q, s.lse, s.k_cache, s.block_tables,
                                   s.context_lens, s.layout, *heads, case["block"],
                                   causal=case["causal"], window=case["window"],
                                   k_scales=s.k_scales)
    kept = ops.evict_tokens(s.weights, s.k_cache, s.v_cache, s.block_tables, s.context_lens,
                            case["keep"], case["block"], sinks=case["sinks"],
                            recent=case["recent"], k_scales=s.k_scales, v_scales=s.v_scales)
    return _evicted(s, kept)


def _evicted(s, kept):
    out = [kept, s.weights, s.k_cache, s.v_cache]
    return out if s.k_scales is None else out + [s.k_scales, s.v_scales]


# ------------------------------------------------------------ plain forms

def _plain_rotated(x, weight, positions, table, pairs):
    """One side's norm and rotation in 32 bits."""
    y = x.to(torch.float32)
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.to(torch.float32)
    rows = table[positions]
    half = rows.shape[1] // 2
    cos, sin = rows[:, None, :half], rows[:, None, half:]
    if pairs:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, y[..., 2 * half:]], -1)


def _bytes(t):
    return t.view(torch.uint8)


def _plain_side(y, cache, scales, block, place, part, filled):
    """Rows y [T, heads, D] to their blocks and places; `part` are blocks with
    `filled` earlier tokens each."""
    H = y.shape[1]
    top = torch.zeros(cache.shape[0], H, device=y.device)
    top.scatter_reduce_(0, block[:, None].expand(-1, H), y.abs().amax(-1), "amax")
    old = _bytes(scales).to(torch.int32) - 127
    e = _page_exponents(top)
    earlier = torch.zeros(cache.shape[0], 1, dtype=torch.bool, device=y.device)
    earlier[part] = True
    e = torch.where(earlier, torch.maximum(e, old), e)
    touched = torch.zeros_like(earlier)
    touched[block] = True
    e = torch.where(touched, e, old)
    # Earlier tokens at the new scale.
    held = cache[part].to(torch.float32)
    moved = torch.ldexp(held, (old - e)[part][:, None, :, None]).to(cache.dtype)
    stay = torch.arange(cache.shape[1], device=y.device)[None] >= filled[:, None]
    moved = torch.where(stay[:, :, None, None], _bytes(cache)[part], _bytes(moved))
    _bytes(cache)[part] = moved
    z = torch.ldexp(y, -e[block][:, :, None]).clamp(-_TOP, _TOP)
    _bytes(cache)[block, place] = _bytes(z.to(cache.dtype))
    _bytes(scales).copy_((e + 127).to(torch.uint8))


def _plain_append(s):
    bs, dev = s.case["block"], s.q.device
    news = torch.tensor(s.news, device=dev)
    before = s.context_lens - news
    seq = torch.repeat_interleave(torch.arange(len(s.news), device=dev), news)
    first = torch.cumsum(news, 0) - news
    pos = torch.arange(seq.numel(), device=dev) - first[seq] + before[seq]
    block, place = s.block_tables[seq, pos // bs].long(), pos % bs
    half_full = (news > 0) & (before % bs > 0)
    page = (before // bs).clamp(max=s.block_tables.shape[1] - 1)
    part = s.block_tables.gather(1, page.long()[:, None])[:, 0].long()[half_full]
    filled = (before % bs)[half_full]
    k = _plain_rotated(s.k, s.k_weight, pos, s.table, s.case["pairs"])
    _plain_side(k, s.k_cache, s.k_scales, block, place, part, filled)
    _plain_side(s.v.to(torch.float32), s.v_cache, s.v_scales, block, place, part, filled)
    q = _plain_rotated(s.q, s.q_weight, pos, s.table, s.case["pairs"])
    return q.to(s.q.dtype), s.k_cache, s.v_cache, s.k_scales, s.v_scales


def _plain_pages(cache, scales, pages, ctx):
    """Keys or values [ctx, heads, D] of a sequence in 32 bits."""
    x = cache[pages].to(torch.float32)
    if scales is not None:
        x *= _scale(scales)[pages][:, None, :, None]
    return x.flatten(0, 1)[:ctx]


def _plain_scores(s, window=0):
    """For each sequence: (rows of q, keys, steps over the KV heads), a step being
    (heads, scores [heads, rows * G, keys], -inf where a row does not see)."""
    case = s.case
    Hk, D, bs = case["kv_heads"], case["dim"], case["block"]
    G = case["q_heads"] // Hk
    at = 0
    for b, (n, before) in enumerate(zip(s.news, s.before)):
        skip = max(0, n - window) if window else 0
        rows = slice(at + skip, at + n)
        at += n
        m, ctx = n - skip, before + n
        if m == 0:
            continue
        pages = s.block_tables[b, :-(-ctx // bs)].long()
        k = _plain_pages(s.k_cache, s.k_scales, pages, ctx).permute(1, 2, 0).contiguous()
        q = s.q[rows].view(m, Hk, G, D).permute(1, 0, 2, 3).reshape(Hk, m * G, D)
        q = q.to(torch.float32) * D ** -0.5
        hidden = None
        if case["causal"] and m > 1:
            row = torch.arange(skip, n, device=q.device).repeat_interleave(G)
            hidden = torch.arange(ctx, device=q.device)[None] > (before + row)[:, None]
        # as many heads as fit, or a part of the rows of one
        step = max(1, _SCORES // (m * G * ctx))
        cut = m * G if m * G * ctx <= _SCORES else max(G, _SCORES // ctx)
        for h in range(0, Hk, step):
            for r in range(0, m * G, cut):
                x = q[h:h + step, r:r + cut] @ k[h:h + step]
                if hidden is not None:
                    x.masked_fill_(hidden[r:r + cut], -math.inf)
                yield b, pages, ctx, rows, slice(h, h + x.shape[0]), slice(r, r + x.shape[1]), x


def _grouped(t, case):
    """[tokens, q heads, ...] as [KV heads, tokens * G, ...], to be written to."""
    Hk = case["kv_heads"]
    return t.unflatten(1, (Hk, -1)).transpose(0, 1).flatten(1, 2)


def _ungrouped(t, case):
    Hk, G = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    return t.unflatten(1, (-1, G)).transpose(0, 1).flatten(1, 2)


def _plain_attend(s):
    case = s.case
    Hk, D, T = case["kv_heads"], case["dim"], s.q.shape[0]
    G = case["q_heads"] // Hk
    out = torch.zeros(Hk, T * G, D, device=s.q.device)
    lse = torch.full((Hk, T * G), -math.inf, device=s.q.device)
    seen = None
    for b, pages, ctx, rows, h, r, x in _plain_scores(s):
        if seen != b:
            seen = b
            v = _plain_pages(s.v_cache, s.v_scales, pages, ctx).transpose(0, 1).contiguous()
        m = x.amax(-1, keepdim=True)
        p = torch.exp(x.sub_(m))
        l = p.sum(-1, keepdim=True)
        to = slice(rows.start * G + r.start, rows.start * G + r.stop)
        out[h, to] = (p @ v[h]) / l
        lse[h, to] = (m + torch.log(l))[..., 0]
    out = _ungrouped(out, case).to(s.q.dtype)
    return (out, _ungrouped(lse, case)) if case["lse"] else out


def _plain_lse(s):
    """Log-sum-exps [T, q heads] of the scores, which a user has from the
    attention."""
    case = s.case
    Hk, T = case["kv_heads"], s.q.shape[0]
    G = case["q_heads"] // Hk
    lse = torch.full((Hk, T * G), -math.inf, device=s.q.device)
    for b, pages, ctx, rows, h, r, x in _plain_scores(s, case["window"]):
        lse[h, rows.start * G + r.start:rows.start * G + r.stop] = torch.logsumexp(x, -1)
    return _ungrouped(lse, case).contiguous()


def _plain_weigh(s):
    case = s.case
    G = case["q_heads"] // case["kv_heads"]
    dev = s.q.device
    before = torch.tensor(s.before, device=dev)[:, None, None]
    new = torch.arange(s.weights.shape[2], device=dev) >= before
    new &= torch.arange(s.weights.shape[2], device=dev) < s.context_lens[:, None, None]
    s.weights.masked_fill_(new, 0)
    lse = _grouped(s.lse, case)
    for b, pages, ctx, rows, h, r, x in _plain_scores(s, case["window"]):
        to = slice(rows.start * G + r.start, rows.start * G + r.stop)
        s.weights[b, h, :ctx] += torch.exp(x.sub_(lse[h, to, None])).sum(1)
    return s.weights


def _plain_evict(s):
    case, dev = s.case, s.weights.device
    Hk, bs, keep = case["kv_heads"], case["block"], case["keep"]
    sinks, recent = case["sinks"], case["recent"]
    B, S = s.weights.shape[0], s.weights.shape[2]
    ctx = s.context_lens.long()[:, None, None]
    slot = torch.arange(S, device=dev).expand(B, Hk, S)
    # The kept: first and last ones, then by weight, the lowest slot first.
    rank = torch.where((slot < sinks) | (slot >= ctx - recent), math.inf, s.weights)
    rank = torch.where(slot < ctx, rank, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :min(keep, S)]
    is_kept = torch.zeros(B, Hk, S, dtype=torch.bool, device=dev).scatter_(-1, order, True)
    is_kept &= slot < ctx
    cut = ctx > keep
    # Where the kept ones go: the last ones to the end, those before stay where
    # they are or fill the places that came free, in order.
    middle = keep - recent
    hole = ~is_kept & (slot < middle)
    tail = is_kept & (slot >= middle) & (slot < ctx - recent)
    holes = torch.sort((~hole).to(torch.uint8), dim=-1, stable=True).indices
    nth = torch.cumsum(tail, -1) - 1
    dest = torch.where(tail, holes.gather(-1, nth.clamp(min=0)), slot)
    dest = torch.where(slot >= ctx - recent, slot - (ctx - keep), dest)
    dest = torch.where(cut, dest, slot)
    dest = torch.where(is_kept, dest, S + keep)  # of no further use
    kept = torch.full((B, Hk, S + keep + 1), -1, dtype=torch.int64, device=dev)
    kept.scatter_(-1, dest, slot)
    kept = kept[..., :keep]
    # Rows that change places.
    b, h, to = torch.nonzero((kept >= 0) & (kept != torch.arange(keep, device=dev)),
                             as_tuple=True)
    src = kept[b, h, to]
    block = [s.block_tables[b, x // bs].long() for x in (src, to)]
    s.weights[b, h, to] = s.weights[b, h, src]
    _plain_move(s.k_cache, s.k_scales, block, src % bs, to % bs, h, s, kept)
    _plain_move(s.v_cache, s.v_scales, block, src % bs, to % bs, h, s, kept)
    return _evicted(s, kept.to(torch.int32))


def _plain_move(cache, scales, block, src, to, h, s, kept):
    if scales is None:
        cache[block[1], to, h] = cache[block[0], src, h]
        return
    # A page that rows come to has the largest scale of its tokens.
    bs, dev = cache.shape[1], cache.device
    old = _bytes(scales).to(torch.int32) - 127
    changed = torch.zeros(old.shape, dtype=torch.bool, device=dev)
    changed[block[1], h] = True
    B, Hk, keep = kept.shape
    at = torch.arange(keep, device=dev).expand(B, Hk, keep)
    valid = kept >= 0
    b, g, place = torch.nonzero(valid, as_tuple=True)
    from_block = s.block_tables[b, kept[valid] // bs].long()
    to_block = s.block_tables[b, at[valid] // bs].long()
    e = torch.full_like(old, -1000)
    e.view(-1).scatter_reduce_(0, to_block * Hk + g, old[from_block, g], "amax")
    e = torch.where(changed, e, old)
    rows = cache[block[0], src, h].to(torch.float32)
    rows = torch.ldexp(rows, (old[block[0], h] - e[block[1], h])[:, None])
    # Rows that stay in such a page.
    stay = valid & (kept == at)
    b, g, place = torch.nonzero(stay, as_tuple=True)
    same = s.block_tables[b, place // bs].long()
    held = torch.ldexp(cache[same, place % bs, g].to(torch.float32),
                       (old[same, g] - e[same, g])[:, None])
    _bytes(cache)[same, place % bs, g] = _bytes(held.to(cache.dtype))
    _bytes(cache)[block[1], to, h] = _bytes(rows.to(cache.dtype))
    _bytes(scales).copy_((e + 127).to(torch.uint8))


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "weigh": _plain_weigh,
          "evict": _plain_evict}


# ------------------------------------------------------------ in 64 bits

def _exact_rotated(x, weight, positions, table, pairs):
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    R = table.shape[1]
    t = table.double()[positions]
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


def _exact_append(s):
    """The cache's payload before its rounding to 8 bits."""
    bs, dev = s.case["block"], s.q.device
    pos = torch.cat([torch.arange(b, b + n, device=dev) for b, n in zip(s.before, s.news)])
    q = _exact_rotated(s.q, s.q_weight, pos, s.table, s.case["pairs"])
    k = _exact_rotated(s.k, s.k_weight, pos, s.table, s.case["pairs"])
    out = []
    for rows, cache, scales in ((k, s.k_cache, s.k_scales), (s.v.double(), s.v_cache, s.v_scales)):
        held, scale = cache.double(), scales.double()
        at = 0
        for b, (n, before) in enumerate(zip(s.news, s.before)):
            # the first page by itself, then the whole ones together
            head = min(n, -before % bs)
            blocks = s.block_tables[b].long()
            if head:
                blk, off = blocks[before // bs], before % bs
                new = rows[at:at + head]
                least = torch.exp2(torch.ceil(torch.log2(new.abs().amax((0, 2)) / 448)))
                wide = torch.maximum(scale[blk], least.clamp(min=2.0 ** -110))
                held[blk, :off] *= (scale[blk] / wide)[:, None]
                held[blk, off:off + head] = new / wide[:, None]
                scale[blk] = wide
            rest = n - head
            if rest:
                pages = -(-rest // bs)
                first = (before + head) // bs
                full = torch.zeros(pages * bs, *rows.shape[1:], dtype=torch.float64, device=dev)
                full[:rest] = rows[at + head:at + n]
                full = full.view(pages, bs, *rows.shape[1:])
                wide = torch.exp2(torch.ceil(torch.log2(full.abs().amax((1, 3)) / 448)))
                wide = wide.clamp(min=2.0 ** -110)
                blk = blocks[first:first + pages]
                there = (torch.arange(pages * bs, device=dev) < rest).view(pages, bs, 1, 1)
                held[blk] = torch.where(there, full / wide[:, None, :, None], held[blk])
                scale[blk] = wide
            at += n
        out.append((held, scale))
    return q, out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_keys(cache, scales, block, place, h):
    x = cache[block, place, h].double()
    return x if scales is None else x * scales.double()[block, h, None]


def _exact_scores(s, b, h, i, j, at):
    """Scores of tokens i to j of sequence b and KV head h, [rows, keys]."""
    case, dev = s.case, s.q.device
    D, bs, before = case["dim"], case["block"], s.before[b]
    G = case["q_heads"] // case["kv_heads"]
    pos = torch.arange(before + s.news[b], device=dev)
    block = s.block_tables[b].long()[pos // bs]
    k = _exact_keys(s.k_cache, s.k_scales, block, pos % bs, h)
    q = s.q[at + i:at + j, h * G:(h + 1) * G].double().reshape(-1, D)
    x = q @ k.t() / math.sqrt(D)
    if case["causal"]:
        own_pos = pos[before + i:before + j].repeat_interleave(G)
        x = torch.where(pos[None] <= own_pos[:, None], x, -math.inf)
    return x


def _exact_evict(s):
    """Sequence by sequence and head by head; payload before its rounding."""
    case, dev = s.case, s.weights.device
    bs, keep, sinks, recent = (case[n] for n in ("block", "keep", "sinks", "recent"))
    weights = s.weights.double()
    kept = torch.full((*weights.shape[:2], keep), -1, dtype=torch.int32, device=dev)
    caches = [(c.double(), None if f is None else f.double())
              for c, f in ((s.k_cache, s.k_scales), (s.v_cache, s.v_scales))]
    for b, ctx in enumerate(s.before):
        blocks = s.block_tables[b].long()
        place = torch.arange(min(ctx, keep), device=dev)
        for h in range(case["kv_heads"]):
            kept[b, h, :place.numel()] = place.int()
            if ctx <= keep:
                continue
            middle = s.weights[b, h, sinks:ctx - recent]
            best = torch.sort(middle, descending=True, stable=True)[1][:keep - sinks - recent]
            best = torch.sort(best + sinks)[0]
            free = torch.ones(keep, dtype=torch.bool, device=dev)
            free[:sinks] = False
            free[keep - recent:] = False
            free[best[best < keep - recent]] = False
            old = place.clone()
            old[free] = best[best >= keep - recent]
            old[keep - recent:] += ctx - keep
            kept[b, h] = old.int()
            weights[b, h, :keep] = weights[b, h, old]
            moved = torch.zeros(-(-keep // bs) * bs, dtype=torch.bool, device=dev)
            moved[:keep] = old != place
            for held, scale in caches:
                rows = held[blocks[old // bs], old % bs, h]
                if scale is not None:
                    mine = scale[blocks[old // bs], h]
                    size = torch.zeros(moved.shape, dtype=torch.float64, device=dev)
                    size[:keep] = mine
                    size = size.view(-1, bs).amax(1)
                    changed = moved.view(-1, bs).any(1)
                    pages = blocks[:size.numel()]
                    size = torch.where(changed, size, scale[pages, h])
                    rows = rows * (mine / size[place // bs])[:, None]
                    scale[pages, h] = size
                held[blocks[place // bs], place % bs, h] = rows
    out = [kept, weights, caches[0][0], caches[1][0]]
    return out if s.k_scales is None else out + [caches[0][1], caches[1][1]]


def exact(case, seed):
    s = _inputs(case, seed)
    Hk, D, bs = case["kv_heads"], case["dim"], case["block"]
    G = case["q_heads"] // Hk
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "evict":
        return _exact_evict(s)
    dev = s.q.device
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=dev)
    lse = torch.full(s.q.shape[:2], -math.inf, dtype=torch.float64, device=dev)
    weights = s.weights.double() if case["op"] == "weigh" else None
    at = 0
    for b, (n, before) in enumerate(zip(s.news, s.before)):
        if case["op"] == "weigh":
            weights[b, :, before:before + n] = 0
        first = max(0, n - case["window"]) if case["window"] else 0
        pos = torch.arange(before + n, device=dev)
        block = s.block_tables[b].long()[pos // bs]
        for h in range(Hk):
            for i in range(first, n, 1024):
                j = min(i + 1024, n)
                x = _exact_scores(s, b, h, i, j, at)
                if case["op"] == "weigh":
                    total = s.lse[at + i:at + j, h * G:(h + 1) * G].double().reshape(-1, 1)
                    weights[b, h, :before + n] += torch.exp(x - total).sum(0)
                    continue
                total = torch.logsumexp(x, -1, keepdim=True)
                v = _exact_keys(s.v_cache, s.v_scales, block, pos % bs, h)
                o = torch.exp(x - total) @ v
                out[at + i:at + j, h * G:(h + 1) * G] = o.view(j - i, G, D)
                lse[at + i:at + j, h * G:(h + 1) * G] = total.view(j - i, G)
        at += n
    if case["op"] == "weigh":
        return weights
    return (out, lse) if case["lse"] else out


# ------------------------------------------------------------------ work

def work(case):
    news, before = _lengths(case)
    T = sum(news)
    Hq, Hk, D, bs = case["q_heads"], case["kv_heads"], case["dim"], case["block"]
    c = case["bits"] // 8
    if case["op"] == "evict":
        keep, ends = case["keep"], case["sinks"] + case["recent"]
        nbytes = flops = 0
        for ctx in before:
            if ctx <= keep:
                nbytes += 4 * Hk * keep
                continue
            # The share of the middle that is given up leaves holes below
            # keep - recent; each takes a row, and so do the last ones.
            gone = (ctx - keep) / max(1, ctx - ends)
            moved = (keep - ends) * gone + case["recent"]
            nbytes += Hk * (4 * ctx + 4 * keep + 2 * moved * (2 * D * c + 4))
            flops += Hk * ctx
        return {"bytes": nbytes, "flops": flops}
    if case["op"] in ("attend", "weigh"):
        pairs = keys = pages = rows = 0
        for n, b in zip(news, before):
            if n:
                m = min(n, case["window"]) if case["window"] else n
                keys += b + n
                pages += -(-(b + n) // bs)
                rows += m
                pairs += m * (b + n) - (m * (m - 1) // 2 if case["causal"] else 0)
        scales = pages * Hk if c == 1 else 0
        if case["op"] == "weigh":
            nbytes = 2 * rows * Hq * D + 4 * rows * Hq + keys * Hk * D * c + scales
            nbytes += 8 * keys * Hk + 4 * pages
            return {"bytes": nbytes, "flops": pairs * Hq * (2 * D + 4)}
        nbytes = 4 * T * Hq * D + 2 * keys * Hk * D * c + 2 * scales + 4 * pages
        if case["lse"]:
            nbytes += 4 * T * Hq
        # two products of D multiply-adds and an exponential for each pair
        return {"bytes": nbytes, "flops": pairs * Hq * (4 * D + 4)}
    e = 4 if case["dtype"] == "fp32" else 2
    rot_rows = min(max((b + n for b, n in zip(before, news)), default=0), T)
    nbytes = 4 * case["rot"] * rot_rows + 2 * e * T * Hq * D  # table, q in and out
    nbytes += 2 * e * T * Hk * D + 2 * T * Hk * D              # k and v in and out
    nbytes += 4 * Hk * (T // bs + len(news))                   # scales in and out
    flops = T * (Hq + Hk) * (3 * case["rot"] + (4 * D if case["norm"] else 0))
    flops += 2 * T * Hk * D * 3
    return {"bytes": nbytes, "flops": flops}
