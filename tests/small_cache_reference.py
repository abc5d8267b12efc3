"""Plain forms in 64 bits of the operators on caches of 8 bits, of the weights of
keys and of eviction, and the bounds of their errors."""
import math

import torch

LOW, HIGH, TOP = -110, 119, 448.0


def scale_bytes(scales):
    return scales.view(torch.uint8).to(torch.int64).cpu()


def to_scales(bytes_):
    return bytes_.to(torch.uint8).view(torch.float8_e8m0fnu)


def values(cache, scales):
    """The values of a cache of 8 bits, in 64 bits; all of a block and head whose
    scale is NaN are."""
    b = scale_bytes(scales)
    f = torch.ldexp(torch.ones(b.shape, dtype=torch.float64), b - 127)
    f[b == 255] = math.nan
    return cache.cpu().double() * f[:, None, :, None]


def exponent(top):
    """Smallest e in LOW .. HIGH with top <= 448 * 2^e."""
    e = LOW
    while e < HIGH and top > TOP * 2.0 ** e:
        e += 1
    return e


def random_cache(g, blocks, bs, H, D, spread=3):
    """Payloads and scales of values of unlike size; no NaN."""
    x = torch.randn(blocks, bs, H, D, generator=g)
    e = torch.randint(-spread, spread + 1, (blocks, H), generator=g)
    return x.to(torch.float8_e4m3fn), to_scales(e + 127)


def appended(y, size, cache, scales, block_tables, context_lens, lens, rel):
    """(low, high, bytes): the least and largest value that each element of the
    cache may have after rows y ([T, H, D], 64 bits) were appended to it, and the
    sets of bytes that each scale may have.  The kernel's rows are y but for rel *
    size of 32-bit arithmetic; a payload is rounded by half a step, 2^-4 of itself
    or 2^-10 below the normal numbers, times the scale.  Earlier tokens of a page
    whose scale grows are rounded once more, from what they were, exactly."""
    bs, nb, H = cache.shape[1], cache.shape[0], cache.shape[2]
    bt, ctx = block_tables.cpu(), context_lens.cpu().tolist()
    have = values(cache, scales)
    low, high = have.clone(), have.clone()
    old = scale_bytes(scales)
    may = [[{int(old[n, h])} for h in range(H)] for n in range(nb)]
    at = 0
    for b, n in enumerate(lens):
        first = ctx[b] - n
        pages = sorted({(first + i) // bs for i in range(n) if first + i >= 0})
        for page in pages:
            if page >= bt.shape[1] or not 0 <= int(bt[b, page]) < nb:
                continue
            blk = int(bt[b, page])
            lo, hi = max(first, page * bs), min(ctx[b], (page + 1) * bs)
            rows = slice(at + lo - first, at + hi - first)
            place = slice(lo - page * bs, hi - page * bs)
            for h in range(H):
                new, err = y[rows, h], rel * size[rows, h]
                fine = new.isfinite()
                top = new.abs()[fine].max().item() if fine.any() else 0.0
                slack = err[fine].max().item() if fine.any() else 0.0
                bytes_ = {exponent(max(0.0, top - slack)) + 127, exponent(top + slack) + 127}
                if place.start > 0:
                    bytes_ = {max(x, int(old[blk, h])) for x in bytes_}
                may[blk][h] = bytes_
                unit = 2.0 ** (max(bytes_) - 127)
                step = torch.maximum((new.abs() + err) * 2.0 ** -4,
                                     torch.full_like(err, unit * 2.0 ** -10))
                bound = new.clamp(-TOP * unit, TOP * unit)
                low[blk, place, h] = torch.where(fine, bound - step - err, math.nan)
                high[blk, place, h] = torch.where(fine, bound + step + err, math.nan)
                if place.start > 0 and max(bytes_) > int(old[blk, h]):
                    both = []
                    for x in bytes_:
                        f = 2.0 ** (int(old[blk, h]) - x)
                        p = (cache[blk, :place.start, h].float() * f).to(cache.dtype).double()
                        both.append(p * 2.0 ** (x - 127))
                    both = torch.stack(both)
                    low[blk, :place.start, h] = both.amin(0)
                    high[blk, :place.start, h] = both.amax(0)
        at += n
    return low, high, may


def check_appended(cache, scales, before, want):
    """`before`: the cache and scales as they were."""
    low, high, may = want
    got, now, was = values(cache, scales), scale_bytes(scales), scale_bytes(before[1])
    for n in range(now.shape[0]):
        for h in range(now.shape[1]):
            assert int(now[n, h]) in may[n][h], (n, h, int(now[n, h]), may[n][h])
    # Rows that nobody asked to change keep their bytes, whatever their scale
    # is now: compare those in blocks whose scale is the same as values.
    nan = low.isnan()
    same = (now == was)[:, None, :, None].expand_as(got)
    held = (low == high) & ~nan
    ok = (got >= low) & (got <= high) | nan & got.isnan()
    kept = cache.cpu().view(torch.uint8) == before[0].cpu().view(torch.uint8)
    assert (ok | (held & ~same & kept)).all(), (~ok & ~(held & ~same & kept)).nonzero()[:5]


def key_weights(weights, q, lse, keys, block_tables, context_lens, lens, G, causal=True,
                scale=None, window=0):
    """(weights, slack) in 64 bits; keys [blocks, bs, H, D] in 64 bits.

    A score's products are summed in 32 bits, D + 8 roundings of sums bounded by a
    = scale sum |q||k|; c = scale log2(e) and lse c / scale are each rounded, 2^-24
    of |score| and 2 2^-24 of |lse|, then the exponent, 2^-24 of itself, and exp2,
    2^-22.  A sum of n terms adds n + 8 roundings.
    """
    w, q = weights.double().cpu().clone(), q.double().cpu()
    lse, bt, ctx = lse.double().cpu(), block_tables.cpu(), context_lens.cpu().tolist()
    slack = torch.zeros_like(w)
    D, bs, nb = q.shape[-1], keys.shape[1], keys.shape[0]
    scale = D ** -0.5 if scale is None else scale
    at, u = 0, 2.0 ** -24
    for b, n in enumerate(lens):
        if n == 0:
            continue
        top = max(0, min(ctx[b], bt.shape[1] * bs))
        first = ctx[b] - n
        if first < top:
            w[b, :, max(0, first):top] = 0
        pos = torch.arange(top)
        blk = bt[b].long()[pos // bs]
        pos, blk = pos[(blk >= 0) & (blk < nb)], blk[(blk >= 0) & (blk < nb)]
        kk = keys[blk, pos % bs]  # [n_keys, H, D]
        count = (min(n, window) if window else n)
        total = torch.zeros(kk.shape[:2], dtype=torch.float64)
        err = torch.zeros_like(total)
        for i in range(n - count, n):
            see = pos <= first + i if causal else torch.ones_like(pos, dtype=torch.bool)
            for h in range(kk.shape[1]):
                for r in range(h * G, (h + 1) * G):
                    if lse[at + i, r] == -math.inf:
                        continue
                    s = kk[:, h] @ q[at + i, r] * scale
                    a = kk[:, h].abs() @ q[at + i, r].abs() * scale
                    t = s - lse[at + i, r]
                    p = torch.where(see, torch.exp(t), 0.0)
                    total[:, h] += p
                    rel = u * ((D + 8) * a + a + 2 * lse[at + i, r].abs() + t.abs()) + 2.0 ** -22
                    err[:, h] += torch.where(see, p * torch.expm1(rel), 0.0)
        for h in range(kk.shape[1]):
            w[b, h, pos] += total[:, h]
            slack[b, h, pos] += (err[:, h] + (count * G + 8) * u * total[:, h]
                                 + u * w[b, h, pos].abs())
        at += n
    return w, slack * 1.05


def evicted(weights, caches, block_tables, context_lens, keep, sinks, recent, scales=None):
    """(kept, weights, caches, scales) of exact copies, head by head."""
    w, bt, ctx = weights.cpu().clone(), block_tables.cpu(), context_lens.cpu().tolist()
    caches = [c.cpu().clone() for c in caches]
    bytes_ = [scale_bytes(s) for s in scales] if scales else None
    bs, nb = caches[0].shape[1], caches[0].shape[0]
    B, H, _ = w.shape
    kept = torch.full((B, H, keep), -1, dtype=torch.int32)
    for b in range(B):
        n = max(0, min(ctx[b], bt.shape[1] * bs))
        for h in range(H):
            if n <= keep:
                kept[b, h, :n] = torch.arange(n)
                continue
            def rank(j):
                x = float(w[b, h, j])
                return (0, 0.0, j) if math.isnan(x) else (1, -x, j)
            middle = sorted(range(sinks, n - recent), key=rank)[:keep - sinks - recent]
            stay = {j for j in middle if j < keep - recent}
            come = iter(sorted(j for j in middle if j >= keep - recent))
            slots = list(range(sinks)) + [j if j in stay else next(come)
                                          for j in range(sinks, keep - recent)]
            slots += list(range(n - recent, n))
            kept[b, h] = torch.tensor(slots)
            src = kept[b, h].long()
            w[b, h, :keep] = w[b, h, src].clone()
            to = torch.arange(keep)
            moved = src != to
            sb, db = bt[b].long()[src // bs], bt[b].long()[to // bs]
            ok = (sb >= 0) & (sb < nb) & (db >= 0) & (db < nb)
            for i, c in enumerate(caches):
                raw = c.view(torch.uint8) if scales else c
                rows = c[sb.clamp(0, nb - 1), src % bs, h].clone()
                if scales:
                    e = bytes_[i][sb.clamp(0, nb - 1), h].clone()
                    e[(sb < 0) | (sb >= nb)] = 0  # no row, so no scale
                    for p in range(-(-keep // bs)):
                        part = slice(p * bs, min((p + 1) * bs, keep))
                        if not moved[part].any() or not 0 <= int(bt[b, p]) < nb:
                            continue
                        top = int(e[part].max())
                        f = torch.ldexp(torch.ones(e[part].shape), (e[part] - top))
                        rows[part] = (rows[part].float() * f[:, None]).to(c.dtype)
                        bytes_[i][int(bt[b, p]), h] = top
                    touched = torch.tensor([bool(moved[j // bs * bs:(j // bs + 1) * bs].any())
                                            for j in range(keep)])
                    put = ok & touched
                    raw[db[put], to[put] % bs, h] = rows.view(torch.uint8)[put]
                else:
                    put = ok & moved
                    raw[db[put], to[put] % bs, h] = rows[put]
    return kept, w, caches, [to_scales(x) for x in bytes_] if scales else None
