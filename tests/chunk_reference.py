"""Plain forms in 64 bits of the operators on chunks of new tokens, and the
bounds of their errors."""
import math

import torch


def half_step(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def rotated(x, weight, positions, table, interleaved, eps):
    """(y, size): norm and rotation of rows [T, H, D] in 64 bits, and
    |a cos| + |b sin| of the terms of each output."""
    x = x.double().cpu()
    T, H, D = x.shape
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + eps) * weight.double().cpu()
    y, size = x.clone(), x.abs()
    if table is not None:
        R = table.shape[1]
        rows = torch.full((T, R), math.nan, dtype=torch.float64)
        for t, p in enumerate(positions.tolist()):
            if 0 <= p < table.shape[0]:
                rows[t] = table[p].double().cpu()
        for i in range(R // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
            c, s = rows[:, None, i], rows[:, None, R // 2 + i]
            y[..., a] = x[..., a] * c - x[..., b] * s
            y[..., b] = x[..., b] * c + x[..., a] * s
            size[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
            size[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, size


def check_rotated(got, want, size, dtype, D):
    """32-bit arithmetic, rounded once to dtype.

    Sum of D squares: at most D roundings of the partial sums and one of each
    square; the mean, eps, the root, the two products with the root and the
    weight and the rotation's products and sum add fewer than 16 more: relative
    (D + 16) 2^-24 of each term.  Then half a step of the result.
    """
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    fp32 = (D + 16) * 2.0 ** -24
    bound = half_step(dtype) * (want.abs() + fp32 * size) + fp32 * size
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25  # half a step of its subnormal numbers
    bad = ((got - want).abs() > bound) & ~want.isnan()
    assert not bad.any(), ((got - want).abs() - bound)[bad].max()


def attend(q, k_cache, v_cache, block_tables, context_lens, lens, G, causal=True, scale=None,
           parts=1):
    """(out, lse, slack, lse_slack) in 64 bits, token by token over exactly the
    keys that each sees; slack bounds the kernel's errors.

    A score's products are summed in 32 bits: D + 8 roundings of sums bounded
    by a = scale sum |q||k|, so a weight is off by 2 (D + 8) 2^-24 a (its own
    score and the reference's), by the roundings of the exponent |x| 2^-23 and
    of exp2 (2^-22), and by half a step of bf16 (2^-8) in the second product,
    whose sum over n keys adds n 2^-24, with 64 roundings for moving
    references and joining splits.  All are relative to sum p |v|; the output
    is then rounded to bf16.  With the weights in two bf16 `parts` half a step of
    half a step is lost (2^-16), and the sum has twice the terms.
    """
    q, kc, vc = q.double().cpu(), k_cache.double().cpu(), v_cache.double().cpu()
    bt, ctx = block_tables.cpu(), context_lens.cpu().tolist()
    T, H_q, D = q.shape
    bs, nb = kc.shape[1], kc.shape[0]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(T, H_q, D, dtype=torch.float64)
    lse = torch.full((T, H_q), -math.inf, dtype=torch.float64)
    slack, lse_slack = torch.zeros_like(out), torch.zeros_like(lse)
    at = 0
    for b, n in enumerate(lens):
        pos = torch.arange(max(0, min(ctx[b], bt.shape[1] * bs)))
        blk = bt[b].long()[pos // bs]
        pos, blk = pos[(blk >= 0) & (blk < nb)], blk[(blk >= 0) & (blk < nb)]
        keys, vals = kc[blk, pos % bs], vc[blk, pos % bs]  # [n_keys, H_kv, D]
        for i in range(n):
            p = ctx[b] - n + i
            seen = int((pos <= p).sum()) if causal else pos.numel()
            if seen:
                kk = keys[:seen].repeat_interleave(G, 1).permute(1, 0, 2)
                vv = vals[:seen].repeat_interleave(G, 1).permute(1, 0, 2)
                qq = q[at + i][:, :, None]
                s = (kk @ qq)[..., 0] * scale                    # [H_q, seen]
                a = ((kk.abs() @ qq.abs())[..., 0] * scale).amax(-1)
                total = torch.logsumexp(s, -1)
                w = torch.exp(s - total[:, None])
                out[at + i] = (w[:, None] @ vv)[:, 0]
                lse[at + i] = total
                x = (s.amax(-1) - s.amin(-1)).clamp(max=150.0) / math.log(2) + 8
                rel = (2 * (D + 8) * 2.0 ** -24 * a + x * 2.0 ** -23 + 2.0 ** -22
                       + (parts * seen + 64) * 2.0 ** -24)
                size = (w[:, None] @ vv.abs())[:, 0]
                slack[at + i] = ((2.0 ** (-8 * parts) + 2 * rel)[:, None] * size
                                 + half_step(torch.bfloat16) * out[at + i].abs())
                lse_slack[at + i] = 2 * rel + 2.0 ** -22 * total.abs()
        at += n
    return out, lse, slack * 1.02, lse_slack * 1.02


def check_attend(got, ref, lse=None):
    out, want_lse, slack, lse_slack = ref
    got = got.double().cpu()
    finite = out.isfinite()
    assert torch.equal(got.isfinite(), finite)
    err = (got - out).abs()
    assert not (err > slack)[finite].any(), (err - slack)[finite].max()
    if lse is not None:
        lse = lse.double().cpu()
        fin = want_lse.isfinite()
        assert torch.equal(lse.isfinite(), fin)
        assert (lse[~fin] == want_lse[~fin]).all() or want_lse[~fin].isnan().any()
        assert not ((lse - want_lse).abs() > lse_slack)[fin].any()


def check_kinds(got, ref):
    """check_attend, and that each output is of its kind: the same infinity, or
    NaN."""
    want = ref[0]
    check_attend(got, ref)
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert inf.any() and torch.equal(got[inf], want[inf])
