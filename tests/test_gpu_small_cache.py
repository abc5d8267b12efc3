"""Caches of 8 bits, weights of the keys and eviction by them on the GPU, each
against its formula in 64 bits, and a run of them together as a serving loop
makes it."""
import math

import pytest
import torch

import chunk_reference as ref
import small_cache_reference as small
from cvsa import ops
from cvsa.backend import CVSABackend
from cvsa.runtime.dense import DenseAttentionBackend
from cvsa.runtime.kv_cache import PagedKVCache, SequenceKVManager

pytestmark = pytest.mark.gpu

EPS = 1e-6
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g)


def _tables(g, totals, bs, W=None, spare=3):
    pages = [-(-t // bs) for t in totals]
    nb = sum(pages) + spare
    W = W or max(1, max(pages))
    perm = torch.randperm(nb, generator=g).int()
    bt = torch.full((len(totals), W), -7, dtype=torch.int32)
    at = 0
    for b, p in enumerate(pages):
        bt[b, :p] = perm[at:at + p]
        at += p
    return bt, torch.tensor(totals, dtype=torch.int32), nb


def _gpu(gpu, *tensors):
    return [None if t is None else t.to(gpu) for t in tensors]


# ------------------------------------------------------------ append

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,bs,Hk,Hq", [(128, 16, 8, 32), (64, 64, 3, 9), (32, 8, 5, 5),
                                        (256, 128, 2, 2), (128, 32, 5, 35), (32, 16, 3, 6),
                                        (64, 8, 3, 3), (128, 8, 2, 4), (32, 128, 1, 1),
                                        (256, 8, 3, 3), (128, 128, 3, 3), (64, 16, 2, 2)])
def test_append(gpu, dtype, D, bs, Hk, Hq):
    g = _gen(D + bs)
    lens = [3, 0, 1, 2 * bs + 1, 1, 5, bs, 2]
    before = [5, 9, 0, bs - 1, 4 * bs, 2 * bs - 2, bs, bs - 1]
    totals = [a + b for a, b in zip(lens, before)]
    bt, ctx, nb = _tables(g, totals, bs)
    T, pad = sum(lens), 4  # rows behind the last sequence
    # Rows of very unlike size, so that scales grow or stay.
    k, v = ((_randn(g, T + pad, Hk, D) * torch.exp(2 * _randn(g, T + pad, 1, 1))).to(dtype)
            for _ in range(2))
    q = _randn(g, T + pad, Hq, D).to(dtype)
    kw, qw = (1 + 0.2 * _randn(g, D) for _ in range(2))
    caches = [small.random_cache(g, nb, bs, Hk, D) for _ in range(2)]
    layout = ops.ChunkLayout(lens, gpu)
    table = ops.RotaryTable.build(D, max(totals), device=gpu)
    (kc, ks), (vc, vs) = [[t.to(gpu) for t in c] for c in caches]
    got = ops.append_chunk_kv(k.to(gpu), v.to(gpu), kc, vc, bt.to(gpu), ctx.to(gpu), layout, bs,
                              table, kw.to(gpu), EPS, q.to(gpu), qw.to(gpu), ks, vs)
    pos = torch.cat([torch.arange(b, b + n) for b, n in zip(before, lens)])
    want, size = ref.rotated(k[:T], kw, pos, table.table, False, EPS)
    rel = (D + 16) * 2.0 ** -24
    small.check_appended(kc, ks, caches[0],
                         small.appended(want, size, *caches[0], bt, ctx, lens, rel))
    y = v[:T].double()
    small.check_appended(vc, vs, caches[1],
                         small.appended(y, y.abs(), *caches[1], bt, ctx, lens, 0.0))
    # The queries are those of the append to a bf16 cache.
    wide = [torch.zeros(nb, bs, Hk, D, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    same = ops.append_chunk_kv(k.to(gpu), v.to(gpu), *wide, bt.to(gpu), ctx.to(gpu), layout, bs,
                               table, kw.to(gpu), EPS, q.to(gpu), qw.to(gpu))
    assert torch.equal(got, same)


@pytest.mark.parametrize("interleaved,R", [(True, 64), (False, 16), (True, 16), (None, 0)])
def test_append_rotations(gpu, interleaved, R):
    g = _gen(R)
    lens, before, bs, Hk, D = [20, 3], [7, 0], 16, 3, 64
    bt, ctx, nb = _tables(g, [27, 3], bs)
    k, v = _randn(g, 23, Hk, D), _randn(g, 23, Hk, D)
    caches = [small.random_cache(g, nb, bs, Hk, D) for _ in range(2)]
    (kc, ks), (vc, vs) = [[t.to(gpu) for t in c] for c in caches]
    table = ops.RotaryTable.build(R, 27, device=gpu, interleaved=interleaved) if R else None
    none = ops.append_chunk_kv(k.to(gpu), v.to(gpu), kc, vc, bt.to(gpu), ctx.to(gpu),
                               ops.ChunkLayout(lens, gpu), bs, table, k_scales=ks, v_scales=vs)
    assert none is None
    pos = torch.cat([torch.arange(7, 27), torch.arange(3)])
    want, size = ref.rotated(k, None, pos, table.table if R else None, interleaved, EPS)
    small.check_appended(kc, ks, caches[0], small.appended(want, size, *caches[0], bt, ctx, lens,
                                                           8 * 2.0 ** -24))
    small.check_appended(vc, vs, caches[1], small.appended(v.double(), v.double().abs(),
                                                           *caches[1], bt, ctx, lens, 0.0))


def test_append_of_extreme_values(gpu):
    """Zeros, subnormal and largest numbers, infinities and NaN, and borders of a
    scale."""
    D, bs, H = 32, 8, 1
    top = torch.finfo(torch.float32).max
    rows = torch.zeros(9, H, D)
    rows[1, 0, :4] = torch.tensor([448.0, -448.0, 1.0, 2.0 ** -9])   # scale 1, exactly
    rows[2, 0, :2] = torch.tensor([448.0001, 1.0])                  # the next
    rows[3, 0, :3] = torch.tensor([top, -top, 1e30])                # past the largest scale
    rows[4, 0, :3] = torch.tensor([1e-45, -1e-40, 1e-38])           # below the least one
    rows[5, 0, :5] = torch.tensor([math.inf, -math.inf, math.nan, 3.0, -2.0])
    rows[6, 0] = math.nan                                           # nothing finite
    # 448 * 2^-110 = 1.75 * 2^-102 < 2^-101 <= 448 * 2^-109: the least but one.
    rows[7, 0, :2] = torch.tensor([2.0 ** -101, 448.0 * 2.0 ** -110])
    rows[8, 0, :2] = torch.tensor([224.0, 7.0 / 1024])
    lens = [1] * 9
    bt = torch.arange(9, dtype=torch.int32)[:, None]
    ctx = torch.ones(9, dtype=torch.int32)
    cache = (torch.zeros(9, bs, H, D).to(torch.float8_e4m3fn),
             small.to_scales(torch.full((9, H), 255)))
    (kc, ks), (vc, vs) = [[t.to(gpu) for t in cache] for _ in range(2)]
    ops.append_chunk_kv(rows.to(gpu), rows.to(gpu), kc, vc, bt.to(gpu), ctx.to(gpu),
                        ops.ChunkLayout(lens, gpu), bs, k_scales=ks, v_scales=vs)
    assert torch.equal(small.scale_bytes(ks), small.scale_bytes(vs))
    assert small.scale_bytes(ks)[:, 0].tolist() == [17, 127, 128, 246, 17, 127 - 7, 17, 18, 126]
    y = rows.double()
    want = small.appended(y, y.abs(), *cache, bt, ctx, lens, 0.0)
    got = small.values(kc, ks)
    assert torch.equal(kc.cpu().view(torch.uint8), vc.cpu().view(torch.uint8))
    ok = (got >= want[0]) & (got <= want[1]) | want[0].isnan() & got.isnan()
    assert ok[:, 0].all(), (~ok[:, 0]).nonzero()
    assert got[5, 0, 0].isnan().tolist()[:5] == [True, True, True, False, False]
    assert got[1, 0, 0, :4].tolist() == [448.0, -448.0, 1.0, 2.0 ** -9]


def test_append_grows_a_scale_step_by_step(gpu):
    """A page filled token by token, each larger than the last, then smaller ones."""
    D, bs, H, n = 64, 16, 2, 16
    g = _gen(1)
    size = [2.0 ** (i if i < 9 else -i) for i in range(n)]
    k = _randn(g, n, H, D) * torch.tensor(size)[:, None, None]
    bt = torch.tensor([[1]], dtype=torch.int32)
    cache = small.random_cache(g, 2, bs, H, D)
    kc, ks = [t.to(gpu) for t in cache]
    vc, vs = [t.to(gpu) for t in cache]
    state = cache
    for i in range(n):
        ctx = torch.tensor([i + 1], dtype=torch.int32)
        ops.append_chunk_kv(k[i:i + 1].to(gpu), k[i:i + 1].to(gpu), kc, vc, bt.to(gpu),
                            ctx.to(gpu), ops.ChunkLayout([1], gpu), bs, k_scales=ks, v_scales=vs)
        y = k[i:i + 1].double()
        small.check_appended(kc, ks, state, small.appended(y, y.abs(), *state, bt, ctx, [1], 0.0))
        state = (kc.cpu(), ks.cpu())
    # Every token within a half step of what it was, at the page's scale.
    unit = torch.ldexp(torch.ones(H), small.scale_bytes(ks)[1] - 127)
    err = (small.values(kc, ks)[1] - k.double()).abs()
    assert (err <= torch.maximum(k.double().abs() * 2.0 ** -4,
                                 2.0 ** -10 * unit[None, :, None].double() * 2)).all()


def test_append_leaves_the_rest_as_it_was(gpu):
    """Tokens at negative positions, past the table or in blocks outside the pool
    are not written, nor the scales of their pages."""
    g = _gen(3)
    D, bs, H = 64, 16, 2
    lens = [5, 4, 40, 3, 30]
    ctx = torch.tensor([3, 4, 100, 3, 30], dtype=torch.int32)  # -2 .. 3; 60 .. 100 of 64
    bt = torch.tensor([[1, -7, -7, -7], [-1, -1, -1, -1], [2, 3, 4, 5], [99, 0, 0, 0],
                       [6, 1000, -7, -7]], dtype=torch.int32)
    T = sum(lens)
    k, v = _randn(g, T, H, D).bfloat16(), _randn(g, T, H, D).bfloat16()
    caches = [small.random_cache(g, 8, bs, H, D) for _ in range(2)]
    (kc, ks), (vc, vs) = [[t.to(gpu) for t in c] for c in caches]
    ops.append_chunk_kv(k.to(gpu), v.to(gpu), kc, vc, bt.to(gpu), ctx.to(gpu),
                        ops.ChunkLayout(lens, gpu), bs, k_scales=ks, v_scales=vs)
    for got, scales, was, y in ((kc, ks, caches[0], k.double()), (vc, vs, caches[1], v.double())):
        small.check_appended(got, scales, was,
                             small.appended(y, y.abs(), *was, bt, ctx, lens, 0.0))
        for n in (0, 7):
            assert torch.equal(got[n].cpu().view(torch.uint8), was[0][n].view(torch.uint8))


def test_append_to_pages_of_the_callers_scales(gpu):
    """Pages that held a token under scales that the append itself does not write: the
    largest powers of two, and the least, which grow."""
    D, bs = 32, 8
    bytes_ = [254, 253, 250, 247, 0, 1, 16]
    n = len(bytes_)
    rows = torch.zeros(n, 1, D)
    for i, b in enumerate(bytes_):
        rows[i, 0, :4] = torch.tensor([1.0, 1.5, -1.75, 0.25]) * 2.0 ** min(b - 127, 127)
    bt = torch.arange(n, dtype=torch.int32)[:, None]
    ctx = torch.full((n,), 2, dtype=torch.int32)
    cache = (torch.ones(n, bs, 1, D).to(torch.float8_e4m3fn),
             small.to_scales(torch.tensor(bytes_)[:, None]))
    (kc, ks), (vc, vs) = [[t.to(gpu) for t in cache] for _ in range(2)]
    ops.append_chunk_kv(rows.to(gpu), rows.to(gpu), kc, vc, bt.to(gpu), ctx.to(gpu),
                        ops.ChunkLayout([1] * n, gpu), bs, k_scales=ks, v_scales=vs)
    y = rows.double()
    for c, s in ((kc, ks), (vc, vs)):
        small.check_appended(c, s, cache, small.appended(y, y.abs(), *cache, bt, ctx, [1] * n, 0.0))
        assert small.scale_bytes(s)[:, 0].tolist() == [254, 253, 250, 247, 17, 17, 17]
        assert torch.equal(small.values(c, s)[:4, 1], y[:4, 0, None])


# ------------------------------------------------------------ attention

def _attend_inputs(g, lens, before, bs, Hk, G, D, W=None):
    totals = [a + b for a, b in zip(lens, before)]
    bt, ctx, nb = _tables(g, totals, bs, W)
    q = (_randn(g, sum(lens), Hk * G, D) * torch.linspace(0.3, 2, Hk * G)[:, None]).bfloat16()
    k = small.random_cache(g, nb, bs, Hk, D, 2)
    v = small.random_cache(g, nb, bs, Hk, D, 2)
    return q, k, v, bt, ctx


def _attend(gpu, q, k, v, bt, ctx, lens, G, bs, **kw):
    kc, ks, vc, vs, qg, btg, cg = _gpu(gpu, *k, *v, q, bt, ctx)
    return ops.chunk_attention(qg, kc, vc, btg, cg, ops.ChunkLayout(lens, gpu), kc.shape[2], G,
                               bs, return_lse=True, k_scales=ks, v_scales=vs, **kw)


def _check_attend(gpu, q, k, v, bt, ctx, lens, G, bs, causal=True, check=ref.check_attend, **kw):
    out, lse = _attend(gpu, q, k, v, bt, ctx, lens, G, bs, causal=causal, **kw)
    want = ref.attend(q, small.values(*k), small.values(*v), bt, ctx, lens, G, causal)
    if check is ref.check_attend:
        check(out, want, lse)
    else:
        check(out, want)
    return out, lse


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("bs", [8, 16, 32, 64, 128])
def test_attend_few_rows(gpu, D, bs):
    """Single tokens and drafts: lengths around the tiles and pages."""
    g = _gen(D + bs)
    for Hk, G, lens, before in ((2, 4, [1, 1, 1, 1, 1], [0, 31, 32, 127, 300]),
                                (1, 1, [1], [0]), (3, 7, [4, 0, 1, 2], [65, 3, 7, 511]),
                                (2, 16, [1, 2, 3, 4], [0, 130, 64, 17])):
        x = _attend_inputs(g, lens, before, bs, Hk, G, D)
        for causal in (True, False):
            _check_attend(gpu, *x, lens, G, bs, causal)


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("bs", [8, 16, 64, 128])
def test_attend_many_rows(gpu, D, bs):
    g = _gen(D * bs)
    for Hk, G, lens, before in ((2, 4, [70, 0, 33, 1], [0, 5, 150, 40]), (1, 8, [40], [600]),
                                (2, 1, [97, 129], [31, 0])):
        x = _attend_inputs(g, lens, before, bs, Hk, G, D)
        for causal in (True, False):
            _check_attend(gpu, *x, lens, G, bs, causal)


@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_attend_over_splits(gpu, D):
    """A wide table: keys of few and of many rows are cut and joined."""
    g = _gen(D)
    x = _attend_inputs(g, [1, 3, 40], [3000, 1000, 2000], 16, 1, 2, D, W=512)
    _check_attend(gpu, *x, [1, 3, 40], 2, 16)
    few = [1] * 3
    y = _attend_inputs(g, few, [2999, 0, 700], 64, 1, 40, D)
    _check_attend(gpu, *y, few, 40, 64)


def test_attend_prompt_of_its_own_tiles(gpu):
    """128-row tiles at D = 64 (from near the start) and 256-row ones."""
    g = _gen(11)
    for n, before in ((300, 0), (260, 4200)):
        x = _attend_inputs(g, [n], [before], 16, 1, 1, 64)
        _check_attend(gpu, *x, [n], 1, 16)


@pytest.mark.parametrize("lens,before", [([2], [40]), ([90], [40])])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_attend_nan_in_unseen_places(gpu, D, lens, before):
    """NaN payloads and scales of NaN behind a context, in blocks that no table
    names, and at keys that some rows do not see."""
    g = _gen(D)
    bs, n = 16, lens[0]
    q, k, v, bt, ctx = _attend_inputs(g, lens, before, bs, 2, 2, D)
    clean, lse = _attend(gpu, q, k, v, bt, ctx, lens, 2, bs)
    total = n + before[0]
    for cache, scales in (k, v):
        last = int(bt[0, (total - 1) // bs])
        cache.view(torch.uint8)[last, (total - 1) % bs + 1:] = 0x7f
        used = set(bt[0].tolist())
        spare = [b for b in range(cache.shape[0]) if b not in used]
        cache.view(torch.uint8)[spare] = 0xff
        scales.view(torch.uint8)[spare] = 255
    out, lse2 = _attend(gpu, q, k, v, bt, ctx, lens, 2, bs)
    assert torch.equal(out, clean) and torch.equal(lse, lse2)
    # The last key's value: only the last token sees it.
    v[0].view(torch.uint8)[int(bt[0, (total - 1) // bs]), (total - 1) % bs, 0, 3] = 0x7f
    out, _ = _attend(gpu, q, k, v, bt, ctx, lens, 2, bs)
    assert torch.equal(out[:n - 1], clean[:n - 1])
    assert out[n - 1, :2, 3].isnan().all() and out[n - 1].isnan().sum() == 2


@pytest.mark.parametrize("n", [1, 60])
def test_attend_scales_of_nan(gpu, n):
    """A block's scale of NaN: its keys' scores, or its values, are NaN for the
    rows that see them."""
    g = _gen(n)
    bs, D, before = 16, 128, 100
    q, k, v, bt, ctx = _attend_inputs(g, [n], [before], bs, 2, 2, D)
    clean, _ = _attend(gpu, q, k, v, bt, ctx, [n], 2, bs)
    last = (before + n - 1) // bs           # the page of the last tokens
    for side, page in ((k, 1), (v, 1), (k, last), (v, last)):
        byte = side[1].view(torch.uint8)
        was = int(byte[int(bt[0, page]), 1])
        byte[int(bt[0, page]), 1] = 255
        out, lse = _attend(gpu, q, k, v, bt, ctx, [n], 2, bs)
        byte[int(bt[0, page]), 1] = was
        sees = torch.arange(before, before + n) >= page * bs
        assert torch.equal(out[:, :2], clean[:, :2])
        assert out[sees][:, 2:].isnan().all()
        assert torch.equal(out[~sees], clean[~sees])


def test_attend_extreme_scales(gpu):
    """Scales of the least and largest exponents, exactly brought to bf16.  With the
    largest a single key: sums over keys are taken before the division, and two
    values of 2.98e38 already pass what 32 bits hold (3.40e38)."""
    D, bs = 64, 16
    q = torch.zeros(1, 1, D)
    q[0, 0, 0] = 1.0
    k = torch.zeros(2, bs, 1, D).to(torch.float8_e4m3fn)
    v = torch.full((2, bs, 1, D), 448.0).to(torch.float8_e4m3fn)
    for byte in (17, 246, 127):
        scales = small.to_scales(torch.full((2, 1), byte))
        out = ops.chunk_attention(*_gpu(gpu, q.bfloat16(), k, v,
                                        torch.tensor([[1]], dtype=torch.int32),
                                        torch.tensor([1 if byte == 246 else 9],
                                                     dtype=torch.int32)),
                                  ops.ChunkLayout([1], gpu), 1, 1, bs,
                                  k_scales=scales.to(gpu), v_scales=scales.to(gpu))
        want = 448.0 * 2.0 ** (byte - 127)
        assert (out.double().cpu() / want - 1).abs().max() <= 2.0 ** -8


def test_attend_rows_without_keys(gpu):
    g = _gen(2)
    bs, D = 16, 128
    q, k, v, bt, ctx = _attend_inputs(g, [1, 80, 2], [20, 9, 5], bs, 2, 2, D)
    bt[0] = -1
    bt[1, 0] = 10 ** 6  # the first 16 keys are none
    out, lse = _check_attend(gpu, q, k, v, bt, ctx, [1, 80, 2], 2, bs)
    assert (out[0] == 0).all() and (lse[0] == -math.inf).all()
    ctx[2] = 0
    _check_attend(gpu, q, k, v, bt, ctx, [1, 80, 2], 2, bs)


def test_attend_strided_queries_and_output_in_place(gpu):
    g = _gen(4)
    lens, bs, D = [3, 70], 16, 128
    q, k, v, bt, ctx = _attend_inputs(g, lens, [40, 100], bs, 2, 4, D)
    want, _ = _attend(gpu, q, k, v, bt, ctx, lens, 4, bs)
    wide = torch.cat([q, q, q], 1).to(gpu)[:, 8:16]
    kc, ks, vc, vs, btg, cg = _gpu(gpu, *k, *v, bt, ctx)
    args = (kc, vc, btg, cg, ops.ChunkLayout(lens, gpu), 2, 4, bs)
    assert torch.equal(ops.chunk_attention(wide, *args, k_scales=ks, v_scales=vs), want)
    qg = q.to(gpu)
    ops.chunk_attention(qg, *args, out=qg, k_scales=ks, v_scales=vs)
    assert torch.equal(qg, want)


@pytest.mark.parametrize("n", [1, 80])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_attend_scales_of_every_size(gpu, n, D):
    """Scales that only a caller's own pages have, of values that bf16 holds."""
    bs = 16
    q = torch.zeros(n, 1, D)
    for byte, payload in ((0, 448.0), (1, 1.5), (8, -2.0), (16, 448.0), (250, 1.75), (254, -1.0)):
        k = torch.zeros(8, bs, 1, D).to(torch.float8_e4m3fn)
        v = torch.full((8, bs, 1, D), payload).to(torch.float8_e4m3fn)
        scales = small.to_scales(torch.full((8, 1), byte))
        # Causal: the first token sees one key, so that no sum passes 32 bits there.
        out = ops.chunk_attention(*_gpu(gpu, q.bfloat16(), k, v,
                                        torch.arange(8, dtype=torch.int32)[None],
                                        torch.tensor([n], dtype=torch.int32)),
                                  ops.ChunkLayout([n], gpu), 1, 1, bs,
                                  k_scales=scales.to(gpu), v_scales=scales.to(gpu))
        want = payload * 2.0 ** (byte - 127)
        got = (out if byte < 200 else out[:1]).double().cpu()
        assert (got / want - 1).abs().max() <= 2.0 ** -8, (byte, got.flatten()[:2], want)


@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_attend_few_rows_keeps_16_bits_of_the_weights(gpu, D):
    """Half of the keys have a weight of 1 and values of 1, the others a weight just
    above 1/2, which one bf16 rounds to it, and values of -2: what is left of the sum
    is what that rounding loses."""
    bs, n = 16, 64
    for lens, before, G in (([1], [n - 1], 4), ([32 // 7], [n - 32 // 7], 7), ([1], [5000], 1)):
        total = lens[0] + before[0]
        bt, ctx, nb = _tables(_gen(D), [total], bs)
        k = torch.zeros(nb, bs, 1, D)
        k[:, 1::2, 0, 0], k[:, 1::2, 0, 1] = -0.6875, -0.1171875
        v = torch.ones(nb, bs, 1, D)
        v[:, 1::2] = -2.0
        q = torch.zeros(sum(lens), G, D)
        q[..., 0], q[..., 1] = 1.0, 2.0 ** -5
        ones = small.to_scales(torch.full((nb, 1), 127))
        k, v = (k.to(torch.float8_e4m3fn), ones), (v.to(torch.float8_e4m3fn), ones)
        out, lse = _attend(gpu, q.bfloat16(), k, v, bt, ctx, lens, G, bs, scale=1.0)
        want = ref.attend(q.bfloat16(), small.values(*k), small.values(*v), bt, ctx, lens, G,
                          scale=1.0, parts=2)
        ref.check_attend(out, want, lse)


@pytest.mark.parametrize("D,most", [(32, 64), (64, 64), (128, 64), (256, 32)])
@pytest.mark.parametrize("G", [1, 4, 7])
def test_attend_few_rows_within_16_bits(gpu, D, most, G):
    """As many rows as count as few, over one workgroup's keys and over many's."""
    g = _gen(D + G)
    bs, Hk = 16, 2
    lens = [most // G, 1, 2]
    x = _attend_inputs(g, lens, [40, 2500, 0], bs, Hk, G, D)
    out, lse = _attend(gpu, *x, lens, G, bs)
    q, k, v, bt, ctx = x
    want = ref.attend(q, small.values(*k), small.values(*v), bt, ctx, lens, G, parts=2)
    ref.check_attend(out, want, lse)


# ------------------------------------------------------------ weights of keys

def _weigh_inputs(g, lens, before, bs, Hk, G, D, bits, W=None):
    q, k, v, bt, ctx = _attend_inputs(g, lens, before, bs, Hk, G, D, W)
    keys = small.values(*k)
    if bits == 16:
        k = (keys.to(torch.bfloat16), None)
        keys = k[0].double()
    B, S = bt.shape[0], bt.shape[1] * bs + 5
    weights = torch.rand(B, Hk, S, generator=g)
    return q, k, keys, bt, ctx, weights


def _lse(q, keys, bt, ctx, lens, G, causal):
    return ref.attend(q, keys, keys, bt, ctx, lens, G, causal)[1].float()


def _weigh(gpu, weights, q, lse, k, bt, ctx, lens, G, bs, **kw):
    kc, ks, wg, qg, lg, btg, cg = _gpu(gpu, *k, weights, q, lse, bt, ctx)
    got = ops.add_key_weights(wg, qg, lg, kc, btg, cg, ops.ChunkLayout(lens, gpu), kc.shape[2], G,
                              bs, k_scales=ks, **kw)
    assert got is wg
    return got


def _check_weigh(got, want, slack, weights):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    err = (got - want).abs()
    fine = want.isfinite()
    assert not (err > slack)[fine].any(), (err - slack)[fine].max()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    still = (slack == 0) & (want == weights.double())
    assert torch.equal(got[still], want[still])


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("D,bs", [(32, 8), (64, 128), (128, 16), (256, 32), (128, 8)])
def test_weigh(gpu, bits, D, bs):
    g = _gen(D + bs + bits)
    for Hk, G, lens, before in ((2, 4, [1, 1, 0, 1, 1], [0, 31, 50, 127, 300]),
                                (1, 1, [1], [0]), (3, 7, [4, 0, 1, 9], [65, 3, 7, 511]),
                                (2, 5, [70, 7, 33, 1], [0, 5, 250, 40])):
        q, k, keys, bt, ctx, w = _weigh_inputs(g, lens, before, bs, Hk, G, D, bits)
        for causal in (True, False):
            lse = _lse(q, keys, bt, ctx, lens, G, causal)
            for window in (0, 1, 6):
                got = _weigh(gpu, w, q, lse, k, bt, ctx, lens, G, bs, causal=causal,
                             window=window)
                _check_weigh(got, *small.key_weights(w, q, lse, keys, bt, ctx, lens, G, causal,
                                                     window=window), w)


@pytest.mark.parametrize("bits", [8, 16])
def test_weigh_in_segments(gpu, bits):
    """More rows than a segment, with a sequence of few rows and one of a single
    segment beside it; and of more segments than there are at 512 rows each."""
    g = _gen(bits)
    for lens, before, G, Hk, D in (([300, 1, 30], [40, 700, 3], 4, 2, 64),
                                   ([700], [0], 32, 1, 32)):
        q, k, keys, bt, ctx, w = _weigh_inputs(g, lens, before, 16, Hk, G, D, bits, W=80)
        lse = _lse(q, keys, bt, ctx, lens, G, True)
        got = _weigh(gpu, w, q, lse, k, bt, ctx, lens, G, 16)
        want = small.key_weights(w, q, lse, keys, bt, ctx, lens, G)
        _check_weigh(got, *want, w)
        again = _weigh(gpu, w, q, lse, k, bt, ctx, lens, G, 16)
        assert torch.equal(got, again)


def test_weigh_sums_to_the_rows(gpu):
    """Each row's weights sum to one over the keys that it sees."""
    g = _gen(8)
    lens, before, bs, Hk, G, D = [1, 200, 17], [600, 100, 0], 16, 2, 4, 128
    q, k, v, bt, ctx = _attend_inputs(g, lens, before, bs, Hk, G, D)
    out, lse = _attend(gpu, q, k, v, bt, ctx, lens, G, bs)
    w = torch.zeros(3, Hk, bt.shape[1] * bs)
    got = _weigh(gpu, w, q, lse, k, bt, ctx, lens, G, bs).double().sum(-1).cpu()
    want = torch.tensor(lens).double()[:, None] * G
    # A weight is off by the attention's and this kernel's errors of the score.
    assert ((got / want) - 1).abs().max() < 1e-4


@pytest.mark.parametrize("n", [1, 3, 60])
def test_weigh_of_what_is_not_finite(gpu, n):
    """Keys outside the pool, rows that saw nothing, infinite and NaN keys behind
    a context and at keys that some rows do not see."""
    g = _gen(n)
    bs, Hk, G, D, before = 16, 2, 4, 64, 70
    q, k, keys, bt, ctx, w = _weigh_inputs(g, [n], [before], bs, Hk, G, D, 16)
    total = before + n
    bt[0, 2] = -5
    lse = _lse(q, keys, bt, ctx, [n], G, True)
    lse[0, 1] = -math.inf
    kc = k[0]
    kc[int(bt[0, -1]), (total - 1) % bs + 1:] = math.nan
    for value in (math.nan, math.inf, -math.inf):
        # the last key: only the last token sees it; its own log-sum-exp is as before
        kc[int(bt[0, (total - 1) // bs]), (total - 1) % bs, 0, 5] = value
        got = _weigh(gpu, w, q, lse, k, bt, ctx, [n], G, bs)
        want, slack = small.key_weights(w, q, lse, kc.double(), bt, ctx, [n], G)
        _check_weigh(got, want, torch.nan_to_num(slack, nan=0.0, posinf=0.0), w)


def test_weigh_strides_and_other_scales(gpu):
    g = _gen(5)
    lens, before, bs, Hk, G, D = [2, 40], [100, 30], 16, 2, 4, 128
    q, k, keys, bt, ctx, w = _weigh_inputs(g, lens, before, bs, Hk, G, D, 8)
    lse = _lse(q, keys, bt, ctx, lens, G, True)
    want = _weigh(gpu, w, q, lse, k, bt, ctx, lens, G, bs)
    wide = torch.cat([q, q], 1).to(gpu)[:, 8:]
    l2 = torch.cat([lse, lse], 1).to(gpu)[:, 8:]
    pad = torch.zeros(3, 8, D, dtype=torch.bfloat16, device=gpu)
    for qq, ll in ((wide, l2), (torch.cat([wide, pad]), torch.cat([l2, torch.ones(3, 8).to(gpu)]))):
        kc, ks, wg, btg, cg = _gpu(gpu, *k, w, bt.long(), ctx.long())
        got = ops.add_key_weights(wg, qq, ll, kc, btg, cg, ops.ChunkLayout(lens, gpu), Hk, G, bs,
                                  k_scales=ks)
        assert torch.equal(got, want)
    lse = torch.zeros_like(lse)
    got = _weigh(gpu, w, q, lse, k, bt, ctx, lens, G, bs, scale=0.01)
    _check_weigh(got, *small.key_weights(w, q, lse, keys, bt, ctx, lens, G, scale=0.01), w)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("n", [1, 60])
def test_weigh_context_past_the_table(gpu, bits, n):
    """Contexts of more keys than the tables hold, which are not a multiple of a
    tile, with weights of the tables' keys and no more."""
    g = _gen(n + bits)
    bs, Hk, G, D = 8, 2, 4, 64
    q, k, keys, bt, ctx, w = _weigh_inputs(g, [n, n], [40 - n, 40 - n] if n == 1 else [12, 20],
                                           bs, Hk, G, D, bits)
    w = w[..., :bt.shape[1] * bs].contiguous()
    ctx = ctx + torch.tensor([300, 5], dtype=torch.int32)
    for causal in (True, False):
        lse = _lse(q, keys, bt, ctx, [n, n], G, causal)
        got = _weigh(gpu, w, q, lse, k, bt, ctx, [n, n], G, bs, causal=causal)
        _check_weigh(got, *small.key_weights(w, q, lse, keys, bt, ctx, [n, n], G, causal), w)


@pytest.mark.parametrize("bits", [8, 16])
def test_weigh_queries_far_apart(gpu, bits):
    """Heads 2^23 values apart (of 65536 tokens, head after head), tokens 2^23 and 2^25
    apart: as the same queries side by side."""
    g = _gen(bits)
    lens, before, bs, Hk, G, D = [1, 40, 3], [100, 30, 200], 16, 2, 4, 128
    q, k, keys, bt, ctx, w = _weigh_inputs(g, lens, before, bs, Hk, G, D, bits)
    lse = _lse(q, keys, bt, ctx, lens, G, True)
    want = _weigh(gpu, w, q, lse, k, bt, ctx, lens, G, bs)
    T, H = q.shape[:2]
    for st, sh in ((D, 1 << 23), (1 << 23, D), (1 << 26, D)):
        far = torch.empty((T - 1) * st + (H - 1) * sh + D, dtype=q.dtype, device=gpu)
        far = far.as_strided((T, H, D), (st, sh, 1))
        far.copy_(q)
        got = _weigh(gpu, w, far, lse, k, bt, ctx, lens, G, bs)
        assert torch.equal(got, want)
        for window in (1, 5):
            assert torch.equal(_weigh(gpu, w, far, lse, k, bt, ctx, lens, G, bs, window=window),
                               _weigh(gpu, w, q, lse, k, bt, ctx, lens, G, bs, window=window))
        del far


@pytest.mark.parametrize("n", [1, 60])
def test_weigh_scales_of_nan_and_the_largest(gpu, n):
    """Log-sum-exps of the caller's own: keys of a block whose scale is NaN get NaN of
    the rows that see them, zeros at the largest scale have a score of zero."""
    g = _gen(n)
    bs, Hk, G, D, before = 16, 2, 4, 64, 100
    q, k, keys, bt, ctx, w = _weigh_inputs(g, [n], [before], bs, Hk, G, D, 8)
    lse = torch.zeros(n, Hk * G)
    k[1].view(torch.uint8)[bt[0, [1, (before + n - 1) // bs]].long(), 1] = 255
    keys = small.values(*k)
    got = _weigh(gpu, w, q, lse, k, bt, ctx, [n], G, bs, scale=0.01)
    want, slack = small.key_weights(w, q, lse, keys, bt, ctx, [n], G, scale=0.01)
    assert want[0, 1, bs:2 * bs].isnan().all() and not want[0, 0].isnan().any()
    _check_weigh(got, want, torch.nan_to_num(slack, nan=0.0), w)
    k = (torch.zeros_like(k[0].float()).to(k[0].dtype), small.to_scales(torch.full(k[1].shape, 246)))
    got = _weigh(gpu, w, q, lse, k, bt, ctx, [n], G, bs, scale=400.0)
    _check_weigh(got, *small.key_weights(w, q, lse, small.values(*k), bt, ctx, [n], G,
                                         scale=400.0), w)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("window", [0, 2, 50])
def test_weigh_chunks_longer_than_their_contexts(gpu, bits, window):
    """Tokens at negative positions see nothing and bring no key."""
    g = _gen(bits + window)
    lens, bs, Hk, G, D = [4, 70, 3, 40, 7], 16, 2, 4, 64
    q, k, keys, bt, ctx, w = _weigh_inputs(g, lens, [0] * 5, bs, Hk, G, D, bits)
    ctx = torch.tensor([2, 33, 0, -9, 7], dtype=torch.int32)
    for causal in (True, False):
        lse = _lse(q, keys, bt, ctx, lens, G, causal)
        got = _weigh(gpu, w, q, lse, k, bt, ctx, lens, G, bs, causal=causal, window=window)
        _check_weigh(got, *small.key_weights(w, q, lse, keys, bt, ctx, lens, G, causal,
                                             window=window), w)


# ------------------------------------------------------------ eviction

def _evict_inputs(g, totals, bs, H, D, bits, W=None):
    bt, ctx, nb = _tables(g, totals, bs, W)
    k, v = (small.random_cache(g, nb, bs, H, D) for _ in range(2))
    if bits == 16:
        k, v = ((small.values(*c).to(torch.bfloat16), None) for c in (k, v))
    w = torch.exp(2 * _randn(g, len(totals), H, bt.shape[1] * bs + 3))
    return bt, ctx, k, v, w


def _check_evict(gpu, bt, ctx, k, v, w, keep, bs, sinks, recent):
    scales = None if k[1] is None else [k[1], v[1]]
    want = small.evicted(w, [k[0], v[0]], bt, ctx, keep, sinks, recent, scales)
    kc, ks, vc, vs, wg, btg, cg = _gpu(gpu, *k, *v, w, bt, ctx)
    kept = ops.evict_tokens(wg, kc, vc, btg, cg, keep, bs, sinks, recent, ks, vs)
    assert kept.dtype == torch.int32 and torch.equal(kept.cpu(), want[0])
    # Bits, so that NaN and zeros of both signs are told apart.
    assert torch.equal(wg.cpu().view(torch.int32), want[1].view(torch.int32))
    if scales:
        for got, s, c, x in ((kc, ks, want[2][0], want[3][0]), (vc, vs, want[2][1], want[3][1])):
            assert torch.equal(small.scale_bytes(s), small.scale_bytes(x))
            a, b = got.cpu().view(torch.uint8), c.view(torch.uint8)
            nan = (a & 0x7f == 0x7f) & (b & 0x7f == 0x7f)  # it has two encodings
            bad = (a != b) & ~nan
            assert not bad.any(), bad.nonzero()[:3]
    else:
        assert torch.equal(kc.cpu().view(torch.int16), want[2][0].view(torch.int16))
        assert torch.equal(vc.cpu().view(torch.int16), want[2][1].view(torch.int16))
    assert torch.equal(btg.cpu(), bt) and torch.equal(cg.cpu(), ctx)
    return kept


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("D,bs,H", [(128, 16, 2), (64, 8, 3), (32, 128, 1), (256, 64, 2),
                                    (32, 8, 2), (128, 32, 3)])
def test_evict(gpu, bits, D, bs, H):
    g = _gen(D + bs + bits)
    bt, ctx, k, v, w = _evict_inputs(g, [300, 0, 1, 97, 150], bs, H, D, bits)
    for keep, sinks, recent in ((97, 4, 16), (1, 0, 0), (1, 0, 1), (1, 1, 0), (128, 0, 128),
                                (96, 0, 0), (150, 10, 140), (149, 3, 100), (299, 1, 64),
                                (300, 0, 0), (400, 4, 8), (64, 64, 0)):
        _check_evict(gpu, bt, ctx, k, v, w, keep, bs, sinks, recent)


@pytest.mark.parametrize("bits", [8, 16])
def test_evict_long_rows(gpu, bits):
    """Several steps of the workgroup's walk, with many equal weights."""
    g = _gen(bits)
    bt, ctx, k, v, w = _evict_inputs(g, [9001, 4100], 16, 1, 32, bits)
    _check_evict(gpu, bt, ctx, k, v, w, 4097, 16, 4, 300)
    w[:, :, ::3] = 0.25
    w[:, :, 1::5] = 0.0
    _check_evict(gpu, bt, ctx, k, v, w, 4000, 16, 4, 300)
    _check_evict(gpu, bt, ctx, k, v, torch.zeros_like(w), 4000, 16, 4, 300)


@pytest.mark.parametrize("bits", [8, 16])
def test_evict_rows_of_chunks(gpu, bits):
    """Tables of more than 16384 keys: rows of several chunks, of one, empty ones, cuts
    in the first chunk and in later ones, equal weights over several chunks."""
    g = _gen(bits)
    bt, ctx, k, v, w = _evict_inputs(g, [20000, 9000, 5, 17000], 64, 2, 32, bits)
    for keep, sinks, recent in ((8192, 4, 256), (16500, 0, 0), (8200, 3, 8000), (100, 100, 0),
                                (1, 0, 0), (30000, 1, 2), (17000, 8192, 8192)):
        _check_evict(gpu, bt, ctx, k, v, w, keep, 64, sinks, recent)
    w[:, :, ::2] = 1.0
    _check_evict(gpu, bt, ctx, k, v, w, 9500, 64, 4, 100)
    _check_evict(gpu, bt, ctx, k, v, torch.zeros_like(w), 8193, 64, 1, 1)
    w[0, 0, :12] = torch.tensor([math.nan, -math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45,
                                 -1e-45, -1.0, 3e38, -3e38, math.nan])
    bt[0, 5], bt[3, 200] = -1, 10 ** 7
    _check_evict(gpu, bt, ctx, k, v, w, 12000, 64, 0, 33)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("D,bs", [(128, 16), (64, 8), (32, 64), (256, 32), (128, 128)])
def test_evict_of_many_sequences(gpu, bits, D, bs):
    """As many sequences and heads as have a workgroup each for everything."""
    g = _gen(D + bs + bits + 1)
    totals = [300, 0, 1, 97, 150, 299, 98, 33, 128, 129, 255, 256, 257, 12, 101, 200, 64, 190]
    bt, ctx, k, v, w = _evict_inputs(g, totals, bs, 4, D, bits)
    for keep, sinks, recent in ((97, 4, 16), (1, 0, 0), (1, 0, 1), (128, 0, 128), (96, 0, 0),
                                (100, 7, 0), (150, 10, 140), (255, 3, 100), (64, 64, 0)):
        _check_evict(gpu, bt, ctx, k, v, w, keep, bs, sinks, recent)
    w[:, :, ::3] = 0.25
    bt[0, 1], bt[4, 0], bt[9, 1] = -1, 10 ** 7, 2 ** 31 - 1
    ctx[5] = bt.shape[1] * bs + 40
    _check_evict(gpu, bt, ctx, k, v, w, 90, bs, 4, 20)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("total", [5000, 9000])
def test_evict_of_many_long_rows(gpu, bits, total):
    """Last tokens of several rounds, which move by less and by more than a page."""
    g = _gen(total + bits)
    totals = [total, total - 3, total - 700] + [20] * 29
    bt, ctx, k, v, w = _evict_inputs(g, totals, 16, 8, 32, bits)
    w[0, :, ::5] = math.nan
    for keep, sinks, recent in ((total - 5, 4, 2500), (total - 1500, 0, 1100), (2000, 1, 1999),
                                (total - 701, 0, 0)):
        _check_evict(gpu, bt, ctx, k, v, w, keep, 16, sinks, recent)


def test_evict_weights_of_every_kind(gpu):
    g = _gen(9)
    bt, ctx, k, v, w = _evict_inputs(g, [200], 16, 2, 64, 8)
    w[0, 0, :12] = torch.tensor([math.nan, -math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45,
                                 -1e-45, -1.0, 3e38, -3e38, math.nan])
    w[0, 1, 100:140] = -torch.rand(40, generator=g)
    w[0, 1, 140:160] = -0.0
    w[0, 1, 160:180] = 0.0
    for keep, sinks, recent in ((120, 0, 0), (5, 0, 0), (6, 2, 2), (170, 0, 20), (197, 3, 1)):
        _check_evict(gpu, bt, ctx, k, v, w, keep, 16, sinks, recent)


@pytest.mark.parametrize("bits", [8, 16])
def test_evict_blocks_outside_the_pool(gpu, bits):
    """Tokens of such blocks are not moved, and nothing outside is touched."""
    g = _gen(bits)
    bt, ctx, k, v, w = _evict_inputs(g, [200, 100], 16, 2, 64, bits)
    bt[0, 1], bt[0, 9], bt[1, 2] = -1, 10 ** 7, 2 ** 31 - 1
    _check_evict(gpu, bt, ctx, k, v, w, 90, 16, 4, 20)


def test_evict_context_past_the_table(gpu):
    g = _gen(6)
    bt, ctx, k, v, w = _evict_inputs(g, [64, 64], 16, 2, 64, 8)
    ctx += 1000
    ctx[1] = -5
    _check_evict(gpu, bt, ctx, k, v, w, 40, 16, 4, 8)


def test_evict_scales_that_far_apart(gpu):
    """Payloads that vanish at the larger scale, NaN payloads and a scale of NaN."""
    g = _gen(12)
    bt, ctx, k, v, w = _evict_inputs(g, [256], 16, 2, 64, 8)
    for c, s in (k, v):
        s.view(torch.uint8).copy_(torch.randint(17, 247, s.shape, generator=g).to(torch.uint8))
        s.view(torch.uint8)[3, 1] = 255
        c.view(torch.uint8)[:, 3, :, 5] = 0x7f
    _check_evict(gpu, bt, ctx, k, v, w, 100, 16, 4, 30)


def test_evict_twice_in_place(gpu):
    """A cut of what a cut left, and one that finds nothing more to do."""
    g = _gen(31)
    bt, ctx, k, v, w = _evict_inputs(g, [260, 90], 16, 2, 64, 8)
    kc, ks, vc, vs, wg, btg, cg = _gpu(gpu, *k, *v, w, bt, ctx)
    caches, scales, weights = [k[0], v[0]], [k[1], v[1]], w
    for keep, recent in ((200, 30), (77, 20), (77, 0)):
        kept = ops.evict_tokens(wg, kc, vc, btg, cg, keep, 16, 3, recent, ks, vs)
        cg.clamp_(max=keep)
        want, weights, caches, scales = small.evicted(weights, caches, bt, ctx, keep, 3, recent,
                                                      scales)
        ctx = ctx.clamp(max=keep)
        assert torch.equal(kept.cpu(), want)
        assert torch.equal(wg.cpu(), weights)
        for got, c in ((kc, caches[0]), (vc, caches[1])):
            x, y = got.cpu().view(torch.uint8), c.view(torch.uint8)
            assert ((x == y) | (x & 0x7f == 0x7f) & (y & 0x7f == 0x7f)).all()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("W,bs,D", [(300, 64, 32), (40, 128, 256), (20, 16, 128)])
def test_evict_keeps_all_that_the_tables_hold(gpu, bits, W, bs, D):
    g = _gen(W + bits)
    bt, ctx, k, v, w = _evict_inputs(g, [W * bs, 0, 77], bs, 1, D, bits)
    ctx[0] += 9  # past the table
    for keep in (W * bs, W * bs + 100):
        for sinks, recent in ((0, 0), (4, 64), (0, keep)):
            _check_evict(gpu, bt, ctx, k, v, w, keep, bs, sinks, recent)


# ------------------------------------------------------------ sizes

def test_more_sequences_than_a_wave_has_lanes(gpu):
    """150 sequences, of none, one and many tokens, in all four."""
    g = _gen(41)
    bs, Hk, G, D = 8, 2, 3, 32
    lens = [(1, 0, 2, 15)[b % 4] for b in range(150)]
    before = [int(x) for x in torch.randint(0, 60, (150,), generator=g)]
    totals = [a + b for a, b in zip(lens, before)]
    q, k, v, bt, ctx = _attend_inputs(g, lens, before, bs, Hk, G, D)
    new = [_randn(g, sum(lens), Hk, D).bfloat16() for _ in range(2)]
    kc, ks, vc, vs, btg, cg = _gpu(gpu, *k, *v, bt, ctx)
    ops.append_chunk_kv(new[0].to(gpu), new[1].to(gpu), kc, vc, btg, cg,
                        ops.ChunkLayout(lens, gpu), bs, k_scales=ks, v_scales=vs)
    for got, scales, was, y in ((kc, ks, k, new[0]), (vc, vs, v, new[1])):
        small.check_appended(got, scales, was, small.appended(
            y.double(), y.double().abs(), *was, bt, ctx, lens, 0.0))
    _check_attend(gpu, q, k, v, bt, ctx, lens, G, bs)
    w = torch.rand(150, Hk, bt.shape[1] * bs, generator=g)
    keys = small.values(*k)
    lse = _lse(q, keys, bt, ctx, lens, G, True)
    _check_weigh(_weigh(gpu, w, q, lse, k, bt, ctx, lens, G, bs),
                 *small.key_weights(w, q, lse, keys, bt, ctx, lens, G), w)
    _check_evict(gpu, bt, ctx, k, v, w, 30, bs, 2, 9)


@pytest.mark.parametrize("n,G", [(1, 128), (9, 33), (40, 6), (3, 100)])
def test_weigh_groups_of_any_size(gpu, n, G):
    """Query heads of a group that no pass of rows is a multiple of, and rows that saw
    nothing among those of which every key is seen."""
    g = _gen(G)
    bs, Hk, D, before = 16, 2, 64, 700
    q, k, keys, bt, ctx, w = _weigh_inputs(g, [n, 2], [before, 5], bs, Hk, G, D, 8)
    lse = _lse(q, keys, bt, ctx, [n, 2], G, True)
    lse[torch.rand(lse.shape, generator=g) < 0.1] = -math.inf
    for causal in (True, False):
        got = _weigh(gpu, w, q, lse, k, bt, ctx, [n, 2], G, bs, causal=causal)
        _check_weigh(got, *small.key_weights(w, q, lse, keys, bt, ctx, [n, 2], G, causal), w)


def test_weigh_with_more_heads_than_compute_units(gpu):
    g = _gen(51)
    bs, Hk, G, D = 16, 300, 1, 32
    for lens, before in (([1, 2], [30, 5]), ([40], [3])):
        q, k, keys, bt, ctx, w = _weigh_inputs(g, lens, before, bs, Hk, G, D, 16)
        lse = _lse(q, keys, bt, ctx, lens, G, True)
        _check_weigh(_weigh(gpu, w, q, lse, k, bt, ctx, lens, G, bs),
                     *small.key_weights(w, q, lse, keys, bt, ctx, lens, G), w)


def test_queries_that_heads_share(gpu):
    """A stride of zero between heads."""
    g = _gen(61)
    bs, Hk, G, D, lens, before = 16, 2, 4, 64, [1, 30], [40, 9]
    q, k, keys, bt, ctx, w = _weigh_inputs(g, lens, before, bs, Hk, G, D, 8)
    one = q[:, :1].to(gpu).expand(-1, Hk * G, -1)
    kc, ks, wg, btg, cg = _gpu(gpu, *k, w, bt, ctx)
    layout = ops.ChunkLayout(lens, gpu)
    got = [ops.chunk_attention(x, kc, kc, btg, cg, layout, Hk, G, bs, return_lse=True, k_scales=ks,
                               v_scales=ks) for x in (one, one.contiguous())]
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    sums = [ops.add_key_weights(wg.clone(), x, got[0][1], kc, btg, cg, layout, Hk, G, bs,
                                k_scales=ks) for x in (one, one.contiguous())]
    assert torch.equal(*sums)


@pytest.mark.parametrize("bits", [8, 16])
def test_pools_past_32_bits(gpu, bits):
    """Blocks whose bytes lie past 2^32 (and values past 2^31): all four as over a
    small pool of the same content."""
    g = _gen(91)
    bs, Hk, G, D = 128, 8, 2, 128 if bits == 8 else 256
    lens, before = [1, 40, 70], [500, 300, 0]
    totals = [a + b for a, b in zip(lens, before)]
    bt, ctx, nb = _tables(g, totals, bs, spare=0)
    per = bs * Hk * D * bits // 8
    far = 2 ** 32 // per + nb
    ids = torch.randperm(nb, generator=g)  # alternately from the start and past 2^32
    where = torch.where(ids % 2 == 0, ids, far - nb + ids).int()
    wide = bt.clone()
    wide[bt >= 0] = where[bt[bt >= 0].long()]
    assert int(wide.max()) * per >= 2 ** 32
    keys, vals = (small.random_cache(g, nb, bs, Hk, D) for _ in range(2))
    if bits == 16:
        keys, vals = ((small.values(*c).to(torch.bfloat16), None) for c in (keys, vals))
    q, k, v = (_randn(g, sum(lens), n, D).bfloat16().to(gpu) for n in (Hk * G, Hk, Hk))
    w = torch.rand(3, Hk, bt.shape[1] * bs, generator=g)
    layout = ops.ChunkLayout(lens, gpu)

    def run(tables, pools):
        (kc, ks), (vc, vs) = pools
        bt, cg, wg = tables.to(gpu), ctx.to(gpu), w.to(gpu)
        ops.append_chunk_kv(k, v, kc, vc, bt, cg, layout, bs, k_scales=ks, v_scales=vs)
        out, lse = ops.chunk_attention(q, kc, vc, bt, cg, layout, Hk, G, bs, return_lse=True,
                                       k_scales=ks, v_scales=vs)
        ops.add_key_weights(wg, q, lse, kc, bt, cg, layout, Hk, G, bs, k_scales=ks)
        kept = ops.evict_tokens(wg, kc, vc, bt, cg, 200, bs, 4, 30, ks, vs)
        return [out, lse, wg, kept]

    def bytes_of(t):
        return None if t is None else t.view(torch.uint8)

    def pool(c, n):
        """c's blocks at `where` of n."""
        x, s = c
        big = torch.zeros(n, *x.shape[1:], dtype=torch.uint8 if bits == 8 else x.dtype, device=gpu)
        big[where.long()] = (bytes_of(x) if bits == 8 else x).to(gpu)
        if s is None:
            return big, None
        scales = torch.full((n, Hk), 127, dtype=torch.uint8, device=gpu)
        scales[where.long()] = bytes_of(s).to(gpu)
        return big.view(x.dtype), scales.view(s.dtype)

    near = [[None if t is None else t.to(gpu) for t in c] for c in (keys, vals)]
    want = run(bt, near)
    pools = [pool(keys, far), pool(vals, far)]
    got = run(wide, pools)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    for c, d in zip(pools, near):
        for x, y in zip(c, d):
            if x is not None:
                at = where.long().to(gpu)
                assert torch.equal(bytes_of(x)[at], bytes_of(y))


# ------------------------------------------------------------ together

@pytest.mark.parametrize("bits", [8, 16])
def test_a_serving_loop(gpu, bits):
    """A manager's prompts, then single tokens, cut again and again: positions that
    the caller counts, every cached value that of the token which should be there, and
    each step's attention by its formula over the cache."""
    g = _gen(71)
    bs, Hk, G, D, B, keep = 16, 2, 4, 64, 3, 48
    cache = PagedKVCache(40, bs, Hk, D, device=gpu,
                         dtype=torch.float8_e4m3fn if bits == 8 else torch.bfloat16)
    mgr = SequenceKVManager(cache, B, 160)
    scales = dict(k_scales=cache.k_scales, v_scales=cache.v_scales)
    table = ops.RotaryTable.build(D, 256, device=gpu)
    weights = torch.zeros(B, Hk, mgr.block_tables.shape[1] * bs, device=gpu)
    norm = (1 + 0.2 * _randn(g, D)).to(gpu)
    tokens = [[] for _ in range(B)]  # (key, value) rows of [Hk, D] as they were appended
    ids = [[[] for _ in range(Hk)] for _ in range(B)]
    seen = [0] * B

    def step(lens):
        layout = ops.ChunkLayout(lens, gpu)
        T = sum(lens)
        q, k, v = ((_randn(g, T, n, D) * torch.exp(_randn(g, T, 1, 1))).bfloat16().to(gpu)
                   for n in (Hk * G, Hk, Hk))
        pos = torch.cat([torch.arange(s, s + n) for s, n in zip(seen, lens)]).to(gpu)
        q, k = ops.qk_norm_rope(q, k, pos, table, norm, norm)
        mgr.append_chunk_kv(k, v, layout)
        at = 0
        for b, n in enumerate(lens):
            for i in range(n):
                for h in range(Hk):
                    ids[b][h].append(len(tokens[b]))
                tokens[b].append((k[at + i].double().cpu(), v[at + i].double().cpu()))
            at += n
            seen[b] += n
        out, lse = ops.chunk_attention(q, cache.k_cache, cache.v_cache, mgr.block_tables,
                                       mgr.context_lens, layout, Hk, G, bs, return_lse=True,
                                       **scales)
        ops.add_key_weights(weights, q, lse, cache.k_cache, mgr.block_tables, mgr.context_lens,
                            layout, Hk, G, bs, k_scales=cache.k_scales)
        values = [small.values(c.cpu(), s.cpu()) if bits == 8 else c.double().cpu() for c, s in
                  ((cache.k_cache, cache.k_scales), (cache.v_cache, cache.v_scales))]
        bt, ctx = mgr.block_tables.cpu(), mgr.context_lens.cpu()
        assert ctx.tolist() == [len(x[0]) for x in ids] == mgr._ctx_host
        ref.check_attend(out, ref.attend(q.cpu(), *values, bt, ctx, lens, G, True), lse)
        for b in range(B):
            slot = torch.arange(int(ctx[b]))
            blk = bt[b].long()[slot // bs]
            for h in range(Hk):
                for i, (got, s) in enumerate(zip(values, scales.values())):
                    want = torch.stack([tokens[b][t][i][h] for t in ids[b][h]])
                    x = got[blk, slot % bs, h]
                    if bits == 16:
                        assert torch.equal(x, want)
                        continue
                    # One rounding to e4m3, then shifts to ever larger scales, each off by
                    # at most half of the smallest step, 2^-10 of its scale: 2 2^-10 of the
                    # last one together.
                    unit = torch.exp2(small.scale_bytes(s).double() - 127)[blk, h][:, None]
                    assert ((x - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -9 * unit).all()

    def cut():
        before = weights.cpu()
        old = mgr.context_lens.cpu()
        kept = mgr.evict_tokens(weights, keep, 4, 16).cpu()
        for b in range(B):
            for h in range(Hk):
                slots = kept[b, h].tolist()[:min(keep, int(old[b]))]
                ids[b][h] = [ids[b][h][j] for j in slots]
                # nothing that is gone weighs more than what stays in the middle
                n = int(old[b])
                middle = set(range(4, max(4, n - 16)))
                gone = [float(before[b, h, j]) for j in middle - set(slots)]
                stay = [float(before[b, h, j]) for j in middle & set(slots)]
                assert not gone or max(gone) <= min(stay)

    step([70, 5, 33])
    cut()
    for n in range(40):
        step([1, int(n % 3 != 0), 2 if n == 7 else 1])
        if n % 8 == 7:
            cut()
    assert mgr.context_lens.tolist() == [48, 31, 48]


def test_two_streams_and_graph_replays(gpu):
    """All four captured once and replayed over new inputs, with eager work in
    between, each replay as the eager calls; then on two streams at once."""
    g = _gen(20)
    lens, before, bs, Hk, G, D, keep = [1, 40, 3], [300, 200, 90], 16, 2, 4, 128, 160
    totals = [a + b for a, b in zip(lens, before)]
    T = sum(lens)
    layout = ops.ChunkLayout(lens, gpu)
    table = ops.RotaryTable.build(D, 512, device=gpu)

    class State:
        def __init__(self, seed):
            h = _gen(seed)
            self.bt, self.ctx, nb = _tables(_gen(1), totals, bs)
            self.bt, self.ctx = self.bt.to(gpu), self.ctx.to(gpu)
            self.q, self.k, self.v = (_randn(h, T, n, D).bfloat16().to(gpu)
                                      for n in (Hk * G, Hk, Hk))
            self.kc, self.ks = [t.to(gpu) for t in small.random_cache(h, nb, bs, Hk, D)]
            self.vc, self.vs = [t.to(gpu) for t in small.random_cache(h, nb, bs, Hk, D)]
            self.w = torch.rand(3, Hk, self.bt.shape[1] * bs, generator=h).to(gpu)

        def load(self, other):
            for name, t in vars(self).items():
                # Byte copies: a copy of float8 tensors must not convert.
                t.view(torch.uint8).copy_(getattr(other, name).view(torch.uint8))

        def run(self):
            q = ops.append_chunk_kv(self.k, self.v, self.kc, self.vc, self.bt, self.ctx, layout,
                                    bs, table, q=self.q, k_scales=self.ks, v_scales=self.vs)
            out, lse = ops.chunk_attention(q, self.kc, self.vc, self.bt, self.ctx, layout, Hk, G,
                                           bs, return_lse=True, k_scales=self.ks,
                                           v_scales=self.vs)
            ops.add_key_weights(self.w, q, lse, self.kc, self.bt, self.ctx, layout, Hk, G, bs,
                                k_scales=self.ks)
            kept = ops.evict_tokens(self.w, self.kc, self.vc, self.bt, self.ctx, keep, bs, 4, 16,
                                    self.ks, self.vs)
            return out, kept

        def state(self):
            return [t.view(torch.uint8).clone() for t in (self.kc, self.vc, self.ks, self.vs,
                                                          self.w)]

    def eager(seed):
        s = State(seed)
        out, kept = s.run()
        return [out, kept] + s.state()

    want = {seed: eager(seed) for seed in (1, 2, 3)}
    s = State(1)
    s.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, kept = s.run()
    for seed in (2, 1, 3, 2):
        s.load(State(seed))
        graph.replay()
        for x, y in zip([out, kept] + s.state(), want[seed]):
            assert torch.equal(x, y)
        eager(1)
        torch.cuda.synchronize()

    states = [State(2), State(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for x, stream in zip(states, streams):
        with torch.cuda.stream(stream):
            got.append(x.run())
    torch.cuda.synchronize()
    for seed, x, (out, kept) in zip((2, 3), states, got):
        for a, b in zip([out, kept] + x.state(), want[seed]):
            assert torch.equal(a, b)


def test_the_managers_other_appends(gpu):
    """Prompts and single tokens without a layout, before and after a cut, are what a
    chunk writes; the backend's prefill is the attention over them."""
    g = _gen(81)
    bs, Hk, D, B = 16, 2, 64, 2
    k, v = (_randn(g, 60, Hk, D).bfloat16().to(gpu) for _ in range(2))
    caches = [PagedKVCache(16, bs, Hk, D, dtype=torch.float8_e4m3fn, device=gpu) for _ in "ab"]
    one, other = (SequenceKVManager(c, B, 96) for c in caches)
    one.prefill_kv(0, k[:37], v[:37])
    one.prefill_kv(1, k[37:42], v[37:42])
    other.append_chunk_kv(k[:37], v[:37], ops.ChunkLayout([37, 0], gpu))
    other.append_chunk_kv(k[37:42], v[37:42], ops.ChunkLayout([0, 5], gpu))
    w = torch.rand(B, Hk, one.block_tables.shape[1] * bs, generator=g).to(gpu)
    for m in (one, other):
        assert m.evict_tokens(w.clone(), 20, 1, 3).shape == (B, Hk, 20)
    one.append_tokens_kv(k[42:44], v[42:44])
    one.append_token_kv(1, k[44], v[44])
    one.append_token_kv(0, k[45], v[45])
    other.append_chunk_kv(k[42:44], v[42:44], ops.ChunkLayout([1, 1], gpu))
    other.append_chunk_kv(k[44:45], v[44:45], ops.ChunkLayout([0, 1], gpu))
    other.append_chunk_kv(k[45:46], v[45:46], ops.ChunkLayout([1, 0], gpu))
    assert one._ctx_host == other._ctx_host == one.context_lens.tolist() == [22, 7]
    a, b = caches
    for x, y in ((a.k_cache, b.k_cache), (a.v_cache, b.v_cache), (a.k_scales, b.k_scales),
                 (a.v_scales, b.v_scales)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    q = _randn(g, 2, 8, D).bfloat16().to(gpu)
    layout = ops.ChunkLayout([1, 1], gpu)
    got = DenseAttentionBackend(Hk, Hk * 4, D, bs).prefill(
        q, a.k_cache, a.v_cache, one.block_tables, one.context_lens, layout, max_context_len=22,
        k_scales=a.k_scales, v_scales=a.v_scales)
    want = ops.chunk_attention(q, a.k_cache, a.v_cache, one.block_tables, one.context_lens, layout,
                               Hk, 4, bs, max_context_len=22, k_scales=a.k_scales,
                               v_scales=a.v_scales)
    assert torch.equal(got, want)


@pytest.mark.parametrize("selector", ["exact", "quest"])
def test_the_sparse_backend_over_a_cut_cache(gpu, selector):
    """Cut, reset: the backend's steps are those of one that never saw the cache before
    the cut, from its selections of pages to Quest's extremes of them."""
    g = _gen(111)
    B, Hk, G, D, bs, keep = 2, 4, 4, 128, 16, 600
    cache = PagedKVCache(300, bs, Hk, D, device=gpu)
    mgr = SequenceKVManager(cache, B, 2048)
    for b, n in enumerate((1900, 1500)):
        mgr.prefill_kv(b, *(_randn(g, n, Hk, D).bfloat16().to(gpu) for _ in range(2)))

    def backend():
        return CVSABackend(Hk, Hk * G, D, bs, num_layers=1, budget_pct=0.25, lazy=True,
                           check_interval=3, selector=selector)

    def step(*backends):
        k, v = (_randn(g, B, Hk, D).bfloat16().to(gpu) for _ in range(2))
        mgr.append_tokens_kv(k, v)
        q = _randn(g, B, Hk * G, D).bfloat16().to(gpu)
        outs = []
        for x in backends:
            outs.append(x(q, cache.k_cache, cache.v_cache, mgr.block_tables, mgr.context_lens, 0))
            x.step_done(0, 1)
        return q, outs

    used = backend()
    meta = ops.QuestPageMeta(cache.k_cache)
    for _ in range(4):
        q, _ = step(used)
        meta.scores(q, mgr.block_tables, mgr.context_lens, Hk, G, bs)
    w = torch.rand(B, Hk, mgr.block_tables.shape[1] * bs, generator=g).to(gpu)
    mgr.evict_tokens(w, keep, 4, 64)
    used.reset()
    meta.invalidate()
    fresh, new = backend(), ops.QuestPageMeta(cache.k_cache)
    for _ in range(7):
        q, (a, b) = step(used, fresh)
        assert torch.equal(a, b)
        assert torch.equal(used._cached_selection[0][0], fresh._cached_selection[0][0])
        x, y = (m.scores(q, mgr.block_tables, mgr.context_lens, Hk, G, bs) for m in (meta, new))
        assert torch.equal(x, y)
    assert used.get_stats() == fresh.get_stats()
    assert mgr.context_lens.tolist() == [keep + 7, keep + 7]
