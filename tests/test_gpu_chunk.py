"""Chunks of new tokens on the GPU: norms with rotation, the append to the
paged cache and the attention over it, each against its formula in 64 bits,
and a run of them together as a serving loop makes it."""
import ctypes
import math

import pytest
import torch

import chunk_reference as ref
from cvsa import ops
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


# ------------------------------------------------------------ norm, rotation

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,R,interleaved", [(128, 128, False), (128, 128, True), (64, 32, False),
                                             (64, 16, True), (32, 32, False), (32, 16, True),
                                             (256, 256, False), (256, 64, True), (256, 16, False),
                                             (128, 96, False), (128, 48, True)])
@pytest.mark.parametrize("norm", [True, False])
def test_qk_norm_rope(gpu, dtype, D, R, interleaved, norm):
    g = _gen(D + R)
    for T, Hq, Hk in ((1, 8, 2), (37, 5, 1), (9, 32, 8), (3, 65, 13)):
        q = (_randn(g, T, Hq, D) * 3).to(dtype)
        k = _randn(g, T, Hk, D).to(dtype)
        w = [(1 + 0.3 * _randn(g, D)).to(torch.bfloat16) for _ in range(2)] if norm else [None] * 2
        table = ops.RotaryTable.build(R, 5000, device=gpu, interleaved=interleaved)
        pos = torch.randint(0, 5000, (T,), generator=g)
        wg = [x if x is None else x.to(gpu) for x in w]
        got = ops.qk_norm_rope(q.to(gpu), k.to(gpu), pos.to(gpu), table, *wg, eps=EPS)
        for x, y, ww in ((q, got[0], w[0]), (k, got[1], w[1])):
            assert y.dtype == dtype and y.is_contiguous()
            want, size = ref.rotated(x, ww, pos, table.table, interleaved, EPS)
            ref.check_rotated(y, want, size, dtype, D)


def test_norm_alone_and_rotation_of_q_alone(gpu):
    g = _gen(5)
    q, k = _randn(g, 7, 4, 64).bfloat16(), _randn(g, 7, 2, 64).bfloat16()
    w = torch.linspace(0.5, 2, 64)
    qn, kn = ops.qk_norm_rope(q.to(gpu), k.to(gpu), None, None, w.to(gpu), None, eps=EPS)
    want, size = ref.rotated(q, w, None, None, False, EPS)
    ref.check_rotated(qn, want, size, torch.bfloat16, 64)
    assert torch.equal(kn.cpu(), k)
    table = ops.RotaryTable.build(64, 10, device=gpu)
    pos = torch.arange(7)
    qr, none = ops.qk_norm_rope(q.to(gpu), None, pos.to(gpu), table)
    assert none is None
    want, size = ref.rotated(q, None, pos, table.table, False, EPS)
    ref.check_rotated(qr, want, size, torch.bfloat16, 64)


def test_rotation_outside_the_table_is_nan_and_leaves_the_rest(gpu):
    q = torch.ones(4, 2, 64, dtype=torch.bfloat16, device=gpu)
    table = ops.RotaryTable.build(32, 8, device=gpu)
    pos = torch.tensor([-1, 0, 7, 8], device=gpu)
    out = ops.qk_norm_rope(q, None, pos, table)[0].float()
    assert out[[0, 3], :, :32].isnan().all() and out[[1, 2]].isfinite().all()
    assert (out[..., 32:] == 1).all()


def test_infinities_and_nan_stay_in_their_rows(gpu):
    g = _gen(6)
    q = _randn(g, 5, 4, 128).bfloat16()
    clean = ops.qk_norm_rope(q.to(gpu), None, torch.arange(5).to(gpu),
                             ops.RotaryTable.build(64, 8, device=gpu),
                             torch.ones(128, device=gpu))[0]
    q[2, 1, 100] = math.inf
    q[3, 0, 3] = math.nan
    q[4, 3, 127] = -math.inf  # past the rotated dimensions, no norm below
    table = ops.RotaryTable.build(64, 8, device=gpu)
    out = ops.qk_norm_rope(q.to(gpu), None, torch.arange(5).to(gpu), table,
                           torch.ones(128, device=gpu))[0]
    same = torch.ones(5, 4, dtype=torch.bool)
    same[2, 1] = same[3, 0] = same[4, 3] = False
    assert torch.equal(out.cpu()[same], clean.cpu()[same])
    plain = ops.qk_norm_rope(q.to(gpu), None, torch.arange(5).to(gpu), table)[0].cpu()
    assert plain[4, 3, 127] == -math.inf and plain[4, 3, :127].isfinite().all()
    assert plain[2, 1, 100] == math.inf and plain[2, 1, :100].isfinite().all()


def test_strided_rows_are_read_in_place(gpu):
    """Views of a fused projection, broadcast heads, and rows that no vector
    load can read in place."""
    g = _gen(7)
    rows = _randn(g, 11, 3 * 40).bfloat16().to(gpu)
    table = ops.RotaryTable.build(32, 64, device=gpu)
    pos = torch.arange(11, device=gpu)
    odd = rows[:, 1:97].view(11, 3, 32)               # not 16-byte aligned
    wide = _randn(g, 11, 9, 32).bfloat16().to(gpu)
    cases = [wide[:, 2:6], wide[:, ::2], wide.transpose(0, 1)[:, :9].contiguous().transpose(0, 1),
             wide[:, :1].expand(11, 4, 32), odd, wide[::2].contiguous()[:5].expand(5, 9, 32)]
    for q in cases:
        want = ops.qk_norm_rope(q.contiguous().clone(), None, pos[:q.shape[0]], table)[0]
        assert torch.equal(ops.qk_norm_rope(q, None, pos[:q.shape[0]], table)[0], want)


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint64])
def test_positions_past_32_bits_are_outside_the_table(gpu, dtype):
    """2^32 + 5 is not position 5."""
    q = torch.ones(4, 2, 64, dtype=torch.bfloat16, device=gpu)
    table = ops.RotaryTable.build(32, 8, device=gpu)
    pos = torch.tensor([2 ** 32 + 5, 5, 2 ** 31, 2 ** 62 + 1], dtype=dtype).to(gpu)
    out = ops.qk_norm_rope(q, None, pos, table)[0].float()
    assert out[[0, 2, 3], :, :32].isnan().all() and out[1].isfinite().all()
    want = ops.qk_norm_rope(q, None, torch.full((4,), 5, dtype=torch.int32, device=gpu), table)[0]
    assert torch.equal(out[1], want[1].float())


# ------------------------------------------------------------ append

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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,bs,Hk,Hq", [(128, 16, 8, 32), (64, 64, 3, 9), (32, 8, 1, 16),
                                        (256, 128, 2, 2), (128, 32, 5, 35)])
def test_append_chunk(gpu, dtype, D, bs, Hk, Hq):
    g = _gen(D + bs)
    lens, before = [3, 0, 1, 2 * bs + 1, 1], [5, 9, 0, bs - 1, 4 * bs]
    totals = [a + b for a, b in zip(lens, before)]
    bt, ctx, nb = _tables(g, totals, bs)
    T = sum(lens)
    pad = 4  # rows behind the last sequence
    k, v = (_randn(g, T + pad, Hk, D).to(dtype) for _ in range(2))
    q = _randn(g, T + pad, Hq, D).to(dtype)
    kw, qw = (1 + 0.2 * _randn(g, D) for _ in range(2))
    kc, vc = (_randn(g, nb, bs, Hk, D).bfloat16() for _ in range(2))
    layout = ops.ChunkLayout(lens, gpu)
    table = ops.RotaryTable.build(D, max(totals), device=gpu)
    kg, vg = kc.to(gpu), vc.to(gpu)
    got = ops.append_chunk_kv(k.to(gpu), v.to(gpu), kg, vg, bt.to(gpu), ctx.to(gpu), layout, bs,
                              table, kw.to(gpu), EPS, q.to(gpu), qw.to(gpu))
    pos = torch.cat([torch.arange(b, b + n) for b, n in zip(before, lens)])
    want, size = ref.rotated(q[:T], qw, pos, table.table, False, EPS)
    ref.check_rotated(got[:T], want, size, dtype, D)
    assert (got[T:] == 0).all()
    want, size = ref.rotated(k[:T], kw, pos, table.table, False, EPS)
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    blk, off = bt[seq, pos // bs].long(), pos % bs
    ref.check_rotated(kg.cpu()[blk, off], want, size, torch.bfloat16, D)
    assert torch.equal(vg.cpu()[blk, off], v[:T].bfloat16())
    kc[blk, off], vc[blk, off] = kg.cpu()[blk, off], vg.cpu()[blk, off]
    assert torch.equal(kc, kg.cpu()) and torch.equal(vc, vg.cpu())  # nothing else written


def test_append_chunk_skips_what_has_no_place(gpu):
    """Blocks outside the pool, positions before the start and past the table
    are not written; the other tokens are."""
    bs, Hk, D = 16, 2, 64
    bt = torch.tensor([[0, 99, 2], [3, -1, 4]], dtype=torch.int32, device=gpu)
    ctx = torch.tensor([52, 10], dtype=torch.int32, device=gpu)  # 48 positions fit; 10 < 14
    lens = [44, 14]
    layout = ops.ChunkLayout(lens, gpu)
    kc = torch.zeros(6, bs, Hk, D, dtype=torch.bfloat16, device=gpu)
    vc = torch.zeros_like(kc)
    rows = torch.arange(1, 59, device=gpu).bfloat16()[:, None, None].expand(58, Hk, D)
    assert ops.append_chunk_kv(rows, rows, kc, vc, bt, ctx, layout, bs) is None
    want = torch.zeros(6, bs, dtype=torch.float32)
    for i in range(44):  # positions 8 .. 51
        p = 8 + i
        if p < 16:
            want[0, p] = i + 1
        elif 32 <= p < 48:
            want[2, p - 32] = i + 1
    for i in range(4, 14):  # positions -4 .. 9
        want[3, i - 4] = 44 + i + 1
    want = want.bfloat16()[:, :, None, None].expand(6, bs, Hk, D)
    assert torch.equal(kc.cpu(), want) and torch.equal(vc.cpu(), want)


@pytest.mark.parametrize("B", [1, 63, 65, 300])
def test_append_chunk_many_sequences(gpu, B):
    """The sequence of each token is found among any number of them."""
    g = _gen(B)
    bs, Hk, D = 8, 1, 32
    lens = torch.randint(0, 4, (B,), generator=g).tolist()
    lens[0] = 1
    before = torch.randint(0, 20, (B,), generator=g).tolist()
    bt, ctx, nb = _tables(g, [a + b for a, b in zip(lens, before)], bs)
    T = sum(lens)
    v = _randn(g, T, Hk, D).bfloat16()
    kc = torch.zeros(nb, bs, Hk, D, dtype=torch.bfloat16, device=gpu)
    vc = torch.zeros_like(kc)
    ops.append_chunk_kv((v * 2).to(gpu), v.to(gpu), kc, vc, bt.to(gpu), ctx.to(gpu),
                        ops.ChunkLayout(lens, gpu), bs)
    pos = torch.cat([torch.arange(b, b + n) for b, n in zip(before, lens)])
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(lens))
    blk, off = bt[seq, pos // bs].long(), pos % bs
    assert torch.equal(vc.cpu()[blk, off], v) and torch.equal(kc.cpu()[blk, off], v * 2)


# ------------------------------------------------------------ attention

def _attend_inputs(g, lens, before, D, bs, Hk, G, W=None):
    totals = [a + b for a, b in zip(lens, before)]
    bt, ctx, nb = _tables(g, totals, bs, W)
    T = sum(lens)
    q = (2 * _randn(g, T, Hk * G, D)).bfloat16()
    kc, vc = (_randn(g, nb, bs, Hk, D).bfloat16() for _ in range(2))
    return q, kc, vc, bt, ctx


def _attend(gpu, q, kc, vc, bt, ctx, lens, G, **kw):
    layout = ops.ChunkLayout(lens, gpu)
    return ops.chunk_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), bt.to(gpu), ctx.to(gpu), layout,
                               kc.shape[2], G, kc.shape[1], **kw)


LENS = [
    ([1], [0]), ([1], [63]), ([1], [64]), ([2], [0]), ([5], [300]), ([33], [31]),
    ([1, 0, 1, 1], [17, 40, 0, 129]),
    ([7, 1, 0, 64], [0, 200, 5, 1]),
    ([130], [70]), ([65, 2], [0, 513]),
]


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("lens,before", LENS)
def test_chunk_attention(gpu, D, lens, before):
    for bs, Hk, G in ((16, 2, 4), (64, 1, 7), (8, 3, 1)):
        g = _gen(D + bs + len(lens))
        q, kc, vc, bt, ctx = _attend_inputs(g, lens, before, D, bs, Hk, G)
        for causal in (True, False):
            out, lse = _attend(gpu, q, kc, vc, bt, ctx, lens, G, causal=causal, return_lse=True)
            ref.check_attend(out, ref.attend(q, kc, vc, bt, ctx, lens, G, causal), lse)


@pytest.mark.parametrize("D,bs,Hk,G,n", [(128, 16, 1, 128, 3), (64, 32, 2, 16, 40),
                                         (128, 128, 1, 4, 300), (256, 16, 1, 8, 33),
                                         (32, 16, 2, 12, 30), (128, 16, 1, 1, 260)])
@pytest.mark.parametrize("W", [None, 5000])
def test_chunk_attention_row_tiles(gpu, D, bs, Hk, G, n, W):
    """Several row tiles and every number of row waves; a wide table takes
    larger tiles and splits."""
    g = _gen(n)
    lens, before = [n, 1], [57, 90]
    q, kc, vc, bt, ctx = _attend_inputs(g, lens, before, D, bs, Hk, G, W)
    out = _attend(gpu, q, kc, vc, bt, ctx, lens, G)
    ref.check_attend(out, ref.attend(q, kc, vc, bt, ctx, lens, G))


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("n,G", [(1, 4), (5, 7), (16, 8), (70, 4)])
def test_chunk_attention_split_keys(gpu, D, n, G):
    """Few rows over many keys: the keys are split and joined."""
    g = _gen(n + D)
    lens, before = [n, 1, 0, n], [4000, 40, 700, 1999]
    q, kc, vc, bt, ctx = _attend_inputs(g, lens, before, D, 16, 1, G, W=300)
    want = ref.attend(q, kc, vc, bt, ctx, lens, G)
    out, lse = _attend(gpu, q, kc, vc, bt, ctx, lens, G, return_lse=True)
    ref.check_attend(out, want, lse)
    for bound in (1000, 4100, 100000):  # a hint below the truth is only slower
        out, lse = _attend(gpu, q, kc, vc, bt, ctx, lens, G, return_lse=True,
                           max_context_len=bound)
        ref.check_attend(out, want, lse)


def test_chunk_attention_equals_dense_decode_for_single_tokens(gpu):
    g = _gen(11)
    lens, before = [1] * 5, [0, 15, 16, 700, 2047]
    q, kc, vc, bt, ctx = _attend_inputs(g, lens, before, 128, 16, 2, 4)
    bt = bt.clamp(min=0)
    out = _attend(gpu, q, kc, vc, bt, ctx, lens, 4)
    want = ref.attend(q, kc, vc, bt, ctx, lens, 4)
    ref.check_attend(out, want)
    dense = ops.dense_decode(q.to(gpu), kc.to(gpu), vc.to(gpu), bt.to(gpu), ctx.to(gpu), 2, 4, 16)
    ref.check_attend(dense, want)


@pytest.mark.parametrize("D,W", [(64, None), (128, None), (256, None), (64, 300)])
@pytest.mark.parametrize("n", [1, 6, 50])
def test_rows_without_keys(gpu, D, n, W):
    """Blocks outside the pool take no part; rows that see no key are zero
    with a log-sum-exp of -inf: a context shorter than the chunk, an empty
    context, a table of bad blocks only."""
    g = _gen(n)
    lens = [n, n, n, n]
    q, kc, vc, bt, ctx = _attend_inputs(g, lens, [40, 40, 40, 40], D, 16, 2, 4, W)
    nb = kc.shape[0]
    bt[0, 1] = -1
    bt[1, :] = nb
    ctx[2] = max(0, n - 3)
    ctx[3] = 0
    for causal in (True, False):
        want = ref.attend(q, kc, vc, bt, ctx, lens, 4, causal)
        assert (want[1][n:2 * n] == -math.inf).all()
        out, lse = _attend(gpu, q, kc, vc, bt, ctx, lens, 4, causal=causal, return_lse=True)
        ref.check_attend(out, want, lse)
        assert (out[want[1].to(gpu) == -math.inf] == 0).all()


def test_context_past_the_table(gpu):
    """Keys past the block table's width take no part."""
    g = _gen(3)
    lens = [20]
    q, kc, vc, bt, ctx = _attend_inputs(g, lens, [44], 64, 16, 1, 2)
    ctx[0] = 100  # positions 80 .. 99, 64 of them in the table
    out, lse = _attend(gpu, q, kc, vc, bt, ctx, lens, 2, return_lse=True)
    ref.check_attend(out, ref.attend(q, kc, vc, bt, ctx, lens, 2), lse)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("D,n,G,W", [(128, 40, 4, None), (64, 9, 1, None), (256, 12, 2, None),
                                     (128, 3, 8, None), (64, 40, 4, None), (64, 40, 4, 300),
                                     (32, 40, 4, None)])
def test_values_that_no_row_sees_do_not_touch_it(gpu, value, D, n, G, W):
    """Behind the context's end, in bad blocks, and keys and values of later
    tokens of the chunk: only the rows that see them feel them."""
    g = _gen(n)
    lens, before = [n, n], [21, 0]
    bs = 16
    q, kc, vc, bt, ctx = _attend_inputs(g, lens, before, D, bs, 2, G, W)
    used = torch.zeros(kc.shape[:2], dtype=torch.bool)
    for b in range(2):
        p = torch.arange(int(ctx[b]))
        used[bt[b, p // bs].long(), p % bs] = True
    kc[~used], vc[~used] = value, value
    want = ref.attend(q, kc, vc, bt, ctx, lens, G)
    assert want[0].isfinite().all()
    ref.check_attend(_attend(gpu, q, kc, vc, bt, ctx, lens, G), want)
    # a late token's value, one element of one head
    at = before[0] + n - 2
    vc[bt[0, at // bs].long(), at % bs, 1, 5] = value
    vc[bt[0, at // bs].long(), at % bs, 1, D - 1] = value
    want = ref.attend(q, kc, vc, bt, ctx, lens, G)
    assert want[0][:n - 2].isfinite().all() and not want[0][n - 1].isfinite().all()
    ref.check_attend(_attend(gpu, q, kc, vc, bt, ctx, lens, G), want)
    # and its key
    kc[bt[0, at // bs].long(), at % bs, 0, 3] = value
    want = ref.attend(q, kc, vc, bt, ctx, lens, G)
    out = _attend(gpu, q, kc, vc, bt, ctx, lens, G).double().cpu()
    early = torch.ones(2 * n, dtype=torch.bool)
    early[n - 2:n] = False
    err = (out - want[0]).abs()
    assert not (err > want[2])[early].any()


def _splits(lens, Hk, G, D, bs, W):
    """(splits, keys of one) that the plan has for sequences of many rows only,
    from the size of its workspace: a part has D sums and two numbers for each
    token and head."""
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    need = ops._lib.load().cvsa_chunk_attention_workspace_bytes(
        (ctypes.c_int32 * len(cu))(*cu), len(lens), Hk * G, Hk, D, bs, W, 0)
    splits = max(1, need // (cu[-1] * Hk * G * (4 * D + 8)))
    return splits, -(-W * bs // (splits * 128)) * 128


MANY = [  # chunks, tokens before, heads of the group, width of the table
    ([600, 80], [1400, 900], 1, 128),    # 128-row tiles at D = 64
    ([70, 300], [5000, 200], 4, 5000),   # the table of a much longer context
    ([100, 17, 40], [3000, 1, 700], 4, 200),
]


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("lens,before,G,W", MANY)
def test_many_rows_in_several_splits(gpu, D, lens, before, G, W):
    """Rows whose keys lie in one split, in several, and in a part of the last;
    some of them tell complete tiles and parts of one call apart."""
    g = _gen(D + W)
    splits, split_len = _splits(lens, 1, G, D, 16, W)
    assert splits > 1 and lens[0] + before[0] > split_len > 128
    q, kc, vc, bt, ctx = _attend_inputs(g, lens, before, D, 16, 1, G, W)
    for causal in (True, False):
        out, lse = _attend(gpu, q, kc, vc, bt, ctx, lens, G, causal=causal, return_lse=True)
        ref.check_attend(out, ref.attend(q, kc, vc, bt, ctx, lens, G, causal), lse)


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("lens,before,G,W", MANY + [([3, 1], [700, 50], 7, None),
                                                    ([40, 40], [60, 0], 4, None),
                                                    ([5, 2], [2000, 900], 4, 600)])
def test_infinite_values_keep_their_kind(gpu, D, lens, before, G, W):
    """Columns of V that hold infinities of either sign and NaN, alone and
    together, at keys that all rows see (in the first split and a later one)
    and at keys that only later tokens see: each row gets what it sees."""
    g = _gen(D + len(lens) + lens[0])
    bs, inf, nan = 16, math.inf, math.nan
    q, kc, vc, bt, ctx = _attend_inputs(g, lens, before, D, bs, 1, G, W)
    columns = [{0: inf}, {0: -inf}, {0: nan}, {0: inf, 1: -inf}, {0: -inf, 1: inf},
               {0: inf, 1: inf}, {0: inf, 1: nan}, {0: nan, 1: -inf}, {1: -inf}]
    n, b0 = lens[0], before[0]
    for i, (early, late) in enumerate(((3, b0 - 5), (b0 // 2, b0 + n // 2), (b0, b0 + n - 1))):
        for j, column in enumerate(columns):
            for at, value in column.items():
                p = late if at else early
                vc[bt[0, p // bs].long(), p % bs, 0, 9 * i + j] = value
    assert 9 * 3 <= D
    for causal in (True, False):
        out = _attend(gpu, q, kc, vc, bt, ctx, lens, G, causal=causal)
        ref.check_kinds(out, ref.attend(q, kc, vc, bt, ctx, lens, G, causal))


def test_scores_of_any_size(gpu):
    """Scores of thousands, all alike or far apart, and a scale of the
    caller's."""
    g = _gen(8)
    lens, before = [6], [90]
    q, kc, vc, bt, ctx = _attend_inputs(g, lens, before, 64, 16, 1, 2)
    for f, scale in ((100.0, None), (1.0, 3.0), (0.0, None), (1e-3, 0.5)):
        qq = (q * f).bfloat16()
        out, lse = _attend(gpu, qq, kc, vc, bt, ctx, lens, 2, scale=scale, return_lse=True)
        ref.check_attend(out, ref.attend(qq, kc, vc, bt, ctx, lens, 2, scale=scale), lse)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B", [65, 150])
def test_chunk_attention_many_sequences(gpu, D, B):
    """More sequences than a wave has lanes: single tokens, drafts, longer
    chunks and none, over contexts from none to many; each class finds its own."""
    g = _gen(B + D)
    kinds = torch.tensor([0, 1, 1, 1, 3, 16, 33])
    lens = kinds[torch.randint(0, 7, (B,), generator=g)].tolist()
    lens[0], lens[-1] = 0, 40
    before = torch.randint(0, 200, (B,), generator=g).tolist()
    before[3] = before[B - 2] = 900
    q, kc, vc, bt, ctx = _attend_inputs(g, lens, before, D, 16, 2, 4)
    out, lse = _attend(gpu, q, kc, vc, bt, ctx, lens, 4, return_lse=True)
    ref.check_attend(out, ref.attend(q, kc, vc, bt, ctx, lens, 4), lse)


@pytest.mark.parametrize("D,Hk,G,n", [(128, 2, 4, 1), (64, 1, 7, 5), (256, 1, 8, 1),
                                      (32, 300, 1, 2)])
@pytest.mark.parametrize("B", [3, 66])
def test_chunk_attention_equal_chunks(gpu, D, Hk, G, n, B):
    """Every sequence brings as many tokens (their places are computed); more
    KV heads than CUs; contexts of one range, several, or a part of one."""
    g = _gen(B + D + n)
    before = torch.randint(0, 60, (B,), generator=g).tolist()
    if Hk < 300:
        before[1] = 1500
    q, kc, vc, bt, ctx = _attend_inputs(g, [n] * B, before, D, 16, Hk, G)
    want = ref.attend(q, kc, vc, bt, ctx, [n] * B, G)
    for bound in (0, 100):  # 100: short contexts promised, without a join
        out, lse = _attend(gpu, q, kc, vc, bt, ctx, [n] * B, G, return_lse=True,
                           max_context_len=bound)
        ref.check_attend(out, want, lse)


@pytest.mark.parametrize("D,n,G", [(32, 2, 4), (64, 5, 7), (128, 1, 8), (256, 3, 4),
                                   (32, 40, 4), (64, 40, 4), (128, 40, 4), (256, 40, 4),
                                   (64, 300, 4)])
def test_scores_that_rise_and_fall(gpu, D, n, G):
    """The reference of a row has to move when later scores outgrow it, by
    little or by far, and to stay when they fall."""
    g = _gen(D + n)
    lens, before, bs = [n], [900], 16
    q, kc, vc, bt, ctx = _attend_inputs(g, lens, before, D, bs, 1, G)
    q = q * 0.25 + 2
    at = torch.arange(int(ctx[0]))
    steps = {"rise": at * 0.25, "fall": -at * 0.25, "jump": (at >= 500) * 40.0,
             "steps": at // 130 * 16.0, "far": (at >= 300) * 3000.0 + (at >= 800) * 1.0}
    for score in steps.values():
        k = kc.clone()
        # q . k / sqrt(D) is score, about
        k[bt[0, at // bs].long(), at % bs, 0] = (
            (score / (2 * math.sqrt(D)))[:, None] + 0.1 * _randn(g, at.numel(), D)).bfloat16()
        out, lse = _attend(gpu, q, k, vc, bt, ctx, lens, G, return_lse=True)
        ref.check_attend(out, ref.attend(q, k, vc, bt, ctx, lens, G), lse)


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_chunk_attention_order_of_tiles(gpu, D, causal):
    """Prompts of many row tiles whose order goes by their keys: alike ones,
    contexts far apart, none, a chunk cut off by its table, and more sequences
    than a wave has lanes; no tile is left out or done twice."""
    g = _gen(D)
    G, bs = 8, 16
    for lens, before in (([100, 100, 100], [0, 0, 0]), ([90, 1, 130, 64], [300, 700, 0, 900]),
                         ([33] * 70, [(37 * b) % 200 for b in range(70)])):
        q, kc, vc, bt, ctx = _attend_inputs(g, lens, before, D, bs, 1, G)
        if len(lens) == 4:
            ctx[0], bt = 1500, bt[:, :50].contiguous()  # positions past the table
            ctx[3] = -5
        out = torch.full(q.shape, math.nan, dtype=torch.bfloat16, device=gpu)
        _attend(gpu, q, kc, vc, bt, ctx, lens, G, causal=causal, out=out)
        ref.check_attend(out, ref.attend(q, kc, vc, bt, ctx, lens, G, causal))


def test_strided_queries_padded_rows_and_out(gpu):
    g = _gen(9)
    lens, before, G, Hk, D = [5, 9], [20, 0], 2, 2, 64
    q, kc, vc, bt, ctx = _attend_inputs(g, lens, before, D, 16, Hk, G)
    want, want_lse = _attend(gpu, q, kc, vc, bt, ctx, lens, G, return_lse=True)
    rows = torch.full((18, 9, D), math.nan, dtype=torch.bfloat16)
    rows[:14, 3:7] = q
    view = rows.to(gpu)[:, 3:7]
    out, lse = _attend(gpu, view, kc, vc, bt, ctx, lens, G, return_lse=True)
    assert torch.equal(out[:14], want) and (out[14:] == 0).all()
    assert torch.equal(lse[:14], want_lse) and (lse[14:] == 0).all()
    mine = torch.full((18, 4, D), 7.0, dtype=torch.bfloat16, device=gpu)
    assert _attend(gpu, view, kc, vc, bt, ctx, lens, G, out=mine) is mine
    assert torch.equal(mine[:14], want) and (mine[14:] == 7).all()
    over = q.to(gpu)
    assert _attend(gpu, over, kc, vc, bt, ctx, lens, G, out=over) is over
    assert torch.equal(over, want)
    none = _attend(gpu, view, kc, vc, bt, ctx, [0, 0], G)
    assert none.shape == (18, 4, D) and (none == 0).all()
    wide = torch.full((2, 40), -1, dtype=torch.int32)
    wide[:, ::2][:, :bt.shape[1]] = bt
    assert torch.equal(_attend(gpu, q, kc, vc, wide[:, ::2], ctx, lens, G), want)


def test_one_token_and_one_sequence_of_any_stride(gpu):
    """A single token's row, and a single sequence's table, whose (unused)
    strides are odd; and a table that sequences share."""
    g = _gen(14)
    Hk, G, D, bs, before = 2, 4, 64, 16, 40
    q, kc, vc, bt, ctx = (x.to(gpu) for x in _attend_inputs(g, [1], [before], D, bs, Hk, G))
    k, v = (_randn(g, 1, Hk, D).bfloat16().to(gpu) for _ in range(2))
    layout, table = ops.ChunkLayout([1], gpu), ops.RotaryTable.build(D, 64, device=gpu)

    def bent(t):
        return t.as_strided(t.shape, (t.stride(0) + 1, *t.stride()[1:]))

    def step(q, k, v, bt):
        c = kc.clone(), vc.clone()
        qr = ops.append_chunk_kv(k, v, *c, bt, ctx, layout, bs, table, q=q)
        qn, kn = ops.qk_norm_rope(q, k, ctx - 1, table)
        return (qr, *c, qn, kn,
                ops.chunk_attention(qr, *c, bt, ctx, layout, Hk, G, bs))

    want = step(q, k, v, bt)
    got = step(bent(q), bent(k), bent(v), bt.as_strided(bt.shape, (1, 1)))
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    three = ops.ChunkLayout([1] * 3, gpu)
    shared = [bt.expand(3, -1), bt.repeat(3, 1)]
    outs = [ops.chunk_attention(q.expand(3, -1, -1), *want[1:3], b, ctx.repeat(3), three, Hk, G, bs)
            for b in shared]
    assert torch.equal(*outs)


def test_offsets_past_32_bits(gpu):
    """A pool of more than 2^32 elements: blocks at its far end."""
    Hk, D, bs = 8, 256, 128
    nb = (1 << 32) // (Hk * D * bs) + 8
    kc = torch.zeros(nb, bs, Hk, D, dtype=torch.bfloat16, device=gpu)
    vc = torch.zeros_like(kc)
    g = _gen(2)
    lens, total = [5], 300
    bt = torch.tensor([[nb - 1, 3, nb - 4]], dtype=torch.int32, device=gpu)
    ctx = torch.tensor([total], dtype=torch.int32, device=gpu)
    layout = ops.ChunkLayout([total], gpu)
    k, v = (_randn(g, total, Hk, D).bfloat16() for _ in range(2))
    ops.append_chunk_kv(k.to(gpu), v.to(gpu), kc, vc, bt, ctx, layout, bs)
    q = _randn(g, 5, Hk, D).bfloat16()
    out = ops.chunk_attention(q.to(gpu), kc, vc, bt, ctx, ops.ChunkLayout(lens, gpu), Hk, 1, bs)
    small = torch.stack([kc[nb - 1], kc[3], kc[nb - 4]]).cpu()
    smallv = torch.stack([vc[nb - 1], vc[3], vc[nb - 4]]).cpu()
    assert torch.equal(small.view(-1, Hk, D)[:total], k)
    assert torch.equal(smallv.view(-1, Hk, D)[:total], v)
    ident = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    ref.check_attend(out, ref.attend(q, small, smallv, ident, ctx, lens, 1))


# ------------------------------------------------------------ together

def _one_by_one(gpu, B, bs, Hk, D, blocks, lens_list):
    """Tables of append_token_kv token by token, sequence after sequence."""
    mgr = SequenceKVManager(PagedKVCache(blocks, bs, Hk, D, device=gpu), B, 512)
    row = torch.zeros(Hk, D, dtype=torch.bfloat16, device=gpu)
    for lens in lens_list:
        for b, n in enumerate(lens):
            for _ in range(n):
                mgr.append_token_kv(b, row, row)
    return mgr


def test_reserve_chunk_follows_the_append_rule(gpu):
    steps = [[5, 0, 40], [1, 1, 1], [16, 30, 0], [0, 0, 0], [11, 1, 64]]
    mgr = SequenceKVManager(PagedKVCache(40, 16, 1, 32, device=gpu), 3, 512)
    for lens in steps:
        mgr.reserve_chunk(ops.ChunkLayout(lens, gpu))
    want = _one_by_one(gpu, 3, 16, 1, 32, 40, steps)
    assert torch.equal(mgr.block_tables, want.block_tables)
    assert torch.equal(mgr.context_lens, want.context_lens)
    assert torch.equal(mgr._pages_allocated_dev, want._pages_allocated_dev)
    assert mgr._ctx_host == want._ctx_host and mgr._pages_allocated == want._pages_allocated
    assert mgr.cache._next_free == want.cache._next_free


@pytest.mark.parametrize("B", [1, 1500])
def test_reserve_chunk_of_any_batch(gpu, B):
    g = _gen(B)
    lens = torch.randint(0, 40, (B,), generator=g).tolist()
    blocks = sum(-(-n // 8) for n in lens) + sum(-(-n // 8) for n in lens)
    mgr = SequenceKVManager(PagedKVCache(blocks, 8, 1, 32, device=gpu), B, 128)
    for _ in range(2):
        mgr.reserve_chunk(ops.ChunkLayout(lens, gpu))
    used = [-(-2 * n // 8) for n in lens]
    assert mgr.context_lens.tolist() == [2 * n for n in lens]
    assert mgr._pages_allocated_dev.tolist() == used == mgr._pages_allocated
    ids = [int(x) for b in range(B) for x in mgr.block_tables[b, :used[b]].tolist()]
    assert sorted(ids) == list(range(sum(used))) and mgr.cache._next_free == sum(used)


@pytest.mark.parametrize("D,bs,Hk,G", [(128, 16, 2, 4), (64, 64, 1, 7)])
def test_prompts_in_pieces_then_decode(gpu, D, bs, Hk, G):
    """Prompts taken in by pieces leave the cache, and give the outputs, of
    prompts taken in at once; decode goes on from there."""
    g = _gen(D)
    lens = [70, 33]
    T = sum(lens)
    q, k, v = _randn(g, T, Hk * G, D), _randn(g, T, Hk, D), _randn(g, T, Hk, D)
    q, k, v = (x.bfloat16().to(gpu) for x in (q, k, v))
    qw, kw = (torch.linspace(0.5, 1.5, D).bfloat16().to(gpu) for _ in range(2))
    table = ops.RotaryTable.build(D, 128, device=gpu)
    backend = DenseAttentionBackend(Hk, Hk * G, D, bs)

    def start():
        return SequenceKVManager(PagedKVCache(32, bs, Hk, D, device=gpu), 2, 128)

    def feed(mgr, lens, q, k, v):
        layout = ops.ChunkLayout(lens, gpu)
        qr = mgr.append_chunk_kv(k, v, layout, table, kw, EPS, q, qw)
        out = backend.prefill(qr, mgr.cache.k_cache, mgr.cache.v_cache, mgr.block_tables,
                              mgr.context_lens, layout)
        return qr, out

    whole = start()
    qr, out = feed(whole, lens, q, k, v)
    cpu = [x.cpu() for x in (whole.cache.k_cache, whole.cache.v_cache, whole.block_tables,
                             whole.context_lens)]
    want = ref.attend(qr.cpu(), *cpu, lens, G)
    ref.check_attend(out, want)

    pieces = start()
    got = torch.empty_like(out)
    done = [0, 0]
    for step in ([7, 33], [0, 0], [1, 0], [62, 0]):
        rows = torch.cat([torch.arange(o + d, o + d + n)
                          for o, d, n in zip((0, 70), done, step)]).to(gpu)
        qp, op = feed(pieces, step, q[rows], k[rows], v[rows])
        assert torch.equal(qp, qr[rows])
        got[rows] = op
        done = [d + n for d, n in zip(done, step)]
    ref.check_attend(got, want)
    for b in range(2):
        for c in ("k_cache", "v_cache"):
            x, y = (getattr(m.cache, c)[m.block_tables[b].long()].flatten(0, 1)[:lens[b]]
                    for m in (whole, pieces))
            assert torch.equal(x, y)

    step_k, step_v = (_randn(g, 2, Hk, D).bfloat16().to(gpu) for _ in range(2))
    step_q = _randn(g, 2, Hk * G, D).bfloat16().to(gpu)
    pieces.append_tokens_kv(step_k, step_v)
    args = (pieces.cache.k_cache, pieces.cache.v_cache, pieces.block_tables, pieces.context_lens)
    want = ref.attend(step_q, *args, [1, 1], G)
    ref.check_attend(backend(step_q, *args, 0), want)
    ref.check_attend(backend.prefill(step_q, *args, ops.ChunkLayout([1, 1], gpu)), want)


@pytest.mark.parametrize("lens,W", [([40, 3], 8), ([2, 2], 256)])
def test_graph_replays_and_other_streams(gpu, lens, W):
    """A captured step (append, attention) replayed over new inputs between
    eager work equals the eager step; so does a step on another stream."""
    g = _gen(12)
    Hk, G, D, bs = 2, 4, 128, 16
    before = [30, 60] if W == 8 else [4000, 1000]
    q, kc, vc, bt, ctx = _attend_inputs(g, lens, before, D, bs, Hk, G, W)
    T = sum(lens)
    layout = ops.ChunkLayout(lens, gpu)
    table = ops.RotaryTable.build(D, W * bs, device=gpu)
    kc, vc, bt, ctx = (x.to(gpu) for x in (kc, vc, bt, ctx))
    sq = torch.zeros(T, Hk * G, D, dtype=torch.bfloat16, device=gpu)
    sk, sv = (torch.zeros(T, Hk, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))

    def step():
        qr = ops.append_chunk_kv(sk, sv, kc, vc, bt, ctx, layout, bs, table, q=sq)
        return ops.chunk_attention(qr, kc, vc, bt, ctx, layout, Hk, G, bs, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, lse = step()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        for s in (sq, sk, sv):
            s.copy_(_randn(g, *s.shape).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        got, got_lse, keys = out.clone(), lse.clone(), kc.clone()
        eager, eager_lse = step()
        assert torch.equal(got, eager) and torch.equal(got_lse, eager_lse)
        assert torch.equal(keys, kc)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()[0]
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, eager)


def test_a_managers_pages_are_not_taken_in_a_graph(gpu):
    """The manager's calls are refused while a graph is captured and leave no
    trace; the append over pages that it reserved before is captured, and
    replays with new rows."""
    g = _gen(15)
    lens, bs, Hk, D = [5, 20], 16, 2, 64
    T = sum(lens)
    mgr = SequenceKVManager(PagedKVCache(8, bs, Hk, D, device=gpu), 2, 64)
    mgr.cache.k_cache.zero_()
    mgr.cache.v_cache.zero_()
    layout, table = ops.ChunkLayout(lens, gpu), ops.RotaryTable.build(D, 64, device=gpu)
    k, v = (torch.zeros(T, Hk, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    mgr.reserve_chunk(layout)
    held = (list(mgr._ctx_host), list(mgr._pages_allocated), mgr.cache._next_free)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    args = (mgr.block_tables, mgr.context_lens, layout, bs, table)
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="captur"):
            mgr.reserve_chunk(layout)
        with pytest.raises(RuntimeError, match="captur"):
            mgr.append_chunk_kv(k, v, layout, table)
        ops.append_chunk_kv(k, v, mgr.cache.k_cache, mgr.cache.v_cache, *args)
    torch.cuda.current_stream().wait_stream(side)
    assert held == (mgr._ctx_host, mgr._pages_allocated, mgr.cache._next_free)
    for _ in range(3):
        k.copy_(_randn(g, T, Hk, D).bfloat16())
        v.copy_(_randn(g, T, Hk, D).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        want = [torch.zeros_like(mgr.cache.k_cache) for _ in range(2)]
        ops.append_chunk_kv(k, v, *want, *args)
        assert torch.equal(mgr.cache.k_cache, want[0])
        assert torch.equal(mgr.cache.v_cache, want[1])
    assert mgr.context_lens.tolist() == lens


def test_calls_on_two_streams_at_once(gpu):
    """Split calls that overlap share no workspace."""
    g = _gen(13)
    lens, before = [3, 3], [6000, 3000]
    q, kc, vc, bt, ctx = (x.to(gpu) for x in _attend_inputs(g, lens, before, 128, 16, 2, 4))
    layout = ops.ChunkLayout(lens, gpu)
    qs = [q, q.flip(0).contiguous()]
    want = [ops.chunk_attention(x, kc, vc, bt, ctx, layout, 2, 4, 16) for x in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.chunk_attention(qs[i], kc, vc, bt, ctx, layout, 2, 4, 16))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
