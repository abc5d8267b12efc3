"""Refusals of the chunk entry points, all on the host before any launch:
cvsa.ops' checks (their device check and launch replaced), the C ABI's, and
the manager's, which leaves its state as it was."""
import ctypes

import pytest
import torch

from cvsa import ops
from cvsa.ops import _lib, chunk
from cvsa.runtime.kv_cache import PagedKVCache, SequenceKVManager

BS, HK, G, D, NB, W = 16, 2, 4, 64, 20, 5
LENS = [3, 0, 20]
T = sum(LENS)


@pytest.fixture
def calls(monkeypatch):
    """Ops on CPU tensors whose launches are only recorded."""
    made = []
    monkeypatch.setattr(chunk, "_device_of", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(chunk, "_same_device", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(chunk, "_call", lambda dev, who, fn, *args, keep=None: made.append((who, args)))

    class Lib:
        cvsa_qk_norm_rope = cvsa_append_chunk_kv = cvsa_reserve_chunk = None
        cvsa_chunk_attention = None

        @staticmethod
        def cvsa_chunk_attention_workspace_bytes(*a):
            return 0

    monkeypatch.setattr(chunk._lib, "load", lambda: Lib)
    return made


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def _append_args():
    return dict(k=_bf(T, HK, D), v=_bf(T, HK, D), k_cache=_bf(NB, BS, HK, D),
                v_cache=_bf(NB, BS, HK, D), block_tables=torch.zeros(3, W, dtype=torch.int32),
                context_lens=torch.tensor(LENS, dtype=torch.int32),
                layout=ops.ChunkLayout(LENS, "cpu"), block_size=BS,
                rotary=ops.RotaryTable.build(D, 80, device="cpu"), k_weight=torch.ones(D),
                q=_bf(T, HK * G, D), q_weight=torch.ones(D))


def _attend_args():
    a = _append_args()
    return dict(q=a["q"], k_cache=a["k_cache"], v_cache=a["v_cache"],
                block_tables=a["block_tables"], context_lens=a["context_lens"],
                layout=a["layout"], num_kv_heads=HK, num_q_per_kv=G, block_size=BS)


def _rope_args():
    return dict(q=_bf(T, HK * G, D), k=_bf(T, HK, D), positions=torch.zeros(T, dtype=torch.int64),
                rotary=ops.RotaryTable.build(D, 80, device="cpu"), q_weight=torch.ones(D),
                k_weight=torch.ones(D))


def test_good_calls_reach_the_library(calls):
    q = ops.append_chunk_kv(**_append_args())
    out, lse = ops.chunk_attention(**_attend_args(), return_lse=True)
    qr, kr = ops.qk_norm_rope(**_rope_args())
    assert [c[0] for c in calls] == ["append_chunk_kv", "chunk_attention", "qk_norm_rope"]
    assert q.shape == out.shape == qr.shape == (T, HK * G, D) and kr.shape == (T, HK, D)
    assert lse.shape == (T, HK * G) and lse.dtype == torch.float32
    for who, args in calls:  # one argument for each of the C entry's, but the stream
        assert len(args) == len(_lib.SIGNATURES["cvsa_" + who][1]) - 1


BAD_APPEND = [
    dict(k=_bf(T, HK, D + 1)), dict(k=_bf(T - 1, HK, D)), dict(v=_bf(T, HK + 1, D)),
    dict(v=torch.zeros(T, HK, D)),                        # another dtype than k's
    dict(k=torch.zeros(T, HK, D, dtype=torch.float64)), dict(k=_bf(T, HK * D)),
    dict(v_cache=_bf(NB + 1, BS, HK, D)), dict(k_cache=torch.zeros(NB, BS, HK, D)),
    dict(k_cache=_bf(NB, BS, HK, 2 * D)[..., ::2]), dict(block_size=32),
    dict(block_tables=torch.zeros(2, W, dtype=torch.int32)),
    dict(context_lens=torch.zeros(4, dtype=torch.int32)),
    dict(layout=ops.ChunkLayout([1, 2], "cpu")),
    dict(layout=ops.ChunkLayout([T + 1, 0, 0], "cpu")),
    dict(k_weight=torch.ones(D + 1)), dict(k_weight=torch.ones(D, dtype=torch.int32)),
    dict(k_weight=torch.ones(D, dtype=torch.bfloat16)),   # q_weight is float32
    dict(q=None), dict(q=torch.zeros(T, HK * G, D)),
    dict(rotary=ops.RotaryTable.build(2 * D, 80, device="cpu")),
]


@pytest.mark.parametrize("bad", BAD_APPEND)
def test_append_refuses(calls, bad):
    with pytest.raises(ValueError):
        ops.append_chunk_kv(**{**_append_args(), **bad})
    assert not calls


BAD_ATTEND = [
    dict(q=_bf(T, HK * G + 1, D)), dict(q=torch.zeros(T, HK * G, D)), dict(q=_bf(T - 1, HK * G, D)),
    dict(num_kv_heads=4), dict(num_q_per_kv=2), dict(block_size=8),
    dict(layout=ops.ChunkLayout([T], "cpu")), dict(max_context_len=-1),
    dict(out=_bf(T - 1, HK * G, D)), dict(out=torch.zeros(T, HK * G, D)),
    dict(out=_bf(T, D, HK * G).transpose(1, 2)),
    dict(context_lens=torch.zeros(3, 1, dtype=torch.int32)),
]


@pytest.mark.parametrize("bad", BAD_ATTEND)
def test_attention_refuses(calls, bad):
    with pytest.raises(ValueError):
        ops.chunk_attention(**{**_attend_args(), **bad})
    assert not calls


BAD_ROPE = [
    dict(k=_bf(T + 1, HK, D)), dict(k=_bf(T, HK, 32)), dict(k=torch.zeros(T, HK, D)),
    dict(k=None), dict(positions=None), dict(positions=torch.zeros(T)),
    dict(positions=torch.zeros(T + 1, dtype=torch.int32)),
    dict(positions=torch.zeros(T, 1, dtype=torch.int32)),
    dict(rotary=None, q_weight=None, k_weight=None), dict(q_weight=torch.ones(1, D)),
]


@pytest.mark.parametrize("bad", BAD_ROPE)
def test_norm_rope_refuses(calls, bad):
    with pytest.raises(ValueError):
        ops.qk_norm_rope(**{**_rope_args(), **bad})
    assert not calls


def test_empty_chunks_launch_nothing(calls):
    a, b = _append_args(), _attend_args()
    a["layout"] = b["layout"] = ops.ChunkLayout([0, 0, 0], "cpu")
    assert (ops.append_chunk_kv(**a) == 0).all()
    assert (ops.chunk_attention(**b) == 0).all()
    assert not calls


def test_layout_and_table_refuse():
    for lens in ([], [-1], [1 << 24, 1]):
        with pytest.raises(ValueError):
            ops.ChunkLayout(lens, "cpu")
    for t in (torch.zeros(4), torch.zeros(4, 32, dtype=torch.float64), torch.zeros(0, 32)):
        with pytest.raises(ValueError):
            ops.RotaryTable(t)
    for r in (8, 24):
        with pytest.raises(NotImplementedError):
            ops.RotaryTable(torch.zeros(4, r))
    with pytest.raises(NotImplementedError):
        ops.RotaryTable(torch.zeros(4, 0))


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU only"):
        ops.chunk_attention(**_attend_args())
    with pytest.raises(ValueError, match="GPU only"):
        ops.append_chunk_kv(**_append_args())
    with pytest.raises(ValueError, match="GPU only"):
        ops.qk_norm_rope(**_rope_args())


def test_rotary_table_keeps_far_angles():
    """The angle of a far position is the 64-bit product's."""
    import math
    t = ops.RotaryTable.build(32, 1 << 17, base=10000.0, device="cpu").table
    for p in (0, 1, 65537, (1 << 17) - 1):
        for i in (0, 1, 15):
            ang = p * 10000.0 ** (-2 * i / 32)
            # half a step of fp32 and the angle's own 64-bit rounding
            assert abs(t[p, i].item() - math.cos(ang)) < 2.0 ** -24 + ang * 2.0 ** -51
            assert abs(t[p, 16 + i].item() - math.sin(ang)) < 2.0 ** -24 + ang * 2.0 ** -51


# ------------------------------------------------------------ C ABI

def _lib_or_skip():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libcvsa_hip.so not built")
    try:
        return _lib.load()
    except OSError as e:  # no HIP runtime on this host
        pytest.skip(f"HIP runtime not loadable: {e}")


P = [1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20, 6 << 20, 7 << 20]  # never dereferenced


def _attention(lib, cu=(0, 3), **over):
    a = dict(q=P[0], st=HK * G * D, sh=D, kc=P[1], vc=P[2], nb=NB, bt=P[3], sb=W, ctx=P[4], cu=P[5],
             host=(ctypes.c_int32 * len(cu))(*cu), B=len(cu) - 1, H_q=HK * G, H_kv=HK, D=D, bs=BS,
             W=W, most=0, scale=0.125, causal=1, out=P[6], lse=None, ws=None, bytes=0)
    a.update(over)
    return lib.cvsa_chunk_attention(*a.values(), None)


@pytest.mark.parametrize("over,code,word", [
    (dict(q=None), _lib.CVSA_ERR_INVALID, b"null"),
    (dict(host=None), _lib.CVSA_ERR_INVALID, b"null"),
    (dict(D=96), _lib.CVSA_ERR_UNSUPPORTED, b"D=96"),
    (dict(bs=12), _lib.CVSA_ERR_UNSUPPORTED, b"block_size=12"),
    (dict(H_q=7), _lib.CVSA_ERR_INVALID, b"head counts"),
    (dict(H_q=HK * 129), _lib.CVSA_ERR_UNSUPPORTED, b"G=129"),
    (dict(W=1 << 19, sb=1 << 19), _lib.CVSA_ERR_UNSUPPORTED, b"W="),
    (dict(sb=W - 1), _lib.CVSA_ERR_INVALID, b"bad sizes"),
    (dict(cu=(1, 3)), _lib.CVSA_ERR_INVALID, b"chunk offsets"),
    (dict(cu=(0, 3, 2)), _lib.CVSA_ERR_INVALID, b"chunk offsets"),
    (dict(cu=(0, 1 << 25)), _lib.CVSA_ERR_INVALID, b"chunk offsets"),
    (dict(scale=0.0), _lib.CVSA_ERR_INVALID, b"scale"),
    (dict(scale=float("inf")), _lib.CVSA_ERR_INVALID, b"scale"),
    (dict(scale=float("nan")), _lib.CVSA_ERR_INVALID, b"scale"),
    (dict(causal=2), _lib.CVSA_ERR_INVALID, b"causal"),
    (dict(most=-1), _lib.CVSA_ERR_INVALID, b"max_context_len"),
    (dict(sh=D + 4), _lib.CVSA_ERR_INVALID, b"aligned"),
    (dict(out=P[6] + 8), _lib.CVSA_ERR_INVALID, b"aligned"),
])
def test_c_attention_refuses(over, code, word):
    lib = _lib_or_skip()
    over = dict(over)
    cu = over.pop("cu", (0, 3)) if isinstance(over.get("cu"), tuple) else (0, 3)
    assert _attention(lib, cu=cu, **over) == code
    assert word in lib.cvsa_last_error()


def test_c_attention_asks_for_its_workspace():
    lib = _lib_or_skip()
    cu = (ctypes.c_int32 * 2)(0, 1)
    need = lib.cvsa_chunk_attention_workspace_bytes(cu, 1, HK * G, HK, D, BS, 4096, 0)
    assert need > 0
    for over in (dict(), dict(ws=256, bytes=need - 1), dict(ws=128, bytes=need)):
        assert _attention(lib, cu=(0, 1), W=4096, sb=4096, **over) == _lib.CVSA_ERR_WORKSPACE
    assert lib.cvsa_chunk_attention_workspace_bytes(cu, 1, HK * G, HK, 96, BS, 4096, 0) == 0
    # a context known to be short needs no split
    assert lib.cvsa_chunk_attention_workspace_bytes(cu, 1, HK * G, HK, D, BS, 4096, 64) == 0
    assert _attention(lib, cu=(0, 0)) == _lib.CVSA_OK  # no tokens: nothing is enqueued


def _append(lib, **over):
    a = dict(k=P[0], kst=HK * D, ksh=D, v=P[1], vst=HK * D, vsh=D, q=None, qst=0, qsh=0, dtype=0,
             kc=P[2], vc=P[3], nb=NB, bt=P[4], sb=W, W=W, ctx=P[5], cu=P[6], B=1, tokens=3,
             table=None, rows=0, rot=0, inter=0, qw=None, kw=None, wd=0, eps=1e-6, H_q=0, H_kv=HK,
             D=D, bs=BS, qo=None)
    a.update(over)
    return lib.cvsa_append_chunk_kv(*a.values(), None)


@pytest.mark.parametrize("over,code,word", [
    (dict(k=None), _lib.CVSA_ERR_INVALID, b"null"),
    (dict(q=P[0], qo=None), _lib.CVSA_ERR_INVALID, b"null"),
    (dict(q=P[0], qo=P[1], H_q=0), _lib.CVSA_ERR_INVALID, b"bad sizes"),
    (dict(D=48), _lib.CVSA_ERR_UNSUPPORTED, b"D=48"),
    (dict(bs=4), _lib.CVSA_ERR_UNSUPPORTED, b"block_size=4"),
    (dict(dtype=3), _lib.CVSA_ERR_INVALID, b"dtype"),
    (dict(kw=P[0], wd=9), _lib.CVSA_ERR_INVALID, b"weight dtype"),
    (dict(kw=P[0] + 4), _lib.CVSA_ERR_INVALID, b"weights"),
    (dict(table=P[0], rows=4, rot=24), _lib.CVSA_ERR_UNSUPPORTED, b"rotated"),
    (dict(table=P[0], rows=4, rot=2 * D), _lib.CVSA_ERR_UNSUPPORTED, b"rotated"),
    (dict(table=P[0], rows=0, rot=D), _lib.CVSA_ERR_INVALID, b"table"),
    (dict(inter=2), _lib.CVSA_ERR_INVALID, b"interleaved"),
    (dict(tokens=0), _lib.CVSA_ERR_INVALID, b"tokens=0"),
    (dict(kst=HK * D + 4), _lib.CVSA_ERR_INVALID, b"aligned"),
    (dict(kc=P[2] + 2), _lib.CVSA_ERR_INVALID, b"aligned"),
    (dict(W=W + 1), _lib.CVSA_ERR_INVALID, b"bad sizes"),
])
def test_c_append_refuses(over, code, word):
    lib = _lib_or_skip()
    assert _append(lib, **over) == code
    assert word in lib.cvsa_last_error()


@pytest.mark.parametrize("size", [0, 2, 16])
def test_c_norm_rope_refuses_positions_of_another_size(size):
    lib = _lib_or_skip()
    args = [P[0], HK * D, D, None, 0, 0, 0, P[1], size, P[2], 8, D, 0, None, None, 0, 1e-6, 3, HK,
            0, D, P[3], None, None]
    assert lib.cvsa_qk_norm_rope(*args) == _lib.CVSA_ERR_INVALID
    assert b"positions" in lib.cvsa_last_error()


def test_c_reserve_refuses():
    lib = _lib_or_skip()
    good = [P[0], W, W, P[1], P[2], P[3], 2, 0, NB, BS]
    for i, bad, word in ((0, None, b"null"), (5, None, b"null"), (6, 0, b"B=0"), (1, W - 1, b"W="),
                         (7, -1, b"bad sizes"), (8, 0, b"bad sizes"), (9, 20, b"block_size=20")):
        args = list(good)
        args[i] = bad
        assert lib.cvsa_reserve_chunk(*args, None) in (_lib.CVSA_ERR_INVALID,
                                                       _lib.CVSA_ERR_UNSUPPORTED)
        assert word in lib.cvsa_last_error()


# ------------------------------------------------------------ manager

def _manager():
    return SequenceKVManager(PagedKVCache(6, BS, HK, D, device="cpu"), 3, 64)


def _state(m):
    return (list(m._ctx_host), list(m._pages_allocated), m.cache._next_free,
            m.context_lens.tolist(), m.block_tables.tolist())


def test_manager_checks_before_it_changes_anything(calls):
    m = _manager()
    m.reserve_chunk(ops.ChunkLayout(LENS, "cpu"))  # 1 + 0 + 2 blocks
    assert [c[0] for c in calls] == ["reserve_chunk"] and m.cache._next_free == 3
    assert m._ctx_host == LENS and m._pages_allocated == [1, 0, 2]
    before = _state(m)
    short = ops.RotaryTable.build(D, 30, device="cpu")
    lay = ops.ChunkLayout(LENS, "cpu")
    cases = [
        (IndexError, dict(layout=ops.ChunkLayout([0, 65, 0], "cpu"))),     # past the table
        (AssertionError, dict(layout=ops.ChunkLayout([0, 64, 0], "cpu"))),  # pool of 6
        (ValueError, dict(layout=ops.ChunkLayout([1], "cpu"))),
        (ValueError, dict(layout=lay, rotary=short)),                       # position 39
        (ValueError, dict(layout=lay, k=_bf(T, HK + 1, D))),
        (ValueError, dict(layout=lay, v=_bf(T - 1, HK, D))),
        (ValueError, dict(layout=lay, q=_bf(T, HK * G, 32))),
    ]
    for error, kw in cases:
        args = dict(k=_bf(T, HK, D), v=_bf(T, HK, D))
        args.update(kw)
        with pytest.raises(error):
            m.append_chunk_kv(**args)
        assert _state(m) == before and len(calls) == 1
    m.append_chunk_kv(_bf(T, HK, D), _bf(T, HK, D), lay)
    assert [c[0] for c in calls[1:]] == ["reserve_chunk", "append_chunk_kv"]
    assert m._ctx_host == [6, 0, 40] and m._pages_allocated == [1, 0, 3]


def test_manager_refuses_a_head_dimension_first(calls):
    m = SequenceKVManager(PagedKVCache(6, BS, HK, 48, device="cpu"), 1, 64)
    with pytest.raises(NotImplementedError):
        m.append_chunk_kv(_bf(3, HK, 48), _bf(3, HK, 48), ops.ChunkLayout([3], "cpu"))
    assert not calls and m._ctx_host == [0]


# ------------------------------------------------------------ positions

def _position_reader(monkeypatch):
    """qk_norm_rope on CPU tensors; the positions that its launch was given."""
    seen = []

    def call(dev, who, fn, *args, keep=None):
        at, size, tokens = args[7], args[8], args[17]
        kind = {4: ctypes.c_int32, 8: ctypes.c_int64}[size]
        seen.append(list((kind * tokens).from_address(at)))

    monkeypatch.setattr(chunk, "_call", call)
    return seen


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint32, torch.uint64])
def test_positions_past_32_bits_stay_outside_the_table(calls, monkeypatch, dtype):
    """A position that int32 cannot hold must not come back as another one."""
    seen = _position_reader(monkeypatch)
    far = {torch.int64: [7, 2 ** 32 + 5, 2 ** 31, 2 ** 62 + 1, 79, -1, -2 ** 32 + 5, -2 ** 63],
           torch.uint32: [7, 2 ** 31, 2 ** 31 + 5, 2 ** 32 - 1, 79],
           torch.uint64: [7, 2 ** 32 + 5, 2 ** 63 + 5, 2 ** 64 - 1, 79]}[dtype]
    T = len(far)
    pos = torch.tensor(far, dtype=dtype)
    table = ops.RotaryTable.build(D, 80, device="cpu")
    for p in (pos, torch.stack([pos, pos], 1)[:, 0]):  # strided too
        ops.qk_norm_rope(_bf(T, 1, D), None, p, table)
    for got in seen:
        for x, y in zip(far, got):
            assert y == x if 0 <= x < 80 else not 0 <= y < 80
    assert [len(got) for got in seen] == [T, T]


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.uint16, torch.int32])
def test_narrow_positions_are_kept(calls, monkeypatch, dtype):
    seen = _position_reader(monkeypatch)
    pos = torch.tensor([0, 5, 79], dtype=dtype)
    ops.qk_norm_rope(_bf(3, 1, D), None, pos, ops.RotaryTable.build(D, 80, device="cpu"))
    assert seen == [[0, 5, 79]]


def test_wide_positions_are_read_in_place(calls):
    """No launch in front of the call's own."""
    pos = torch.arange(3)
    ops.qk_norm_rope(_bf(3, 1, D), None, pos, ops.RotaryTable.build(D, 80, device="cpu"))
    assert calls[0][1][7:9] == (pos.data_ptr(), 8)


@pytest.mark.parametrize("dtype", [torch.bool, torch.complex64, torch.float32])
def test_positions_that_are_no_integers_are_refused(calls, dtype):
    with pytest.raises(ValueError, match="positions"):
        ops.qk_norm_rope(_bf(3, 1, D), None, torch.zeros(3, dtype=dtype),
                         ops.RotaryTable.build(D, 80, device="cpu"))
    assert not calls


# ------------------------------------------------------------ strides

def _bent(t, stride):
    """t (one entry along its first dimension) with another stride there: torch
    calls it contiguous, whatever the stride is."""
    assert t.shape[0] == 1
    return t.as_strided(t.shape, (stride, *t.stride()[1:]))


def test_the_stride_of_one_token_and_of_one_sequence_does_not_matter(calls):
    """One token of rows that are no multiple of 16 bytes apart, and the table
    of one sequence: no second row is read, so no stride refuses them."""
    a = _append_args()
    a["layout"] = ops.ChunkLayout([1], "cpu")
    a["block_tables"] = _bent(torch.zeros(1, W, dtype=torch.int32), 1)
    a["context_lens"] = torch.ones(1, dtype=torch.int32)
    a.update(k=_bent(_bf(1, HK, D), HK * D + 3), v=_bent(_bf(1, HK, D), 1),
             q=_bent(_bf(1, HK * G, D), HK * G * D + 1))
    ops.append_chunk_kv(**a)
    b = _attend_args()
    b.update({n: a[n] for n in ("q", "layout", "block_tables", "context_lens")})
    ops.chunk_attention(**b)
    r = _rope_args()
    # one head: its stride is none either
    one = _bf(1, 1, D).as_strided((1, 1, D), (D + 5, 7, 1))
    r.update(q=a["q"], k=one, positions=torch.zeros(1, dtype=torch.int64))
    ops.qk_norm_rope(**r)
    ops.reserve_chunk(a["block_tables"], a["context_lens"], torch.zeros(1, dtype=torch.int32),
                      a["layout"], 0, NB, BS)
    got = {who: dict(zip(range(len(args)), args)) for who, args in calls}
    # (stride of the tokens, stride of the heads) in elements, multiples of 8
    for who, places in (("append_chunk_kv", (1, 4, 7)), ("chunk_attention", (1,)),
                        ("qk_norm_rope", (1, 4))):
        for i in places:
            assert got[who][i] % 8 == 0 and got[who][i + 1] % 8 == 0
    assert got["append_chunk_kv"][14] >= W and got["append_chunk_kv"][15] == W
    assert got["chunk_attention"][7] >= W and got["reserve_chunk"][1] >= W


def test_a_table_that_sequences_share_is_read(calls):
    """One row of blocks for every sequence, as a broadcast view."""
    b = _attend_args()
    b["block_tables"] = torch.zeros(1, W, dtype=torch.int32).expand(3, W)
    ops.chunk_attention(**b)
    assert calls[0][1][7] >= W


# ------------------------------------------------------------ before any state changes

@pytest.mark.parametrize("error,bad", [
    (TypeError, dict(eps=None)), (ValueError, dict(eps="small")),
    (ValueError, dict(q=_bf(1, 1, D).expand(T, 65537, D))),
])
def test_manager_refuses_before_pages_are_taken(calls, error, bad):
    """What only the launch looked at: by then the pages were taken."""
    m = _manager()
    before = _state(m)
    with pytest.raises(error):
        m.append_chunk_kv(_bf(T, HK, D), _bf(T, HK, D), ops.ChunkLayout(LENS, "cpu"), **bad)
    assert _state(m) == before and not calls


def test_a_prepared_append_reads_the_tables_at_its_launch(calls, monkeypatch):
    """The tables that grow between the checks and the launch, in a form that
    the kernel needs copied: the copy is the launch's."""
    a = _append_args()
    a["context_lens"], a["block_tables"] = a["context_lens"].long(), a["block_tables"].long()
    launch, _ = ops.prepare_append_chunk(**a)
    a["context_lens"] += 9
    a["block_tables"] += 4
    got = []

    def call(dev, who, fn, *args, keep=None):
        got.append((list((ctypes.c_int32 * 3).from_address(args[16])),
                    list((ctypes.c_int32 * (3 * W)).from_address(args[13]))))

    monkeypatch.setattr(chunk, "_call", call)
    launch()
    assert got == [([n + 9 for n in LENS], [4] * (3 * W))]


# ------------------------------------------------------------ captured graphs

def test_manager_refuses_to_be_captured(calls, monkeypatch):
    """A replay would hand out the same blocks again, and the manager's
    lengths would stay behind."""
    m = _manager()
    before = _state(m)
    lay = ops.ChunkLayout(LENS, "cpu")
    monkeypatch.setattr(chunk, "capturing", lambda dev: True)
    with pytest.raises(RuntimeError, match="captur"):
        m.reserve_chunk(lay)
    with pytest.raises(RuntimeError, match="captur"):
        m.append_chunk_kv(_bf(T, HK, D), _bf(T, HK, D), lay)
    assert _state(m) == before and not calls
    ops.append_chunk_kv(**_append_args())  # over tables of the caller's: may be captured
    ops.chunk_attention(**_attend_args())
    assert len(calls) == 2
