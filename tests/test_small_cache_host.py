"""Refusals of the operators on caches of 8 bits, of the weights of keys and of
eviction, all on the host before any launch, and the manager's rules."""
import ctypes

import pytest
import torch

from cvsa import ops
from cvsa.ops import _lib, chunk, eviction
from cvsa.runtime import kv_cache
from cvsa.runtime.kv_cache import PagedKVCache, SequenceKVManager

BS, HK, G, D, NB, W = 16, 2, 4, 64, 20, 5
LENS = [3, 0, 20]
T = sum(LENS)
F8, SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.fixture
def calls(monkeypatch):
    """Ops on CPU tensors whose launches are only recorded."""
    made = []

    def call(dev, who, fn, *args, keep=None):
        made.append((fn, args))

    for module in (chunk, eviction):
        monkeypatch.setattr(module, "_same_device", lambda *t: torch.device("cpu"))
        monkeypatch.setattr(module, "_call", call)
    monkeypatch.setattr(chunk, "_device_of", lambda *t: torch.device("cpu"))

    class Lib:
        cvsa_append_chunk_kv8 = "cvsa_append_chunk_kv8"
        cvsa_chunk_attention8 = "cvsa_chunk_attention8"
        cvsa_add_key_weights = "cvsa_add_key_weights"
        cvsa_evict_tokens = "cvsa_evict_tokens"
        cvsa_append_chunk_kv = "cvsa_append_chunk_kv"
        cvsa_chunk_attention = "cvsa_chunk_attention"
        cvsa_reserve_chunk = "cvsa_reserve_chunk"
        cvsa_chunk_attention_workspace_bytes = cvsa_chunk_attention8_workspace_bytes = \
            cvsa_add_key_weights_workspace_bytes = cvsa_evict_tokens_workspace_bytes = \
            staticmethod(lambda *a: 0)

    monkeypatch.setattr(chunk._lib, "load", lambda: Lib)
    return made


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def _f8(*shape):
    return torch.zeros(*shape, dtype=F8)


def _scales(*shape):
    return torch.full(shape, 127, dtype=torch.uint8).view(SCALE)


def _cache():
    return dict(k_cache=_f8(NB, BS, HK, D), v_cache=_f8(NB, BS, HK, D),
                block_tables=torch.zeros(3, W, dtype=torch.int32),
                context_lens=torch.tensor(LENS, dtype=torch.int32), k_scales=_scales(NB, HK),
                v_scales=_scales(NB, HK))


def _append_args():
    return dict(k=_bf(T, HK, D), v=_bf(T, HK, D), layout=ops.ChunkLayout(LENS, "cpu"),
                block_size=BS, **_cache())


def _attend_args():
    return dict(q=_bf(T, HK * G, D), layout=ops.ChunkLayout(LENS, "cpu"), num_kv_heads=HK,
                num_q_per_kv=G, block_size=BS, **_cache())


def _weigh_args():
    a = _attend_args()
    del a["v_cache"], a["v_scales"]
    return dict(weights=torch.zeros(3, HK, W * BS), lse=torch.zeros(T, HK * G), **a)


def _evict_args():
    return dict(weights=torch.zeros(3, HK, W * BS), keep=20, block_size=BS, sinks=2, recent=4,
                **_cache())


def test_good_calls_reach_the_library(calls):
    ops.append_chunk_kv(**_append_args())
    out, lse = ops.chunk_attention(**_attend_args(), return_lse=True)
    w = _weigh_args()
    assert ops.add_key_weights(**w) is w["weights"]
    kept = ops.evict_tokens(**_evict_args())
    assert kept.shape == (3, HK, 20) and kept.dtype == torch.int32
    assert out.dtype == torch.bfloat16 and lse.dtype == torch.float32
    names = ["cvsa_append_chunk_kv8", "cvsa_chunk_attention8", "cvsa_add_key_weights",
             "cvsa_evict_tokens"]
    assert [c[0] for c in calls] == names
    for name, args in calls:  # one argument for each of the C entry's, but the stream
        assert len(args) == len(_lib.SIGNATURES[name][1]) - 1
    # bf16 caches for the last two
    b = dict(k_cache=_bf(NB, BS, HK, D), k_scales=None)
    ops.add_key_weights(**{**_weigh_args(), **b})
    ops.evict_tokens(**{**_evict_args(), **b, "v_cache": _bf(NB, BS, HK, D), "v_scales": None})
    assert [c[0] for c in calls][4:] == names[2:]


BAD_CACHE = [
    dict(k_scales=None), dict(v_scales=None), dict(k_scales=None, v_scales=None),
    dict(k_cache=_bf(NB, BS, HK, D)), dict(v_cache=_bf(NB, BS, HK, D)),
    dict(k_cache=_bf(NB, BS, HK, D), v_cache=_bf(NB, BS, HK, D)),
    dict(k_cache=torch.zeros(NB, BS, HK, D, dtype=torch.float8_e5m2)),
    dict(k_cache=_f8(NB, BS, HK, 2 * D)[..., ::2]), dict(v_cache=_f8(NB + 1, BS, HK, D)),
    dict(v_cache=_f8(NB + 1, BS, HK, D), v_scales=_scales(NB + 1, HK)),
    dict(k_cache=_f8(NB * BS, HK, D)), dict(k_cache=_f8(NB * BS * HK * D + 1)[1:].view(
        NB, BS, HK, D)),
    dict(k_scales=_scales(NB, HK + 1)), dict(k_scales=_scales(NB + 1, HK)),
    dict(k_scales=torch.ones(NB, HK)), dict(v_scales=torch.ones(NB, HK, dtype=torch.uint8)),
    dict(v_scales=_scales(HK, NB).t()), dict(block_size=32),
    dict(block_tables=torch.zeros(2, W, dtype=torch.int32)),
    dict(context_lens=torch.zeros(4, dtype=torch.int32)),
]


@pytest.mark.parametrize("bad", BAD_CACHE)
@pytest.mark.parametrize("op,args", [(ops.append_chunk_kv, _append_args),
                                     (ops.chunk_attention, _attend_args),
                                     (ops.evict_tokens, _evict_args)])
def test_caches_are_refused(calls, op, args, bad):
    with pytest.raises(ValueError):
        op(**{**args(), **bad})
    assert not calls


BAD_WEIGH = [
    dict(k_scales=None), dict(k_cache=_bf(NB, BS, HK, D)), dict(k_scales=_scales(NB, HK + 1)),
    dict(weights=torch.zeros(3, HK, W * BS - 1)), dict(weights=torch.zeros(2, HK, W * BS)),
    dict(weights=torch.zeros(3, HK + 1, W * BS)), dict(weights=torch.zeros(3, HK * W * BS)),
    dict(weights=torch.zeros(3, HK, W * BS, dtype=torch.float64)),
    dict(weights=torch.zeros(3, HK, 2 * W * BS)[..., ::2]),
    dict(lse=torch.zeros(T - 1, HK * G)), dict(lse=torch.zeros(T, HK)),
    dict(lse=torch.zeros(T, HK * G, dtype=torch.float64)), dict(lse=torch.zeros(T * HK * G)),
    dict(q=_bf(T - 1, HK * G, D)), dict(q=torch.zeros(T, HK * G, D)), dict(num_kv_heads=4),
    dict(num_q_per_kv=2), dict(window=-1), dict(block_size=8),
    dict(layout=ops.ChunkLayout([T], "cpu")), dict(context_lens=torch.zeros(2, dtype=torch.int32)),
]


@pytest.mark.parametrize("bad", BAD_WEIGH)
def test_weights_are_refused(calls, bad):
    with pytest.raises(ValueError):
        ops.add_key_weights(**{**_weigh_args(), **bad})
    assert not calls


BAD_EVICT = [
    dict(keep=0), dict(keep=-3), dict(sinks=-1), dict(recent=-1), dict(sinks=17, recent=4),
    dict(weights=torch.zeros(3, HK, W * BS - 1)), dict(weights=torch.zeros(2, HK, W * BS)),
    dict(weights=_bf(3, HK, W * BS)), dict(block_tables=torch.zeros(3 * W, dtype=torch.int32)),
]


@pytest.mark.parametrize("bad", BAD_EVICT)
def test_evictions_are_refused(calls, bad):
    with pytest.raises(ValueError):
        ops.evict_tokens(**{**_evict_args(), **bad})
    assert not calls


def test_empty_chunks_launch_nothing(calls):
    a, b, c = _append_args(), _attend_args(), _weigh_args()
    a["layout"] = b["layout"] = c["layout"] = ops.ChunkLayout([0, 0, 0], "cpu")
    assert ops.append_chunk_kv(**a) is None
    assert (ops.chunk_attention(**b) == 0).all()
    assert ops.add_key_weights(**c) is c["weights"]
    assert not calls


def test_cpu_tensors_are_refused():
    for op, args in ((ops.append_chunk_kv, _append_args), (ops.chunk_attention, _attend_args),
                     (ops.add_key_weights, _weigh_args), (ops.evict_tokens, _evict_args)):
        with pytest.raises(ValueError, match="GPU only"):
            op(**args())


# ------------------------------------------------------------ C ABI

def _lib_or_skip():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libcvsa_hip.so not built")
    try:
        return _lib.load()
    except OSError as e:  # no HIP runtime on this host
        pytest.skip(f"HIP runtime not loadable: {e}")


P = [i << 20 for i in range(1, 12)]  # never dereferenced
INVALID, UNSUPPORTED = _lib.CVSA_ERR_INVALID, _lib.CVSA_ERR_UNSUPPORTED


def _attention(lib, cu=(0, 3), **over):
    a = dict(q=P[0], st=HK * G * D, sh=D, kc=P[1], vc=P[2], ks=P[7], vs=P[8], nb=NB, bt=P[3], sb=W,
             ctx=P[4], cu=P[5], host=(ctypes.c_int32 * len(cu))(*cu), B=len(cu) - 1, H_q=HK * G,
             H_kv=HK, D=D, bs=BS, W=W, most=0, scale=0.125, causal=1, out=P[6], lse=None, ws=None,
             bytes=0)
    a.update(over)
    return lib.cvsa_chunk_attention8(*a.values(), None)


@pytest.mark.parametrize("over,code,word", [
    (dict(q=None), INVALID, b"null"), (dict(ks=None), INVALID, b"null"),
    (dict(vs=None), INVALID, b"null"), (dict(D=96), UNSUPPORTED, b"D=96"),
    (dict(bs=12), UNSUPPORTED, b"block_size=12"), (dict(H_q=7), INVALID, b"head counts"),
    (dict(sb=W - 1), INVALID, b"bad sizes"), (dict(scale=0.0), INVALID, b"scale"),
    (dict(causal=2), INVALID, b"causal"), (dict(kc=P[1] + 8), INVALID, b"aligned"),
])
def test_c_attention_refuses(over, code, word):
    lib = _lib_or_skip()
    assert _attention(lib, **over) == code
    said = lib.cvsa_last_error()
    assert word in said and b"chunk_attention8" in said


def test_c_attention_asks_for_its_workspace():
    lib = _lib_or_skip()
    cu = (ctypes.c_int32 * 2)(0, 1)
    need = lib.cvsa_chunk_attention8_workspace_bytes(cu, 1, HK * G, HK, D, BS, 4096, 0)
    assert need > 0
    for over in (dict(), dict(ws=256, bytes=need - 1), dict(ws=128, bytes=need)):
        assert _attention(lib, cu=(0, 1), W=4096, sb=4096, **over) == _lib.CVSA_ERR_WORKSPACE
    assert _attention(lib, cu=(0, 0)) == _lib.CVSA_OK  # no tokens: nothing is enqueued


def _append(lib, **over):
    a = dict(k=P[0], kst=HK * D, ksh=D, v=P[1], vst=HK * D, vsh=D, q=None, qst=0, qsh=0, dtype=0,
             kc=P[2], vc=P[3], ks=P[7], vs=P[8], nb=NB, bt=P[4], sb=W, W=W, ctx=P[5], cu=P[6], B=1,
             tokens=3, table=None, rows=0, rot=0, inter=0, qw=None, kw=None, wd=0, eps=1e-6, H_q=0,
             H_kv=HK, D=D, bs=BS, qo=None)
    a.update(over)
    return lib.cvsa_append_chunk_kv8(*a.values(), None)


@pytest.mark.parametrize("over,code,word", [
    (dict(k=None), INVALID, b"null"), (dict(ks=None), INVALID, b"null"),
    (dict(vs=None), INVALID, b"null"), (dict(q=P[0], qo=None), INVALID, b"null"),
    (dict(D=48), UNSUPPORTED, b"D=48"), (dict(bs=4), UNSUPPORTED, b"block_size=4"),
    (dict(dtype=3), INVALID, b"dtype"), (dict(kc=P[2] + 8), INVALID, b"aligned"),
    (dict(tokens=0), INVALID, b"tokens=0"), (dict(sb=W - 1), INVALID, b"bad sizes"),
    (dict(vst=HK * D + 4), INVALID, b"aligned"),
    (dict(table=P[9], rows=4, rot=24), UNSUPPORTED, b"rotated"),
    (dict(B=1 << 30, H_kv=65536), UNSUPPORTED, b"too many"),
])
def test_c_append_refuses(over, code, word):
    lib = _lib_or_skip()
    assert _append(lib, **over) == code
    said = lib.cvsa_last_error()
    assert word in said and b"append_chunk_kv8" in said


def _weigh(lib, cu=(0, 3), **over):
    a = dict(w=P[0], S=W * BS, q=P[1], st=HK * G * D, sh=D, lse=P[2], kc=P[3], ks=None, nb=NB,
             bt=P[4], sb=W, ctx=P[5], cu=P[6], host=(ctypes.c_int32 * len(cu))(*cu),
             B=len(cu) - 1, H_q=HK * G, H_kv=HK, D=D, bs=BS, W=W, scale=0.125, causal=1, window=0,
             ws=None, bytes=0)
    a.update(over)
    return lib.cvsa_add_key_weights(*a.values(), None)


@pytest.mark.parametrize("over,code,word", [
    (dict(w=None), INVALID, b"null"), (dict(lse=None), INVALID, b"null"),
    (dict(host=None), INVALID, b"null"), (dict(D=96), UNSUPPORTED, b"D=96"),
    (dict(bs=12), UNSUPPORTED, b"block_size=12"), (dict(H_q=7), INVALID, b"head counts"),
    (dict(H_q=HK * 129), UNSUPPORTED, b"G=129"), (dict(S=W * BS - 1), INVALID, b"weights of"),
    (dict(sb=W - 1), INVALID, b"bad sizes"), (dict(window=-1), INVALID, b"bad sizes"),
    (dict(scale=float("nan")), INVALID, b"scale"), (dict(causal=3), INVALID, b"causal"),
    (dict(sh=D + 4), INVALID, b"aligned"), (dict(kc=P[3] + 8), INVALID, b"aligned"),
])
def test_c_weigh_refuses(over, code, word):
    lib = _lib_or_skip()
    assert _weigh(lib, **over) == code
    assert word in lib.cvsa_last_error()


def test_c_weigh_asks_for_its_workspace():
    lib = _lib_or_skip()
    for cu in ((1, 3), (0, 3, 2), (0, 1 << 25)):
        assert _weigh(lib, cu=cu) == INVALID
    assert _weigh(lib, cu=(0, 0)) == _lib.CVSA_OK
    cu = (ctypes.c_int32 * 2)(0, 2000)
    need = lib.cvsa_add_key_weights_workspace_bytes(cu, 1, HK * G, HK, D, W * BS, 0)
    assert need > 0
    for over in (dict(), dict(ws=P[9], bytes=need - 1)):
        assert _weigh(lib, cu=(0, 2000), **over) == _lib.CVSA_ERR_WORKSPACE
    # more tiles than a launch has workgroups of 256 threads
    many = tuple(40 * b for b in range(4001))
    wide = dict(W=(1 << 18) - 1, sb=1 << 18, bs=128, S=1 << 25, H_q=1, H_kv=1)
    assert _weigh(lib, cu=many, **wide) == UNSUPPORTED
    assert b"too many" in lib.cvsa_last_error()
    # the last few tokens alone need none
    assert lib.cvsa_add_key_weights_workspace_bytes(cu, 1, HK * G, HK, D, W * BS, 8) == 0


def _evict(lib, **over):
    a = dict(w=P[0], S=W * BS, kc=P[1], vc=P[2], ks=None, vs=None, nb=NB, bt=P[3], sb=W, W=W,
             ctx=P[4], B=1, H_kv=HK, D=D, bs=BS, keep=20, sinks=2, recent=4, kept=P[5], ws=P[6],
             bytes=1 << 40)
    a.update(over)
    return lib.cvsa_evict_tokens(*a.values(), None)


@pytest.mark.parametrize("over,code,word", [
    (dict(w=None), INVALID, b"null"), (dict(kept=None), INVALID, b"null"),
    (dict(ks=P[7]), INVALID, b"scales"), (dict(vs=P[7]), INVALID, b"scales"),
    (dict(D=48), UNSUPPORTED, b"D=48"), (dict(bs=4), UNSUPPORTED, b"block_size=4"),
    (dict(W=1 << 19, sb=1 << 19), UNSUPPORTED, b"W="), (dict(keep=0), INVALID, b"keep=0"),
    (dict(sinks=18), INVALID, b"sinks=18"), (dict(recent=-1), INVALID, b"recent=-1"),
    (dict(B=0), INVALID, b"B=0"), (dict(sb=W - 1), INVALID, b"bad sizes"),
    (dict(S=W * BS - 1), INVALID, b"weights of"), (dict(vc=P[2] + 8), INVALID, b"aligned"),
    (dict(B=1 << 19, H_kv=16), UNSUPPORTED, b"too many"),
    (dict(vc=P[1]), INVALID, b"of their own"),
    (dict(bytes=16), _lib.CVSA_ERR_WORKSPACE, b"workspace"),
    (dict(ws=None), _lib.CVSA_ERR_WORKSPACE, b"workspace"),
    (dict(ws=P[6] + 128), _lib.CVSA_ERR_WORKSPACE, b"workspace"),
])
def test_c_evict_refuses(over, code, word):
    lib = _lib_or_skip()
    assert _evict(lib, **over) == code
    assert word in lib.cvsa_last_error()


def test_c_evict_asks_for_a_workspace_only_where_two_launches_share_it():
    lib = _lib_or_skip()

    def need(B, D=128, bs=16, W=260, keep=4096, recent=256, bits=8):
        return lib.cvsa_evict_tokens_workspace_bytes(B, 8, D, bs, W, bits, keep, 4, recent)
    assert need(32) == need(64) == need(16) == need(32, bits=16) == 0
    assert need(1) > 0 and need(32, W=1025) > 0 and need(32, bs=128) > 0
    assert need(32, D=256, bits=16) > 0 and need(16, W=1024, keep=8192) > 0


# ------------------------------------------------------------ the manager

def _manager(dtype=F8, batch=2):
    cache = PagedKVCache(NB, BS, HK, D, dtype=dtype, device="cpu")
    return cache, SequenceKVManager(cache, batch, 5 * BS)


def test_a_cache_of_8_bits_has_scales():
    cache, _ = _manager()
    assert cache.k_scales.shape == cache.v_scales.shape == (NB, HK)
    assert cache.k_scales.dtype == SCALE and (cache.k_scales.float() == 1).all()
    assert cache.k_scales.data_ptr() != cache.v_scales.data_ptr()
    for call in (lambda: cache.write_kv(0, 0, _bf(HK, D), _bf(HK, D)),
                 lambda: cache.write_kv_block(0, _bf(BS, HK, D), _bf(BS, HK, D), 3)):
        with pytest.raises(ValueError, match="scale"):
            call()
    assert PagedKVCache(NB, BS, HK, D, device="cpu").k_scales is None


def test_the_manager_appends_to_8_bits(calls):
    cache, mgr = _manager()
    rows = _bf(2, HK, D)
    assert not mgr.fusable_rows(rows, rows)
    mgr.prefill_kv(1, _bf(20, HK, D), _bf(20, HK, D))
    assert mgr._ctx_host == [0, 20] and mgr.context_lens.tolist() == [0, 20]
    mgr.append_tokens_kv(rows, rows)
    mgr.append_token_kv(0, rows[0], rows[0])
    assert mgr._ctx_host == [2, 21]
    done = [c[0] for c in calls if c[0] != "cvsa_reserve_chunk"]
    assert done == ["cvsa_append_chunk_kv8"] * 3
    # the layouts of single tokens are kept
    first = dict(mgr._token_layouts)
    assert {k: x.lens for k, x in first.items()} == {(0, 2): (1, 1), (0, 1): (1, 0)}
    mgr.append_tokens_kv(rows, rows)
    mgr.append_token_kv(1, rows[0], rows[0])
    assert all(mgr._token_layouts[k] is x for k, x in first.items())
    assert mgr._token_layouts[1, 1].lens == (0, 1) and mgr._ctx_host == [3, 23]


def test_a_refused_prompt_takes_no_block(calls):
    cache, mgr = _manager()
    for k, v in ((_bf(20, HK, D), _bf(19, HK, D)), (_bf(20, HK, D), _bf(20, HK, D).float()),
                 (_bf(20, HK, D + 8), _bf(20, HK, D + 8)), (_bf(20, HK + 1, D), _bf(20, HK, D))):
        with pytest.raises(ValueError):
            mgr.prefill_kv(0, k, v)
    assert cache._next_free == 0 and mgr._ctx_host == [0, 0] and not calls
    assert mgr.context_lens.tolist() == [0, 0]
    mgr.prefill_kv(1, _bf(0, HK, D), _bf(0, HK, D))
    assert mgr._ctx_host == [0, 0] and not calls
    mgr.prefill_kv(-1, _bf(17, HK, D), _bf(17, HK, D))  # the last sequence
    assert mgr._ctx_host == [0, 17] and len(calls) == 1


def test_the_manager_cuts(calls, monkeypatch):
    cache, mgr = _manager()
    mgr.prefill_kv(0, _bf(40, HK, D), _bf(40, HK, D))
    mgr.prefill_kv(1, _bf(7, HK, D), _bf(7, HK, D))
    w = torch.zeros(2, HK, 5 * BS)
    kept = mgr.evict_tokens(w, 12, 2, 4)
    assert kept.shape == (2, HK, 12) and calls[-1][0] == "cvsa_evict_tokens"
    assert mgr._ctx_host == [12, 7] and mgr.context_lens.tolist() == [12, 7]
    assert mgr._pages_allocated == [3, 1]  # theirs still
    mgr.cut(100.5)
    assert mgr._ctx_host == [12, 7]
    mgr.evict_tokens(w, 12.75)
    assert mgr._ctx_host == [12, 7] and all(type(c) is int for c in mgr._ctx_host)
    n = len(calls)
    for call in (lambda: mgr.cut(0), lambda: mgr.evict_tokens(w, 0),
                 lambda: mgr.evict_tokens(w, 5, 3, 3)):
        with pytest.raises(ValueError):
            call()
    monkeypatch.setattr(kv_cache.ops.chunk, "capturing", lambda dev: True)
    for call in (lambda: mgr.cut(5), lambda: mgr.evict_tokens(w, 5)):
        with pytest.raises(RuntimeError, match="captured"):
            call()
    assert mgr._ctx_host == [12, 7] and len(calls) == n


def test_a_token_of_no_sequence_is_refused(calls):
    cache, mgr = _manager()
    row = _bf(HK, D)
    for s in (-1, -2, 2, 7):
        with pytest.raises(IndexError):
            mgr.append_token_kv(s, row, row)
    with pytest.raises(ValueError):
        mgr.append_tokens_kv(_bf(2, HK, D), _bf(3, HK, D))
    assert mgr._ctx_host == [0, 0] and cache._next_free == 0 and not calls
    assert not mgr._token_layouts
    mgr.append_token_kv(1, row, row)
    assert mgr._ctx_host == [0, 1]


def test_a_prompt_past_the_tables_takes_no_block(calls):
    cache, mgr = _manager()
    with pytest.raises(IndexError, match="block table"):
        mgr.prefill_kv(0, _bf(5 * BS + 1, HK, D), _bf(5 * BS + 1, HK, D))
    assert cache._next_free == 0 and mgr._ctx_host == [0, 0] and not calls
    assert mgr.context_lens.tolist() == [0, 0]
    mgr.prefill_kv(0, _bf(5 * BS, HK, D), _bf(5 * BS, HK, D))
    assert cache._next_free == 5 and mgr._ctx_host == [5 * BS, 0]


def test_c_weigh_refuses_queries_that_32_bits_cannot_span():
    lib = _lib_or_skip()
    most = (1 << 31) - 1
    for g, st, sh in ((4, HK * G * D, most // 3 // 8 * 8 + 8), (4, most // 32 // 8 * 8 + 8, D),
                      (1, most // 127 // 8 * 8 + 8, D), (4, 1 << 40, D), (4, 8, 1 << 40)):
        assert _weigh(lib, cu=(0, 2000), H_q=HK * g, st=st, sh=sh) == UNSUPPORTED
        assert b"too far apart" in lib.cvsa_last_error()
    # Those that it can are asked for their workspace.
    for g, st, sh in ((4, D, 1 << 23), (4, 1 << 25, D), (1, 1 << 24, D), (4, 1 << 24, 1 << 28)):
        assert _weigh(lib, cu=(0, 2000), H_q=HK * g, st=st, sh=sh) == _lib.CVSA_ERR_WORKSPACE
    # Groups of one head: none is far from its group's first.
    assert _weigh(lib, cu=(0, 2000), H_q=HK, st=D, sh=1 << 40) == _lib.CVSA_ERR_WORKSPACE
    assert _weigh(lib, st=-8) == INVALID


def test_queries_far_apart_are_copied(calls, monkeypatch):
    """What the kernel's 32 bits cannot span is made contiguous, nothing else is."""
    w = _weigh_args()
    where = w["q"].data_ptr()
    for st, sh, copied in ((HK * G * D, 1 << 23, False), (1 << 25, D, False),
                           (1 << 26, D, True), (HK * G * D, 1 << 30, True)):
        monkeypatch.setattr(eviction, "_rows", lambda *a: (a[2], where, st, sh))
        ops.add_key_weights(**w)
        at, st_, sh_ = calls[-1][1][2:5]
        assert (st_, sh_) == ((HK * G * D, D) if copied else (st, sh))


def test_c_caches_that_are_written_are_not_shared():
    """Keys and values would write one row, or one byte of a scale, each its own."""
    lib = _lib_or_skip()
    for over in (dict(vc=P[2]), dict(vs=P[7])):
        assert _append(lib, **over) == INVALID
        assert b"of their own" in lib.cvsa_last_error()
    assert _evict(lib, ks=P[7], vs=P[7]) == INVALID
    assert b"of their own" in lib.cvsa_last_error()


def test_caches_that_are_written_are_not_shared(calls):
    a = _append_args()
    for over in (dict(v_cache=a["k_cache"]), dict(v_scales=a["k_scales"])):
        with pytest.raises(ValueError, match="of their own"):
            ops.append_chunk_kv(**{**a, **over})
    assert not calls
    b = _attend_args()  # reading one is fine
    ops.chunk_attention(**{**b, "v_cache": b["k_cache"], "v_scales": b["k_scales"]})
    assert len(calls) == 1


def test_the_backends_prefill_returns_what_the_weights_need(calls):
    from cvsa.runtime.dense import DenseAttentionBackend
    a = _attend_args()
    dense = DenseAttentionBackend(HK, HK * G, D, BS)
    args = [a[x] for x in ("q", "k_cache", "v_cache", "block_tables", "context_lens", "layout")]
    kw = dict(k_scales=a["k_scales"], v_scales=a["v_scales"])
    assert dense.prefill(*args, **kw).shape == (T, HK * G, D)
    out, lse = dense.prefill(*args, **kw, return_lse=True)
    assert out.shape == (T, HK * G, D) and lse.shape == (T, HK * G)
    assert lse.dtype == torch.float32
    w = _weigh_args()
    ops.add_key_weights(**{**w, "lse": lse})
    assert [c[0] for c in calls] == ["cvsa_chunk_attention8"] * 2 + ["cvsa_add_key_weights"]


def test_c_evict_of_long_rows_takes_a_number_for_each_kept_slot():
    lib = _lib_or_skip()

    def need(keep):
        return lib.cvsa_evict_tokens_workspace_bytes(1, 8, 128, 16, 2048, 16, keep, 0, 0)
    assert need(8192) - need(4096) == 4096 * 8 * 4


def test_c_evict_of_tables_that_hold_no_more_than_is_kept_needs_nothing():
    lib = _lib_or_skip()
    for W, bs, D, bits in ((2048, 16, 128, 16), (260, 16, 128, 8), (40, 128, 256, 16)):
        for keep in (W * bs, W * bs + 1, 1 << 24):
            assert lib.cvsa_evict_tokens_workspace_bytes(1, 8, D, bs, W, bits, keep, 4, 256) == 0
        assert lib.cvsa_evict_tokens_workspace_bytes(1, 8, D, bs, W, bits, W * bs - 1, 4, 256) > 0


def test_no_append_of_the_managers_to_8_bits_is_captured(calls, monkeypatch):
    """Refused before a layout is copied from the host, which would end the capture."""
    cache, mgr = _manager()
    rows = _bf(2, HK, D)

    def layout(*a):
        raise AssertionError("a copy to the device in a capture")
    monkeypatch.setattr(kv_cache.ops.chunk, "capturing", lambda dev: True)
    monkeypatch.setattr(kv_cache.ops, "ChunkLayout", layout)
    for call in (lambda: mgr.append_tokens_kv(rows, rows),
                 lambda: mgr.append_token_kv(1, rows[0], rows[0]),
                 lambda: mgr.prefill_kv(0, _bf(20, HK, D), _bf(20, HK, D))):
        with pytest.raises(RuntimeError, match="captured"):
            call()
    assert mgr._ctx_host == [0, 0] and cache._next_free == 0 and not calls
    assert not mgr._token_layouts
