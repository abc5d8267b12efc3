"""Chunks of new tokens: several per sequence, taken into the paged cache and
attended from it.

A prompt, a piece of one, a draft to be verified or a decode step is a ragged
batch of new tokens (:class:`ChunkLayout`).  :func:`append_chunk_kv` writes
its keys, normed and rotated on the way, and its values to the cache, and can
rotate the queries in the same launch; :func:`chunk_attention` attends the
queries over the cache.  :func:`qk_norm_rope` is the norm and rotation alone,
for keys that stay outside the cache.

The cache is bf16, or holds 8 bits a value: e4m3 payloads with a power of two
for each block and head (``k_scales`` and ``v_scales``, see
:func:`append_chunk_kv`), half the bytes to keep and to read.

None of these has a counterpart in the reference, whose harness leaves
prefill to the model it wraps.  They serve; there is no backward pass.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import (_DTYPE_CODE, _block_tables, _check_cache, _check_count, _check_seqs, _device_of,
               _i32, _lib, _ptr, check)

_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
_F8, _SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu
_INTEGERS = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8, torch.uint16,
             torch.uint32, torch.uint64)


class ChunkLayout:
    """Which rows of a chunk's q, k and v belong to which sequence.

    ``query_lens[b]`` new tokens of sequence b, 0 allowed; their rows follow
    each other.  Made once per step and kept by the caller for all layers:
    ``cu_seqlens`` ([B + 1] int32) on the device and the same offsets on the
    host, from which the launches are shaped.
    """

    __slots__ = ("lens", "batch", "total", "longest", "cu_seqlens", "cu_host", "device",
                 "_workspace_bytes")

    def __init__(self, query_lens: Sequence[int], device="cuda"):
        lens = tuple(int(n) for n in query_lens)
        if not lens:
            raise ValueError("chunk layout: no sequences")
        if min(lens) < 0:
            raise ValueError(f"chunk layout: negative chunk length {min(lens)}")
        if sum(lens) > 1 << 24:
            raise ValueError(f"chunk layout: {sum(lens)} tokens (at most {1 << 24})")
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        self.lens = lens
        self.batch = len(lens)
        self.total = cu[-1]
        self.longest = max(lens)
        self.cu_host = (ctypes.c_int32 * len(cu))(*cu)
        self.cu_seqlens = torch.tensor(cu, dtype=torch.int32, device=device)
        self.device = self.cu_seqlens.device
        self._workspace_bytes = {}  # by the call's sizes


class RotaryTable:
    """Cosines and sines of every position's angles, kept by the caller.

    ``table``: [positions, rot_dim] fp32, the cosines of the rot_dim / 2
    angles, then their sines.  ``rot_dim`` is a multiple of 16; a head's
    dimensions past it are not rotated.  Pair i is (i, i + rot_dim / 2) of
    the head, or (2i, 2i + 1) with ``interleaved``.
    """

    __slots__ = ("table", "rot_dim", "max_positions", "interleaved")

    def __init__(self, table: torch.Tensor, interleaved: bool = False):
        if table.dim() != 2 or table.dtype != torch.float32:
            raise ValueError("rotary table must be [positions, rot_dim] float32, got "
                             f"{tuple(table.shape)} {table.dtype}")
        if table.shape[0] < 1:
            raise ValueError("rotary table holds no position")
        if table.shape[1] < 16 or table.shape[1] % 16:
            raise NotImplementedError(f"rotary table: rot_dim {table.shape[1]} is not a "
                                      "multiple of 16")
        self.table = table.contiguous()
        if self.table.data_ptr() % 16:
            self.table = self.table.clone()
        self.max_positions, self.rot_dim = table.shape
        self.interleaved = bool(interleaved)

    @classmethod
    def build(cls, rot_dim: int, max_positions: int, base: float = 10000.0, device="cuda",
              interleaved: bool = False) -> "RotaryTable":
        """Angles position * base^(-2i / rot_dim), taken in 64 bits (32 lose
        the angle of far positions) and rounded once."""
        i = torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device)
        ang = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] \
            * base ** (-i / rot_dim)
        return cls(torch.cat([ang.cos(), ang.sin()], 1).to(torch.float32), interleaved)


def _same_device(*tensors: Optional[torch.Tensor]) -> torch.device:
    """_device_of for the calls of every step: one look at each tensor."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != index or index < 0):
            return _device_of(*tensors)  # raises
    return tensors[0].device


def capturing(dev: torch.device) -> bool:
    """Whether dev's current stream records a graph."""
    if dev.type != "cuda":
        return False
    if torch._C._cuda_getDevice() == dev.index:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(dev):
        return torch.cuda.is_current_stream_capturing()


def _call(dev: torch.device, who: str, fn, *args, keep=None) -> None:
    """fn(*args, stream) on dev's current stream, whatever the current device;
    `keep` lives until the launch."""
    index = dev.index
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, who)


def _rows(who: str, name: str, t: torch.Tensor, rows: Optional[int], heads: Optional[int], D: int,
          dtype=None):
    """t as [>= rows, heads, D] rows that the kernels can read: (t, address,
    token stride, head stride)."""
    shape, dt = t.shape, t.dtype
    if len(shape) != 3 or shape[2] != D or (heads is not None and shape[1] != heads) \
            or (rows is not None and shape[0] < rows):
        raise ValueError(f"{who}: {name} must be [{'tokens' if rows is None else rows}, "
                         f"{'heads' if heads is None else heads}, {D}], got {tuple(shape)}")
    if (dt is not dtype) if dtype is not None else (dt not in _DTYPE_CODE):
        raise ValueError(f"{who}: {name} must be {dtype or 'bfloat16, float16 or float32'}, "
                         f"got {dt}")
    st, sh, sd = t.stride()
    at = t.data_ptr()
    if sd != 1 or (st | sh) & (3 if dt is _F32 else 7) or at & 15:
        t = t.contiguous()
        if t.data_ptr() & 15:
            t = t.clone()
        # Not t's own: the stride of a single token or head can be any number.
        st, sh = shape[1] * D, D
        at = t.data_ptr()
    return t, at, st, sh


def _weights(who: str, D: int, q_weight, k_weight):
    """Norm weights [D] of one dtype (None: no norm), and its code."""
    if q_weight is None and k_weight is None:
        return None, None, 0
    if q_weight is not None and k_weight is not None:
        dt = k_weight.dtype
        if q_weight.dtype is not dt:
            raise ValueError(f"{who}: q_weight and k_weight differ in dtype")
        if dt in _DTYPE_CODE and q_weight.shape == k_weight.shape == (D,) \
                and q_weight.is_contiguous() and k_weight.is_contiguous() \
                and not (q_weight.data_ptr() | k_weight.data_ptr()) & 15:
            return q_weight, k_weight, _DTYPE_CODE[dt]
    return (_weight(who, "q_weight", q_weight, D), _weight(who, "k_weight", k_weight, D),
            _DTYPE_CODE[(k_weight if q_weight is None else q_weight).dtype])


def _weight(who: str, name: str, w, D: int):
    if w is None:
        return None
    if w.dim() != 1 or w.shape[0] != D or w.dtype not in _DTYPE_CODE:
        raise ValueError(f"{who}: {name} must be [{D}] of a float dtype, got "
                         f"{tuple(w.shape)} {w.dtype}")
    if not w.is_contiguous() or w.data_ptr() & 15:
        w = w.contiguous().clone()
    return w


def _rotary(who: str, rotary: Optional[RotaryTable], D: int):
    if rotary is None:
        return None, 0, 0, 0
    if rotary.rot_dim > D:
        raise ValueError(f"{who}: rot_dim {rotary.rot_dim} exceeds the head dimension {D}")
    return (rotary.table.data_ptr(), rotary.max_positions, rotary.rot_dim,
            int(rotary.interleaved))


def _tables(who: str, layout: ChunkLayout, dev: torch.device, block_tables, context_lens):
    """Block tables, their row stride and context lengths as the kernels read
    them."""
    strides = block_tables.stride()
    if block_tables.dtype is not _I32 or len(strides) != 2 or strides[1] != 1:
        block_tables = _block_tables(block_tables)
        strides = block_tables.stride()
    if context_lens.dtype is not _I32 or not context_lens.is_contiguous():
        context_lens = _i32(context_lens)
    B = layout.batch
    if layout.device != dev:
        raise ValueError(f"{who}: the layout is on {layout.device}, the tensors on {dev}")
    rows, W = block_tables.shape
    if rows != B:
        raise ValueError(f"{who}: the layout has {B} sequences, the tables {rows}")
    if context_lens.shape != (B,):
        _check_seqs(who, B, None, context_lens)
    # The stride of a single row can be any number.
    return block_tables, strides[0] if B > 1 else W, context_lens


def _positions(t: torch.Tensor) -> torch.Tensor:
    """Positions as the kernel reads them: int32 or int64, never narrowed to
    another position."""
    if t.dtype is torch.uint64:
        t = t.view(torch.int64)  # those past its range: negative, outside the table
    elif t.dtype is torch.uint32:
        t = t.to(torch.int64)
    elif t.dtype is not torch.int64:
        t = t.to(torch.int32)
    return t.contiguous()


def qk_norm_rope(q: torch.Tensor, k: Optional[torch.Tensor],
                 positions: Optional[torch.Tensor], rotary: Optional[RotaryTable] = None,
                 q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """Norms of queries and keys for each head, with the position rotation.

    q [T, H_q, D] and k [T, H_kv, D] (or None), bf16, fp16 or fp32, any token
    and head strides (views of a fused projection are read in place).  Every
    head's row becomes x * rsqrt(mean(x^2) + eps) * weight where a weight [D]
    is given, then is rotated by ``rotary``'s entry of positions[t] ([T]
    integers; None without rotation); a position outside the table gives NaN.
    In 32 bits, rounded once to the inputs' dtype.  Returns contiguous
    (q_out, k_out).
    """
    who = "qk_norm_rope"
    dev = _same_device(q, k, positions, rotary.table if rotary else None, q_weight, k_weight)
    q, *q_at = _rows(who, "q", q, None, None, q.shape[-1])
    T, H_q, D = q.shape
    H_kv, k_at = 0, (None, 0, 0)
    if k is not None:
        k, *k_at = _rows(who, "k", k, T, None, D, q.dtype)
        if k.shape[0] != T:
            raise ValueError(f"{who}: k has {k.shape[0]} tokens, q {T}")
        H_kv = k.shape[1]
    elif k_weight is not None:
        raise ValueError(f"{who}: k_weight without k")
    if rotary is None and q_weight is None and k_weight is None:
        raise ValueError(f"{who}: neither a rotation nor a norm is asked for")
    qw, kw, wcode = _weights(who, D, q_weight, k_weight)
    rot = _rotary(who, rotary, D)
    if rotary is not None:
        if positions is None or positions.dim() != 1 or positions.dtype not in _INTEGERS:
            raise ValueError(f"{who}: positions must be [{T}] integers")
        _check_count(who, "positions", positions, T)
        if positions.dtype is not torch.int32 or not positions.is_contiguous():
            positions = _positions(positions)
    q_out = q.new_empty((T, H_q, D))
    k_out = None if k is None else q.new_empty((T, H_kv, D))
    if T:
        _call(dev, who, _lib.load().cvsa_qk_norm_rope, *q_at, *k_at, _DTYPE_CODE[q.dtype],
              *((positions.data_ptr(), positions.element_size()) if rotary else (None, 4)), *rot,
              _ptr(qw), _ptr(kw), wcode, float(eps), T, H_q, H_kv, D, q_out.data_ptr(),
              _ptr(k_out))
    return q_out, k_out


def _check_cache8(who, name, cache, scales):
    """A cache of 8 bits and its scales."""
    if cache.dim() != 4 or cache.dtype is not _F8 or not cache.is_contiguous() \
            or cache.data_ptr() & 15:
        raise ValueError(f"{who}: {name}_cache must be contiguous, 16-byte aligned float8_e4m3fn "
                         "[num_blocks, block_size, H_kv, D] with scales, got "
                         f"{tuple(cache.shape)} {cache.dtype}")
    want = (cache.shape[0], cache.shape[2])
    if scales is None:
        raise ValueError(f"{who}: {name}_cache is of 8 bits, {name}_scales are missing")
    if scales.shape != want or scales.dtype is not _SCALE or not scales.is_contiguous():
        raise ValueError(f"{who}: {name}_scales must be contiguous float8_e8m0fnu {want}, got "
                         f"{tuple(scales.shape)} {scales.dtype}")


def _check_caches(who, k_cache, v_cache, block_size, k_scales=None, v_scales=None):
    """The caches' (num_blocks, H_kv, D)."""
    shape = k_cache.shape
    if k_scales is not None and v_scales is not None and len(shape) == 4 \
            and k_cache.dtype is v_cache.dtype is _F8 \
            and k_scales.dtype is v_scales.dtype is _SCALE \
            and k_scales.shape == v_scales.shape == (shape[0], shape[2]) \
            and k_cache.is_contiguous() and v_cache.is_contiguous() \
            and k_scales.is_contiguous() and v_scales.is_contiguous() \
            and not (k_cache.data_ptr() | v_cache.data_ptr()) & 15:
        pass  # as _check_cache8 wants them: one look at each
    elif k_scales is not None or v_scales is not None or k_cache.dtype is _F8:
        _check_cache8(who, "k", k_cache, k_scales)
        _check_cache8(who, "v", v_cache, v_scales)
    elif len(shape) != 4 or k_cache.dtype is not _BF16 or v_cache.dtype is not _BF16 \
            or not k_cache.is_contiguous() or not v_cache.is_contiguous():
        _check_cache(k_cache)
        _check_cache(v_cache, "v_cache")
    if v_cache.shape != shape:
        raise ValueError("k_cache and v_cache shapes differ")
    if shape[1] != block_size:
        raise ValueError(f"{who}: cache block_size mismatch")
    return shape[0], shape[2], shape[3]


def prepare_append_chunk(k, v, k_cache, v_cache, block_tables, context_lens, layout, block_size,
                         rotary=None, k_weight=None, eps=1e-6, q=None, q_weight=None,
                         k_scales=None, v_scales=None):
    """The checks of :func:`append_chunk_kv` without its launch: returns
    (launch, q_out); launch() enqueues it, on the same stream.  The tables may
    change in place in between; k, v, q and the weights may not."""
    who = "append_chunk_kv"
    dev = _same_device(k, v, k_cache, v_cache, block_tables, context_lens, q, q_weight, k_weight,
                       rotary.table if rotary else None, k_scales, v_scales)
    num_blocks, H_kv, D = _check_caches(who, k_cache, v_cache, block_size, k_scales, v_scales)
    if k_scales is not None and (k_cache.data_ptr() == v_cache.data_ptr()
                                 or k_scales.data_ptr() == v_scales.data_ptr()):
        raise ValueError(f"{who}: keys and values must have caches and scales of their own")
    bt, bt_stride, ctx = _tables(who, layout, dev, block_tables, context_lens)
    B, W = bt.shape
    T, eps = layout.total, float(eps)
    k, *k_at = _rows(who, "k", k, T, H_kv, D)
    v, *v_at = _rows(who, "v", v, T, H_kv, D, k.dtype)
    if q is None and q_weight is not None:
        raise ValueError(f"{who}: q_weight without q")
    qw, kw, wcode = _weights(who, D, q_weight, k_weight)
    rot = _rotary(who, rotary, D)
    q_out, H_q, q_at = None, 0, (None, 0, 0)
    if q is not None:
        q, *q_at = _rows(who, "q", q, T, None, D, k.dtype)
        rows, H_q, _ = q.shape
        q_out = q.new_empty((rows, H_q, D))
        if rows > T:
            q_out[T:].zero_()
    if D not in (32, 64, 128, 256):
        raise NotImplementedError(f"{who}: D={D} not in {{32, 64, 128, 256}}")
    if max(H_q, H_kv) > 65536:
        raise ValueError(f"{who}: {H_q} and {H_kv} heads (at most 65536)")
    copied = bt is not block_tables or ctx is not context_lens

    def launch(at_once: bool = False):
        if T == 0:
            return
        b, stride, c = bt, bt_stride, ctx
        if copied and not at_once:
            b, stride, c = _tables(who, layout, dev, block_tables, context_lens)
        L = _lib.load()
        fn, scales = (L.cvsa_append_chunk_kv, ()) if k_scales is None else (
            L.cvsa_append_chunk_kv8, (k_scales.data_ptr(), v_scales.data_ptr()))
        # k, v and q are held here: they may be copies.
        _call(dev, who, fn, *k_at, *v_at, *q_at,
              _DTYPE_CODE[k.dtype], k_cache.data_ptr(), v_cache.data_ptr(), *scales, num_blocks,
              b.data_ptr(), stride, W, c.data_ptr(), layout.cu_seqlens.data_ptr(), B, T,
              *rot, _ptr(qw), _ptr(kw), wcode, eps, H_q, H_kv, D, block_size,
              _ptr(q_out), keep=(k, v, q, rotary))
    return launch, q_out


def append_chunk_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                    v_cache: torch.Tensor, block_tables: torch.Tensor,
                    context_lens: torch.Tensor, layout: ChunkLayout, block_size: int,
                    rotary: Optional[RotaryTable] = None,
                    k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                    q: Optional[torch.Tensor] = None,
                    q_weight: Optional[torch.Tensor] = None,
                    k_scales: Optional[torch.Tensor] = None,
                    v_scales: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Write a chunk's keys and values [T, H_kv, D] to the paged cache.

    ``context_lens`` counts the chunk's tokens already and the block tables
    hold their pages (SequenceKVManager.reserve_chunk, or a scheduler of the
    caller's): token i of sequence b goes to position context_lens[b] -
    layout.lens[b] + i.  Nothing but the cache rows is changed, so one layout
    and one set of tables serve all layers.  Keys are normed (``k_weight``)
    and rotated (``rotary``) on the way as in :func:`qk_norm_rope`, and with
    ``q`` ([T, H_q, D]) the queries' norm and rotation by the same positions
    are returned.  bf16, fp16 or fp32 rows, any token and head strides; the
    cache is bf16.  A token whose position is negative, past the block table
    or in a block outside the pool is not written.  Rows past layout.total
    are not read; the returned q is zero there.

    With ``k_scales`` and ``v_scales`` ([num_blocks, H_kv] float8_e8m0fnu,
    powers of two) the caches are float8_e4m3fn, and a value is payload times
    its block's and head's scale.  A page whose first token is written gets
    the smallest scale 2^e, -110 <= e <= 119, with which its new finite values
    do not pass 448 (larger ones become 448 * 2^119); one that held tokens
    before keeps its scale, or takes a larger one if the new tokens need it,
    to which its tokens are brought (a shift, exact but for values that become
    subnormal).  Payloads are rounded to nearest even; infinite and NaN values
    become NaN.  No two sequences may append to one block, and keys and values
    have caches and scales of their own.
    """
    launch, q_out = prepare_append_chunk(k, v, k_cache, v_cache, block_tables, context_lens,
                                         layout, block_size, rotary, k_weight, eps, q, q_weight,
                                         k_scales, v_scales)
    launch(at_once=True)
    return q_out


def reserve_chunk(block_tables: torch.Tensor, context_lens: torch.Tensor,
                  pages_allocated: torch.Tensor, layout: ChunkLayout, next_free_block: int,
                  num_blocks: int, block_size: int) -> None:
    """Pages for a chunk, by the rule of append_token_kv
    (cvsa/runtime/kv_cache.py:133-150) for each of its tokens: context_lens
    grows by the chunk's lengths and new pages take the blocks from
    next_free_block on.  The three tensors are contiguous int32 and updated in
    place; the caller has checked that tables and pool hold the chunk
    (SequenceKVManager.reserve_chunk does).  next_free_block is the call's own
    number: replays of a captured call give the same blocks out again, so
    capture it only where no sequence needs a new page (pages_allocated)."""
    who = "reserve_chunk"
    dev = _device_of(block_tables, context_lens, pages_allocated)
    for name, t in (("block_tables", block_tables), ("context_lens", context_lens),
                    ("pages_allocated", pages_allocated)):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"{who}: {name} must be contiguous int32")
    block_tables, bt_stride, context_lens = _tables(who, layout, dev, block_tables, context_lens)
    B = layout.batch
    _check_count(who, "pages_allocated", pages_allocated, B)
    _call(dev, who, _lib.load().cvsa_reserve_chunk, block_tables.data_ptr(),
          bt_stride, block_tables.shape[1], context_lens.data_ptr(),
          pages_allocated.data_ptr(), layout.cu_seqlens.data_ptr(), B, next_free_block,
          num_blocks, block_size)


def chunk_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_tables: torch.Tensor, context_lens: torch.Tensor,
                    layout: ChunkLayout, num_kv_heads: int, num_q_per_kv: int, block_size: int,
                    causal: bool = True, scale: Optional[float] = None,
                    max_context_len: int = 0, return_lse: bool = False,
                    out: Optional[torch.Tensor] = None,
                    k_scales: Optional[torch.Tensor] = None,
                    v_scales: Optional[torch.Tensor] = None):
    """Attention of a chunk's queries over the paged cache -> [T, H_q, D] bf16.

    q [T, H_q, D] bf16, any token and head strides.  ``context_lens`` counts
    the chunk's tokens: query i of sequence b has position context_lens[b] -
    layout.lens[b] + i and sees the keys up to it, or with ``causal=False``
    the whole context (an encoder's states, a bidirectional chunk).  Keys of
    blocks outside the pool or past the block table take no part; a query
    that sees no key gives zeros and a log-sum-exp of -inf.  ``scale``
    defaults to D^-0.5.  ``max_context_len`` (most keys of a sequence, where
    the caller knows) only shapes the launch: without it chunks of more than a
    few tokens are cut for contexts that fill the block table, and take up to
    several times as long where the table is much wider.  With ``return_lse`` the natural
    log-sum-exps [T, H_q] fp32 of the scaled scores are returned too.  Rows
    past layout.total are zero in a new output and left as they are in ``out``
    (contiguous bf16 of q's shape; a contiguous q itself will do).

    Scores, sums and outputs are held in 32 bits; the weights of the second
    product are rounded to bf16 (:func:`dense_decode`, for batches of single
    tokens, keeps 16 bits of them).

    With ``k_scales`` and ``v_scales`` the caches are of 8 bits (see
    :func:`append_chunk_kv`); their values are brought to bf16, exactly, and
    the rest is the same, but that sequences of up to 64 rows (tokens times
    num_q_per_kv; 32 at D = 256) keep 16 bits of the weights: single tokens
    and drafts, which no decode kernel takes over such caches.  A scale of NaN
    makes its block's values NaN; under one past 2^119, which the append does not
    write, values that bf16 does not hold make their outputs infinite or NaN.
    """
    who = "chunk_attention"
    dev = _same_device(q, k_cache, v_cache, block_tables, context_lens, out, k_scales, v_scales)
    num_blocks, H_kv, D = _check_caches(who, k_cache, v_cache, block_size, k_scales, v_scales)
    if H_kv != num_kv_heads:
        raise ValueError(f"{who}: head counts do not match the caches")
    bt, bt_stride, ctx = _tables(who, layout, dev, block_tables, context_lens)
    B, W = bt.shape
    if bt_stride < W:  # a row that sequences share
        bt, bt_stride = bt.contiguous(), W
    T, H_q = layout.total, num_kv_heads * num_q_per_kv
    q, *q_at = _rows(who, "q", q, T, H_q, D, _BF16)
    max_context_len = int(max_context_len)
    if max_context_len < 0:
        raise ValueError(f"{who}: max_context_len must not be negative")
    scale = D ** -0.5 if scale is None else float(scale)
    rows = q.shape[0]
    if out is None:
        out = q.new_empty((rows, H_q, D))
        if rows > T:
            out[T:].zero_()
    elif out.shape != q.shape or out.dtype != torch.bfloat16 or not out.is_contiguous() \
            or out.data_ptr() % 16:
        raise ValueError(f"{who}: out must be contiguous bfloat16 {tuple(q.shape)}")
    lse = None
    if return_lse:
        lse = torch.empty(rows, H_q, device=dev, dtype=torch.float32)
        if rows > T:
            lse[T:].zero_()
    if T:
        L = _lib.load()
        # Allocated for the call, so no two calls, streams or captured graphs
        # share it.
        sizes = (H_q, H_kv, D, block_size, W, max_context_len)
        key = sizes if k_scales is None else (*sizes, 8)
        need = layout._workspace_bytes.get(key)
        if need is None:
            size_of = L.cvsa_chunk_attention_workspace_bytes if k_scales is None \
                else L.cvsa_chunk_attention8_workspace_bytes
            need = layout._workspace_bytes[key] = size_of(layout.cu_host, B, *sizes)
        ws = torch.empty(need, device=dev, dtype=torch.uint8) if need else None
        fn, scales = (L.cvsa_chunk_attention, ()) if k_scales is None else (
            L.cvsa_chunk_attention8, (k_scales.data_ptr(), v_scales.data_ptr()))
        _call(dev, who, fn, *q_at, k_cache.data_ptr(), v_cache.data_ptr(), *scales,
              num_blocks, bt.data_ptr(), bt_stride, ctx.data_ptr(), layout.cu_seqlens.data_ptr(),
              layout.cu_host, B, H_q, num_kv_heads, D, block_size, W, max_context_len, scale,
              int(bool(causal)), out.data_ptr(), _ptr(lse), _ptr(ws), need)
    return (out, lse) if return_lse else out
