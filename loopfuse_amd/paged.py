"""Key / value caches in pages for requests of different lengths: their tables, the storing of new tokens, attention over them.

A serving step over a batch of requests, nothing of which waits for the lengths, which live on the GPU:

    step = extend_tables(lengths, new, table, free, page_size, total)    # pages for the new tokens, and each one's slot
    store_kv(k, v, k_pool, v_pool, step.slots)                           # their keys and values into the pools
    o = attention_shared(q, k_pool, v_pool, plan, table, step.lengths,   # one new token per request over its keys,
                         prefix_table=prefix, prefix_len=n)              # and over a prefix that all requests share

Pools are ``[pages, page, Hkv, D]`` (or ``[pages, Hkv, D]`` for one-token pages), as ``lowering.attention`` takes them; a table
row names a request's pages in the order of its tokens.  ``append_kv`` norms and rotates the new queries and keys on the way to the pools.

Pools in 4 bits (``pool4``) hold nearly four times as many tokens and are read in a quarter of the time:

    q = append_kv(q, k, v, k_pool, v_pool, step.slots, step.positions, table_of_angles)
    o = attention_cached(q, k_pool, v_pool, plan, table, step.lengths, step.offsets, step.positions)      # one token per request or several

The reference reads caches of one length through
``paged_load`` (reference loopfuse/torch_backend/__init__.py:46-56) and leaves tables and stores to its user.
"""
from __future__ import annotations

import ctypes
import dataclasses
import math
import operator
from typing import NamedTuple, Optional, Union

import torch

from . import lowering
from .lowering import AttnPlan, UnsupportedPlan

_TABLE_DTYPES = (torch.int32, torch.int64)
MAX_REQUESTS = 1 << 22      # of extend_tables, in which each forms its sums over all of them: a second or two for so many


class _TablesParams(ctypes.Structure):
    """Mirror of ``struct LfTablesParams`` in csrc/kernels/lf_paged_tables.hip."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("cached", "fresh", "table", "free", "offsets", "lengths", "slots", "positions", "pages")]
                + [("table_stride", ctypes.c_longlong)] + [(n, ctypes.c_int) for n in ("B", "width", "count", "T", "shift")])


class _StoreParams(ctypes.Structure):
    """Mirror of ``struct LfStoreParams`` in csrc/kernels/lf_store_kv.hip."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("k", "v", "k_pool", "v_pool", "slots")]
                + [(n, ctypes.c_longlong) for n in ("k_ss", "k_sh", "v_ss", "v_sh", "kp_sb", "kp_ss", "kp_sh", "vp_sb", "vp_ss", "vp_sh", "last")]
                + [(n, ctypes.c_int) for n in ("T", "heads", "per_head", "shift")])


class SharedParams(lowering.AttnParams):
    """Mirror of ``struct LfSharedParams`` in csrc/kernels/lf_shared.hip.h."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("lengths", "prefix_k", "prefix_v", "pre_acc", "pre_ml")]
                + [(n, ctypes.c_int) for n in ("room", "units", "pre_units", "pre_blocks", "target_log2", "least")])


class _ReadParams(ctypes.Structure):
    """Mirror of ``struct LfReadParams`` in csrc/kernels/lf_read_kv.hip."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("k_pool", "v_pool", "k_scales", "v_scales", "k", "v", "slots")]
                + [(n, ctypes.c_longlong) for n in ("kp_sb", "kp_ss", "kp_sh", "vp_sb", "vp_ss", "vp_sh", "last")]
                + [(n, ctypes.c_int) for n in ("T", "heads", "per_head", "shift")])


class CachedParams(ctypes.Structure):
    """Mirror of ``struct LfCachedParams`` in csrc/kernels/lf_cached.hip."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "o", "k", "v", "k_scales", "v_scales", "table", "lengths", "offsets", "positions", "part_acc", "part_ml")]
                + [(n, ctypes.c_longlong) for n in ("q_ss", "q_sh", "o_ss", "o_sh", "page_bytes", "table_stride")]
                + [(n, ctypes.c_int) for n in ("T", "B", "Hkv", "group")] + [("per_group", ctypes.c_uint)]
                + [(n, ctypes.c_int) for n in ("room", "shift", "window", "fixed", "least", "workgroups", "slots", "clear")] + [("scale", ctypes.c_float), ("softcap", ctypes.c_float)])


@dataclasses.dataclass(frozen=True, eq=False)
class Pool4:
    """A page pool of keys or values held in 4 bits (``pool4``)."""

    codes: torch.Tensor        # uint8 [pages, heads, page / 16, 8 * D]
    scales: torch.Tensor       # uint8 [pages, heads, page / 16, D / 2]
    dtype: torch.dtype         # of the rows that it stands for

    @property
    def shape(self) -> tuple:
        """(pages, page size, heads, D)"""
        n, heads, tiles, row = self.codes.shape
        return n, 16 * tiles, heads, row // 8

    @property
    def device(self) -> torch.device:
        return self.codes.device


class PagedStep(NamedTuple):
    """What ``extend_tables`` leaves."""

    offsets: torch.Tensor      # int32 [B + 1]: request b's new tokens are rows offsets[b] ... offsets[b + 1]
    lengths: torch.Tensor      # int32 [B]: tokens of each request with the new ones that have a slot
    slots: torch.Tensor        # int32 [total]: page * page_size + place in the page, -1 for rows of no token
    positions: torch.Tensor    # int32 [total]: place in the request, -1 for rows of no token
    pages: torch.Tensor        # int32 [1]: free pages that the new tokens need


def _on_gpu(name: str, t: torch.Tensor, dtypes, dim: int, device=None) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.dim() != dim:
        raise UnsupportedPlan(f"{name} must be a tensor of {dim} dim(s), {' or '.join(str(d).replace('torch.', '') for d in dtypes)}")
    if not t.is_cuda:
        raise RuntimeError(f"loopfuse_amd: {name} is not on the GPU; the HIP path has no CPU fallback")
    if device is not None and t.device != device:
        raise RuntimeError(f"loopfuse_amd: {name} is on {t.device}, not on {device}")


def _whole(name: str, n) -> int:
    """A size that the host knows (a tensor would have to be waited for)."""
    if isinstance(n, torch.Tensor):
        raise UnsupportedPlan(f"{name} must be a number of the host's")
    return operator.index(n)


def _shift(page_size: int) -> int:
    if not isinstance(page_size, int) or page_size < 1 or page_size & (page_size - 1) or page_size > 1 << 30:
        raise UnsupportedPlan("page size must be a power of two, 2**30 at most")
    return page_size.bit_length() - 1


@lowering.outside_graphs
def extend_tables(cached: torch.Tensor, new: torch.Tensor, table: torch.Tensor, free: torch.Tensor, page_size: int, total: int) -> PagedStep:
    """Pages for the new tokens of a batch, and the slot of each of them, from lengths on the GPU.

    cached, new : int32 [B], tokens that a request has in its pages and tokens that come (0 for both: an empty place of the batch);
    below 0 counts as 0.  table : [B, width], int32 or int64, rows contiguous; request ``b``'s first ``ceil(cached / page_size)`` entries are
    read, those of its new pages are WRITTEN, the others stay as they are.  free : pages to take, [count], of the table's dtype; the
    requests take ``pages`` of them from the front, in the order of the batch.  total : rows of the step's packed tensors (a padded
    size will do).

    Nothing is raised for what only the GPU knows: where no free page is left, the row of the table is too short or a token lies behind
    ``total``, the token's slot (and the new entry) is -1, which ``store_kv`` leaves out, and ``lengths`` ends in front of it;
    ``pages`` above ``len(free)`` says so.  Slots are numbers in 32 bits: a page behind those counts as none, and so does one below 0
    (``LOOPFUSE_CHECK_TABLES=1`` raises for all of these)."""
    done = _host.extend_tables(cached, new, table, free, page_size, total)
    if done is not None:
        return done
    _on_gpu("cached", cached, (torch.int32,), 1)
    dev, B = cached.device, cached.shape[0]
    _on_gpu("new", new, (torch.int32,), 1, dev)
    _on_gpu("table", table, _TABLE_DTYPES, 2, dev)
    _on_gpu("free", free, (table.dtype,), 1, dev)
    if new.shape[0] != B or table.shape[0] != B:
        raise UnsupportedPlan(f"new and table must be of {B} requests")
    if B > MAX_REQUESTS:
        raise UnsupportedPlan(f"more than {MAX_REQUESTS} requests")
    if table.shape[1] and B and table.stride(1) != 1 or (B > 1 and table.stride(0) < table.shape[1]):
        raise UnsupportedPlan("rows of the table must be contiguous and apart")
    shift, total = _shift(page_size), _whole("total", total)
    if total < 0 or total >= 1 << 31:
        raise UnsupportedPlan("the number of rows must be between 0 and 2**31 - 1")
    with torch.cuda.device(dev):
        if lowering._checks_tables():
            _check_extension(cached, new, table, free, page_size, total)
        packed = [t if t.is_contiguous() else t.contiguous() for t in (cached, new, free)]
        P = _TablesParams(table_stride=table.stride(0), B=B, width=table.shape[1], count=free.shape[0], T=total, shift=shift)
        spec = lowering._spec("paged_tables", 0, 64, table_i64=table.dtype == torch.int64)
        # a block per request and 1024 rows of the mean one
        share = max(1, min(64, total // (1024 * max(B, 1))))
        repeat = lowering._Repeat(P, [(lowering.get_kernel(spec, spec.entry()), (max(B, 1), share, 1), 256)], {"kernels": [spec.entry()]},
                                  (2 * B + 2 + 2 * total, (B + 1, B, 1, total, total)))
        step = _tables(packed[0], packed[1], table, packed[2], total, repeat)
        if packed[0] is cached and packed[1] is new and packed[2] is free:
            lowering._keep_call(lowering._call_key("t", (), (cached, new, table, free), None, (page_size, total)), repeat, (repeat.more[0], *repeat.more[1]))
    return step


def _check_extension(cached, new, table, free, page_size, total) -> None:
    c, n = cached.clamp(min=0).long(), new.clamp(min=0).long()
    pages = (c + n + page_size - 1) // page_size
    need, width, rows = int((pages - (c + page_size - 1) // page_size).sum()), int(pages.max()) if len(c) else 0, int(n.sum())
    if need > free.shape[0] or width > table.shape[1] or rows > total:
        raise ValueError(f"loopfuse_amd: {need} pages of {free.shape[0]} free ones, tables of {width} of {table.shape[1]} entries, {rows} of {total} rows")
    if need and (int(free[:need].min()) < 0 or int(free[:need].max()) > ((1 << 31) - 1) // page_size):
        raise ValueError(f"loopfuse_amd: free pages must be between 0 and {((1 << 31) - 1) // page_size}")


def _tables(cached, new, table, free, total, repeat) -> PagedStep:
    size, parts = repeat.more
    made = cached.new_empty(size)
    offsets, lengths, pages, slots, positions = made.split_with_sizes(parts)
    P = _TablesParams.from_buffer_copy(repeat.block)
    P.cached, P.fresh, P.table, P.free = cached.data_ptr(), new.data_ptr(), table.data_ptr(), free.data_ptr()
    P.offsets = at = made.data_ptr()
    P.lengths = at = at + 4 * parts[0]
    P.pages = at = at + 4 * parts[1]
    P.slots = at = at + 4
    P.positions = at + 4 * total
    repeat.launches.launch(P)
    lowering._last_launch.set(repeat.record)
    return PagedStep(offsets, lengths, slots, positions, pages)


def _pool(name: str, t: torch.Tensor) -> tuple:
    """(pages, page size, heads, D, page stride, token stride, head stride) of a page pool."""
    if t.dim() == 3:
        return t.shape[0], 1, t.shape[1], t.shape[2], t.stride(0), 0, t.stride(1)
    if t.dim() == 4:
        return (*t.shape, *t.stride()[:3])
    raise UnsupportedPlan(f"{name} pool must be [N, Hkv, D] or [N, P, Hkv, D]")


def pool4(pages: int, page_size: int, heads: int, D: int, dtype: torch.dtype, device=None) -> Pool4:
    """A pool of ``pages`` pages of keys, or of values, in 4 bits, holding zeros.  page_size: a power of two, 16 at least; D 64 or 128; ``dtype``:
    bf16 or fp16, of the rows that it stands for.

    A value is 0 0.5 1 1.5 2 3 4 or 6 with a sign, times a power of two that 32 neighbours of a row share, the least one of which their largest size is below the
    7-fold: 4.25 bits an element, off by a fifth of the largest size of its 32 at most.  Sizes beyond ``6 * 2 ** 125`` (fp16: ``6 * 2 ** 13``) count as that; 32
    neighbours with a NaN or an infinity among them are NaN.  Keys and values lie in different orders: a pool of the one is not read as the other."""
    shift = _shift(page_size)
    if shift < 4 or D not in (64, 128) or heads < 1 or pages < 0 or dtype not in lowering._DTYPE_CODE:
        raise UnsupportedPlan("a pool in 4 bits has pages of 16 tokens or more, head dim 64 or 128, and stands for bf16 or fp16 rows")
    lead = (pages, heads, page_size // 16)
    return Pool4(torch.zeros((*lead, 8 * D), dtype=torch.uint8, device=device), torch.zeros((*lead, D // 2), dtype=torch.uint8, device=device), dtype)


def _pool4(name: str, pool: Pool4, dtype, device) -> tuple:
    """(pages, page size, heads, D) of a pool in 4 bits that the kernels serve."""
    if not isinstance(pool, Pool4):
        raise UnsupportedPlan("pools of K and V must both be in 4 bits, or both not")
    codes, scales = pool.codes, pool.scales
    for t in (codes, scales):
        _on_gpu(f"{name} pool", t, (torch.uint8,), 4, device)
    n, heads, tiles, row = codes.shape
    if pool.dtype != dtype:
        raise UnsupportedPlan(f"{name} pool stands for {pool.dtype} rows, not for {dtype}")
    if row not in (512, 1024) or tuple(scales.shape) != (n, heads, tiles, row // 16) or heads < 1 or tiles < 1 or tiles & (tiles - 1):
        raise UnsupportedPlan(f"{name} pool: not the shapes that pool4 makes")
    for t in (codes, scales):
        if n and not t[0].is_contiguous() or t.data_ptr() % 16 or (n > 1 and (t.stride(0) % 16 or t.stride(0) < t[0].numel())):
            raise UnsupportedPlan(f"{name} pool: pages must be contiguous and apart, on 16-byte borders")
    return pool.shape


def _two_pools4(k_pool, v_pool, dtype, device) -> tuple:
    shape = _pool4("K", k_pool, dtype, device)
    if _pool4("V", v_pool, dtype, device) != shape:
        raise UnsupportedPlan("the pools must agree in pages, page size, heads and head dim")
    return shape


def _parts(k_pool, v_pool, dtype):
    """Pools as the host module takes them: K, V, scales of K, of V; None: not for it."""
    if isinstance(k_pool, Pool4):
        if not isinstance(v_pool, Pool4) or k_pool.dtype is not dtype or v_pool.dtype is not dtype:
            return None
        return k_pool.codes, v_pool.codes, k_pool.scales, v_pool.scales
    return k_pool, v_pool, None, None


def _two_pools(k_pool, v_pool, dtype, device, heads: int, D: int, written=True) -> tuple:
    """(pages, page size, strides of K's pages, tokens and heads, V's) of pools of 16-bit rows."""
    for name, t in (("K pool", k_pool), ("V pool", v_pool)):
        if not isinstance(t, torch.Tensor):
            raise UnsupportedPlan("pools of K and V must both be in 4 bits, or both not")
        lowering._check_tensor(name, t, dtype)
        if t.device != device:
            raise RuntimeError(f"loopfuse_amd: {name} is on {t.device}, not on {device}")
    pages, page, hk, dk, *ks = _pool("K", k_pool)
    pages_v, page_v, hv, dv, *vs = _pool("V", v_pool)
    if (pages, page) != (pages_v, page_v) or (hk, dk) != (heads, D) or (hv, dv) != (heads, D):
        raise UnsupportedPlan("the pools must agree in pages and page size with each other, in heads and head dim with K and V")
    if written and any(n > 1 and s == 0 for p in (k_pool, v_pool) for n, s in zip(p.shape, p.stride())):
        raise UnsupportedPlan("every element of a pool must have a place of its own")
    return pages, page, ks, vs


def _checked_slots(slots, last, positions=None, places=0) -> None:
    if lowering._checks_tables():
        kept = slots[slots >= 0 if positions is None else (slots >= 0) & (positions >= 0) & (positions < places)]
        if len(kept) and (int(kept.max()) >= last or len(torch.unique(kept)) < len(kept)):
            raise ValueError(f"loopfuse_amd: slots must be distinct and below {last}")


@lowering.outside_graphs
def append_kv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pool: Union[torch.Tensor, Pool4], v_pool: Union[torch.Tensor, Pool4], slots: torch.Tensor,
              positions: torch.Tensor, table: Optional[torch.Tensor], *, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
              eps: Optional[float] = None, pairs: bool = False) -> torch.Tensor:
    """The new tokens' keys, normed and rotated, and their values into the page pools, and their queries, normed and rotated, as a new tensor: what
    ``rotary.rotate_heads`` and ``store_kv`` do, in one pass.  No gradients are recorded.

    q ``[rows, Hq, D]``, k and v ``[rows, Hkv, D]``, ``positions``, ``table``, weights, ``eps`` and ``pairs`` as ``rotate_heads`` takes them; slots int32 ``[rows]`` and
    the pools as ``store_kv``: ``PagedStep.slots`` and ``.positions`` of ``extend_tables``.  A row whose position is below 0 or behind the table's last is one of no token:
    zeros among the queries, left out of the pools whatever its slot.  Without a table and a norm rows stay as they are."""
    if positions is None:
        raise UnsupportedPlan("positions must be given")
    parts = _parts(k_pool, v_pool, getattr(q, "dtype", None))
    done = None if parts is None else _host.append_kv(q, k, v, *parts, table, q_weight, k_weight, slots, positions, eps, bool(pairs))
    if done is not None:
        return done
    return _append(q, k, v, k_pool, v_pool, slots, positions, table, q_weight, k_weight, eps, bool(pairs))


@lowering._on_device_of_first_argument
def _append(q, k, v, k_pool, v_pool, slots, positions, table, q_weight, k_weight, eps, pairs):
    """``positions`` None: only keys and values, into pools in 4 bits; ``q`` then stands for nothing."""
    lowering._no_tangents(q, k, v, table, q_weight, k_weight)
    keys_only = positions is None
    T, Hq, Hkv, D, R, wide = rotary.check_operands(q, k, positions, table, q_weight, k_weight, eps, (("V", v),), plain=True)
    _on_gpu("slots", slots, (torch.int32,), 1, q.device)
    if slots.shape[0] != T:
        raise UnsupportedPlan(f"slots must be int32 [{T}]")
    P = rotary.params(q, k, table, T, Hq, Hkv, D, R, wide, eps, pairs)
    P.v_ss, P.v_sh = v.stride()[:2]
    if isinstance(k_pool, Pool4) or isinstance(v_pool, Pool4):
        pages, page, heads, d = _two_pools4(k_pool, v_pool, q.dtype, q.device)
        if (heads, d) != (Hkv, D):
            raise UnsupportedPlan("the pools must have the heads and head dim of K and V")
        P.kp_sb, P.kp_ss, P.vp_sb, P.vp_ss = k_pool.codes.stride(0), k_pool.scales.stride(0), v_pool.codes.stride(0), v_pool.scales.stride(0)
        store = 2
    else:
        lowering._no_tangents(k_pool, v_pool)
        pages, page, (P.kp_sb, P.kp_ss, P.kp_sh), (P.vp_sb, P.vp_ss, P.vp_sh) = _two_pools(k_pool, v_pool, q.dtype, q.device, Hkv, D)
        store = 1
    P.shift, P.last = _shift(page), pages * page
    if P.q_blocks + 2 * P.k_blocks >= 1 << 24:
        raise UnsupportedPlan(f"a launch for {T} rows of {Hq} and {Hkv} heads of {D} is too large")
    if T == 0:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _checked_slots(slots, P.last, positions, P.places)
    if not keys_only:
        rotary._checked_positions(positions, P.places)
    if keys_only:
        P.q_blocks = 0
    spec = rotary.kernel_spec(q.dtype, D, store)
    repeat = lowering._Repeat(P, [(lowering.get_kernel(spec, spec.entry()), (P.q_blocks + 2 * P.k_blocks, 1, 1), 256)], {"kernels": [spec.entry()]})
    given = slots, positions, q_weight, k_weight
    even = slots.contiguous(), None if keys_only else positions.contiguous(), rotary.even_weight(q_weight), rotary.even_weight(k_weight)
    res = _append_again(q, k, v, k_pool, v_pool, even[0], even[1], table, even[2], even[3], repeat)
    if all(a is b for a, b in zip(even, given)):
        lowering._keep_call(lowering._call_key("a", (q, k, v, *_parts(k_pool, v_pool, q.dtype), table, q_weight, k_weight), (slots, positions), None, (eps, pairs)), repeat, ())
    return res


def _append_again(q, k, v, k_pool, v_pool, slots, positions, table, q_weight, k_weight, repeat):
    P = rotary.RotateParams.from_buffer_copy(repeat.block)
    out = None if positions is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    P.q, P.k, P.v, P.slots = q.data_ptr(), k.data_ptr(), v.data_ptr(), slots.data_ptr()
    if positions is not None:
        P.q_out, P.positions = out.data_ptr(), positions.data_ptr()
    _set_pools(P, "k_out", "v_out", k_pool, v_pool)
    rotary.set_tables(P, table, q_weight, k_weight)
    repeat.launches.launch(P)
    lowering._last_launch.set(repeat.record)
    return out


def _set_pools(P, k_name, v_name, k_pool, v_pool) -> None:
    for name, scales, pool in ((k_name, "k_scales", k_pool), (v_name, "v_scales", v_pool)):
        if isinstance(pool, Pool4):
            setattr(P, name, pool.codes.data_ptr())
            setattr(P, scales, pool.scales.data_ptr())
        else:
            setattr(P, name, pool.data_ptr())


@lowering.outside_graphs
def read_kv(k_pool: Union[torch.Tensor, Pool4], v_pool: Union[torch.Tensor, Pool4], slots: torch.Tensor) -> tuple:
    """Rows of keys and values out of the page pools, what ``store_kv`` and ``append_kv`` have put there: ``(k, v)``, each ``[rows, Hkv, D]``, row t of slot ``slots[t]``
    (int32 ``[rows]`` on the GPU, any number of times), zeros where it is below 0 or behind the pool's last.  From pools in 4 bits the values that they stand for,
    rounded to the type (those of fp16 have less than a bit below its least normal number).  For keys that go on elsewhere: into another cache, or beside
    those of a prompt's next part.  No gradients are recorded."""
    dtype = k_pool.dtype if isinstance(k_pool, (Pool4, torch.Tensor)) else None
    parts = _parts(k_pool, v_pool, dtype)
    done = None if parts is None else _host.read_kv(*parts, slots, dtype is torch.float16)
    if done is not None:
        return done
    if dtype not in lowering._DTYPE_CODE:
        raise UnsupportedPlan("pools must be of bf16 or fp16 rows")
    return _read(slots, k_pool, v_pool, parts)


@lowering._on_device_of_first_argument
def _read(slots, k_pool, v_pool, parts):
    _on_gpu("slots", slots, (torch.int32,), 1)
    P, dtype = _ReadParams(), k_pool.dtype
    if isinstance(k_pool, Pool4):
        pages, page, heads, D = _two_pools4(k_pool, v_pool, dtype, slots.device)
        P.kp_sb, P.kp_ss, P.vp_sb, P.vp_ss = k_pool.codes.stride(0), k_pool.scales.stride(0), v_pool.codes.stride(0), v_pool.scales.stride(0)
        spec = lowering._spec("read_kv", lowering._DTYPE_CODE[dtype], D, extra=("-DLF_READ4=1",))
    else:
        lowering._no_tangents(k_pool, v_pool)
        _, _, heads, D, *_ = _pool("K", k_pool)
        if D % 8:
            raise UnsupportedPlan("head dim must be a multiple of 8")
        pages, page, (P.kp_sb, P.kp_ss, P.kp_sh), (P.vp_sb, P.vp_ss, P.vp_sh) = _two_pools(k_pool, v_pool, dtype, slots.device, heads, D, False)
        spec = lowering._spec("read_kv", lowering._DTYPE_CODE[dtype], 64)
    T = slots.shape[0]
    P.last, P.T, P.heads, P.per_head, P.shift = pages * page, T, heads, D // 8, _shift(page)
    pieces = T * heads * (D // 8)
    if pieces + 256 >= 1 << 32:
        raise UnsupportedPlan(f"a launch for {T} rows of {heads} heads of {D} is too large")
    if pieces == 0:
        return tuple(torch.empty((T, heads, D), dtype=dtype, device=slots.device) for _ in range(2))
    repeat = lowering._Repeat(P, [(lowering.get_kernel(spec, spec.entry()), (-(-pieces // 256), 1, 1), 256)], {"kernels": [spec.entry()]}, (T, heads, D))
    even = slots.contiguous()
    res = _read_again(k_pool, v_pool, even, repeat)
    if even is slots:
        lowering._keep_call(lowering._call_key("g", parts, (slots,), None, (dtype is torch.float16,)), repeat, (T, heads, D))
    return res


def _read_again(k_pool, v_pool, slots, repeat):
    P = _ReadParams.from_buffer_copy(repeat.block)
    k, v = (torch.empty(repeat.more, dtype=k_pool.dtype, device=slots.device) for _ in range(2))
    P.k, P.v, P.slots = k.data_ptr(), v.data_ptr(), slots.data_ptr()
    _set_pools(P, "k_pool", "v_pool", k_pool, v_pool)
    repeat.launches.launch(P)
    lowering._last_launch.set(repeat.record)
    return k, v


@lowering.outside_graphs
def store_kv(k: torch.Tensor, v: torch.Tensor, k_pool: Union[torch.Tensor, Pool4], v_pool: Union[torch.Tensor, Pool4], slots: torch.Tensor) -> None:
    """Write rows of new keys and values, k and v ``[rows, Hkv, D]``, into the page pools: row t into token ``slots[t] % page`` of page
    ``slots[t] // page``, in pools in 4 bits (``pool4``) rounded as those say.  bf16 / fp16, D a multiple of 8; views will do.  ``slots``: int32 [rows] (``PagedStep.slots``); rows whose slot is below 0 or
    behind the pool's last are left out.  Slots that are not left out are distinct, as those of ``extend_tables`` are:
    of two rows with one slot, either may be found there afterwards, or a part of each."""
    if _host.store_kv(k, v, k_pool, v_pool, slots):
        return
    if isinstance(k_pool, Pool4) or isinstance(v_pool, Pool4):
        parts = _parts(k_pool, v_pool, k.dtype)
        if parts is None or _host.append_kv(k, k, v, *parts, None, None, None, slots, None, None, False) is None:
            _append(k, k, v, k_pool, v_pool, slots, None, None, None, None, None, False)
        return
    lowering._no_tangents(k, v, k_pool, v_pool)
    if k.dtype not in lowering._DTYPE_CODE:
        raise UnsupportedPlan(f"dtype {k.dtype} not supported (bf16/fp16 only)")
    for name, t in (("K", k), ("V", v), ("K pool", k_pool), ("V pool", v_pool)):
        lowering._check_tensor(name, t, k.dtype)
        if t.device != k.device:
            raise RuntimeError(f"loopfuse_amd: {name} is on {t.device}, K on {k.device}")
    _on_gpu("slots", slots, (torch.int32,), 1, k.device)
    if k.dim() != 3 or k.shape != v.shape or slots.shape[0] != k.shape[0] or k.shape[2] % 8:
        raise UnsupportedPlan("K and V must be [rows, Hkv, D], D a multiple of 8, slots [rows]")
    T, heads, D = k.shape
    pages, page, hk, dk, *ks = _pool("K", k_pool)
    pages_v, page_v, hv, dv, *vs = _pool("V", v_pool)
    if (pages, page) != (pages_v, page_v) or (hk, dk) != (heads, D) or (hv, dv) != (heads, D):
        raise UnsupportedPlan("the pools must agree in pages and page size with each other, in heads and head dim with K and V")
    if any(n > 1 and s == 0 for p in (k_pool, v_pool) for n, s in zip(p.shape, p.stride())):
        raise UnsupportedPlan("every element of a pool must have a place of its own")
    shift = _shift(page)
    if T == 0 or pages == 0 or heads == 0 or D == 0:
        return
    # (the kernel numbers rows in 32 bits, up to the end of the last block)
    blocks = -(-T // max(256 // (heads * D // 8), 1))
    if T > (1 << 31) - 256 or blocks * 256 >= 1 << 32:
        raise UnsupportedPlan(f"a launch for {T} rows of {heads} heads of {D} is too large")
    with torch.cuda.device(k.device):
        if lowering._checks_tables():
            kept_slots = slots[slots >= 0]
            if len(kept_slots) and (int(kept_slots.max()) >= pages * page or len(torch.unique(kept_slots)) < len(kept_slots)):
                raise ValueError(f"loopfuse_amd: slots must be distinct and below {pages * page}")
        packed = slots.contiguous()
        P = _StoreParams(0, 0, 0, 0, 0, *(x // 8 for x in (*k.stride()[:2], *v.stride()[:2], *ks, *vs)), pages * page, T, heads, D // 8, shift)
        spec = lowering._spec("store_kv", 0, 64)
        repeat = lowering._Repeat(P, [(lowering.get_kernel(spec, spec.entry()), (blocks, 1, 1), 256)], {"kernels": [spec.entry()]})
        _store(k, v, k_pool, v_pool, packed, repeat)
        if packed is slots:
            lowering._keep_call(lowering._call_key("s", (k, v, k_pool, v_pool), (slots,), None, ()), repeat, ())


def _store(k, v, k_pool, v_pool, slots, repeat) -> None:
    P = _StoreParams.from_buffer_copy(repeat.block)
    P.k, P.v, P.k_pool, P.v_pool, P.slots = k.data_ptr(), v.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), slots.data_ptr()
    repeat.launches.launch(P)
    lowering._last_launch.set(repeat.record)


def own_loads(D: int, Hkv: int, tiles: bool, requests: int, keys: int) -> int:
    """Heads whose waves load whole token rows of the own keys together (``-DLF_COOP=1``), where the pools allow it: 4 at head dimension 128, 8 at 64 (0: four
    waves share a head).  ``keys`` = that a call can have in all, without a prefix on ``tiles`` (whose workgroups have 4 waves).  Each wave then walks
    its head's keys alone: four times the steps for a fourth of the workgroups, which pays where there are many (request, head) pairs or many keys.  GPU time,
    us, none / together: 128, 32/8 heads, without a prefix 3 requests up to 128 keys 8.8 / 11.3, 14 up to 510 11.3 / 12.7, 20 up to 60 7.9 / 7.8, 95 up to 512 27.6 / 22.3, 238
    of 6 21.3 / 11.8; behind 1000 ... 12 000 on tiles 3 up to 1008 15.7 / 15.6, 12 up to 1088 20.1 / 16.3, 38 up to 64 27.7 / 22.7, 157 up to 64 59.9 / 31.7; 64, 32/8
    heads, 4 up to 110 7.0 / 10.6, 134 of 16 12.7 / 9.2, 55 up to 1904 32.5 / 25.7."""
    if D == 128:
        return 4 if requests * Hkv >= (100 if tiles else 300) or keys * Hkv > (32_000 if tiles else 64_000) else 0
    return 8 if not tiles and (requests * Hkv >= 500 or keys > 24_000) else 0


def own_pieces(coop: int, workgroups: int, room: int, keys: int) -> tuple:
    """(log2 of the workgroups that the own keys are cut for, least length of a piece).  ``workgroups`` = with one piece per request, ``room`` = keys that a
    request can have, ``keys`` = all of them.  About one or two workgroups per CU, four from 150 000 keys on, and of 8 waves half as many of the small calls; pieces of 128 keys,
    or of 256 where the requests fill the GPU in one piece each and where ends of pieces are few.  300 drawn batches, 1 ... 256 requests of 5 ... 8000 keys, with own_loads:
    1.025 of the best choice's time in the mean, 1.3 at most; us, by log2: 72 up to 2432
    keys, 32/8 heads, 8 158, 9 136, 10 123, 134 of 16, D 64, 9.2, 10.7, 13.4; by least length, 128 / 256: 214 of 178, 2/2 heads, 28.3 / 17.5, 78 of 157, 64/8, 25.9 / 17.5, 55 up to
    1904, D 64, 31.0 / 25.7, 2 up to 3819, 16/4, 15.2 / 20.8."""
    least = 256 if workgroups >= 128 and room <= 256 else 128
    if coop == 8:
        return (8, least) if keys < 50_000 else (9, 256)
    return (9, least) if keys < 150_000 else (10, least if coop else 256)


def prefix_on_tiles(rows: int, prefix_len: int) -> bool:
    """Does a prefix run on tiles of 128 query rows (one read of it for so many), or as the own keys do, for 16?  ``rows`` = B * group.
    GPU time, us, tiles / 16 rows: 8 rows behind 1000 keys 11.7 / 10.2, 4 behind 4096 13.9 / 17.2, 32 behind 2000 15.1 / 18.0, 64 behind 1000 14 /
    16, 128 behind 500 17.3 / 24.0, behind 8000 27 / 60, 512 behind 2000 29 / 48."""
    return rows > lowering.DECODE_QROWS or prefix_len >= 2048


def prefix_splits(units: int, keys: int, rows: int, D: int, prefix_bytes: int, own_bytes: int) -> int:
    """Splits of a prefix on 128-row tiles, the least of a sum: ``units`` workgroups per split, ``keys`` tiles of 64 keys, ``rows`` (request, head)
    pairs, bytes of K and V of the prefix and of what the own keys have room for.  A tile of a chain takes 1.3 us (0.86 at head dimension 64), more
    with more than one workgroup per CU; chains gain nothing below what HBM takes for the prefix and part of the own keys; a split leaves its
    partial results, 0.46 us per 1000 rows.  300 drawn batches, 2 ... 256 requests of 20 ... 2000 keys behind 500 ... 16 000: 1.025 of the best number's
    time in the mean, 1.2 at most.  GPU time, us, by splits, 32/8 heads: 64 requests up to 1024 behind 2048 keys 2 42.5, 3 37.3, 4 38.6, 8 43.7; 128 up to 300
    behind 8208 4 61.5, 8 45.2, 9 42.9, 10 49.8, 15 55.8; 32 up to 100 behind 8000 8 36.2, 16 25.4, 21 28.1, 32 30.0; 8/2 heads, 11 up to 194 behind 4154 8 22.5, 17
    15.3, 33 13.5."""
    tile, best = 1.3 if D == 128 else 0.86, (math.inf, 1)
    stream = (prefix_bytes + own_bytes / 5) / 4.2e6
    for n in range(1, min(64, keys) + 1):
        chain = -(-keys // n) * tile * (1 + 0.4 * max(0.0, units * n / 256 - 1))
        best = min(best, (max(chain, stream) + n * (0.025 + 0.46e-3 * rows * D / 128), n))
    return best[1]


def _checked_choice(choice: dict) -> dict:
    """An override of the rules of the work split whose values the kernels serve: pieces begin at whole steps of 16 keys, in pairs, and are rounded up
    in 32 bits; partial results are kept for every piece that the own keys are cut for."""
    number = lambda lo, hi: lambda x: isinstance(x, int) and not isinstance(x, bool) and lo <= x <= hi
    served = {"prefix": lambda x: x in ("tiles", "stream"), "splits": number(0, 1 << 30), "target_log2": number(0, 24), "coop": lambda x: number(0, 8)(x) and x % 4 == 0,
              "least": lambda x: number(0, 1 << 30)(x) and x % 32 == 0, "near": lambda x: isinstance(x, bool)}
    for name, x in choice.items():
        if name not in served or not served[name](x):
            raise UnsupportedPlan(f"choice {name!r}: {x!r} not served")
    return choice


def scratch_parts(own: int, pre: int, D: int) -> tuple:
    """Floats of partial results, ``own`` rows of the requests' keys and ``pre`` of the prefix, and the bytes in front of part_ml, pre_acc and pre_ml: the sums
    with V of both come first, whose rows of 4 D bytes stay on borders of 16, then the pairs of offset and sum."""
    return (own + pre) * (D + 2), 4 * (own + pre) * D, 4 * own * D, 4 * (own + pre) * D + 8 * own


def combine_grid(B: int, Hq: int, D: int) -> int:
    """Blocks of lf_shared_combine: 1024 / D rows of one request each, or one row whose parts the block's groups of threads share."""
    return B * Hq if B * Hq <= 1024 else B * -(-Hq // (1024 // D))


@lowering.outside_graphs
def attention_shared(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, plan: AttnPlan, table: torch.Tensor, lengths: torch.Tensor, *,
                     prefix_table: Optional[torch.Tensor] = None, prefix_len: int = 0, v_table: Optional[torch.Tensor] = None,
                     prefix_v_table: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                     choice: Optional[dict] = None) -> torch.Tensor:
    """Attention of one new token per request over a prefix that all requests share and over the request's own keys.

    q : [B, Hq, 1, D], bf16 / fp16, D 64 or 128.  k_pool, v_pool : page pools of one page size.  table : [B, width], int32 or int64,
    the pages of each request's own keys, of which it has ``lengths[b]`` (int32 [B], on the GPU; what a row of the table has no room for is
    left out); entries behind the last page are not read.  prefix_table : [ceil(prefix_len / page)], the pages of the prefix, of
    the table's dtype.  ``v_table`` / ``prefix_v_table``: those of V where they differ from K's.  ``plan``: scale and softcap, no mask.
    Returns O [B, Hq, 1, D], of which no gradients are recorded; a request without a key, e.g. an empty place of a padded batch, gets zeros.

    The prefix is read once for all requests together: its keys meet the rows of the whole batch as a matrix product, the requests'
    own keys are streamed, and the partial results are joined in a second launch.  Page ids are trusted, as those of
    ``lowering.attention`` are (``LOOPFUSE_CHECK_TABLES=1`` looks at them).  ``choice`` overrides the rules of the work split: ``{"prefix": "tiles" | "stream", "splits": n,
    "target_log2": n, "least": n, "coop": n, "near": bool}``: splits 64 at most, target_log2 0 ... 24, least a multiple of 32, coop 0, or 4 or 8 heads where
    ``own_loads`` could have its own."""
    if not choice:
        done = _host.attention_shared(q, k_pool, v_pool, out, table, lengths, prefix_table, v_table, prefix_v_table, plan, prefix_len)
        if done is not None:
            return done
    return _shared(q, k_pool, v_pool, plan, table, lengths, prefix_table, _whole("prefix_len", prefix_len), v_table, prefix_v_table, out, _checked_choice(choice or {}))


@lowering._on_device_of_first_argument
def _shared(q, k_pool, v_pool, plan, table, lengths, prefix_table, prefix_len, v_table, prefix_v_table, out, choice):
    if isinstance(k_pool, Pool4) or isinstance(v_pool, Pool4):
        raise UnsupportedPlan("pools in 4 bits are attended over by attention_cached")
    given = (table, lengths, prefix_table, v_table, prefix_v_table)
    lowering._no_tangents(q, k_pool, v_pool)
    dtype = q.dtype
    if dtype not in lowering._DTYPE_CODE:
        raise UnsupportedPlan(f"dtype {dtype} not supported by the MFMA kernels (bf16/fp16 only)")
    if q.dim() != 4 or q.shape[2] != 1 or q.shape[3] not in (64, 128):
        raise UnsupportedPlan("Q must be [B, Hq, 1, D] with head dim 64 or 128")
    B, Hq, _, D = q.shape
    lowering._check_tensor("Q", q, dtype)
    for name, t in (("K pool", k_pool), ("V pool", v_pool)):
        lowering._check_tensor(name, t, dtype)
        if t.device != q.device:
            raise RuntimeError(f"loopfuse_amd: {name} is on {t.device}, Q on {q.device}")
    if plan.mask not in (None, "none") or plan.denom_add != 0.0:
        raise UnsupportedPlan("attention over a shared prefix takes no mask and the plain softmax denominator")
    if not (plan.scale > 0.0) or not math.isfinite(plan.scale):
        raise UnsupportedPlan("score scale must be positive and finite")
    softcap = None
    if plan.softcap is not None:
        softcap = abs(float(plan.softcap))
        if not (softcap > 0.0) or not math.isfinite(softcap):
            raise UnsupportedPlan("softcap must be finite and non-zero")
    pages, page, Hkv, Dk, *ks = _pool("K", k_pool)
    pages_v, page_v, Hkv_v, Dv, *vs = _pool("V", v_pool)
    if page != page_v or Hkv != Hkv_v or Dk != D or Dv != D:
        raise UnsupportedPlan("the pools must have one page size, the same kv heads and Q's head dim")
    _shift(page)
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise UnsupportedPlan("Hq must be a multiple of Hkv")
    group = Hq // Hkv
    _on_gpu("table", table, _TABLE_DTYPES, 2, q.device)
    _on_gpu("lengths", lengths, (torch.int32,), 1, q.device)
    v_table = table if v_table is None else v_table
    _on_gpu("V table", v_table, (table.dtype,), 2, q.device)
    if table.shape[0] != B or v_table.shape != table.shape or lengths.shape[0] != B:
        raise UnsupportedPlan(f"tables and lengths must be of {B} requests, the tables of one width")
    # (the kernels round keys up to pieces, 2**30 keys at most, in 32 bits)
    if prefix_len < 0 or max(prefix_len, table.shape[1] * page) > 1 << 30:
        raise UnsupportedPlan("a request or the prefix has room for more than 2**30 keys")
    if prefix_len:
        if prefix_table is None:
            raise UnsupportedPlan("a prefix needs its table")
        prefix_v_table = prefix_table if prefix_v_table is None else prefix_v_table
        for name, t in (("prefix table", prefix_table), ("V prefix table", prefix_v_table)):
            _on_gpu(name, t, (table.dtype,), 1, q.device)
            if t.shape[0] * page < prefix_len:
                raise UnsupportedPlan(f"{name} has room for {t.shape[0] * page} of {prefix_len} keys")
        prefix_table, prefix_v_table = prefix_table.contiguous(), prefix_v_table.contiguous()
    # (the kernels have 32 bits for the distance of a table's rows)
    table, v_table = (t if t.stride(1) == 1 and t.stride(0) < 1 << 31 else t.contiguous() for t in (table, v_table))
    lengths = lengths.contiguous()
    if out is not None:
        lowering._check_tensor("O", out, dtype)
        if tuple(out.shape) != (B, Hq, 1, D) or out.device != q.device or any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
            raise UnsupportedPlan(f"O must be [{B}, {Hq}, 1, {D}] on the device of Q, every element with a place of its own")
    if B == 0:
        return torch.empty(q.shape, dtype=dtype, device=q.device) if out is None else out
    if lowering._checks_tables():
        used = torch.arange(table.shape[1], device=q.device) < ((lengths.clamp(min=0).long() + page - 1) // page)[:, None]
        named = [(table[used], pages), (v_table[used], pages_v)]
        if prefix_len:
            named += [(t[:-(-prefix_len // page)], n) for t, n in ((prefix_table, pages), (prefix_v_table, pages_v))]
        if any(len(t) and (int(t.min()) < 0 or int(t.max()) >= n) for t, n in named) or (B and int(lengths.max()) > table.shape[1] * page):
            raise ValueError(f"loopfuse_amd: page ids outside 0 ... {pages - 1} (V: {pages_v - 1}), or a length beyond its row of the table")
    P = SharedParams()
    P.q_sb, P.q_sh, P.q_ss = q.stride(0), group * q.stride(1), q.stride(1)
    o_sb, o_sh = (Hq * D, D) if out is None else out.stride()[:2]
    P.o_sb, P.o_sh, P.o_ss = o_sb, group * o_sh, o_sh
    P.k_sb, P.k_ss, P.k_sh = ks
    P.v_sb, P.v_ss, P.v_sh = vs
    P.kt_stride, P.vt_stride = table.stride(0), v_table.stride(0)
    P.B, P.Hq, P.Hkv, P.rows, P.Sq = B, Hq, Hkv, group, 1
    P.scale, P.softcap = float(plan.scale), softcap or 0.0
    P.room = table.shape[1] * page
    P.Sk = prefix_len
    rows = B * group
    # direct-to-LDS loads with 32-bit offsets, in the pools or else in a page
    spans = [sum((n - 1) * abs(st) for n, st in zip(t.shape, t.stride())) + 1 for t in (k_pool, v_pool)]
    near = max(spans) < (1 << 31) - 64
    tiles = prefix_len > 0 and all(st >= 0 for t in (k_pool, v_pool) for st in t.stride()) and \
        (near or (page % 8 == 0 and page * max(P.k_ss, P.v_ss) < 1 << 30)) and \
        choice.get("prefix", "tiles" if prefix_on_tiles(rows, prefix_len) else "stream") == "tiles"
    if tiles and not choice.get("near", True) and page % 8 == 0:
        near = False
    coop = lowering._decode_coop_waves(3, page, 0, 0, Hkv, P, D)
    if choice.get("coop") and (not coop or Hkv % choice["coop"] or choice["coop"] * D < 512 or (tiles and choice["coop"] != 4)):
        raise UnsupportedPlan(f"choice 'coop': {choice['coop']} heads of {Hkv} of {D}")
    if coop:
        coop = choice.get("coop", own_loads(D, Hkv, tiles, B, B * P.room + (0 if tiles else prefix_len)))
    chunks = -(-group // lowering.DECODE_QROWS)
    heads = Hkv // coop if coop else Hkv
    P.units = heads * chunks
    target, least = own_pieces(coop, B * P.units, P.room, B * P.room)
    P.target_log2, P.least = choice.get("target_log2", target), choice.get("least", least)
    items = (1 << P.target_log2) // P.units + B if P.room else 0
    splits = 0
    P.nsplit = P.pre_units = 1
    if prefix_len:
        if tiles:
            P.pre_units, keys = Hkv * -(-rows // 128), -(-prefix_len // 64)
            splits = max(1, min(64, keys, choice.get("splits", prefix_splits(P.pre_units, keys, B * Hq, D, 4 * prefix_len * Hkv * D, 4 * B * P.room * Hkv * D))))
            P.split_len = 64 * -(-keys // splits)
            splits = -(-prefix_len // P.split_len)
            P.k_span, P.v_span = spans if near else (1, 1)
        else:
            P.pre_units = heads * -(-rows // lowering.DECODE_QROWS)
            splits = max(1, min(64, prefix_len // 32, choice.get("splits", 512 // P.pre_units)))
            splits, P.split_len = lowering._split_lengths(splits, prefix_len)
        P.nsplit, P.pre_blocks = splits, splits * P.pre_units
    if (P.pre_blocks + items * P.units) * 64 * max(4, coop) >= 1 << 32:
        raise UnsupportedPlan(f"a launch for {B} requests of {Hq} heads is too large")
    args = dict(rows=lowering.DECODE_QROWS, waves=coop or 4, headwave=coop > 0, coop=coop > 0,
                rowload=not coop and lowering._decode_rowload(3, page, 0, 0))
    steps, spec = [], lowering._spec("decode", lowering._DTYPE_CODE[dtype], D, lowering.MASK_NONE, softcap is not None, 3, page,
                                     table.dtype == torch.int64, shared=(2 if near else 3) if tiles else 1, **args)
    if splits or items:
        steps.append((lowering.get_kernel(spec, "lf_attn_decode"), (P.pre_blocks + items * P.units, 1, 1), 64 * args["waves"]))
    spec = lowering._spec("shared_combine", lowering._DTYPE_CODE[dtype], D)
    steps.append((lowering.get_kernel(spec, spec.entry()), (combine_grid(B, Hq, D), 1, 1), 256))
    repeat = lowering._Repeat(P, steps, {"kernels": [k.symbol for k, _, _ in steps], "prefix": "tiles" if tiles else "stream", "splits": splits},
                              scratch_parts(items * Hq, splits * B * Hq, D))
    res = _again(q, k_pool, v_pool, table, lengths, prefix_table if prefix_len else None, v_table, prefix_v_table, out, repeat)
    if not choice and all(a is b for a, b in zip(given[:3], (table, lengths, prefix_table))) and (given[3] is None or given[3] is v_table) \
            and (given[4] is None or given[4] is prefix_v_table):
        lowering._keep_call(lowering._call_key("h", (q, k_pool, v_pool, out), given, plan, (prefix_len,)), repeat, repeat.more)
    return res


def _again(q, k_pool, v_pool, table, lengths, prefix_table, v_table, prefix_v_table, out, repeat):
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    P = SharedParams.from_buffer_copy(repeat.block)
    P.q, P.k, P.v, P.o = q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr()
    P.k_table = table.data_ptr()
    P.v_table = P.k_table if v_table is None else v_table.data_ptr()
    P.lengths = lengths.data_ptr()
    if prefix_table is not None:
        P.prefix_k = prefix_table.data_ptr()
        P.prefix_v = P.prefix_k if prefix_v_table is None else prefix_v_table.data_ptr()
    floats, ml, pre_acc, pre_ml = repeat.more
    with lowering._scratch_lock:        # no other thread's step on this stream between the launches
        scratch = lowering._get_scratch(q.device, floats)
        at = scratch.data_ptr()
        P.part_acc, P.part_ml, P.pre_acc, P.pre_ml = at, at + ml, at + pre_acc, at + pre_ml
        repeat.launches.launch(P)
    lowering._last_launch.set(repeat.record)
    return out


def cached_build(rows: float, all_rows: int, keys: int, D: int) -> tuple:
    """(blocks of 16 rows of a wave, do a workgroup's waves have rows of their own) for so many rows of a kv head per request, ``all_rows`` of all heads and up to ``keys`` keys.
    Up to 16 rows are taken by four waves that share their keys; more of them 32 at a time in the same way, whose keys and values are converted once for both blocks, where the work is enough for
    half the workgroups (at head dimension 64, of which two run on a CU where four of the others do, also for pairs of blocks or long keys only); many 128 at a time, whose keys and
    values are converted once for four waves.  us, 16 / 32: 32/8 heads of 128, 16 requests of 2048 keys, 8 new tokens each 17.5 / 21.3, 16 22.4 / 21.9, 64 65 / 53; 4 of 8192, 8 21.5 / 22.2, 32 46 / 38; 64 of
    1500, 8 35 / 28; 64 up to 8192, 5 99 / 74; 2 of 100 000, 5 80 / 57; 64/2 heads, 64 up to 8192, 1 38 / 29; 4/4 of 64, 100 of 1200, 40 26 / 33.  32 / 128: 32/8 heads of 128, 16 of 2048, 96 82 / 91, 128 99 / 94,
    512 390 / 273; 4 of 8192, 128 87 / 98, 256 166 / 159; 1 of 32 768, 256 182 / 159; 1 of 1000, all 36 / 42; 2 of 1500, all 122 / 70; 32 of 700, 64 57 / 43; 16/16 of 64, 32 of 1024, 64 28 / 38, 128 51 / 40."""
    if rows > 64 and (all_rows >= 65536 or all_rows * keys >= 2 * 10 ** 8):
        return 2, True
    if rows > 16 and all_rows * keys >= 16 * 10 ** 6 and (D == 128 or keys > 4096 or math.ceil(rows / 16) % 2 == 0):
        return 2, False
    return 1, False


def cached_spec(dtype: torch.dtype, D: int, mask: int, softcap: bool, table_i64: bool, blocks: int, rowwaves: bool) -> lowering.KernelSpec:
    return lowering._spec("cached", lowering._DTYPE_CODE[dtype], D, mask, softcap, table_i64=table_i64,
                          extra=(f"-DLF_CACHED_CB={blocks}",) + (("-DLF_CACHED_ROWWAVES=1",) if rowwaves else ()))


def cached_shares(units: int, keys: int, rows: float, build: tuple, D: int) -> tuple:
    """(workgroups, what a unit costs besides its pairs of tiles or -1, least share of a workgroup) for at most so many units of up to ``keys`` keys that a row can see, ``rows`` as
    above; -1: each workgroup has a unit.  Shares cost a second launch, 4 us, and the begin of every part of a unit; a unit of its own the chain of its pairs, 0.6 us a
    pair of each wave (1.2 us in 128 rows), and what the longest lasts longer than the others, which differ less where a request has many; under a causal mask the first of a request's new tokens
    have fewer keys than shares are cut for.  As many workgroups as run at once: two on a CU (16 rows of 128, 32 rows), three (128 rows of 128; 16 rows of 64), four.
    us, shares / units: 16 rows, 2 requests up to 1000, 32/8 heads of 128, 12.5 / 10.8, 64 up to 8192 65 / 76, 4 up to 100 000 58 / 620, 75 up to 2063, 8/8, 32 / 30, 16 of 2048 with 8 new tokens each 21 / 18, 48 up to 1029 in a window,
    16/4 of 64, 21 / 17, 53 of 1681 with 75 new tokens each, 4/4, 54 / 40; workgroups, 512 / 768 / 1024: 64 up to 8192 64 / 66 / 73, 48 up to 12 341, 32/8 of 64, 57 / 52 / 50.  128 rows, 32/8 of
    128: 16 of 2048 with 128 new each 108 / 92, 8 of 4096 with 128 108 / 147, 4 up to 6001 with up to 1000 286 / 235, 1 of 12 000 with 1000 231 / 407, 1 of 32 768 with 3500 1820 / 2341, with 6144
    2965 / 2854; workgroups, 512 / 768 / 1024: 4 of 8192 with 256 new each 195 / 161 / 199.  32 rows, 32/8 of 128: 64 up to 8192 with 5 new each 74 / 91, 24 of 1900 with 5 25 / 21, 32 of 4096 with 8
    42 / 43, with 10 57 / 54, 4 of 8192 with 128 96 / 87, 1 of 32 768 with 256 182 / 221."""
    if build == (2, True):
        if units >= (256 if keys <= 1536 else 512 if keys <= 4096 else 768 if keys <= 12288 else 1536):
            return units, -1, 1
        return 768 if D == 128 else 1024, 8, 20
    if build == (2, False):
        return (units, -1, 1) if keys <= 2100 or (units >= 512 and (rows >= 32 or keys <= 4096)) else (512, 16, 20)
    if keys <= 1536 or (units >= 512 and rows >= 64) or (units >= 256 and keys <= 2100):
        return units, -1, 1
    return 512 if D == 128 else 768, 16, 20


@lowering.outside_graphs
def attention_cached(q: torch.Tensor, k_pool: Pool4, v_pool: Pool4, plan: AttnPlan, table: torch.Tensor, lengths: torch.Tensor,
                     offsets: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the new tokens of requests of different lengths, one each or several, over their keys and values in page pools held in 4 bits.

    q : [rows, Hq, D], bf16 / fp16, Hq a multiple of the pools' heads, D 64 or 128 (views will do).  table : [B, width], int32 or int64, each request's pages, of which it
    has ``lengths[b]`` keys (int32 [B], on the GPU; what a row of the table has no room for is left out), those of its new tokens among them; entries behind the last
    page are not read.  ``offsets``: int32 [B + 1], request b's new tokens are rows offsets[b] ... offsets[b + 1]; ``positions``: int32 [rows], of each in its request, not
    descending within it; below 0: a row of no token.  Both as ``extend_tables`` leaves them (``PagedStep``); without offsets row b is request b's, without
    positions (for one row per request at most) its last key's.  ``plan``: scale and softcap, and the mask: causal (a token sees the keys up to its own position), sliding, or
    none (all keys of its request).

    Returns O [rows, Hq, D], of which no gradients are recorded.  Rows of no token, and those without a key, are zeros; rows of no request are zeros too, or stay as they
    are in an ``out`` that is given.  A prompt's next part, behind what the cache has of it, is such a call; a prompt of which the cache has nothing attends over
    its own unrounded keys by ``packed.attention_packed``.  Page ids are trusted, as those of ``lowering.attention`` are (``LOOPFUSE_CHECK_TABLES=1`` looks at them)."""
    parts = _parts(k_pool, v_pool, q.dtype)
    if parts is not None and parts[2] is not None:
        done = _host.attention_cached(q, *parts, out, table, lengths, offsets, positions, plan)
        if done is not None:
            return done
    return _cached(q, k_pool, v_pool, plan, table, lengths, offsets, positions, out)


@lowering._on_device_of_first_argument
def _cached(q, k_pool, v_pool, plan, table, lengths, offsets, positions, out):
    given = (table, lengths, offsets, positions)
    lowering._no_tangents(q)
    dtype = q.dtype
    if dtype not in lowering._DTYPE_CODE:
        raise UnsupportedPlan(f"dtype {dtype} not supported by the MFMA kernels (bf16/fp16 only)")
    if q.dim() != 3 or q.shape[2] not in (64, 128):
        raise UnsupportedPlan("Q must be [rows, Hq, D] with head dim 64 or 128")
    lowering._check_tensor("Q", q, dtype)
    T, Hq, D = q.shape
    pages, page, Hkv, Dk = _two_pools4(k_pool, v_pool, dtype, q.device)
    if pages > 1 and not k_pool.codes.stride(0) == v_pool.codes.stride(0) == 16 * k_pool.scales.stride(0) == 16 * v_pool.scales.stride(0):
        raise UnsupportedPlan("pages must be as far apart in V's pool as in K's, those of codes 16 times as far as those of scales")
    if page * Hkv * Dk >= 1 << 32:
        raise UnsupportedPlan("a page of 2 GiB of codes or more")
    if Dk != D or Hq < 1 or Hq % Hkv:
        raise UnsupportedPlan("the pools must have Q's head dim, Hq a multiple of their heads")
    if plan.mask not in lowering._MASK_NAMES or plan.denom_add != 0.0:
        raise UnsupportedPlan("attention over a cache in 4 bits takes no mask, a causal or a sliding one, and the plain softmax denominator")
    mask = lowering._MASK_NAMES[plan.mask]
    if mask == lowering.MASK_SLIDING and plan.window < 1:
        raise UnsupportedPlan("sliding mask needs window >= 1")
    narrow = lambda x: ctypes.c_float(x).value       # (as the kernels take it: masked scores, -inf, must not meet a scale of 0)
    if not (narrow(plan.scale) > 0.0) or not math.isfinite(narrow(plan.scale)):
        raise UnsupportedPlan("score scale must be positive and finite in 32 bits")
    softcap = None
    if plan.softcap is not None:
        softcap = abs(float(plan.softcap))
        if not (narrow(softcap) > 0.0) or not math.isfinite(narrow(softcap)) or not math.isfinite(narrow(plan.scale / softcap)):
            raise UnsupportedPlan("softcap, and the scale over it, must be finite, the cap non-zero, in 32 bits")
    _on_gpu("table", table, _TABLE_DTYPES, 2, q.device)
    _on_gpu("lengths", lengths, (torch.int32,), 1, q.device)
    B = table.shape[0]
    if lengths.shape[0] != B:
        raise UnsupportedPlan(f"table and lengths must be of as many requests, not {B} and {lengths.shape[0]}")
    if offsets is not None:
        _on_gpu("offsets", offsets, (torch.int32,), 1, q.device)
        if offsets.shape[0] != B + 1:
            raise UnsupportedPlan(f"offsets must be int32 [{B + 1}]")
    elif T != B:
        raise UnsupportedPlan(f"without offsets there is a row for each of the {B} requests, not {T}")
    if positions is not None:
        _on_gpu("positions", positions, (torch.int32,), 1, q.device)
        if positions.shape[0] != T:
            raise UnsupportedPlan(f"positions must be int32 [{T}]")
    elif offsets is not None and T > B:
        raise UnsupportedPlan("requests with several rows need positions")
    room = table.shape[1] * page if pages else 0
    if room > 1 << 30:
        raise UnsupportedPlan("a request has room for more than 2**30 keys")
    if out is not None:
        lowering._check_tensor("O", out, dtype)
        if tuple(out.shape) != (T, Hq, D) or out.device != q.device or any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
            raise UnsupportedPlan(f"O must be [{T}, {Hq}, {D}] on the device of Q, every element with a place of its own")
    if T == 0 or B == 0:
        return torch.zeros(q.shape, dtype=dtype, device=q.device) if out is None else out
    if lowering._checks_tables():
        used = torch.arange(table.shape[1], device=q.device) < ((lengths.clamp(min=0).long() + page - 1) // page)[:, None]
        ids = table[used]
        if len(ids) and (int(ids.min()) < 0 or int(ids.max()) >= pages) or int(lengths.max()) > room:
            raise ValueError(f"loopfuse_amd: page ids outside 0 ... {pages - 1}, or a length beyond its row of the table")
        if offsets is not None and (bool((offsets[1:] < offsets[:-1]).any()) or int(offsets[0]) < 0 or int(offsets[-1]) > T):
            raise ValueError(f"loopfuse_amd: offsets must not descend, within 0 ... {T}")
    P = CachedParams()
    P.q_ss, P.q_sh = q.stride()[:2]
    P.o_ss, P.o_sh = (Hq * D, D) if out is None else out.stride()[:2]
    P.page_bytes = k_pool.codes.stride(0)
    P.T, P.B, P.Hkv, P.group = T, B, Hkv, Hq // Hkv
    P.room, P.shift, P.clear = room, _shift(page), int(out is None)
    P.window = min(int(plan.window), 1 << 30) if mask == lowering.MASK_SLIDING else 0
    P.scale, P.softcap = plan.scale, softcap or 0.0
    keys, per = min(room, P.window + T) if P.window else room, T * P.group / B
    blocks, rowwaves = build = cached_build(per, T * Hq, keys, D)
    rows = 16 * blocks * (4 if rowwaves else 1)
    units = (T * P.group // rows + min(T, B)) * Hkv       # (at most: a chunk that is not full for each request)
    P.workgroups, P.fixed, P.least = cached_shares(units, keys, per, build, D)
    if P.workgroups * 256 >= 1 << 32:
        raise UnsupportedPlan(f"a launch for {T} rows of {Hq} heads, of {B} requests, is too large")
    P.per_group = (-(-(1 << 32) // P.group)) & 0xffffffff
    # (the line of all units, and rows times their division's error, are numbers in 32 bits)
    if units * (-(-room // 32) + 64) >= 1 << 31 or T * P.group ** 2 >= 1 << 32 or T * P.group >= 1 << 30:
        raise UnsupportedPlan(f"a launch for {T} rows of {Hq} heads, of {B} requests of up to {room} keys, is too large")
    table = table if table.shape[1] == 0 or table.stride(1) == 1 else table.contiguous()
    lengths, offsets, positions = (t if t is None else t.contiguous() for t in (lengths, offsets, positions))
    P.table_stride = table.stride(0)
    spec = cached_spec(dtype, D, mask, softcap is not None, table.dtype == torch.int64, blocks, rowwaves)
    steps = [(lowering.get_kernel(spec, "lf_cached"), (P.workgroups, 1, 1), 256)]
    if P.fixed >= 0:
        per = 1024 // D
        grid = T * Hq if T * Hq <= 1024 else T * -(-Hq // per)
        if grid * 256 >= 1 << 32:
            raise UnsupportedPlan(f"a launch for {T} rows of {Hq} heads is too large")
        steps.append((lowering.get_kernel(spec, "lf_cached_combine"), (grid, 1, 1), 256))
    P.slots = units + P.workgroups if P.fixed >= 0 else 0
    slots = P.slots * rows
    repeat = lowering._Repeat(P, steps, {"kernels": [k.symbol for k, _, _ in steps]}, (slots * (D + 2), 4 * slots * D))
    res = _cached_again(q, k_pool, v_pool, table, lengths, offsets, positions, out, repeat)
    if all(a is b for a, b in zip(given, (table, lengths, offsets, positions))):
        lowering._keep_call(lowering._call_key("c", (q, *_parts(k_pool, v_pool, dtype), out), given, plan, ()), repeat, repeat.more)
    return res


def _cached_again(q, k_pool, v_pool, table, lengths, offsets, positions, out, repeat):
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    P = CachedParams.from_buffer_copy(repeat.block)
    P.q, P.o, P.table, P.lengths = q.data_ptr(), out.data_ptr(), table.data_ptr(), lengths.data_ptr()
    for name, t in (("offsets", offsets), ("positions", positions)):
        if t is not None:
            setattr(P, name, t.data_ptr())
    _set_pools(P, "k", "v", k_pool, v_pool)
    floats, ml = repeat.more
    if floats:
        with lowering._scratch_lock:        # no other thread's step on this stream between the launches
            at = lowering._get_scratch(q.device, floats).data_ptr()
            P.part_acc, P.part_ml = at, at + ml
            repeat.launches.launch(P)
    else:
        repeat.launches.launch(P)
    lowering._last_launch.set(repeat.record)
    return out


from . import rotary  # noqa: E402  (either module's host module knows PagedStep)

_host = lowering._host()
