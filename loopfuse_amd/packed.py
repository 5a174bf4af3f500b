"""Attention over sequences of different lengths packed into one tensor, forward and backward.

A batch whose sequences differ in length stands here as one tensor ``[rows, heads, D]``, one sequence behind the other, with
their bounds ``offsets`` (``N + 1`` numbers on the GPU): no padding is stored, read or computed.

    layout = packed_layout(offsets, total)                  # once per batch, for all layers
    o = attention_packed(q, k, v, AttnPlan("causal", scale=D ** -0.5), layout)

Every query sees the keys of its own sequence under the plan's mask (none, causal, causal sliding window; positions count from the
sequence's first row).  The kernels are those of the dense operators (``lowering.attention``, ``lowering.attention_backward``)
built with ``-DLF_PACKED=1``: their workgroups take the tiles of a list that ``packed_layout`` leaves on the GPU, so that nothing
waits for the lengths.  The reference has no counterpart: its graphs hold one length for a batch (reference README.md:62-99).
"""
from __future__ import annotations

import ctypes
import dataclasses
import math
import operator
from typing import Optional

import torch

from . import lowering, runtime
from .lowering import AttnPlan, UnsupportedPlan

TILE_HEIGHTS = (32, 64, 128, 256)      # rows of a tile, lists by lists
GROUP_SIZES = (1, 2, 4, 8)             # sequences whose tiles come together, list by list
MAX_ROWS = (1 << 31) - 1024            # of a packed batch
MAX_SEQUENCES = 1 << 22                # each is ranked among all of them, some seconds for so many


class _PlanParams(ctypes.Structure):
    """Mirror of ``struct LfPackedPlanParams`` in csrc/kernels/lf_packed_plan.hip."""

    _fields_ = [("offsets", ctypes.c_void_p), ("tiles", ctypes.c_void_p), ("sorted", ctypes.c_void_p), ("N", ctypes.c_int), ("T", ctypes.c_int),
                ("cap", ctypes.c_int * 4)]


class PackedAttnParams(lowering.AttnParams):
    """Mirror of ``struct LfPackedAttnParams`` in csrc/kernels/lf_packed.hip.h."""

    _fields_ = [("tiles", ctypes.c_void_p), ("low", ctypes.c_void_p), ("clear", ctypes.c_int)]


class PackedBwdParams(lowering.AttnBwdParams):
    """Mirror of ``struct LfPackedBwdParams`` in csrc/kernels/lf_attn_bwd.hip."""

    _fields_ = [("dkdv_tiles", ctypes.c_void_p), ("dq_tiles", ctypes.c_void_p), ("low", ctypes.c_void_p), ("dkdv_blocks", ctypes.c_int)]


@dataclasses.dataclass(frozen=True, eq=False)
class PackedLayout:
    """Where the sequences of a packed batch lie, and the lists of their tiles (``packed_layout``)."""

    offsets: torch.Tensor      # int32 [N + 1]
    total: int                 # rows of the packed tensors
    tiles: torch.Tensor        # int32 [entries of all lists, 4]
    caps: tuple                # entries of each list

    @property
    def count(self) -> int:
        return self.offsets.shape[0] - 1

    def tiles_of(self, rows: int, units: int) -> tuple:
        """(first byte in ``tiles``, entries) of the list of tiles of so many rows in groups of about ``units`` sequences."""
        i, g = TILE_HEIGHTS.index(rows), max(j for j, n in enumerate(GROUP_SIZES) if n <= max(1, units))
        return 16 * (len(GROUP_SIZES) * sum(self.caps[:i]) + g * self.caps[i]), self.caps[i]


@lowering.outside_graphs
def packed_layout(offsets: torch.Tensor, total: int) -> PackedLayout:
    """The layout of a batch of ``N`` packed sequences, ``MAX_SEQUENCES`` at most: sequence ``n`` is rows ``offsets[n] ... offsets[n + 1]`` of
    tensors of ``total`` rows, ``MAX_ROWS`` at most.  ``offsets``: int32 or int64 ``[N + 1]`` on the GPU, not descending (as a cumulative sum of the lengths is); sequences may be
    empty.  Two launches on the current stream, nothing waits for them; the layout serves every call over this batch, forward and
    backward, on that stream or on one that waits for it.  Offsets beyond ``0 ... total`` count as the nearer bound
    (``LOOPFUSE_CHECK_TABLES=1`` raises for them and for descending ones)."""
    done = _host.packed_layout(offsets, total)
    if done is not None:
        return PackedLayout(offsets, total, *done)
    if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.shape[0] < 1 or offsets.dtype not in (torch.int32, torch.int64):
        raise UnsupportedPlan("offsets must be an int32 or int64 tensor of one more than the number of sequences")
    if not offsets.is_cuda:
        raise RuntimeError("loopfuse_amd: offsets are not on the GPU; the HIP path has no CPU fallback")
    if isinstance(total, torch.Tensor):
        raise UnsupportedPlan("the number of rows must be a number of the host's")
    total = operator.index(total)
    # (the kernels round rows up to tiles, and walk a few tiles ahead, in 32 bits)
    if total < 0 or total > MAX_ROWS:
        raise UnsupportedPlan(f"the number of rows must be between 0 and {MAX_ROWS}")
    if offsets.shape[0] > MAX_SEQUENCES + 1:
        raise UnsupportedPlan(f"more than {MAX_SEQUENCES} sequences")
    with torch.cuda.device(offsets.device):
        count = offsets.shape[0] - 1
        if lowering._checks_tables():
            ends = offsets.tolist()
            if any(a > b for a, b in zip(ends, ends[1:])) or ends[0] < 0 or ends[-1] > total:
                raise ValueError(f"loopfuse_amd: offsets must not descend, within 0 ... {total}")
        given, offsets = offsets, offsets.clamp(0, total).to(torch.int32) if offsets.dtype == torch.int64 else offsets.contiguous()
        # a sequence ends with a tile that is not full; so do the rows of no sequence at either end
        caps = tuple(total // rows + count + 2 for rows in TILE_HEIGHTS)
        made = torch.empty(4 * len(GROUP_SIZES) * sum(caps) + (3 + len(caps)) * (count + 2), dtype=torch.int32, device=offsets.device)
        tiles = made[:4 * len(GROUP_SIZES) * sum(caps)].view(-1, 4)
        P = _PlanParams(offsets.data_ptr(), tiles.data_ptr(), tiles.data_ptr() + 16 * tiles.shape[0], count, total, caps)
        spec = lowering._spec("packed_plan", 0, 64)
        repeat = lowering._Repeat(P, [(lowering.get_kernel(spec, "lf_packed_sort"), (-(-(count + 2) // 256), 1, 1), 256),
                                      (lowering.get_kernel(spec, "lf_packed_plan"), (-(-(count + 2) // 4), len(caps) * len(GROUP_SIZES), 1), 256)], None)
        repeat.launches.launch(P)
        if given is offsets:
            lowering._keep_call(lowering._call_key("l", (), (offsets,), None, (total,)), repeat, (tiles.shape[0], made.shape[0]), (repeat, caps))
    return PackedLayout(offsets, total, tiles, caps)


def _rows(name: str, t: torch.Tensor, layout: PackedLayout, dtype, D: Optional[int] = None) -> None:
    if t.dim() != 3 or t.shape[0] != layout.total:
        raise UnsupportedPlan(f"{name} must be [{layout.total}, heads, D]")
    if D is not None and t.shape[2] != D:
        raise UnsupportedPlan(f"{name} has head dim {t.shape[2]}, Q has {D}")
    lowering._check_tensor(name, t, dtype)
    if t.device != layout.tiles.device:
        raise RuntimeError(f"loopfuse_amd: {name} is on {t.device}, the layout on {layout.tiles.device}")


def _row_stride(t: torch.Tensor) -> int:
    """Elements from a row to the next.  The stride of a dimension of one element can be any number: of one row its length, so that what is read
    behind it lies outside."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2]


def _constants(plan: AttnPlan, total: int) -> tuple:
    """(mask, window, scale, softcap or None) of a plan that the packed kernels serve."""
    if plan.k_paged or plan.v_paged or plan.denom_add != 0.0:
        raise UnsupportedPlan("packed sequences go with dense K/V and the plain softmax denominator")
    if plan.mask not in lowering._MASK_NAMES:
        raise UnsupportedPlan(f"mask {plan.mask!r} not served")
    mask = lowering._MASK_NAMES[plan.mask]
    if mask == lowering.MASK_SLIDING and plan.window < 1:
        raise UnsupportedPlan("sliding mask needs window >= 1")
    if not (plan.scale > 0.0) or not math.isfinite(plan.scale):
        raise UnsupportedPlan("score scale must be positive and finite")
    cap = None
    if plan.softcap is not None:
        cap = abs(float(plan.softcap))
        if not (cap > 0.0) or not math.isfinite(cap):
            raise UnsupportedPlan("softcap must be finite and non-zero")
    # (a window beyond all rows keeps what one of their number keeps; the kernels add it to positions in 32 bits)
    return mask, min(int(plan.window), max(total, 1)) if mask == lowering.MASK_SLIDING else 0, float(plan.scale), cap


def _heads(q, k, v, layout) -> tuple:
    dtype = q.dtype
    if dtype not in lowering._DTYPE_CODE:
        raise UnsupportedPlan(f"dtype {dtype} not supported by the MFMA kernels (bf16/fp16 only)")
    if q.dim() != 3 or q.shape[2] not in (64, 128):
        raise UnsupportedPlan("Q must be [rows, Hq, D] with head dim 64 or 128")
    D = q.shape[2]
    for name, t in (("Q", q), ("K", k), ("V", v)):
        _rows(name, t, layout, dtype, D)
    Hq, Hkv = q.shape[1], k.shape[1]
    if v.shape[1] != Hkv or Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise UnsupportedPlan(f"{Hq} query heads over {Hkv} / {v.shape[1]} kv heads")
    return dtype, D, Hq, Hkv


def _grid(entries: int, heads: int, threads: int) -> int:
    if entries * heads * threads >= 1 << 32:
        raise UnsupportedPlan(f"a launch of {entries} tiles x {heads} heads is too large")
    return entries * heads


@lowering.outside_graphs
def attention_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: AttnPlan, layout: PackedLayout, *,
                     out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of every packed sequence over itself: q ``[rows, Hq, D]``, k and v ``[rows, Hkv, D]`` (views will do: rows of a
    fused projection) to O ``[rows, Hq, D]``.  bf16 / fp16, Hq a multiple of Hkv, D 64 or 128, any other below 128 by zero-padding;
    ``plan``: mask, window, scale and softcap.  Rows of no sequence, in front of the first offset or behind the last,
    come out as zeros, or stay as they are in an ``out`` that is given.  ``lse``: float32 ``[Hq, rows]``, contiguous, to be given the
    rows' log-sum-exp in log2 units, as ``lowering.attention`` does.

    Inside ``torch.compile`` the call runs as it is, between two graphs.

    Differentiable where gradients are recorded and neither ``out`` nor ``lse`` is given; gradients of rows of no sequence are zero.  Forward-mode
    derivatives are refused.
    Under graph capture a leaf that another autograd graph holds is refused, and what a graph made outside the capture computed: capture forward and
    backward with no eager graph of them alive.
    Kept for the backward besides Q, K, V and O: lse, and what rounding takes from O, as large as O (it halves what delta is off by)."""
    if not isinstance(layout, PackedLayout):
        raise UnsupportedPlan("layout must come from packed_layout")
    grads = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if grads and (out is not None or lse is not None):
        raise UnsupportedPlan("out and lse are for calls without gradients")
    if grads and torch.cuda.is_current_stream_capturing() and any(t.requires_grad and (in_a_graph(t) if t.is_leaf else _host.elsewhere(t)) for t in (q, k, v)):
        raise UnsupportedPlan("under capture, Q, K and V must not be leaves of an autograd graph that lives, nor come from one that was made outside: its "
                              "stream would be waited for. Drop what that graph computed, or take detached tensors")
    if q.dim() == 3 and q.shape[2] not in (64, 128) and 1 <= q.shape[2] < 128:
        if out is not None or lse is not None or k.dim() != 3 or v.dim() != 3 or k.shape[2] != q.shape[2] or v.shape[2] != q.shape[2]:
            raise UnsupportedPlan(f"head dim {q.shape[2]}: by zero-padding, without out and lse")
        D = q.shape[2]
        q, k, v = (torch.nn.functional.pad(t, (0, (64 if D < 64 else 128) - D)) for t in (q, k, v))
        return attention_packed(q, k, v, plan, layout)[..., :D].contiguous()
    if grads:
        lowering._no_tangents(q, k, v)      # (not to be seen inside)
        return _Packed.apply(q, k, v, plan, layout)
    done = _host.attention_packed(q, k, v, out, lse, layout.tiles, plan, layout.total, layout.caps[-1], False)
    return _forward(q, k, v, plan, layout, out, lse) if done is None else done


def in_a_graph(leaf: torch.Tensor) -> bool:
    """Does an autograd graph hold the leaf's accumulation node?  The leaf itself does not, so that without one the node that is marked here is
    gone when it is looked for again.  (Such a node belongs to the stream that it was made on.  Gradients that a captured backward hands to a node of
    the default stream would have that stream wait inside the capture, which ends the process.)"""
    edge = torch.autograd.graph.get_gradient_edge
    edge(leaf).node.metadata["loopfuse_amd"] = True
    return edge(leaf).node.metadata.pop("loopfuse_amd", False)


def _forward_again(q, k, v, layout, out, lse, low, repeat):
    P = PackedAttnParams.from_buffer_copy(repeat.block)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    P.q, P.k, P.v, P.o = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    if lse is not None:
        P.part_ml = lse.data_ptr()
    if low is not None:
        P.low = low.data_ptr()
    P.tiles = layout.tiles.data_ptr() + repeat.more
    repeat.launches.launch(P)
    lowering._last_launch.set(repeat.record)
    return out


@lowering._on_device_of_first_argument
def _forward(q, k, v, plan, layout, out, lse, low=None):
    lowering._no_tangents(q, k, v)
    dtype, D, Hq, Hkv = _heads(q, k, v, layout)
    mask, window, scale, cap = _constants(plan, layout.total)
    T = layout.total
    for name, t in (("K", k), ("V", v)):
        # direct-to-LDS loads address a sequence, of whatever part of the rows, with unsigned 32-bit byte offsets, up to three tiles past its end
        if _row_stride(t) < 0 or 2 * (T + 192) * _row_stride(t) + 2 * D >= 1 << 32:
            raise UnsupportedPlan(f"{name}: {T} rows of stride {t.stride(0)} are beyond the direct loads' reach")
    if out is not None:
        _rows("O", out, layout, dtype, D)
        if out.shape[1] != Hq or any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
            raise UnsupportedPlan(f"O must be [{T}, {Hq}, {D}], every element with a place of its own")
    if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != (Hq, T) or not lse.is_contiguous() or lse.device != q.device):
        raise UnsupportedPlan(f"lse must be a contiguous float32 [{Hq}, {T}] tensor on the device of Q")
    if T == 0:
        return torch.empty(q.shape, dtype=dtype, device=q.device) if out is None else out
    P = PackedAttnParams()
    P.q_ss, P.q_sh = _row_stride(q), q.stride(1)
    P.k_ss, P.k_sh = _row_stride(k), k.stride(1)
    P.v_ss, P.v_sh = _row_stride(v), v.stride(1)
    P.o_ss, P.o_sh = (Hq * D, D) if out is None else out.stride()[:2]
    P.B, P.Hq, P.Hkv, P.Sq, P.Sk, P.window = 1, Hq, Hkv, T, T, window
    P.scale, P.softcap = scale, cap or 0.0
    P.nsplit, P.rows = 1, 1
    P.clear = int(out is None)
    group = Hq // Hkv
    pack = heads_per_workgroup(group)
    bm, heads = 128 // (pack or 1), Hq // (pack or 1)
    tiles_at, entries = layout.tiles_of(bm, group_size(mask, 64 // heads))
    mean = T // max(1, layout.count)
    spec = lowering._spec("prefill_swp", lowering._DTYPE_CODE[dtype], D, mask, cap is not None, pack=pack, packed=True,
                          bn=lowering.prefill_kv_tile(D, 0, None, heads * (T // bm + layout.count // 2),
                                                      min(mean, window) if mask == lowering.MASK_SLIDING else mean),
                          stay=lowering.prefill_out_stays(2 * T * Hq * D))
    grid = _grid(entries, heads, 256)
    record = {"kernels": [spec.entry()], "grid": grid, "block": 256, "q_tile_rows": bm, "kv_tile_rows": spec.bn or 64, "heads_per_workgroup": pack or 1}
    repeat = lowering._Repeat(P, [(lowering.get_kernel(spec, spec.entry()), (grid, 1, 1), 256)], record, tiles_at)
    key = lowering._call_key("p", (q, k, v, out), (None if low is not None else lse, layout.tiles), plan, (T, layout.caps[-1], low is not None))
    out = _forward_again(q, k, v, layout, out, lse, low, repeat)
    lowering._keep_call(key, repeat, (tiles_at,))
    return out


def group_size(mask: int, causal: int) -> int:
    """Sequences whose tiles come together by their work: under a causal mask ``causal``, so that an XCD has 8 (sequence, head) pairs at a time,
    under a window, where K and V of a tile are few, 8, and 1 without a mask, where all tiles of a sequence are alike.
    Forward, us, 1 / 2 / 4 / 8, 32/8 heads: causal 3 up to 6000 430 / 435 / 422 / 422, 4 of 500 18.2 / 18.2 / 15.8 / 15.9; 32/32 heads 8 up to 2048
    120 / 120 / 127 / 121; window 256 8 up to 2048 55.4 / 56.9 / 54.6 / 52.5, 5 up to 4001 with a softcap 84 / 84 / 83 / 79; unmasked 8 up to 2048 206 /
    214 / 222 / 230.  All backward launches: causal 8 up to 2048, 32/8 466 / 487 / 491 / 430, 32/32 441 / 447 / 452 / 443; 24 up to 1000, D 64, 16/4
    93 / 93 / 94 / 96, 3 up to 4001 305 / 306 / 299 / 299; window 256 286 / 287 / 285 / 281; unmasked 738 / 785 / 790 / 850."""
    return 1 if mask == lowering.MASK_NONE else 8 if mask == lowering.MASK_SLIDING else causal


def heads_per_workgroup(group: int) -> int:
    """Query heads of a group that share a workgroup's K and V, as in ``lowering.attention``.  1 / 2 / 4, us, 32/8 heads: 12 sequences up to 2048
    174 / 167 / 162, 64 up to 300 50 / 42 / 37, window 256 8 up to 2048 74 / 59 / 52."""
    return 4 if group % 4 == 0 else 2 if group % 2 == 0 else 0


@lowering.outside_graphs
def attention_packed_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor, dout: torch.Tensor,
                              plan: AttnPlan, layout: PackedLayout):
    """Gradients of ``attention_packed(q, k, v, plan, layout)``: ``(dq, dk, dv)`` in the operands' dtype, zeros in rows of no
    sequence.  ``o`` and ``lse`` are the forward's output and row log-sum-exp; Q, K, V and dO whose rows are not apart (one row expanded)
    are copied.  As ``lowering.attention_backward``: delta with dQ or in front of it, dK and dV, no atomics."""
    if not isinstance(layout, PackedLayout):
        raise UnsupportedPlan("layout must come from packed_layout")
    return _backward(q, k, v, o, lse, dout, plan, layout)


def rows_apart(t):
    """``t`` or, where rows lie closer than a row is long (one row expanded over all), a copy.  The kernels take what lies behind a sequence's last
    row for zeros, which the ranges of their buffers make of it only where it lies behind that row's last element too."""
    return t if t.dim() != 3 or _row_stride(t) >= t.shape[2] else t.clone(memory_format=torch.contiguous_format)


def _backward(q, k, v, o, lse, dout, plan, layout, low=None):
    done = _host.attention_packed_backward(q, k, v, o, dout, low, lse, layout.tiles, plan, layout.total, layout.caps[-1])
    if done is None:      # (operands with rows that are not apart are of no signature that is kept)
        apart = [rows_apart(t) for t in (q, k, v, dout)]
        if any(a is not b for a, b in zip(apart, (q, k, v, dout))):
            q, k, v, dout = apart
            done = _host.attention_packed_backward(q, k, v, o, dout, low, lse, layout.tiles, plan, layout.total, layout.caps[-1])
    # (False: there was no room for dS)
    return done or _backward_general(q, k, v, o, lse, dout, plan, layout, low, done is None)


def _backward_again(q, k, v, o, lse, dout, layout, low, repeat):
    P = PackedBwdParams.from_buffer_copy(repeat.block)
    dtype, dev = q.dtype, q.device
    dq, dk, dv = torch.empty(q.shape, dtype=dtype, device=dev), torch.empty(k.shape, dtype=dtype, device=dev), torch.empty(k.shape, dtype=dtype, device=dev)
    delta = torch.empty(lse.shape, dtype=torch.float32, device=dev)
    P.q, P.k, P.v, P.o, P.dout = q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), dout.data_ptr()
    P.dq, P.dk, P.dv, P.lse, P.delta = dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), lse.data_ptr(), delta.data_ptr()
    if low is not None:
        P.low = low.data_ptr()
    at = layout.tiles.data_ptr()
    P.dkdv_tiles, P.dq_tiles = at + repeat.more[0], at + repeat.more[1]
    if repeat.more[2]:
        # last: it may take what room is left, which the results need and it does not
        try:
            ds = torch.empty(repeat.more[2], dtype=dtype, device=dev)
        except torch.OutOfMemoryError:
            return None
        P.ds = ds.data_ptr()
    repeat.launches.launch(P)
    lowering._last_launch.set(repeat.record)
    return dq, dk, dv


@lowering._on_device_of_first_argument
def _backward_general(q, k, v, o, lse, dout, plan, layout, low, room=True):
    lowering._no_tangents(q, k, v, o, dout)
    dtype, D, Hq, Hkv = _heads(q, k, v, layout)
    mask, window, scale, cap = _constants(plan, layout.total)
    T, dev = layout.total, q.device
    for name, t in (("O", o), ("dO", dout)):
        _rows(name, t, layout, dtype, D)
        if t.shape[1] != Hq:
            raise UnsupportedPlan(f"{name} must have the shape of Q")
    if lse.dtype != torch.float32 or tuple(lse.shape) != (Hq, T) or not lse.is_contiguous() or lse.device != dev:
        raise UnsupportedPlan(f"lse must be a contiguous float32 [{Hq}, {T}] tensor on the device of Q")
    if low is not None:
        _rows("what rounding took from O", low, layout, dtype, D)
        if low.shape != o.shape or low.stride() != o.stride():
            raise UnsupportedPlan("what rounding took from O must have its shape and strides")
    for name, t in (("Q", q), ("dO", dout), ("K", k), ("V", v)):
        if _row_stride(t) < D or 2 * (T + 64) * _row_stride(t) + 2 * D >= 1 << 32:
            raise UnsupportedPlan(f"{name}: {T} rows of stride {t.stride(0)} are beyond the direct loads' reach")
    if T == 0:
        return tuple(torch.empty(t.shape, dtype=dtype, device=dev) for t in (q, k, v))
    P = PackedBwdParams()
    for name, t in (("q", q), ("k", k), ("v", v), ("o", o), ("do", dout)):
        setattr(P, name + "_ss", _row_stride(t))
        setattr(P, name + "_sh", t.stride(1))
    for name, heads in (("dq", Hq), ("dk", Hkv), ("dv", Hkv)):
        setattr(P, name + "_ss", heads * D)
        setattr(P, name + "_sh", D)
    P.B, P.Hq, P.Hkv, P.Sq, P.Sk, P.window = 1, Hq, Hkv, T, T, window
    P.scale, P.softcap = scale, cap or 0.0
    count = max(1, layout.count)
    mean = max(1, T // count)
    keys = lowering.bwd_key_blocks(D, mask, cap is not None, count * Hkv, mean)
    nt = bwd_dq_threads(D, mask, count * Hq * -(-mean // 256))
    q_split = bwd_q_split(D, mask, Hkv, T, layout.count)
    if q_split:
        keys = 1
    blocks = ds_blocks(mask, window, T, layout.count)
    wants_ds = bwd_keep_ds(D, cap is not None, Hq * blocks)
    keep_ds = room and wants_ds
    rows = 64 if q_split else 128 * keys
    both = bwd_both(D, nt, keep_ds)
    spec = bwd_spec(dtype, D, mask, cap is not None, keys, nt, q_split, lowering.bwd_grads_stay(2 * T * Hq * D), keep_ds, both)
    P.ds_sh = blocks * lowering.BWD_DS_BLOCK
    dkdv_at, dkdv_entries = layout.tiles_of(rows, group_size(mask, 64 // Hkv if Hkv <= 16 else 1))
    dq_at, dq_entries = layout.tiles_of(nt // 2, group_size(mask, 64 // Hkv if Hkv <= 16 else 1))
    steps = {"lf_attn_bwd_delta": (-(-Hq * T // (4096 // D)), 256), "lf_attn_bwd_dkdv": (_grid(dkdv_entries, Hkv, 256), 256),
             "lf_attn_bwd_dq": (_grid(dq_entries, Hq, nt), nt)}
    names = ["lf_attn_bwd_dq", "lf_attn_bwd_dkdv"] if nt == 256 and not keep_ds else list(steps)
    if both:
        P.dkdv_blocks = steps["lf_attn_bwd_dkdv"][0]
        steps["lf_attn_bwd_both"] = _grid(1, P.dkdv_blocks + steps["lf_attn_bwd_dq"][0], 256), 256
        names = ["lf_attn_bwd_delta", "lf_attn_bwd_both"]
    named = lowering._kernels_of(spec)
    launches = [(lowering.get_kernel(spec, name, named), (steps[name][0], 1, 1), steps[name][1]) for name in names]
    repeat = lowering._Repeat(P, launches, {"kernels": names}, (dkdv_at, dq_at, P.ds_sh * Hq if keep_ds else 0))
    res = _backward_again(q, k, v, o, lse, dout, layout, low, repeat)
    if res is None:
        return _backward_general(q, k, v, o, lse, dout, plan, layout, low, False)
    key = lowering._call_key("b", (q, k, v, o, dout, low), (lse, layout.tiles), plan, (T, layout.caps[-1]))
    # an allocation that fails makes the allocator give back what it holds and wait for the device: the form without dS is kept, and room for dS looked
    # for again once in many calls
    lowering._keep_call(key, repeat, (*repeat.more, -1 if keep_ds or not wants_ds else lowering._NO_ROOM_CALLS))
    return res


def bwd_spec(dtype: torch.dtype, D: int, mask: int, softcap: bool = False, key_blocks: int = 1, dq_threads: int = 512, q_split: bool = False,
             stay: bool = False, keep_ds: bool = False, both: bool = False) -> lowering.KernelSpec:
    spec = lowering.bwd_spec(dtype, D, mask, softcap, key_blocks, dq_threads, keep_ds, q_split, stay)
    return dataclasses.replace(spec, packed=True, **({"family": "bwd_both", "extra": spec.extra + ("-DLF_BW_BOTH=1",)} if both else {}))


def bwd_q_split(D: int, mask: int, Hkv: int, total: int, count: int) -> bool:
    """``lowering.bwd_q_split``, and at head dimension 128 under a causal mask up to 320 workgroups of 128 keys instead of 192: sequences of different lengths
    leave the longest chain alone for longer.  us, whole / split: 8 up to 3511, 8/2 heads (254) 554 / 387, 11 up to 1776, 4/4 (248) 93 / 72, 3 up to 2051, 64/8 (264) 666 /
    476, 4 up to 3931, 4/4 (312) 0.77 of the time, 31 up to 183, 32/8 (296) 1.00, 8 up to 171, 64/32 (288) 1.04, 14 of 349, 32/8 (360) 1.07; with a narrow window 0.89 ...
    1.17 from 184 on."""
    if D == 128 and mask == lowering.MASK_CAUSAL:
        return Hkv * (total // 128 + count // 2) <= 320
    return lowering.bwd_q_split(D, mask, max(1, count) * Hkv, max(1, total // max(1, count)))


def bwd_both(D: int, dq_threads: int, keep_ds: bool) -> bool:
    """All gradients in one launch behind delta's (``-DLF_BW_BOTH=1``), where dQ forms dS itself and two workgroups of it and of dK and dV fit a CU (head
    dimension 64)?  The longest chain of tiles of dK and dV is several times the mean where sequences differ or are few, and dQ fills what it leaves empty.  us, dQ then dK and dV /
    delta then all: 24 sequences up to 1000, 16/4 heads 98 / 77, 3 up to 4001, 16/4 304 / 248, 2 up to 4708, 2/1 197 / 121, 5 of 576, 2/2 26 / 17, 28 up to 208, 2/2 17 / 12, 16
    of 300, 32/8 66 / 64, 64 up to 500, 16/16 88 / 91, 8 of 2048, 32/8 588 / 585, 32/32 608 / 616; 35 batches 0.84 of the time in the mean."""
    return D == 64 and dq_threads == 256 and not keep_ds


def bwd_dq_threads(D: int, mask: int, tiles: int) -> int:
    """Workgroup size of lf_attn_bwd_dq (``lowering.bwd_dq_threads``), ``tiles`` = of 256 queries in all heads: 512 threads at head dimension 128
    once all CUs have work, else 256.  All backward launches, us, 512 / 256, recomputed and with dS kept: D 128 causal, 8 sequences up to 2048,
    H32 487 / 523 and 454 / 458, 32/8 505 / 558 and 489 / 482, window 256 343 / 378 and 290 / 299; D 64 24 up to 1000, 16/4 113 / 104, 3 up to 4001 320 / 304,
    with a softcap 110 / 98 and 85 / 83."""
    return 512 if D == 128 and tiles > (256 if mask == lowering.MASK_CAUSAL else 128) else 256


def ds_blocks(mask: int, window: int, total: int, count: int) -> int:
    """Blocks of dS of one head: those in front of a sequence that begins behind the last row (``lf_bw_ds_before`` in
    csrc/kernels/lf_attn_bwd.hip); under a window the blocks in front of the first key that the last row's start leaves out."""
    n = -(-total // 32)
    per = n if mask == lowering.MASK_NONE else (n + 2) // 2 if mask == lowering.MASK_CAUSAL else (window + 30) // 32 + 1
    return (total // 32 + count + 1) * per


def bwd_keep_ds(D: int, softcap: bool, blocks: int) -> bool:
    """Does dS stay in memory between the two product kernels (``lowering.bwd_keep_ds``)?  ``blocks`` = of dS in all that the rows have room
    for, 2 KB each, as if they were one sequence; what the real ones need of them is touched.  Up to 9 GiB, a 32nd of the memory: 16 384 rows
    of 32 heads under a causal mask.  All launches, us, recomputed / kept: D 128 causal, 8 sequences up to 2048, H32 487 / 454, 32/8 505 / 482, 40 up
    to 300, 32/8 150 / 124, window 256 343 / 290, unmasked H16 186 / 170; D 64 with a softcap 98 / 83, without 104 / 103 and 304 / 324."""
    return 2 * lowering.BWD_DS_BLOCK * blocks <= 9 << 30 and (D == 128 or softcap)


def _gradients(ctx, dout):
    q, k, v, out, lse, low = ctx.saved_tensors
    if low.stride() != out.stride():      # (hooks of saved tensors may give them back with strides of their own)
        out, low = (t.clone(memory_format=torch.contiguous_format) for t in (out, low))
    if dout.stride(-1) != 1 or dout.data_ptr() % 16 or any(n > 1 and s % 8 for n, s in zip(dout.shape[:-1], dout.stride()[:-1])):
        dout = dout.contiguous()
    return (*_backward(q, k, v, out, lse, dout, ctx.plan, ctx.layout, low), None, None)


_gradients_once = torch.autograd.function.once_differentiable(_gradients)


class _Packed(torch.autograd.Function):
    """As the fused training graphs: gradients can be asked for with ``create_graph=True`` but not differentiated again.  (Only then do
    they go through the wrapper that says so, which costs 10 us.)"""

    @staticmethod
    def forward(ctx, q, k, v, plan, layout):
        done = _host.attention_packed(q, k, v, None, None, layout.tiles, plan, layout.total, layout.caps[-1], True)
        if done is None:
            _heads(q, k, v, layout)
            lse = torch.empty((q.shape[1], layout.total), dtype=torch.float32, device=q.device)
            low = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            done = _forward(q, k, v, plan, layout, None, lse, low), lse, low
        out, lse, low = done
        ctx.save_for_backward(q, k, v, out, lse, low)
        # (the caller may change a plan)
        ctx.plan = AttnPlan(plan.mask, plan.window, plan.scale, plan.softcap, plan.k_paged, plan.v_paged, plan.denom_add)
        ctx.layout = layout
        return out

    @staticmethod
    def backward(ctx, dout):
        return (_gradients_once if torch.is_grad_enabled() else _gradients)(ctx, dout)


_host = lowering._host()
