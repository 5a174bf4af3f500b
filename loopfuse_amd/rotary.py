"""Norms of queries and keys for each head and their rotation by position, in one pass, forward and backward.

    table = rotary_table(length, D, device=q.device)                     # once per model
    q, k = rotate_heads(q, k, positions, table, q_weight=wq, k_weight=wk, eps=1e-6)
    o = attention_packed(q, k, v, plan, layout)

``positions`` are those of the tokens in their sequences: ``packed_positions`` of a packed batch, ``PagedStep.positions`` of a serving step
(whose keys and values ``paged.append_kv`` takes into the page pools in the same pass).  The reference has no counterpart: its graphs take queries and keys
as they are (reference README.md:62-99).
"""
from __future__ import annotations

import ctypes
import math
import operator
from typing import Optional

import torch

from . import lowering
from .lowering import UnsupportedPlan

MAX_HEAD_DIM = 256
_ALL = (1 << 31) - 1      # places of a call without a table


class RotateParams(ctypes.Structure):
    """Mirror of ``struct LfRotateParams`` in csrc/kernels/lf_rotate.hip."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "q_out", "k_out", "v_out", "k_scales", "v_scales", "table", "q_weight", "k_weight", "positions", "slots")]
                + [(n, ctypes.c_longlong) for n in ("q_ss", "q_sh", "k_ss", "k_sh", "v_ss", "v_sh", "kp_sb", "kp_ss", "kp_sh", "vp_sb", "vp_ss", "vp_sh",
                                                    "table_stride", "last")]
                + [(n, ctypes.c_int) for n in ("T", "Hq", "Hkv", "D", "R", "places", "q_chunks", "k_chunks", "q_blocks", "k_blocks", "shift", "pairs", "norm", "wide")]
                + [("eps", ctypes.c_float)])


class RotateBwdParams(ctypes.Structure):
    """Mirror of ``struct LfRotateBwdParams`` in csrc/kernels/lf_rotate.hip."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "dq_out", "dk_out", "dq", "dk", "table", "q_weight", "k_weight", "dq_weight", "dk_weight", "parts", "positions")]
                + [(n, ctypes.c_longlong) for n in ("q_ss", "q_sh", "k_ss", "k_sh", "dqo_ss", "dqo_sh", "dko_ss", "dko_sh", "table_stride")]
                + [(n, ctypes.c_int) for n in ("T", "Hq", "Hkv", "D", "R", "places", "q_chunks", "k_chunks", "q_blocks", "k_blocks", "pairs", "norm", "wide")]
                + [("eps", ctypes.c_float)])


def rotary_table(length: int, dim: int, base: float = 10000.0, *, device=None, frequencies: Optional[torch.Tensor] = None) -> torch.Tensor:
    """float32 ``[length, dim]``: of each position the cosines of its ``dim / 2`` angles, then their sines.  Angle i is ``position * base ** (-2 i / dim)``, or
    ``position * frequencies[i]``; formed in 64 bits, as angles of far positions have no digits left in 32.  On ``device``, or where the
    frequencies are."""
    length, dim = operator.index(length), operator.index(dim)
    if length < 0 or dim < 2 or dim % 2:
        raise UnsupportedPlan("a table has 0 positions or more and an even number of rotated elements")
    if frequencies is None:
        frequencies = base ** (torch.arange(dim // 2, dtype=torch.float64, device=device) * (-2.0 / dim))
    elif frequencies.shape != (dim // 2,):
        raise UnsupportedPlan(f"frequencies must be [{dim // 2}]")
    elif device is None:
        device = frequencies.device
    angles = torch.arange(length, dtype=torch.float64, device=device)[:, None] * frequencies.to(device=device, dtype=torch.float64)
    return torch.cat((torch.cos(angles), torch.sin(angles)), 1).float()


def slots_of(D: int) -> int:
    """Threads that share a head's row of D elements, 16 each: a power of two."""
    return 1 << (D // 16 - 1).bit_length()


def kernel_spec(dtype: torch.dtype, D: int, store: int = 0) -> lowering.KernelSpec:
    return lowering._spec("rotate", lowering._DTYPE_CODE[dtype], 16 * slots_of(D), extra=(f"-DLF_ROT_STORE={store}",) if store else ())


def check_operands(q, k, positions, table, q_weight, k_weight, eps, extra=(), plain=False) -> tuple:
    """What ``rotate_heads`` and ``paged.append_kv`` ask of their operands: (T, Hq, Hkv, D, R, weights in 32 bits).  ``extra``: further rows of the
    keys' shape, ``(name, tensor)``; ``plain``: with neither a table nor a norm there is something to do."""
    if not isinstance(q, torch.Tensor) or q.dtype not in lowering._DTYPE_CODE:
        raise UnsupportedPlan("Q must be a bf16 or fp16 tensor")
    for name, t in (("Q", q), ("K", k)) + tuple(extra):
        if not isinstance(t, torch.Tensor) or t.dim() != 3 or t.shape[0] != q.shape[0]:
            raise UnsupportedPlan(f"{name} must be [{q.shape[0] if q.dim() else 'rows'}, heads, D]")
        lowering._check_tensor(name, t, q.dtype)
        if t.device != q.device:
            raise RuntimeError(f"loopfuse_amd: {name} is on {t.device}, Q on {q.device}")
        if name != "Q" and t.shape[1:] != k.shape[1:]:
            raise UnsupportedPlan(f"{name} must have the heads of K")
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    if k.shape[2] != D or D % 16 or not 16 <= D <= MAX_HEAD_DIM or Hq < 1 or Hkv < 1:
        raise UnsupportedPlan(f"head dim must be that of Q and K, a multiple of 16, {MAX_HEAD_DIM} at most")
    if positions is not None:
        if not isinstance(positions, torch.Tensor) or positions.dtype != torch.int32 or tuple(positions.shape) != (T,):
            raise UnsupportedPlan(f"positions must be int32 [{T}]")
        _beside("positions", positions, q)
    R = 0
    if table is not None:
        if not isinstance(table, torch.Tensor) or table.dtype != torch.float32 or table.dim() != 2:
            raise UnsupportedPlan("the table must be float32 [positions, rotated elements]")
        _beside("the table", table, q)
        R = table.shape[1]
        if R % 16 or not 16 <= R <= D or table.stride(1) != 1 or (table.shape[0] > 1 and (table.stride(0) % 4 or table.stride(0) < R)) or table.data_ptr() % 16:
            raise UnsupportedPlan("rows of the table: a multiple of 16 rotated elements, head dim at most, contiguous and apart, on 16-byte borders")
        if table.shape[0] > _ALL:
            raise UnsupportedPlan(f"a table of more than {_ALL} positions")
    weights = [(n, w) for n, w in (("q_weight", q_weight), ("k_weight", k_weight)) if w is not None]
    if eps is None:
        if weights:
            raise UnsupportedPlan("weights are those of norms: they need eps")
        if table is None and not plain:
            raise UnsupportedPlan("neither a table nor a norm")
    elif not (float(eps) >= 0.0) or not math.isfinite(eps):
        raise UnsupportedPlan("eps must be finite, 0 at least")
    for name, w in weights:
        if not isinstance(w, torch.Tensor) or w.dtype not in (q.dtype, torch.float32) or w.dtype != weights[0][1].dtype or tuple(w.shape) != (D,):
            raise UnsupportedPlan(f"{name} must be [{D}], of Q's dtype or float32, both alike")
        _beside(name, w, q)
    if T >= 1 << 31:
        raise UnsupportedPlan("the number of rows must be below 2**31")
    return T, Hq, Hkv, D, R, bool(weights) and weights[0][1].dtype == torch.float32


def _beside(name, t, q) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"loopfuse_amd: {name} is not on the GPU; the HIP path has no CPU fallback")
    if t.device != q.device:
        raise RuntimeError(f"loopfuse_amd: {name} is on {t.device}, Q on {q.device}")


def even_weight(w):
    """A weight that is read 16 bytes at a time."""
    return w if w is None or (w.is_contiguous() and w.data_ptr() % 16 == 0) else w.clone(memory_format=torch.contiguous_format)


def even_rows(t):
    """Rows that are read 16 bytes at a time."""
    unit = 16 // t.element_size() if t is not None else 0
    if t is None or (t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and not any(n > 1 and s % unit for n, s in zip(t.shape[:-1], t.stride()[:-1]))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def grid(T: int, heads: int, D: int) -> tuple:
    """(groups of two heads of a token, workgroups for all tokens')."""
    chunks, groups = -(-heads // 2), 256 // slots_of(D)
    blocks = -(-T * chunks // groups)
    # (the kernels number items, up to the end of the last workgroup, in 32 bits)
    if blocks * groups >= 1 << 32 or blocks * 256 >= 1 << 32:
        raise UnsupportedPlan(f"a launch for {T} rows of {heads} heads of {D} is too large")
    return chunks, blocks


def grids(T: int, Hq: int, Hkv: int, D: int) -> tuple:
    """``grid`` of the queries and of the keys, which one launch has together."""
    (q_chunks, q_blocks), (k_chunks, k_blocks) = grid(T, Hq, D), grid(T, Hkv, D)
    if (q_blocks + k_blocks) * 256 >= 1 << 32:
        raise UnsupportedPlan(f"a launch for {T} rows of {Hq} and {Hkv} heads of {D} is too large")
    return q_chunks, q_blocks, k_chunks, k_blocks


def _checked_positions(positions, places) -> None:
    if lowering._checks_tables() and len(positions) and int(positions.max()) >= places:
        raise ValueError(f"loopfuse_amd: positions must be below {places}")


@lowering.outside_graphs
def rotate_heads(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: Optional[torch.Tensor], *, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: Optional[float] = None, pairs: bool = False) -> tuple:
    """Q and K of new tokens with each head normed and rotated: ``(q, k)``, new contiguous tensors.

    q : ``[rows, Hq, D]``, k : ``[rows, Hkv, D]``, bf16 / fp16 (views will do: parts of a fused projection), D a multiple of 16, 256 at most.
    positions : int32 ``[rows]`` on the GPU, the rows of ``table`` (float32 ``[places, R]``, ``rotary_table``) that tokens are rotated by; below 0, or behind the
    table's last: a row of no token, which comes out as zeros and gives no gradient (``LOOPFUSE_CHECK_TABLES=1`` raises for positions behind the last).
    The first R elements of a head, a multiple of 16, are rotated, element i with i + R / 2, or with ``pairs`` neighbours, 2 i with 2 i + 1; ``table=None``: none.
    eps : with it each head is divided by its root mean square, ``sqrt(mean(x ** 2) + eps)``, and multiplied with ``q_weight`` / ``k_weight``
    (``[D]``, of Q's dtype or float32; none: ones), before the rotation.  Sums and products in 32 bits, rounded once.

    Differentiable in q, k and the weights, as ``packed.attention_packed`` is: once, not forward-mode, and under graph capture not for leaves that another
    autograd graph holds, nor for what a graph made outside the capture computed.  A table
    that asks for a gradient is refused.  Kept for the backward: q and k as given where there is a norm."""
    done = _host.rotate(q, k, table, q_weight, k_weight, positions, eps, bool(pairs), _differentiate)      # (gradients neither under capture nor with tangents)
    if done is not None:
        return done
    operands = [t for t in (q, k, q_weight, k_weight) if isinstance(t, torch.Tensor)]
    if torch.is_grad_enabled() and isinstance(table, torch.Tensor) and table.requires_grad:
        raise UnsupportedPlan("no gradient of the table is formed")
    if torch.is_grad_enabled() and any(t.requires_grad for t in operands):
        from . import packed
        packed.refuse_outside_capture(operands, "Q, K and the weights")
        lowering._no_tangents(*operands, table)      # (not to be seen inside)
        return _Rotate.apply(q, k, _given(positions), table, q_weight, k_weight, eps, bool(pairs))
    return _general(q, k, positions, table, q_weight, k_weight, eps, bool(pairs))


def _forward(q, k, positions, table, q_weight, k_weight, eps, pairs):
    done = _host.rotate_heads(q, k, table, q_weight, k_weight, positions, eps, pairs)
    return _general(q, k, positions, table, q_weight, k_weight, eps, pairs) if done is None else done


def _given(positions):
    if positions is None:
        raise UnsupportedPlan("positions must be given")
    return positions


@lowering._on_device_of_first_argument
def _general(q, k, positions, table, q_weight, k_weight, eps, pairs):
    lowering._no_tangents(q, k, table, q_weight, k_weight)
    T, Hq, Hkv, D, R, wide = check_operands(q, k, _given(positions), table, q_weight, k_weight, eps)
    if T:
        _checked_positions(positions, table.shape[0] if table is not None else _ALL)
    P = params(q, k, table, T, Hq, Hkv, D, R, wide, eps, pairs)
    if T == 0:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)
    spec = kernel_spec(q.dtype, D)
    repeat = lowering._Repeat(P, [(lowering.get_kernel(spec, spec.entry()), (P.q_blocks + P.k_blocks, 1, 1), 256)], {"kernels": [spec.entry()]})
    even = positions.contiguous(), even_weight(q_weight), even_weight(k_weight)
    res = _forward_again(q, k, even[0], table, *even[1:], repeat)
    if all(a is b for a, b in zip(even, (positions, q_weight, k_weight))):
        lowering._keep_call(lowering._call_key("r", (q, k, table, q_weight, k_weight), (positions,), None, (eps, pairs)), repeat, ())
    return res


def params(q, k, table, T, Hq, Hkv, D, R, wide, eps, pairs) -> RotateParams:
    """The parameter block of a call, its pointers and what it stores still to be set."""
    P = RotateParams()
    P.q_ss, P.q_sh, P.k_ss, P.k_sh = *q.stride()[:2], *k.stride()[:2]
    P.T, P.Hq, P.Hkv, P.D, P.R, P.pairs, P.norm, P.wide = T, Hq, Hkv, D, R, int(pairs), int(eps is not None), int(wide)
    P.eps = 0.0 if eps is None else float(eps)
    P.places, P.table_stride = (table.shape[0], table.stride(0)) if table is not None else (_ALL, 0)
    P.q_chunks, P.q_blocks, P.k_chunks, P.k_blocks = grids(T, Hq, Hkv, D)
    return P


def _forward_again(q, k, positions, table, q_weight, k_weight, repeat):
    P = RotateParams.from_buffer_copy(repeat.block)
    q_out, k_out = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    P.q, P.k, P.q_out, P.k_out, P.positions = q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), positions.data_ptr()
    set_tables(P, table, q_weight, k_weight)
    repeat.launches.launch(P)
    lowering._last_launch.set(repeat.record)
    return q_out, k_out


def set_tables(P, table, q_weight, k_weight) -> None:
    for name, t in (("table", table), ("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None:
            setattr(P, name, t.data_ptr())


def _backward(dq_out, dk_out, q, k, positions, table, q_weight, k_weight, eps, pairs, sums):
    """Gradients of q and k, and where the ``sums`` say so of q_weight and k_weight; q and k none without a norm."""
    done = _host.rotate_backward(dq_out, dk_out, q, k, table, q_weight, k_weight, positions, eps, pairs, *sums)
    return _backward_general(dq_out, dk_out, q, k, positions, table, q_weight, k_weight, eps, pairs, sums) if done is None else done


@lowering._on_device_of_first_argument
def _backward_general(dq_out, dk_out, q, k, positions, table, q_weight, k_weight, eps, pairs, sums):
    lowering._no_tangents(dq_out, dk_out)
    given = dq_out, dk_out, q, k, table, q_weight, k_weight, positions
    # (hooks of saved tensors may give them back laid out otherwise, or as something else)
    dq_out, dk_out, q, k = (even_rows(t) for t in given[:4])
    table, q_weight, k_weight, positions = even_rows(table), even_weight(q_weight), even_weight(k_weight), positions.contiguous()
    saved = (q, k) if eps is not None else (dq_out, dk_out)
    check_operands(*saved, positions, table, q_weight, k_weight, eps)
    T, Hq, D = dq_out.shape
    Hkv, dev, dtype = dk_out.shape[1], dq_out.device, dq_out.dtype
    for t, g in zip(saved, (dq_out, dk_out)):
        if t.shape != g.shape or t.dtype != g.dtype or t.device != g.device:
            raise UnsupportedPlan("gradients must be of the results' shape and dtype, with Q and K")
    weights, sizes = [w for w in (q_weight, k_weight) if w is not None], grids(T, Hq, Hkv, D)
    dq, dk = (torch.empty(t.shape, dtype=dtype, device=dev) for t in (dq_out, dk_out))
    dw = [torch.empty(D, dtype=weights[0].dtype, device=dev) if x else None for x in sums]
    if T == 0:
        return dq, dk, *(None if w is None else w.zero_() for w in dw)
    P = RotateBwdParams()
    if eps is not None:
        P.q_ss, P.q_sh, P.k_ss, P.k_sh = *q.stride()[:2], *k.stride()[:2]
    P.dqo_ss, P.dqo_sh, P.dko_ss, P.dko_sh = *dq_out.stride()[:2], *dk_out.stride()[:2]
    P.T, P.Hq, P.Hkv, P.D, P.R, P.pairs, P.norm = T, Hq, Hkv, D, 0 if table is None else table.shape[1], int(pairs), int(eps is not None)
    P.wide, P.eps = int(bool(weights) and weights[0].dtype == torch.float32), 0.0 if eps is None else float(eps)
    P.places, P.table_stride = (table.shape[0], table.stride(0)) if table is not None else (_ALL, 0)
    P.q_chunks, P.q_blocks, P.k_chunks, P.k_blocks = sizes
    if any(sums):
        P.q_blocks, P.k_blocks = min(P.q_blocks, BWD_BLOCKS), min(P.k_blocks, BWD_BLOCKS)
    spec = kernel_spec(dtype, D)
    floats = (P.q_blocks + P.k_blocks) * D if any(sums) else 0
    steps = [(lowering.get_kernel(spec, "lf_rotate_bwd"), (P.q_blocks + P.k_blocks, 1, 1), 256)]
    if any(sums):
        steps.append((lowering.get_kernel(spec, "lf_rotate_dw"), (D // 16, 2, 1), 256))
    repeat = lowering._Repeat(P, steps, {"kernels": [x.symbol for x, _, _ in steps]})
    if floats:
        parts = torch.empty(floats, dtype=torch.float32, device=dev)
        P.parts = parts.data_ptr()
    P.dq_out, P.dk_out, P.dq, P.dk, P.positions = dq_out.data_ptr(), dk_out.data_ptr(), dq.data_ptr(), dk.data_ptr(), positions.data_ptr()
    if eps is not None:
        P.q, P.k = q.data_ptr(), k.data_ptr()
    set_tables(P, table, q_weight, k_weight)
    for name, w in zip(("dq_weight", "dk_weight"), dw):
        if w is not None:
            setattr(P, name, w.data_ptr())
    repeat.launches.launch(P)
    lowering._last_launch.set(repeat.record)
    if all(a is b for a, b in zip(given, (dq_out, dk_out, q, k, table, q_weight, k_weight, positions))):
        lowering._keep_call(lowering._call_key("R", (dq_out, dk_out, q, k, table, q_weight, k_weight), (positions,), None, (eps, pairs, *sums)), repeat, (floats,))
    return dq, dk, *dw


# Workgroups that sum the weights' gradients, of the queries and of the keys: few leave some memory idle, many more parts to add.  us, 256 / 512 / 1024 / 2048, 32/8 heads of 128, both
# launches: 4096 rows 33 / 28 / 29 / 32, 8192 58 / 47 / 48 / 51, 16384 111 / 98 / 98 / 96; 8192 of 32/32, 512 / 1024, 90 / 82.
BWD_BLOCKS = 1024


def _gradients(ctx, dq_out, dk_out):
    q, k, positions, table, q_weight, k_weight = ctx.saved_tensors
    dq, dk, dqw, dkw = _backward(dq_out, dk_out, q, k, positions, table, q_weight, k_weight, ctx.eps, ctx.pairs, (q_weight is not None and ctx.needs_input_grad[4], k_weight is not None and ctx.needs_input_grad[5]))
    return dq, dk, None, None, dqw, dkw, None, None


_gradients_once = torch.autograd.function.once_differentiable(_gradients)
_backward_once = torch.autograd.function.once_differentiable(lambda ctx, dq_out, dk_out, rest: _backward(dq_out, dk_out, *rest))


def _differentiate(dq_out, dk_out, q, k, table, q_weight, k_weight, positions, eps, pairs, of_q_weight, of_k_weight):
    """As ``_gradients``, for the host module's own node."""
    return _backward_once(None, dq_out, dk_out, (q, k, positions, table, q_weight, k_weight, eps, pairs, (of_q_weight, of_k_weight)))


class _Rotate(torch.autograd.Function):
    """As ``packed._Packed``: gradients can be asked for with ``create_graph=True`` but not differentiated again."""

    @staticmethod
    def forward(ctx, q, k, positions, table, q_weight, k_weight, eps, pairs):
        positions, q_weight, k_weight = positions.contiguous(), even_weight(q_weight), even_weight(k_weight)
        out = _forward(q, k, positions, table, q_weight, k_weight, eps, pairs)
        kept = (q, k) if eps is not None else (None, None)
        ctx.save_for_backward(*kept, positions, table, q_weight, k_weight)
        ctx.eps, ctx.pairs = eps, pairs
        return out

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        return (_gradients_once if torch.is_grad_enabled() else _gradients)(ctx, dq_out, dk_out)


_host = lowering._host()
