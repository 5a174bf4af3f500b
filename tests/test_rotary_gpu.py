"""``rotary.rotate_heads``, forward and backward, against the formulas in 64 bits.

Tolerances.  With e the half step of the operands' type (2^-8 bf16, 2^-11 fp16), and what is computed in 32 bits: a rotated element is off by
2^-22 (|z0 c| + |z1 s|) (three roundings of 2^-24 at most), with a norm by 2^-19 of the same, as a row's root mean square is off by less than 2^-20 (256 squares summed by 16 at a time,
their half, 2^-22 for the root) and two products follow; then e |y| for the result and for fp16 half of the least step, 2^-25.  The gradients in the same
way, each step's bound carried on: dz by 2^-22 of its terms, h = dz w, the mean of h n by those of both factors, dx by what its two terms are off by and 2^-18
of their sizes.  dw sums |dz n| (2^-18 each) in 32 bits: a thread some dozens of rows, a workgroup and the parts by halves, 2^-17 of the sum of sizes at most."""
import threading

import pytest
import torch
import torch.utils.checkpoint

from loopfuse_amd import packed, paged, rotary
from loopfuse_amd.lowering import AttnPlan, UnsupportedPlan

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def rnd(shape, seed, dtype=BF):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def halves(t, R, pairs):
    t = t[..., :R]
    return (t[..., 0::2], t[..., 1::2]) if pairs else (t[..., :R // 2], t[..., R // 2:])


def joined(a, b, rest, pairs):
    return torch.cat((torch.stack((a, b), -1).flatten(-2) if pairs else torch.cat((a, b), -1), rest), -1)


def oracle(x, g, positions, table, w, eps, pairs):
    """{"y", "dx", "dw": (value, bound)} for rows x with a gradient g of the result, in 64 bits."""
    e, least = torch.finfo(x.dtype).eps / 2, 2.0 ** -25 if x.dtype == HF else 0.0
    R, D = (0 if table is None else table.shape[1]), x.shape[-1]
    places, positions = 1 << 31 if table is None else table.shape[0], positions.long()
    live = ((positions >= 0) & (positions < places))[:, None, None]
    x, g = torch.where(live, x.double(), 0.0), torch.where(live, g.double(), 0.0)       # (rows of no token may hold anything)
    if R:
        a = table.double()[torch.where(live[:, 0, 0], positions, 0).long()][:, None]
        c, s = a[..., :R // 2], a[..., R // 2:]
    else:
        c = s = x.new_zeros((x.shape[0], 1, 0))
    z, w64 = x, (1.0 if w is None else w.double())
    if eps is not None:
        r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
        n = torch.where(live, x * r, 0.0)
        z = n * w64
    off = 2.0 ** -22 if eps is None else 2.0 ** -19
    z0, z1 = halves(z, R, pairs)
    y = joined(z0 * c - z1 * s, z1 * c + z0 * s, z[..., R:], pairs) * live
    by = off * joined((z0 * c).abs() + (z1 * s).abs(), (z1 * c).abs() + (z0 * s).abs(), z[..., R:].abs(), pairs) + e * y.abs() + least
    g0, g1 = halves(g, R, pairs)
    dz = joined(g0 * c + g1 * s, g1 * c - g0 * s, g[..., R:], pairs) * live
    bz = 2.0 ** -22 * joined((g0 * c).abs() + (g1 * s).abs(), (g1 * c).abs() + (g0 * s).abs(), g[..., R:].abs(), pairs)
    res = {"y": (y, by * live)}
    if eps is None:
        res["dx"] = dz, (bz + e * dz.abs() + least) * live
        return res
    h, bh = dz * w64, bz * abs(w64) + 2.0 ** -23 * (dz * w64).abs()
    m = (h * n).mean(-1, keepdim=True)
    bm = (bh * n.abs() + 2.0 ** -18 * (h * n).abs()).mean(-1, keepdim=True)
    dx = torch.where(live, (h - n * m) * r, 0.0)
    bx = torch.where(live, r * (bh + n.abs() * bm + 2.0 ** -18 * ((n * m).abs() + h.abs())), 0.0)
    res["dx"] = dx, (bx + e * dx.abs() + least) * live
    if w is not None:
        dw, size = (dz * n).sum((0, 1)), (bz * n.abs() + 2.0 ** -18 * (dz * n).abs()).sum((0, 1)) + 2.0 ** -17 * (dz * n).abs().sum((0, 1))
        ew = torch.finfo(w.dtype).eps / 2
        res["dw"] = dw, size + ew * dw.abs() + (least if w.dtype == HF else 0.0)
    return res


def check(got, want, what):
    value, bound = want
    assert not torch.isnan(got).any(), f"{what}: NaN"
    err = (got.double() - value).abs()
    worst = (err - 1.01 * bound).max().item() if err.numel() else 0.0
    assert worst <= 0, f"{what}: {worst} beyond its bound, at an error of {err.max().item()}"


CASES = [
    # rows, query heads, kv heads, D, R (0: no table), type, weights' type ("" without a norm, None a norm without weights), pairs
    (1, 1, 1, 16, 16, BF, "", False),
    (3, 2, 1, 32, 32, HF, HF, True),
    (17, 4, 4, 48, 16, BF, BF, False),
    (70, 5, 3, 80, 80, HF, F32, False),
    (33, 7, 1, 96, 48, BF, F32, True),
    (129, 3, 2, 112, 64, HF, "", True),
    (200, 8, 2, 64, 64, BF, BF, False),
    (65, 32, 8, 128, 128, BF, "", False),
    (257, 6, 6, 128, 32, HF, None, False),
    (41, 4, 2, 256, 256, BF, BF, False),
    (19, 3, 3, 208, 208, HF, F32, True),
    (90, 8, 8, 128, 0, BF, F32, False),
    (1000, 33, 7, 128, 128, BF, F32, False),       # several heads to a thread, some groups of them not full
    (4000, 17, 17, 128, 96, HF, HF, True),
]


def operands(T, Hq, Hkv, D, R, dtype, wtype, seed, views=False):
    if views:       # parts of a fused projection, with the values' behind them
        rows = rnd((T, Hq + 2 * Hkv, D), seed, dtype)
        q, k = rows[:, :Hq], rows[:, Hq:Hq + Hkv]
    else:
        q, k = rnd((T, Hq, D), seed, dtype), 3 * rnd((T, Hkv, D), seed + 1, dtype)
    places = 50
    positions = torch.randint(-3, places + 3, (T,), generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(torch.int32)       # some of no token
    table = rotary.rotary_table(places, R, device=DEV) if R else None
    norm = {}
    if wtype != "":
        norm = {"eps": 1e-3}
        if wtype is not None:
            norm.update(q_weight=(1 + 0.3 * rnd((D,), seed + 2, F32)).to(wtype), k_weight=rnd((D,), seed + 3, F32).to(wtype))
    return q, k, positions, table, norm


@pytest.mark.parametrize("T,Hq,Hkv,D,R,dtype,wtype,pairs", CASES)
def test_rotated_rows_and_their_gradients_are_the_formulas(T, Hq, Hkv, D, R, dtype, wtype, pairs):
    for views in (False, True):
        q, k, positions, table, norm = operands(T, Hq, Hkv, D, R, dtype, wtype, T + D, views)
        if views:       # rows of no token are not looked at
            q[(positions < 0) | (positions >= 50) & bool(R)] = float("nan")
        leaves = [t.requires_grad_() for t in (q.detach(), k.detach(), *(norm[n] for n in ("q_weight", "k_weight") if n in norm))]
        norm.update({n: t for n, t in zip(("q_weight", "k_weight"), leaves[2:])})
        gq, gk = rnd(q.shape, 5, dtype), rnd(k.shape, 6, dtype)
        with torch.no_grad():
            plain = rotary.rotate_heads(leaves[0], leaves[1], positions, table, pairs=pairs, **norm)
        y = rotary.rotate_heads(leaves[0], leaves[1], positions, table, pairs=pairs, **norm)
        grads = torch.autograd.grad(y, leaves, (gq, gk))
        for i, (x, g, name) in enumerate(((q, gq, "q_weight"), (k, gk, "k_weight"))):
            w = norm.get(name)
            want = oracle(x, g, positions, table, None if w is None else w.detach(), norm.get("eps"), pairs)
            check(y[i], want["y"], "y")
            assert torch.equal(y[i], plain[i])
            check(grads[i], want["dx"], "dx")
            if w is not None:
                check(grads[2 + i], want["dw"], "dw")
                assert grads[2 + i].dtype == w.dtype


def test_no_rows_and_rows_of_no_token():
    table, w = rotary.rotary_table(4, 64, device=DEV), rnd((64,), 1, F32).requires_grad_()
    for T, positions in ((0, []), (5, [-1] * 5), (3, [4, 2 ** 31 - 1, -2 ** 31])):
        q, k = rnd((T, 2, 64), 2).fill_(float("nan")).requires_grad_(), rnd((T, 1, 64), 3).requires_grad_()
        y = rotary.rotate_heads(q, k, torch.tensor(positions, dtype=torch.int32, device=DEV), table, q_weight=w, k_weight=w, eps=1e-6)
        grads = torch.autograd.grad(y, (q, k, w), [torch.ones_like(t) for t in y])
        assert all(int(torch.count_nonzero(t)) == 0 for t in (*y, *grads))


def test_weights_of_queries_alone_and_of_both():
    q, k, positions, table, norm = operands(100, 4, 2, 64, 64, BF, F32, 3)
    w = norm["q_weight"].requires_grad_()
    # one of them; the same tensor for both; a view off the borders of 16 bytes
    y = rotary.rotate_heads(q, k, positions, table, q_weight=w, eps=1e-6)
    assert torch.equal(y[1], rotary.rotate_heads(k, k, positions, table, eps=1e-6)[0])
    one = torch.autograd.grad(y, w, [torch.ones_like(t) for t in y])[0]
    y = rotary.rotate_heads(q, k, positions, table, q_weight=w, k_weight=w, eps=1e-6)
    both = torch.autograd.grad(y, w, [torch.ones_like(t) for t in y])[0]
    y = rotary.rotate_heads(q, k, positions, table, k_weight=w, eps=1e-6)
    other = torch.autograd.grad(y, w, [torch.ones_like(t) for t in y])[0]
    assert torch.equal(both, one + other)
    off = torch.cat((w.detach()[:1], w.detach()))[1:]
    assert off.data_ptr() % 16
    assert torch.equal(rotary.rotate_heads(q, k, positions, table, q_weight=off, eps=1e-6)[0], rotary.rotate_heads(q, k, positions, table, q_weight=w.detach(), eps=1e-6)[0])


def test_gradients_of_broadcast_rows_and_of_a_sum():
    """One row expanded over all, and the expanded gradient that a sum gives: those of a copy."""
    _, _, positions, table, norm = operands(30, 4, 2, 64, 32, BF, BF, 4)
    a, b = rnd((1, 4, 64), 1).requires_grad_(), rnd((30, 1, 64), 2).requires_grad_()
    q, k = a.expand(30, 4, 64), b.expand(30, 2, 64)
    y = rotary.rotate_heads(q, k, positions, table, **norm)
    got = torch.autograd.grad(y[0].sum() + y[1].sum(), (a, b))
    q, k = (t.detach().contiguous().requires_grad_() for t in (q, k))
    y = rotary.rotate_heads(q, k, positions, table, **norm)
    dq, dk = torch.autograd.grad(y, (q, k), [torch.ones_like(t) for t in y])
    # (autograd's own sums over the expanded dimension)
    assert torch.equal(got[0], dq.sum(0, keepdim=True)) and torch.equal(got[1], dk.sum(1, keepdim=True))


def test_saved_tensors_that_hooks_lay_out_otherwise():
    q, k, positions, table, norm = operands(70, 4, 2, 64, 64, BF, BF, 8)
    leaves = [t.requires_grad_() for t in (q, k, norm["q_weight"], norm["k_weight"])]
    grads = [rnd(t.shape, 30 + i) for i, t in enumerate((q, k))]
    y = rotary.rotate_heads(q, k, positions, table, **norm)
    want = torch.autograd.grad(y, leaves, grads)

    def apart(t):       # columns of a wider tensor that begins off the borders of 16 bytes
        wide = torch.empty((*t.shape, 3), dtype=t.dtype, device=t.device)
        wide[..., 1] = t.detach()
        return wide[..., 1]

    for unpack in (apart, lambda t: torch.cat((t.detach().flatten()[:1], t.detach().flatten()))[1:].view(t.shape)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = rotary.rotate_heads(q, k, positions, table, **norm)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, grads), want))


def test_results_do_not_change_from_call_to_call():
    q, k, positions, table, norm = operands(3000, 16, 4, 128, 128, BF, F32, 9)
    leaves = [t.requires_grad_() for t in (q, k, norm["q_weight"], norm["k_weight"])]
    runs = []
    for _ in range(3):
        y = rotary.rotate_heads(q, k, positions, table, **norm)
        runs.append((*y, *torch.autograd.grad(y, leaves, [t.detach() for t in y])))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


def test_gradients_are_not_differentiated_again():
    q, k, positions, table, norm = operands(10, 2, 2, 64, 64, BF, BF, 1)
    q.requires_grad_()
    y = rotary.rotate_heads(q, k, positions, table, **norm)
    dq, = torch.autograd.grad(y[0].float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.float().sum(), q)


def test_gradients_of_repeated_calls():
    """The graph's node that repeated calls make gives what the first call's does, and behaves as it in what autograd asks of a node."""
    q, k, positions, table, norm = operands(70, 4, 2, 64, 32, BF, BF, 8)
    leaves = [t.requires_grad_() for t in (q, k, norm["q_weight"], norm["k_weight"])]
    grads = [rnd(t.shape, 30 + i) for i, t in enumerate((q, k))]

    def call(first=False, **change):
        if first:
            rotary._host.clear()
        return rotary.rotate_heads(q, k, positions, table, **{**norm, **change})

    first = call(True)
    want = torch.autograd.grad(first, leaves, grads)
    call(), torch.autograd.grad(call(), leaves, grads)
    y = call()
    assert y[0].grad_fn is y[1].grad_fn and y[0].grad_fn.name() == "RotateHeadsBackward" != first[0].grad_fn.name() and torch.equal(y[0], first[0]) and torch.equal(y[1], first[1])
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, grads, retain_graph=True), want))
    torch.autograd.grad(y, leaves, grads)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaves, grads)
    # one result alone, some of the leaves
    for i in range(2):
        want_i = torch.autograd.grad(call(True)[i], leaves, grads[i], allow_unused=True)
        call(), torch.autograd.grad(call(), leaves, grads)
        got = torch.autograd.grad(call()[i], leaves, grads[i], allow_unused=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want_i))
        got, = torch.autograd.grad(call()[i], leaves[2 + i], grads[i])
        assert torch.equal(got, want[2 + i])
    # without norms nothing of q and k is kept
    want_plain = torch.autograd.grad(rotary.rotate_heads(q, k, positions, table), leaves[:2], grads)
    y = rotary.rotate_heads(q, k, positions, table)
    assert y[0].grad_fn.name() == "RotateHeadsBackward" and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves[:2], grads), want_plain))
    # not differentiated again, though a graph may be asked for
    y = call()
    dq, = torch.autograd.grad(y[0].float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.float().sum(), q)
    # written to meanwhile
    y = call()
    with torch.no_grad():
        q.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, leaves, grads)
    # what hooks give back, in the order of 16 bytes or off it
    for unpack in (lambda t: t.detach().clone(), lambda t: torch.cat((t.detach().flatten()[:1], t.detach().flatten()))[1:].view(t.shape)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = call()
        assert y[0].grad_fn.name() == "RotateHeadsBackward" and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, grads), want))
    # or that are none of them: elsewhere, of another type or shape
    for unpack in (lambda t: t.detach().cpu(), lambda t: t.detach().double(), lambda t: t.detach()[:1], lambda t: t.detach()[None]):
        for again in (False, True):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                y = call(not again)
            rotary._host.clear()
            with pytest.raises((UnsupportedPlan, RuntimeError)):
                torch.autograd.grad(y, leaves, grads)
            call(True), torch.autograd.grad(call(True), leaves, grads)
    assert call()[0].grad_fn.name() == "RotateHeadsBackward"
    # into leaves, on a stream of their own, from threads
    wrong = []

    def run():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = torch.autograd.grad(call(), leaves, grads)
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    wrong.append(got)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    torch.autograd.backward(call(), grads)
    assert all(torch.equal(t.grad, g) for t, g in zip(leaves, want))


def test_repeated_calls_follow_their_operands():
    """Calls of one signature, each with its own operands, on streams of their own and in threads."""
    sets = [operands(64, 8, 2, 128, 128, BF, BF, seed) for seed in range(6)]
    want = [rotary._general(*s[:4], s[4]["q_weight"], s[4]["k_weight"], s[4]["eps"], False) for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def run(s, w):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = rotary.rotate_heads(*s[:4], **s[4])
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, w)):
                    wrong.append(s)

    threads = [threading.Thread(target=run, args=x) for x in zip(sets, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_captured_training_step_replays_with_other_rows():
    q, k, positions, table, norm = operands(300, 8, 2, 128, 64, BF, F32, 2)
    gq, gk = rnd(q.shape, 11), rnd(k.shape, 12)
    leaves = [t.requires_grad_() for t in (q, k, norm["q_weight"], norm["k_weight"])]

    def step():
        y = rotary.rotate_heads(q, k, positions, table, **norm)
        return (*y, *torch.autograd.grad(y, leaves, (gq, gk)))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        with torch.no_grad():
            q.copy_(rnd(q.shape, 20 + i))
            positions.copy_(torch.randint(-1, 50, positions.shape, device=DEV))
        for t in got:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_a_captured_call_refuses_leaves_of_a_living_eager_graph():
    q, k, positions, table, norm = operands(30, 4, 2, 64, 64, BF, BF, 5)
    leaves = [t.requires_grad_() for t in (q, k, norm["q_weight"], norm["k_weight"])]
    for i in range(4):
        eager = leaves[i] * 2
        outside = (leaves[0] * 2, leaves[1]) if i == 0 else (leaves[0], leaves[1])
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            table.add_(0)
            with pytest.raises(UnsupportedPlan, match="leaves"):
                rotary.rotate_heads(*outside, positions, table, **norm)
            with torch.no_grad():
                rotary.rotate_heads(q, k, positions, table, **norm)
        del eager, outside


def test_positions_of_packed_sequences_and_attention_over_rotated_rows():
    """Scores of rotated rows depend on the distance alone: attention over a packed batch gives the same with every position shifted."""
    lengths, D = [40, 0, 1, 100], 64
    offsets = torch.tensor([3, 43, 43, 44, 144], dtype=torch.int32, device=DEV)
    layout = packed.packed_layout(offsets, 150)
    positions = packed.packed_positions(layout)
    assert positions.tolist() == [-1] * 3 + [p for n in lengths for p in range(n)] + [-1] * 6
    table = rotary.rotary_table(5000, D, device=DEV)
    q, k, v = (rnd((150, h, D), h, HF) for h in (4, 2, 2))
    plan = AttnPlan("causal", scale=D ** -0.5)
    out = []
    for shift in (0, 4000):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        rq, rk = rotary.rotate_heads(leaves[0], leaves[1], torch.where(positions < 0, -1, positions + shift).to(torch.int32), table)
        o = packed.attention_packed(rq, rk, leaves[2], plan, layout)
        out.append((o, *torch.autograd.grad(o, leaves, torch.ones_like(o))))
    # roundings of 2^-11 each in rotated rows (twice in a score of size 1 or so), the probabilities, the results and, backwards, the same again
    for a, b in zip(*out):
        assert (a.double() - b.double()).norm() <= 8 * 2.0 ** -11 * a.double().norm()


def test_inside_a_compiled_function():
    q, k, positions, table, norm = operands(40, 4, 2, 64, 64, BF, BF, 6)
    want = rotary.rotate_heads(q * 2, k, positions, table, **norm)
    got = torch.compile(lambda q, k: rotary.rotate_heads(q * 2, k, positions, table, **norm), backend="eager")(q, k)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("eps", [0.0, 1e-50])       # (the second is 0 in 32 bits)
@pytest.mark.parametrize("T,Hq,Hkv,D,R,dtype,wtype,pairs", [(7, 3, 1, 64, 64, BF, BF, False), (300, 5, 8, 128, 0, HF, F32, False), (65, 2, 3, 80, 48, BF, F32, True)])
def test_weights_gradients_without_eps(T, Hq, Hkv, D, R, dtype, wtype, pairs, eps):
    """Rows of no token, odd numbers of heads and the last workgroup's rest add nothing to the weights' gradients, whose norms would divide by zero there."""
    q, k, positions, table, norm = operands(T, Hq, Hkv, D, R, dtype, wtype, T)
    positions[::3] = -1
    norm["eps"] = eps
    leaves = [t.requires_grad_() for t in (q, k, norm["q_weight"], norm["k_weight"])]
    grads = [rnd(t.shape, 40 + i, dtype) for i, t in enumerate((q, k))]
    rotary._host.clear()
    for _ in range(3):       # the general path, then the host module's node
        y = rotary.rotate_heads(q, k, positions, table, pairs=pairs, **norm)
        got = torch.autograd.grad(y, leaves, grads)
        for i, name in enumerate(("q_weight", "k_weight")):
            want = oracle(leaves[i].detach(), grads[i], positions, table, norm[name].detach(), 0.0, pairs)
            check(y[i], want["y"], "y")
            check(got[i], want["dx"], "dx")
            check(got[2 + i], want["dw"], "dw")
    assert y[0].grad_fn.name() == "RotateHeadsBackward"


@pytest.mark.parametrize("power", [-62, -64, -70])
def test_norms_of_rows_whose_squares_are_below_the_least_normal_number(power):
    """Elements of 2^p and -2^p: squares of 2^(2 p), exact in 32 bits, have a mean of the same, and rows are signs after the norm, off by the root's 2^-22, which a
    rounding to 16 bits takes away.  With one element's gradient 1 and the others' 0, dx is 2^-p times (1 - 1 / D) there and the signs' product by -1 / D elsewhere, all exact but for 2^-21,
    which 2^-8 of each covers."""
    D = 64
    sign = torch.where(rnd((5, 2, D), 1, F32) < 0, -1.0, 1.0)
    x = (sign * 2.0 ** power).to(BF).requires_grad_()
    w = torch.ones(D, device=DEV).requires_grad_()
    positions = torch.zeros(5, dtype=torch.int32, device=DEV)
    g = torch.zeros_like(x.detach())
    g[..., 7] = 1
    n = sign.double()
    want = (g.double() - n * n[..., 7:8] / D) * 2.0 ** -power
    for _ in range(2):
        y = rotary.rotate_heads(x, x, positions, None, q_weight=w, eps=0.0)
        assert torch.equal(y[0], sign.to(BF)) and torch.equal(y[1], sign.to(BF))
        dx, dw = torch.autograd.grad(y[0], (x, w), g)
        assert ((dx.double() - want).abs() <= 2.0 ** -8 * want.abs()).all()
        assert ((dw.double() - (g.double() * n).sum((0, 1))).abs() <= 10 * 2.0 ** -20).all()
    pools = [torch.zeros((1, 8, 2, D), dtype=BF, device=DEV) for _ in range(2)]
    slots = torch.arange(5, dtype=torch.int32, device=DEV)
    q = paged.append_kv(x.detach(), x.detach(), x.detach(), *pools, slots, positions, None, eps=0.0)
    assert torch.equal(q, sign.to(BF)) and torch.equal(pools[0][0, :5], sign.to(BF)) and torch.equal(pools[1][0, :5], x.detach())


def test_a_repeated_call_refuses_a_table_that_asks_for_a_gradient():
    q, k, positions, table, norm = operands(30, 4, 2, 64, 64, BF, BF, 5)
    for _ in range(3):       # (the signature of a call does not say whether gradients are asked for)
        want = rotary.rotate_heads(q, k, positions, table, **norm)
    table.requires_grad_()
    for leaf in (None, q):
        if leaf is not None:
            leaf.requires_grad_()
        with pytest.raises(UnsupportedPlan, match="table"):
            rotary.rotate_heads(q, k, positions, table, **norm)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(rotary.rotate_heads(q, k, positions, table, **norm), want))


@pytest.mark.parametrize("norms", [True, False])
@pytest.mark.parametrize("again", [False, True])
def test_a_checkpointed_step_gives_the_gradients_of_a_plain_one(again, norms):
    """What is saved in the forward is matched, one by one, with what the recomputation saves, which a call that is kept since then takes through the host module's node."""
    q, k, positions, table, norm = operands(50, 4, 2, 64, 64, BF, BF, 9)
    norm = norm if norms else {}
    leaves = [t.requires_grad_() for t in (q, k, *(norm[n] for n in ("q_weight", "k_weight") if n in norm))]
    grads = [rnd(t.shape, 30 + i) for i, t in enumerate((q, k))]
    want = torch.autograd.grad(rotary.rotate_heads(q, k, positions, table, **norm), leaves, grads)
    if not again:
        rotary._host.clear()
    for early in (True, False):
        with torch.utils.checkpoint.set_checkpoint_early_stop(early):
            y = torch.utils.checkpoint.checkpoint(lambda q, k: rotary.rotate_heads(q, k, positions, table, **norm), q, k, use_reentrant=False)
            got = torch.autograd.grad(y, leaves, grads)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        if again:       # a recomputation whose call is no longer kept
            y = torch.utils.checkpoint.checkpoint(lambda q, k: rotary.rotate_heads(q, k, positions, table, **norm), q, k, use_reentrant=False)
            rotary._host.clear()
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, grads), want))
