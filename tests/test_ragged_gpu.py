"""The operators for requests of different lengths as they are used: together, from graphs, on other streams and threads, over
views, shared and broadcast operands, and over pools beyond 32 bits."""
import math
import threading

import pytest
import torch

from loopfuse_amd import lowering, packed, paged
from loopfuse_amd.lowering import AttnPlan, UnsupportedPlan

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


def rnd(shape, seed, dtype=BF):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def dense(q, k, v, scale, causal, cap=None):
    """[rows, heads, D] of one sequence, in 64 bits; keys in front of the queries are seen by all."""
    g = q.shape[1] // k.shape[1]
    q, k, v = q.double().transpose(0, 1), k.double().transpose(0, 1).repeat_interleave(g, 0), v.double().transpose(0, 1).repeat_interleave(g, 0)
    s = q @ k.transpose(1, 2).contiguous() * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    if causal:
        i = torch.arange(q.shape[1], device=q.device)[:, None] + k.shape[1] - q.shape[1]
        s = s.masked_fill(torch.arange(k.shape[1], device=q.device)[None] > i, -math.inf)
    return (torch.softmax(s, -1) @ v).transpose(0, 1)


def rel(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


# A result's error against 64 bits, relative in the 2-norm: two roundings (probabilities, result) of half a step at most each, 2^-8 for bf16
TOL = 2 * 2.0 ** -8


def test_a_serving_loop_is_attention_over_the_whole_history():
    """Prompts through extend_tables, store_kv and attention_packed, then single tokens through extend_tables, store_kv and
    attention_shared behind a prefix: every result is that of plain attention over the request's tokens so far."""
    Hq, Hkv, D, page, prefix, B = 8, 2, 128, 16, 37, 5
    scale, steps = D ** -0.5, 20
    prompts = [40, 0, 1, 100, 16]          # (request 1 begins with its first single token)
    pool = [torch.full((64, page, Hkv, D), math.nan, dtype=BF, device=DEV) for _ in range(2)]
    free = torch.randperm(64, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(DEV)
    # the prefix in pages of its own, through the same operators
    pk, pv = rnd((prefix, Hkv, D), 1), rnd((prefix, Hkv, D), 2)
    prefix_table = torch.full((1, 3), -1, dtype=torch.int32, device=DEV)
    step = paged.extend_tables(i32([0]), i32([prefix]), prefix_table, free, page, prefix)
    paged.store_kv(pk, pv, *pool, step.slots)
    free = free[int(step.pages):]
    table = torch.full((B, 8), -1, dtype=torch.int32, device=DEV)
    lengths = i32([0] * B)
    history = [(rnd((0, Hkv, D), 0), rnd((0, Hkv, D), 0)) for _ in range(B)]
    total = sum(prompts) + 11              # a padded step
    q, k, v = rnd((total, Hq, D), 3), rnd((total, Hkv, D), 4), rnd((total, Hkv, D), 5)
    step = paged.extend_tables(lengths, i32(prompts), table, free, page, total)
    paged.store_kv(k, v, *pool, step.slots)
    out = packed.attention_packed(q, k, v, AttnPlan("causal", scale=scale), packed.packed_layout(step.offsets, total))
    assert (out[sum(prompts):] == 0).all()
    ends = step.offsets.tolist()
    for b in range(B):
        rows = slice(ends[b], ends[b + 1])
        history[b] = (k[rows], v[rows])
        if prompts[b]:
            assert rel(out[rows], dense(q[rows], k[rows], v[rows], scale, True)) <= TOL
    free, lengths = free[int(step.pages):], step.lengths
    plan = AttnPlan(scale=scale, k_paged=True, v_paged=True)
    for t in range(steps):
        active = [int((b + t) % 4 != 0) for b in range(B)]
        q, k, v = rnd((B, Hq, 1, D), 100 + t), rnd((B, Hkv, D), 200 + t), rnd((B, Hkv, D), 300 + t)
        step = paged.extend_tables(lengths, i32(active), table, free, page, B)
        at = step.offsets.tolist()
        rows_k, rows_v = torch.zeros_like(k), torch.zeros_like(v)
        for b in range(B):
            if active[b]:
                rows_k[at[b]], rows_v[at[b]] = k[b], v[b]
                history[b] = tuple(torch.cat((h, x[b:b + 1])) for h, x in zip(history[b], (k, v)))
        paged.store_kv(rows_k, rows_v, *pool, step.slots)
        free, lengths = free[int(step.pages):], step.lengths
        out = paged.attention_shared(q, *pool, plan, table, lengths, prefix_table=prefix_table[0], prefix_len=prefix)
        for b in range(B):
            hk, hv = torch.cat((pk, history[b][0])), torch.cat((pv, history[b][1]))
            assert rel(out[b].transpose(0, 1), dense(q[b].transpose(0, 1), hk, hv, scale, False)) <= TOL
    assert lengths.tolist() == [len(h[0]) for h in history]


def packed_args(seed, lengths=(70, 5, 200), Hq=4, Hkv=2, D=64):
    T = sum(lengths) + 3
    bounds = [0]
    for n in lengths:
        bounds.append(bounds[-1] + n)
    return rnd((T, Hq, D), seed), rnd((T, Hkv, D), seed + 1), rnd((T, Hkv, D), seed + 2), rnd((T, Hq, D), seed + 3), packed.packed_layout(i32(bounds), T)


def shared_args(seed, lengths=(33, 0, 500, 16), prefix=100, page=16, Hq=16, Hkv=4, D=128):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    B, width, pre = len(lengths), -(-max(lengths) // page), -(-prefix // page)
    ids = torch.randperm(B * width + pre, generator=gen, device=DEV).to(torch.int32)
    return (rnd((B, Hq, 1, D), seed), rnd((len(ids), page, Hkv, D), seed + 1), rnd((len(ids), page, Hkv, D), seed + 2),
            ids[pre:].view(B, width).contiguous(), i32(lengths), ids[:pre].contiguous(), prefix)


def run_shared(a):
    q, kp, vp, table, n, pre, prefix = a
    return paged.attention_shared(q, kp, vp, AttnPlan(scale=0.1, k_paged=True, v_paged=True), table, n, prefix_table=pre, prefix_len=prefix)


def run_train(a):
    q, k, v, g, layout = a
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = packed.attention_packed(*leaves, AttnPlan("causal", scale=0.1), layout)
    return (out.detach(), *torch.autograd.grad(out, leaves, g))


def run_tables(a):
    cached, new, table, free = a
    table = table.clone()
    return (table, *paged.extend_tables(cached, new, table, free, 16, 60))


def run_store(a):
    k, v, kp, vp, slots = a
    kp, vp = kp.clone(), vp.clone()
    paged.store_kv(k, v, kp, vp, slots)
    return kp, vp


FORMS = {
    "packed": (lambda s: packed_args(s), lambda a: (packed.attention_packed(*a[:3], AttnPlan("sliding", window=20, scale=0.1, softcap=9.0), a[4]),)),
    "packed training": (lambda s: packed_args(s, D=128), run_train),
    "layout": (lambda s: (i32([0, 3 + s % 5, 9, 40]),), lambda a: (packed.packed_layout(a[0], 50).tiles,)),
    "shared": (lambda s: shared_args(s), lambda a: (run_shared(a),)),
    "shared, no prefix": (lambda s: shared_args(s, prefix=0), lambda a: (run_shared(a),)),
    "shared, one row": (lambda s: shared_args(s, lengths=(9,), Hq=8, Hkv=8, D=64, page=1), lambda a: (run_shared(a),)),
    "tables": (lambda s: (i32([s % 20, 0, 33]), i32([1, 20, s % 7]), torch.arange(30, dtype=torch.int32, device=DEV).view(3, 10), i32(list(range(40, 60)))), run_tables),
    "store": (lambda s: (rnd((20, 2, 64), s), rnd((20, 2, 64), s + 1), rnd((4, 8, 2, 64), s + 2), rnd((4, 8, 2, 64), s + 3),
                         torch.randperm(32, generator=torch.Generator().manual_seed(s)).to(torch.int32)[:20].to(DEV)), run_store),
}


@pytest.mark.parametrize("form", FORMS)
def test_repeated_captured_and_on_another_stream(form):
    """The launches recorded for a signature give the bits of the general path on tensors that were not there when they were recorded;
    so do a graph's replays, between eager calls of other inputs, and a call on another stream."""
    make, run = FORMS[form]
    run(make(1))
    args, other = make(11), make(21)
    again = run(args)
    paged._host.clear()
    want = run(args)
    assert all(torch.equal(x, y) for x, y in zip(again, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = run(args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(there, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(args)
    for _ in range(4):
        for t in got:
            t.zero_()
        graph.replay()
        run(other)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_a_captured_step_replays_with_other_lengths():
    """One graph of a serving step and of a packed batch: what it replays follows the lengths, new tokens and offsets that its buffers hold then."""
    Hq, Hkv, D, page, B, width = 16, 4, 128, 16, 4, 40
    pool = [rnd((B * width + 38, page, Hkv, D), s) for s in (1, 2)]
    prefix_table = i32(list(range(B * width + 30, B * width + 37)))
    plan = AttnPlan(scale=0.1, k_paged=True, v_paged=True)

    def run(a):
        step = paged.extend_tables(a["cached"], a["new"], a["table"], a["free"], page, 50)
        paged.store_kv(a["k"][:, :Hkv], a["k"][:, Hkv:], *a["pool"], step.slots)
        out = paged.attention_shared(a["q"], *a["pool"], plan, a["table"], step.lengths, prefix_table=prefix_table, prefix_len=100)
        rows = packed.attention_packed(a["k"].repeat(1, 2, 1), a["k"][:, :Hkv], a["k"][:, Hkv:], AttnPlan("causal", scale=0.1),
                                       packed.packed_layout(step.offsets, 50))
        return (*step, out, rows, *a["pool"], a["table"])

    def inputs(cached, new, seed):
        ids = torch.randperm(B * width + 30, generator=torch.Generator().manual_seed(seed)).to(torch.int32).to(DEV)
        return {"cached": i32(cached), "new": i32(new), "table": ids[30:].view(B, width).clone(), "free": ids[:30].clone(), "q": rnd((B, Hq, 1, D), seed), "k": rnd((50, 2 * Hkv, D), seed + 1),
                "pool": [p.clone() for p in pool]}

    steps = [([0, 3, 600, 16], [1, 1, 1, 1]), ([0, 0, 0, 0], [0, 0, 0, 0]), ([100, 20, 0, 33], [0, 50, 0, 0]), ([639, 1, 1, 500], [1, 20, 9, 20]), ([5, 6, 7, 8], [40, 40, 40, 40])]
    wants = [run(inputs(c, n, 10 + i)) for i, (c, n) in enumerate(steps)]
    held = inputs(*steps[0], 10)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(held)
    for i in (3, 1, 4, 0, 2, 3):
        for name, x in inputs(*steps[i], 10 + i).items():
            for to, t in zip(held[name], x) if name == "pool" else ((held[name], x),):
                to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for j, (x, y) in enumerate(zip(got, wants[i])):
            assert torch.equal(x, y), (i, j)


def test_a_captured_call_refuses_leaves_of_a_living_eager_graph():
    q, k, v, g, layout = packed_args(5)
    leaves, plan = [t.requires_grad_(True) for t in (q, k, v)], AttnPlan("causal", scale=0.1)
    eager = packed.attention_packed(*leaves, plan, layout)
    want = torch.autograd.grad(eager, leaves, g, retain_graph=True)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        g.add_(0)
        with pytest.raises(UnsupportedPlan, match="leaves"):
            packed.attention_packed(*leaves, plan, layout)
        padded = [t[..., :40].contiguous().detach().requires_grad_(True) for t in leaves]
        held = [t * 2 for t in padded]
        with pytest.raises(UnsupportedPlan, match="leaves"):
            packed.attention_packed(*padded, plan, layout)
        del held
        with torch.no_grad():
            packed.attention_packed(*leaves, plan, layout)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(packed.attention_packed(*leaves, plan, layout), leaves, g)
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_two_graphs_and_a_larger_eager_call_do_not_share_room():
    """Partial results of captured calls live in the graphs, those of eager calls in a buffer that a larger call replaces."""
    a, b = shared_args(1), shared_args(2, lengths=(700, 3))
    want = [run_shared(x) for x in (a, b)]
    graphs, got = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    torch.cuda.synchronize()
    for g, x in zip(graphs, (a, b)):
        with torch.cuda.graph(g):
            got.append(run_shared(x))
    big = shared_args(3, lengths=(400,) * 60, prefix=1000)
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        run_shared(big)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_threads_share_a_stream():
    args = [shared_args(s, lengths=(100 * s, 7, 300)) for s in range(1, 5)]
    want = [run_shared(a) for a in args]
    bad = []

    def work(a, w):
        for _ in range(20):
            if not torch.equal(run_shared(a), w):
                bad.append(1)

    threads = [threading.Thread(target=work, args=x) for x in zip(args, want)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_threads_on_streams_of_their_own_and_a_cache_that_is_emptied():
    forms = ["packed", "packed training", "shared", "shared, no prefix", "tables", "store"]
    args = {f: [FORMS[f][0](s) for s in (1, 11, 21)] for f in forms}
    want = {f: [FORMS[f][1](a) for a in args[f]] for f in forms}
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream() if i % 2 else torch.cuda.default_stream()
        with torch.cuda.stream(stream):
            for n in range(30):
                f, j = forms[(n + i) % len(forms)], (n * 7 + i) % 3
                got = FORMS[f][1](args[f][j])
                stream.synchronize()
                if not all(torch.equal(x, y) for x, y in zip(got, want[f][j])):
                    bad.append((i, n, f))
                if n % 8 == i:
                    paged._host.clear()
                torch.cuda.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_packed_operands_that_are_views_of_one_projection():
    """Q, K and V as slices of [rows, (Hq + 2 Hkv) D]; an output and a gradient of other strides."""
    lengths, Hq, Hkv, D = (100, 31), 8, 2, 64
    q, k, v, g, layout = packed_args(5, lengths, Hq, Hkv, D)
    plan = AttnPlan("causal", scale=0.1)
    one = torch.cat([t.reshape(len(t), -1) for t in (q, k, v)], 1).requires_grad_(True)
    views = [x.view(len(one), -1, D) for x in one.split((Hq * D, Hkv * D, Hkv * D), 1)]
    out = packed.attention_packed(*views, plan, layout)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want = packed.attention_packed(*leaves, plan, layout)
    assert torch.equal(out, want)
    wide = torch.zeros((len(q), 2 * Hq, D), dtype=BF, device=DEV)
    wide[:, ::2] = g
    grads = torch.autograd.grad(want, leaves, wide[:, ::2])
    got, = torch.autograd.grad(out, one, g.transpose(0, 1).contiguous().transpose(0, 1))
    assert torch.equal(got, torch.cat([t.reshape(len(t), -1) for t in grads], 1))
    head_major = torch.zeros((Hq, len(q), D), dtype=BF, device=DEV).transpose(0, 1)
    packed.attention_packed(q, k, v, plan, layout, out=head_major)
    assert torch.equal(head_major, want)


def test_gradients_of_broadcast_operands_and_of_a_sum():
    """K and V of one head expanded to several (their gradient is the sum over them), an output gradient without memory of its own."""
    q, k, v, _, layout = packed_args(7, (50, 80), 4, 1, 64)
    plan = AttnPlan("causal", scale=0.1)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    packed.attention_packed(leaves[0], leaves[1].expand(-1, 4, -1), leaves[2].expand(-1, 4, -1), plan, layout).sum().backward()
    full = [t.detach().expand(-1, h, -1).contiguous().requires_grad_(True) for t, h in zip((q, k, v), (4, 4, 4))]
    packed.attention_packed(*full, plan, layout).sum().backward()
    assert torch.equal(leaves[0].grad, full[0].grad)
    for a, b in zip(leaves[1:], full[1:]):
        # four gradients of bf16, added up in bf16: half a step, 2^-8, per addition
        total = b.grad.double().sum(1, keepdim=True)
        assert ((a.grad.double() - total).abs() <= 3 * 2.0 ** -8 * b.grad.double().abs().sum(1, keepdim=True) + 1e-30).all()


def test_gradients_are_differences():
    """dQ, dK and dV against central differences of a loss in 64 bits over the oracle's forward, along random directions; fp16, so that what
    the gradients' own roundings add (2^-11 each, two per product) stays below the tolerance."""
    q, k, v, g, layout = packed_args(9, (20, 45), 4, 2, 64)
    q, k, v, g = (t.half() for t in (q, k, v, g))
    grads = run_train((q, k, v, g, layout))[1:]

    def loss(q, k, v):
        return sum((dense(q[a:b], k[a:b], v[a:b], 0.1, True) * g[a:b].double()).sum().item() for a, b in ((0, 20), (20, 65)))

    for i, grad in enumerate(grads):
        d = rnd(grad.shape, 50 + i, torch.float32).double()
        x = [t.double() for t in (q, k, v)]
        ends = []
        for sign in (1, -1):
            y = list(x)
            y[i] = x[i] + sign * 1e-5 * d
            ends.append(loss(*y))
        slope = (ends[0] - ends[1]) / 2e-5
        dot = (grad.double() * d).sum().item()
        assert abs(dot - slope) <= 4 * 2.0 ** -11 * (grad.double().norm() * d.norm()).item()


def test_gradients_are_not_differentiated_again():
    q, k, v, g, layout = packed_args(9)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    plan = AttnPlan("causal", scale=0.1)
    out = packed.attention_packed(*leaves, plan, layout)
    plan.scale = 5.0                                    # the call's plan is the one it was given
    grads = torch.autograd.grad(out, leaves, g, create_graph=True, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(grads, run_train((q, k, v, g, layout))[1:]))
    with pytest.raises(RuntimeError):
        grads[0].float().sum().backward()
    grads = torch.autograd.grad(out, leaves, g.clone().requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grads[0].float().sum().backward()


def test_other_head_dims_are_padded():
    q, k, v, g, layout = packed_args(3, (30, 40), 4, 2, 40)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = packed.attention_packed(*leaves, AttnPlan("causal", scale=0.1), layout)
    assert out.shape == q.shape and out.is_contiguous()
    assert rel(out[:30], dense(q[:30], k[:30], v[:30], 0.1, True)) <= TOL and rel(out[30:70], dense(q[30:70], k[30:70], v[30:70], 0.1, True)) <= TOL
    grads = torch.autograd.grad(out, leaves, g)
    assert all(a.shape == b.shape and torch.isfinite(a).all() for a, b in zip(grads, leaves))


def test_offsets_in_64_bits_beyond_the_rows_and_descending():
    q, k, v, _, _ = packed_args(1, (40, 60), 2, 2, 64)
    plan = AttnPlan("causal", scale=0.1)
    T = len(q)
    want = packed.attention_packed(q, k, v, plan, packed.packed_layout(i32([0, 40, T]), T))
    for offsets in (torch.tensor([0, 40, 1 << 40], device=DEV), torch.tensor([-5, 40, T], device=DEV), i32([0, 40, T + 9]), i32([-1, 40, T])):
        assert torch.equal(packed.attention_packed(q, k, v, plan, packed.packed_layout(offsets, T)), want)
    # descending ones overlap: no result is promised, but nothing outside the tensors is touched and the call ends
    guard = torch.full((T + 64, 2, 64), 3.0, dtype=BF, device=DEV)
    packed.attention_packed(q, k, v, plan, packed.packed_layout(i32([0, 90, 10, 100, 20, T]), T), out=guard[32:32 + T])
    assert (guard[:32] == 3).all() and (guard[32 + T:] == 3).all()
    # no sequence at all
    assert (packed.attention_packed(q, k, v, plan, packed.packed_layout(i32([0]), T)) == 0).all()
    empty = packed.attention_packed(q[:0], k[:0], v[:0], plan, packed.packed_layout(i32([0, 0]), 0))
    assert empty.shape == (0, 2, 64)


def test_many_sequences():
    """More than a block of lf_packed_sort holds, of lengths 0 ... 9, one long one among them."""
    lengths = [(i * 7) % 10 for i in range(1500)]
    lengths[700] = 3000
    q, k, v, _, layout = packed_args(2, tuple(lengths), 2, 1, 64)
    out = packed.attention_packed(q, k, v, AttnPlan("causal", scale=0.1), layout)
    at = 0
    for i, n in enumerate(lengths):
        if n and (i % 50 == 0 or i == 700):
            assert rel(out[at:at + n], dense(q[at:at + n], k[at:at + n], v[at:at + n], 0.1, True)) <= TOL
        at += n
    assert (out[at:] == 0).all() and torch.isfinite(out).all()


def test_dS_is_formed_again_where_there_is_no_room(monkeypatch):
    q, k, v, g, layout = packed_args(4, (300, 100), 4, 4, 128)
    plan, lse = AttnPlan("causal", scale=0.1), torch.empty((4, len(q)), device=DEV)
    o = packed.attention_packed(q, k, v, plan, layout, lse=lse)
    want = packed.attention_packed_backward(q, k, v, o, lse, g, plan, layout)
    assert "lf_attn_bwd_delta" in lowering._last_launch["kernels"]
    real = torch.empty

    def full(*size, **kw):
        if size and isinstance(size[0], int) and size[0] > 1 << 18:      # the scratch of dS: one number
            raise torch.OutOfMemoryError("no room")
        return real(*size, **kw)

    monkeypatch.setattr(torch, "empty", full)
    for _ in range(2):
        paged._host.clear()
        got = packed.attention_packed_backward(q, k, v, o, lse, g, plan, layout)
        assert lowering._last_launch["kernels"] == ["lf_attn_bwd_dq", "lf_attn_bwd_dkdv"]
        # dK and dV keep their bits but for delta, which is summed in another order; dQ its value: products of the same 16-bit dS
        assert all(rel(x, y.double()) <= 2.0 ** -8 for x, y in zip(got, want))


def test_dS_is_formed_again_where_a_repeated_call_has_no_room():
    q, k, v, g, layout = packed_args(4, (4000,), 16, 16, 128)
    plan, lse = AttnPlan("causal", scale=0.1), torch.empty((16, len(q)), device=DEV)
    o = packed.attention_packed(q, k, v, plan, layout, lse=lse)
    for _ in range(2):
        want = packed.attention_packed_backward(q, k, v, o, lse, g, plan, layout)
    assert "lf_attn_bwd_delta" in lowering._last_launch["kernels"]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    # room for the results, 100 MB with those of the call before, and not for 266 MB of dS
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (200 << 20)) / torch.cuda.get_device_properties(0).total_memory)
    try:
        got = [(packed.attention_packed_backward(q, k, v, o, lse, g, plan, layout), lowering._last_launch["kernels"]) for _ in range(2)]
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    for grads, kernels in got:
        assert kernels == ["lf_attn_bwd_dq", "lf_attn_bwd_dkdv"]
        assert all(rel(x, y.double()) <= 2.0 ** -8 for x, y in zip(grads, want))


def test_repeated_calls_are_taken_by_the_host_module(monkeypatch):
    """... for plain operands of a signature that ran before; others, and those under another environment, take the general path to the same bits."""
    paged._host.clear()
    a = shared_args(7)
    want = run_shared(a)
    assert paged._host.size() == 1
    monkeypatch.setattr(paged, "_shared", None)
    assert torch.equal(run_shared(a), want)
    b = shared_args(8)                              # other tensors of the same sizes
    assert torch.equal(run_shared(b), run_shared(b)) and not torch.equal(run_shared(b), want)
    out = torch.empty_like(want)
    monkeypatch.undo()
    plan = AttnPlan(scale=0.1, k_paged=True, v_paged=True)
    given = lambda: paged.attention_shared(*a[:3], plan, *a[3:5], prefix_table=a[5], prefix_len=a[6], out=out)
    assert given() is out and given() is out and torch.equal(out, want)
    size = paged._host.size()
    assert size == 2
    for change in ({"LOOPFUSE_DECODE_COOP": "0"}, {"LOOPFUSE_CHECK_TABLES": "1"}):
        for name, value in change.items():
            monkeypatch.setenv(name, value)
        assert rel(run_shared(a), want.double()) <= TOL
        monkeypatch.undo()
    assert paged._host.size() == size + 1           # (the first of the two is a signature of its own)
    assert torch.equal(run_shared(a), want)
    # a plan that is changed, and one whose fields are no plain numbers
    other = AttnPlan(scale=torch.tensor(0.1), k_paged=True, v_paged=True)
    kept = paged._host.size()
    with torch.inference_mode():
        assert torch.equal(run_shared(a), want)
    assert rel(paged.attention_shared(*a[:3], other, *a[3:5], prefix_table=a[5], prefix_len=a[6]), want.double()) <= TOL
    assert paged._host.size() == kept

    class Sub(torch.Tensor):
        pass

    assert torch.equal(run_shared((a[0].as_subclass(Sub), *a[1:])).as_subclass(torch.Tensor), want) and paged._host.size() == kept


def test_the_parts_of_a_step_are_tensors_of_their_own():
    cached, new = i32([3, 0, 40]), i32([1, 20, 5])
    table, free = torch.zeros((3, 8), dtype=torch.int32, device=DEV), i32(list(range(20)))
    for _ in range(3):
        step = paged.extend_tables(cached, new, table, free, 16, 30)
        assert type(step) is paged.PagedStep and [t.shape[0] for t in step] == [4, 3, 30, 30, 1]
        assert step.offsets.tolist() == [0, 1, 21, 26] and step.lengths.tolist() == [4, 20, 45] and step.pages.tolist() == [2]
        assert all(t.dtype == torch.int32 and t.is_contiguous() and not t.requires_grad for t in step)
        lengths = step.lengths
        before = step.slots.clone()
        lengths += 1
        assert torch.equal(step.slots, before) and (lengths - 1).tolist() == [4, 20, 45]
        assert lengths.storage_offset() == 4 and step.positions[-4:].tolist() == [-1] * 4
        del step
        assert lengths.tolist() == [5, 21, 46]


@pytest.mark.parametrize("mask,window,cap", [("causal", 0, None), ("sliding", 100, None), (None, 0, None), ("causal", 0, 20.0)])
def test_gradients_in_one_launch_by_both_splits(monkeypatch, mask, window, cap):
    """At head dimension 64 all gradients come from one launch; whole keys or queries shared by two waves, dQ keeps its bits and the others differ by the order
    of their sums.  With a softcap, dS formed again."""
    q, k, v, g, layout = packed_args(6, (700, 0, 64, 333, 1, 129), 8, 2, 64)
    plan, lse = AttnPlan(mask, window=window, scale=0.125, softcap=cap), torch.empty((8, len(q)), device=DEV)
    o = packed.attention_packed(q, k, v, plan, layout, lse=lse)
    monkeypatch.setattr(packed, "bwd_keep_ds", lambda *a: False)
    res = []
    for q_split in (False, True):
        monkeypatch.setattr(lowering, "bwd_q_split", lambda *a: q_split)
        paged._host.clear()
        res.append(packed.attention_packed_backward(q, k, v, o, lse, g, plan, layout))
        assert lowering._last_launch["kernels"] == ["lf_attn_bwd_delta", "lf_attn_bwd_both"]
    paged._host.clear()
    assert torch.equal(res[0][0], res[1][0])
    for x, y in zip(*res):
        assert rel(x, y.double()) <= 2.0 ** -8


def test_pools_beyond_32_bits():
    """A pool of 5 GiB whose last pages are used, by stores and by both forms of the prefix."""
    pages, page, Hkv, D = 170_000, 16, 8, 128
    kp, vp = (torch.empty((pages, page, Hkv, D), dtype=BF, device=DEV) for _ in range(2))
    prefix, n = 70, 45
    ids = torch.arange(pages - 1, pages - 9, -1, dtype=torch.int32, device=DEV)
    pre, table = ids[:5].contiguous(), ids[5:8].view(1, 3).contiguous()
    k, v = rnd((prefix + n, Hkv, D), 1), rnd((prefix + n, Hkv, D), 2)
    t = torch.arange(prefix + n, device=DEV)
    slots = torch.where(t < prefix, ids[(t // page).clamp(max=4)] * page + t % page, ids[(5 + (t - prefix) // page).clamp(0, 7)] * page + (t - prefix) % page)
    paged.store_kv(k, v, kp, vp, slots.to(torch.int32))
    assert torch.equal(kp[pages - 1, 3], k[3])
    q = rnd((1, 32, 1, D), 3)
    plan = AttnPlan(scale=0.1, k_paged=True, v_paged=True)
    want = dense(q[0].transpose(0, 1), k, v, 0.1, False)
    for choice in ({"prefix": "tiles"}, {"prefix": "stream"}, None):
        out = paged.attention_shared(q, kp, vp, plan, table, i32([n]), prefix_table=pre, prefix_len=prefix, choice=choice)
        assert rel(out[0].transpose(0, 1), want) <= TOL


def test_rows_of_a_table_far_apart():
    a = shared_args(9, lengths=(40, 90))
    want, wide = run_shared(a), torch.empty(2 ** 31 + 64, dtype=torch.int32, device=DEV)
    far = wide.as_strided((2, a[3].shape[1]), (2 ** 31 + 8, 1))
    far.copy_(a[3])
    for _ in range(2):
        assert torch.equal(run_shared((*a[:3], far, *a[4:])), want)
    table = wide.as_strided((2, 8), (2 ** 31 + 8, 1))
    table.fill_(-1)
    step = paged.extend_tables(i32([0, 20]), i32([17, 13]), table, i32(list(range(5))), 16, 30)
    assert table.tolist() == [[0, 1] + [-1] * 6, [-1, -1, 2] + [-1] * 5] and step.slots[:17].tolist() == list(range(17))


def test_tables_of_v_of_their_own_and_views_of_tables():
    q, kp, vp, table, n, pre, prefix = shared_args(6)
    want = run_shared((q, kp, vp, table, n, pre, prefix))
    order = torch.randperm(len(vp), generator=torch.Generator().manual_seed(2)).to(DEV)
    moved = torch.empty_like(vp)
    moved[order] = vp
    plan = AttnPlan(scale=0.1, k_paged=True, v_paged=True)
    wide = torch.full((2 * len(table), table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    wide[::2, :table.shape[1]] = table
    got = paged.attention_shared(q, kp, moved, plan, wide[::2, :table.shape[1]], n, prefix_table=pre, prefix_len=prefix,
                                 v_table=order[table.long()].to(torch.int32), prefix_v_table=order[pre.long()].to(torch.int32))
    assert torch.equal(got, want)
    # pools stored head by head
    hk, hv = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kp, vp))
    got = paged.attention_shared(q, hk, hv, plan, table, n, prefix_table=pre, prefix_len=prefix)
    assert rel(got, want.double()) <= 2 * TOL
    # lengths beyond the table's room count as that room, below zero as none
    room = table.shape[1] * kp.shape[1]
    full = [int(x) for x in n]
    got = run_shared((q, kp, vp, table, i32([room + 1000, -3, *full[2:]]), pre, prefix))
    assert torch.equal(got, run_shared((q, kp, vp, table, i32([room, 0, *full[2:]]), pre, prefix)))


def test_infinite_and_nan_keys_stay_with_their_request():
    q, kp, vp, table, n, pre, prefix = shared_args(8, prefix=0)
    want = run_shared((q, kp, vp, table, n, pre, prefix))
    bad_k, bad_v = kp.clone(), vp.clone()
    bad_k[table[2, 0].long()] = math.inf
    bad_v[table[2, 1].long()] = math.nan
    got = run_shared((q, bad_k, bad_v, table, n, pre, prefix))
    for b in (0, 1, 3):
        assert torch.equal(got[b], want[b])
    assert torch.isnan(got[2]).any()
    a = packed_args(3, (40, 70, 30), 2, 2, 64)
    clean = run_train(a)
    for t in a[:4]:
        t[40:110] = math.nan
    got = run_train(a)
    for x, y in zip(got, clean):
        assert torch.equal(x[:40], y[:40]) and torch.equal(x[110:], y[110:])


def test_checked_tables(monkeypatch):
    monkeypatch.setenv("LOOPFUSE_CHECK_TABLES", "1")
    q, kp, vp, table, n, pre, prefix = shared_args(4)
    run_shared((q, kp, vp, table, n, pre, prefix))
    bad = table.clone()
    bad[0, 0] = len(kp)
    with pytest.raises(ValueError):
        run_shared((q, kp, vp, bad, n, pre, prefix))
    bad = table.clone()
    bad[1] = -1                                   # a request without keys: its row is not looked at
    run_shared((q, kp, vp, bad, n, pre, prefix))
    with pytest.raises(ValueError):
        run_shared((q, kp, vp, table, n + 10000, pre, prefix))
    with pytest.raises(ValueError):
        packed.packed_layout(i32([0, 5, 3]), 9)
    with pytest.raises(ValueError):
        packed.packed_layout(i32([0, 5, 10]), 9)
    packed.packed_layout(i32([0, 5, 9]), 9)
    k = rnd((2, 4, 128), 1)
    for slots in ([3, 3], [0, len(kp) * 16]):
        with pytest.raises(ValueError):
            paged.store_kv(k, k, kp, vp, i32(slots))
    paged.store_kv(k, k, kp, vp, i32([-1, -1]))
    with pytest.raises(ValueError):
        paged.extend_tables(i32([0]), i32([17]), i32([[0, 0]]), i32([1]), 16, 17)


def test_inside_a_compiled_function():
    q, k, v, _, layout = packed_args(3)
    plan = AttnPlan("causal", scale=0.1)
    fn = torch.compile(lambda q, k, v: packed.attention_packed(q * 2, k, v, plan, layout) + 1)
    assert torch.equal(fn(q, k, v), packed.attention_packed(q * 2, k, v, plan, layout) + 1)
    a = shared_args(2)
    fn = torch.compile(lambda q: run_shared((q + 0, *a[1:])) * 2)
    assert torch.equal(fn(a[0]), run_shared(a) * 2)


def test_refused_again_after_a_call_that_ran():
    q, k, v, _, layout = packed_args(1)
    packed.attention_packed(q, k, v, AttnPlan("causal", scale=0.1), layout)
    for _ in range(2):
        with pytest.raises(UnsupportedPlan):
            packed.attention_packed(q, k, v.half(), AttnPlan("causal", scale=0.1), layout)
        with pytest.raises(UnsupportedPlan):
            packed.attention_packed(q, k, v, AttnPlan("causal", scale=math.nan), layout)
