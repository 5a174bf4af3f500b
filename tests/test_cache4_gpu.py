"""Page pools in 4 bits: what rows become in them, appends with norms and rotation, reads, and attention over them, against plain implementations in
Python and the formulas in 64 bits.

Tolerance of an attention result, e the half step of the type (2^-8 bf16, 2^-11 fp16), over the values that the pools stand for (which read_kv gives, and a plain
implementation tests): e (P |V|) for the probabilities, which are rounded for the second product, and e |O| for the result; besides, in 32 bits, a
probability is off by 2^-17 scale |Q| |K| (128 products) + 2^-20 of itself, with a softcap by 2^-19 cap more (its tanh is off by 2^-22), and the sums by 2^-17 of the sizes of
their terms.  A result below bf16's least normal number is off by half of the least step, 2^-134.  fp16: half of the least step, 2^-25, per probability relative to the largest, and per key and value in 4 bits that is below the least normal number."""
import math
import threading

import pytest
import torch

from loopfuse_amd import lowering, packed, paged, rotary
from loopfuse_amd.lowering import AttnPlan
from loopfuse_amd.paged import Pool4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def rnd(shape, seed, dtype=BF):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---- what rows become ----------------------------------------------------------------------------------------

def plain4(block, most):
    """32 numbers in 4 bits: the least power of two of which the largest is below the 7-fold, each to the nearest value, ties to the even code."""
    if any(math.isnan(x) or math.isinf(x) for x in block):
        return [math.nan] * 32
    top, e = max(abs(x) for x in block), -127
    while top >= 7 * 2.0 ** e and e < most:
        e += 1
    res = []
    for x in block:
        y = min(abs(x) / 2.0 ** e, 6.0)
        d = [abs(y - v) for v in GRID]
        near = [i for i in range(8) if d[i] == min(d)]
        res.append(math.copysign(GRID[near[0] if len(near) == 1 or near[0] % 2 == 0 else near[1]] * 2.0 ** e, x))
    return res


def special(dtype):
    most = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).tiny
    blocks = [[0.0] * 32, [-0.0] * 31 + [1.0], [x / 8 for x in range(-16, 16)], [x / 4 for x in range(32)], [7.0 * 2 ** -3] + [x / 64 for x in range(31)],
              [6.96875 if dtype == BF else 6.996] + [x / 4 for x in range(31)], [3.5] + [0.25, 0.75, 1.25, 1.75, 2.5] * 6 + [-3.5], [most] + [x * most / 32 for x in range(31)],
              [-most] * 32, [tiny] * 16 + [-tiny / 2] * 16, [tiny / 64] + [0.0] * 31, [math.inf] + [1.0] * 31, [1.0] * 31 + [-math.inf], [1.0] * 16 + [math.nan] + [2.0] * 15,
              [1000.0] + [1.0] * 31, [3.0, -5.0, 0.2, -0.24, 0.26, 0.74, 0.76] + [1.1] * 25]
    return torch.tensor(blocks, dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_in_4_bits_are_the_nearest_values(dtype, D):
    blocks = torch.cat((special(dtype), rnd((48, 32), 1, dtype).cpu(), (rnd((32, 32), 2, F32) * torch.exp(3 * rnd((32, 1), 3, F32))).to(dtype).cpu()))
    heads = 3
    rows = blocks.reshape(-1, D)
    rows = rows[:rows.shape[0] // heads * heads].reshape(-1, heads, D)
    T = rows.shape[0]
    k, v = rows.to(DEV), rows.flip(0).contiguous().to(DEV)
    kp, vp = (paged.pool4(3, 16, heads, D, dtype, DEV) for _ in range(2))
    slots = torch.randperm(48, generator=torch.Generator().manual_seed(D))[:T].to(torch.int32).to(DEV)
    paged.store_kv(k, v, kp, vp, slots)
    got = paged.read_kv(kp, vp, slots)
    for g, x in zip(got, (k, v)):
        want = torch.tensor([plain4(b, 125 if dtype == BF else 13) for b in x.reshape(-1, 32).double().tolist()], dtype=torch.float64).reshape(x.shape).to(dtype)
        assert torch.equal(torch.isnan(g.cpu()), torch.isnan(want)) and torch.equal(torch.nan_to_num(g.cpu()), torch.nan_to_num(want))
    # places of no row hold what they held: zeros
    rest = torch.tensor(sorted(set(range(48)) - set(slots.tolist())), dtype=torch.int32, device=DEV)
    assert all(int(torch.count_nonzero(t)) == 0 for t in paged.read_kv(kp, vp, rest))
    # what is held stays when it is stored again
    again = [paged.pool4(3, 16, heads, D, dtype, DEV) for _ in range(2)]
    paged.store_kv(*got, *again, slots)
    for a, b in zip(paged.read_kv(*again, slots), got):
        assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


def test_reads_of_slots_that_are_none_and_of_one_slot_twice():
    for pools in ([paged.pool4(4, 32, 2, 128, HF, DEV) for _ in range(2)], [rnd((4, 32, 2, 128), i, HF) for i in range(2)], [rnd((128, 2, 40), i, BF)[:, :, ::1] for i in range(2)]):
        if isinstance(pools[0], Pool4):
            paged.store_kv(rnd((128, 2, 128), 1, HF), rnd((128, 2, 128), 2, HF), *pools, torch.arange(128, dtype=torch.int32, device=DEV))
        every = paged.read_kv(*pools, torch.arange(128, dtype=torch.int32, device=DEV))
        if not isinstance(pools[0], Pool4):
            assert all(torch.equal(a, b.reshape(a.shape)) for a, b in zip(every, pools))
        slots = [5, -1, 127, 128, 5, 2 ** 31 - 1, -2 ** 31, 0]
        for got, x in zip(paged.read_kv(*pools, i32(slots)), every):
            want = torch.stack([x[s] if 0 <= s < 128 else torch.zeros_like(x[0]) for s in slots])
            assert torch.equal(got, want)


# ---- append_kv -------------------------------------------------------------------------------------------------

APPEND = [
    # rows, query heads, kv heads, D, R, pages, page, type, weights' type ("": no norm), pairs
    (1, 1, 1, 64, 64, 1, 16, BF, "", False),
    (37, 4, 2, 128, 64, 3, 32, HF, HF, True),
    (100, 7, 3, 64, 16, 9, 16, BF, F32, False),
    (300, 32, 8, 128, 128, 5, 64, BF, BF, False),
    (65, 3, 1, 80, 48, 70, 1, HF, F32, False),
    (50, 2, 2, 256, 256, 8, 8, BF, "", True),
    (2000, 32, 8, 128, 128, 130, 16, HF, "", False),
    (2500, 40, 16, 64, 64, 40, 64, BF, BF, False),
    (64, 5, 1, 64, 0, 4, 16, BF, BF, False),
]


@pytest.mark.parametrize("T,Hq,Hkv,D,R,pages,page,dtype,wtype,pairs", APPEND)
def test_appends_are_rotations_and_stores(T, Hq, Hkv, D, R, pages, page, dtype, wtype, pairs):
    gen = torch.Generator(device=DEV).manual_seed(T + D)
    rows = rnd((T, Hq + 2 * Hkv, D), T, dtype)            # views of a fused projection
    q, k, v = rows[:, :Hq], rows[:, Hq:Hq + Hkv], rows[:, Hq + Hkv:]
    places = 40
    table = rotary.rotary_table(places, R, device=DEV) if R else None
    norm = {} if wtype == "" else {"eps": 1e-5, "q_weight": (1 + 0.3 * rnd((D,), 1, F32)).to(wtype), "k_weight": (1 + 0.3 * rnd((D,), 2, F32)).to(wtype)}
    positions = torch.randint(-2, places + (2 if R else 0), (T,), generator=gen, device=DEV).to(torch.int32)
    slots = torch.randperm(max(pages * page, T), generator=gen, device=DEV)[:T].to(torch.int32)       # some behind the last
    slots[::7] = -1
    live = (positions >= 0) & (positions < (places if R else 1 << 30))
    if R or norm:
        want_q, want_k = rotary.rotate_heads(q, k, positions, table, pairs=pairs, **norm)
    else:
        want_q, want_k = torch.where(live[:, None, None], q, 0.0).to(dtype), k
    kept = torch.where(live, slots, -1).to(torch.int32)
    kinds = ["16", "4"] if D in (64, 128) and page >= 16 else ["16"]
    for kind in kinds:
        if kind == "16":      # a layer's pools among others', token-major and one behind the other
            shape = (pages, page, Hkv, D) if page > 1 else (pages, Hkv, D)
            layers = [rnd((3, *shape), 5 + i, dtype) for i in range(2)]
            pools, other = [x[1] for x in layers], [x.clone()[1] for x in layers]
        else:
            layers = [torch.randint(0, 126, (3, pages, Hkv, page // 16, n), generator=gen, device=DEV).to(torch.uint8) for n in (8 * D, D // 2) for _ in range(2)]
            pools = [Pool4(layers[i][1], layers[2 + i][1], dtype) for i in range(2)]
            other = [Pool4(layers[i].clone()[1], layers[2 + i].clone()[1], dtype) for i in range(2)]
        before = [x.clone() for x in layers]
        got = paged.append_kv(q, k, v, *pools, slots, positions, table, pairs=pairs, **norm)
        assert torch.equal(got, want_q)
        paged.store_kv(want_k, v, *other, kept)
        for a, b in zip(pools, other):
            for x, y in ((a, b),) if kind == "16" else ((a.codes, b.codes), (a.scales, b.scales)):
                assert torch.equal(x, y)
        for x, y in zip(layers, before):      # the other layers are as they were
            assert torch.equal(x[0], y[0]) and torch.equal(x[2], y[2])
        if kind == "16":                       # (stores are tested against plain loops elsewhere; here against one)
            flat, old = pools[0].reshape(-1, Hkv, D), before[0][1].reshape(-1, Hkv, D).clone()
            at = [(s, t) for t, s in enumerate(kept.tolist()) if 0 <= s < pages * page]
            for s, t in at:
                old[s] = want_k[t]
            assert torch.equal(flat, old)


def test_stores_into_few_and_many_heads():
    for T, Hkv, D, page in ((5, 1, 64, 16), (3, 48, 128, 16), (700, 2, 64, 64), (9000, 8, 128, 32)):
        k, v = rnd((T, Hkv, D), T, HF), rnd((T, Hkv, D), T + 1, HF)
        pools = [paged.pool4(-(-T // page), page, Hkv, D, HF, DEV) for _ in range(2)]
        slots = torch.randperm(-(-T // page) * page, device=DEV)[:T].to(torch.int32)
        paged.store_kv(k, v, *pools, slots)
        for got, x in zip(paged.read_kv(*pools, slots), (k, v)):
            # an element's error in units of its block's power of two, of which the largest has 3.5 ... 7: up to 4 half of the step below, 0.5 at most (a seventh of 3.5);
            # between 4 and 6 half of the step of 2, 1 at most, at 5, where the largest is 5 at least: a fifth of it; beyond 6 what it has more, below 1 (a seventh)
            top = x.double().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
            assert ((got.double() - x.double()).unflatten(-1, (-1, 32)).abs() <= top / 5 + 2.0 ** -24).all()


# ---- attention_cached ------------------------------------------------------------------------------------------

def batch(lengths, new, page, Hkv, D, dtype, seed, table_dtype=torch.int32, before=0, behind=0, width=None, spare=3, big=False):
    """Pools, table, lengths, offsets and positions of requests whose new tokens come last; what no request has holds NaN."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    width = width or max(1, *need)
    pages = sum(need) + spare
    ids = torch.randperm(pages, generator=gen, device=DEV)
    table = torch.full((len(lengths), width), -1, dtype=table_dtype, device=DEV)
    slots, at = [], 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    pools = []
    for i in range(2):
        pool = paged.pool4(pages, page, Hkv, D, dtype, DEV)
        pool.scales.fill_(255)
        pool.codes.fill_(0x77)
        pools.append(pool)
    ends = torch.tensor(lengths, device=DEV)
    tok = torch.arange(width * page, device=DEV)
    slots = torch.where(tok < ends[:, None], table.long()[:, tok // page] * page + tok % page, -1)
    slots = slots[slots >= 0].to(torch.int32)
    k = torch.randn((len(slots), Hkv, D), generator=gen, device=DEV)
    k = (k * torch.exp(0.8 * torch.randn((1, Hkv, D), generator=gen, device=DEV))).to(dtype)        # columns of different sizes
    v = torch.randn((len(slots), Hkv, D), generator=gen, device=DEV).to(dtype)
    paged.store_kv(k, v, *pools, slots)
    offsets, positions = [before], [-1] * before
    for n, m in zip(lengths, new):
        offsets.append(offsets[-1] + m)
        positions += range(n - m, n)
    return pools, table, i32(lengths), i32(offsets), i32(positions + [-1] * behind)


def oracle(q, pools, plan, table, lengths, offsets, positions, dtype):
    T, Hq, D = q.shape
    page, Hkv = pools[0].shape[1:3]
    g, e = Hq // Hkv, torch.finfo(dtype).eps / 2
    least = 2.0 ** -25 if dtype == HF else 0.0
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    ends = offsets.tolist()
    room = table.shape[1] * page
    for b, n in enumerate(lengths.tolist()):
        lo, hi, n = ends[b], ends[b + 1], min(n, room)
        if lo == hi or n <= 0:
            continue
        t = torch.arange(n, device=q.device)
        k, v = (x.double() for x in paged.read_kv(*pools, (table[b].long()[t // page] * page + t % page).to(torch.int32)))
        p = positions[lo:hi].long()[:, None]
        hidden = (p < 0).expand(hi - lo, n)
        if plan.mask is not None:
            hidden = hidden | (t > p)
        if plan.mask == "sliding":
            hidden = hidden | (p - t >= plan.window)
        blind = hidden.all(-1)
        for h in range(Hkv):
            qh = q[lo:hi, h * g:(h + 1) * g].double().transpose(0, 1)                # [g, rows, D]
            s = qh @ k[:, h].t().contiguous() * plan.scale
            if plan.softcap:
                s = plan.softcap * torch.tanh(s / plan.softcap)
            w = torch.softmax(s.masked_fill(hidden, -math.inf), -1).masked_fill(blind[:, None], 0.0)
            er = e + 2.0 ** -17 * plan.scale * (qh.abs() @ k[:, h].abs().t().contiguous()) + 2.0 ** -20 + (2.0 ** -19 * plan.softcap if plan.softcap else 0.0)
            o = w @ v[:, h]
            out[lo:hi, h * g:(h + 1) * g] = o.transpose(0, 1)
            x = (w * (2 * er - e + 2.0 ** -17) + least * ~hidden) @ v[:, h].abs() + e * o.abs() + (2 * least or 2.0 ** -134)
            bound[lo:hi, h * g:(h + 1) * g] = x.transpose(0, 1) * ~blind[:, None, None]
    return out, 1.01 * bound


def check(got, want, what="out"):
    value, bound = want
    assert not torch.isnan(got).any(), f"{what}: NaN"
    err = (got.double() - value).abs()
    worst = (err - bound).max().item()
    assert worst <= 0, f"{what}: {worst} beyond its bound, at an error of {err.max().item()}"


CACHED = [
    # lengths, new tokens, page, Hkv, group, D, type, mask, window, softcap
    ([1], [1], 16, 1, 1, 64, BF, "causal", 0, None),
    ([0], [0], 16, 2, 2, 128, HF, "causal", 0, None),
    ([17, 0, 16, 1, 33], [1, 0, 1, 1, 1], 16, 8, 4, 128, BF, "causal", 0, None),
    ([1000, 500], [1, 1], 16, 8, 4, 128, BF, "causal", 0, None),
    ([4000, 1, 2100], [1, 1, 1], 64, 2, 8, 128, HF, "causal", 0, 30.0),
    ([9000], [1], 16, 1, 16, 64, BF, None, 0, None),
    ([300, 5, 77], [5, 5, 5], 16, 4, 4, 64, HF, "sliding", 40, 20.0),
    ([3000, 2500, 7], [3, 1, 7], 32, 3, 3, 64, BF, "sliding", 1000, None),
    ([50, 60, 3], [50, 20, 3], 16, 2, 4, 128, BF, "causal", 0, None),           # a whole prompt among them
    ([700, 300], [200, 300], 64, 2, 4, 128, HF, "causal", 0, None),             # rows of their own for the waves
    ([1500, 129, 40], [129, 129, 40], 16, 4, 1, 64, BF, None, 0, 15.0),
    ([2000, 2000], [128, 127], 16, 1, 8, 128, BF, "sliding", 100, None),
    ([90 + 7 * i for i in range(150)], [1 + i % 3 for i in range(150)], 16, 2, 2, 64, HF, "causal", 0, None),       # more than 64 requests
    ([40 * (i % 5) for i in range(131)], [min(1, i % 5) for i in range(131)], 16, 1, 40, 128, BF, "causal", 0, None),
    ([20000, 33], [30, 33], 64, 1, 1, 128, BF, "causal", 0, None),
    ([64] * 70, [1] * 70, 16, 16, 1, 64, BF, "causal", 0, None),
    ([500, 400], [40, 17], 16, 1, 5, 64, HF, "causal", 0, None),
]


@pytest.mark.parametrize("lengths,new,page,Hkv,group,D,dtype,mask,window,cap", CACHED)
def test_attention_over_a_cache_is_the_formula(lengths, new, page, Hkv, group, D, dtype, mask, window, cap, monkeypatch):
    before, behind = (2, 5) if len(lengths) % 2 else (0, 0)
    pools, table, n, offsets, positions = batch(lengths, new, page, Hkv, D, dtype, len(lengths) + D, torch.int64 if page == 64 and D == 128 else torch.int32, before, behind)
    T = before + sum(new) + behind
    q = rnd((T, Hkv * group + 1, D), 3, dtype)[:, 1:]          # (a view)
    plan = AttnPlan(mask, window, D ** -0.5, cap, True, True)
    want = oracle(q, pools, plan, table, n, offsets, positions, dtype)
    out = paged.attention_cached(q, *pools, plan, table, n, offsets, positions)
    check(out, want)
    assert torch.equal(out, paged.attention_cached(q, *pools, plan, table, n, offsets, positions))        # the repeated call
    if set(new) == {1} and not before:         # the same without offsets, and without positions
        assert torch.equal(out, paged.attention_cached(q, *pools, plan, table, n))
        assert torch.equal(out, paged.attention_cached(q, *pools, plan, table, n, None, positions))
    # an output that is given: rows of no request stay
    wide = torch.full((T, 2 * Hkv * group, D), 7.0, dtype=dtype, device=DEV)
    given = wide[:, ::2]
    assert paged.attention_cached(q, *pools, plan, table, n, offsets, positions, out=given) is given
    inside = slice(before, before + sum(new))
    assert torch.equal(given[inside], out[inside]) and bool((wide[:, 1::2] == 7).all()) and bool((given[:before] == 7).all()) and bool((given[before + sum(new):] == 7).all())
    # other shares, and other builds
    for choice in ((97, 3, 5), (1, 0, 1), None):
        for build in ((1, False), (2, False), (2, True)):
            monkeypatch.setattr(paged, "cached_build", lambda *a: build)
            monkeypatch.setattr(paged, "cached_shares", lambda units, *a: choice or (units, -1, 1))
            paged._host.clear()
            check(paged.attention_cached(q, *pools, plan, table, n, offsets, positions), want, f"{choice} {build}")
    monkeypatch.undo()
    paged._host.clear()


def test_lengths_that_tables_have_no_room_for_and_rows_of_no_token():
    pools, table, n, offsets, positions = batch([70, 40, 64], [3, 2, 1], 16, 2, 64, BF, 1, width=5)
    plan = AttnPlan("causal", 0, 0.125, None, True, True)
    q = rnd((6, 4, 64), 2)
    short = table[:, :4]                                      # room for 64 keys: the first request's last 6 are left out
    n = i32([70, -5, 64])                                      # (and a length below 0 is none)
    positions = i32([67, -1, 69, 38, 39, 63])
    out = paged.attention_cached(q, *pools, plan, short, n, offsets, positions)
    want = oracle(q, pools, plan, short, n, offsets, positions, BF)
    check(out, want)
    assert int(torch.count_nonzero(out[1])) == 0 and int(torch.count_nonzero(out[3:5])) == 0
    assert int(torch.count_nonzero(paged.attention_cached(q, *pools, plan, table[:, :0], n, offsets, positions))) == 0
    # a pool without a page has none
    empty = [Pool4(p.codes[:0], p.scales[:0], p.dtype) for p in pools]
    assert int(torch.count_nonzero(paged.attention_cached(q, *empty, plan, table, n, offsets, positions))) == 0


@pytest.mark.parametrize("D,dtype,group", [(128, BF, 4), (64, HF, 20)])
def test_many_keys_pass_the_caches_by(D, dtype, group):
    """Requests that share their pages count as if each had its own: 64 of 4100 keys are beyond the 128 MB from which codes are loaded so."""
    B, Hkv = 64 if D == 128 else 128, 8
    pools, table, n, _, _ = batch([4100], [1], 16, Hkv, D, dtype, 3)
    assert B * (4100 // 32 * Hkv) * 34 * D > 128 << 20
    table, n = table.expand(B, -1).contiguous(), n.expand(B).contiguous()
    q, plan = rnd((B, Hkv * group, D), 4, dtype), AttnPlan("causal", 0, 0.1, None, True, True)
    positions, offsets = torch.full((B,), 4099, dtype=torch.int32, device=DEV), i32(range(B + 1))
    out = paged.attention_cached(q, *pools, plan, table, n, offsets, positions)
    assert "lf_cached_combine" in lowering._last_launch["kernels"]
    check(out, oracle(q, pools, plan, table, n, offsets, positions, dtype))


@pytest.mark.parametrize("build", [(1, False), (2, False), (2, True)])
def test_rows_of_no_token_in_front_of_others_in_a_window(build, monkeypatch):
    monkeypatch.setattr(paged, "cached_build", lambda *a: build)
    pools, table, n, offsets, positions = batch([700, 90], [6, 3], 16, 2, 64, BF, 5)
    plan = AttnPlan("sliding", 100, 0.1, None, True, True)
    q = rnd((9, 4, 64), 2)
    for none in (-1, -2 ** 31, -2 ** 31 + 50):
        positions[0] = positions[6] = positions[7] = none
        out = paged.attention_cached(q, *pools, plan, table, n, offsets, positions)
        check(out, oracle(q, pools, plan, table, n, offsets, positions, BF), f"{none} {build}")
        assert int(torch.count_nonzero(out[0])) == 0 and int(torch.count_nonzero(out[6:8])) == 0


def test_offsets_that_descend_stay_within_the_rows_and_the_room():
    """Offsets that are none (they say of more rows than there are): numbers come out, and nothing beside O and the parts is written."""
    pools, table, n, _, _ = batch([5000] * 6, [1] * 6, 16, 2, 64, BF, 1)
    T, plan = 40, AttnPlan("causal", 0, 0.1, None, True, True)
    q, positions = rnd((T, 4, 64), 1), torch.full((T,), 4999, dtype=torch.int32, device=DEV)
    for offsets in ([0, 40, 0, 40, 0, 40, 0], [-5, 60, 20, 10, 50, 30, 20], [40, 30, 20, 10, 5, 3, 0], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 0, 2 ** 31 - 1, -1, 40]):
        out = torch.zeros((T + 2, 4, 64), dtype=BF, device=DEV)
        paged.attention_cached(q, *pools, plan, table, n, i32(offsets), positions, out=out[1:-1])
        assert int(torch.count_nonzero(out[0])) == 0 and int(torch.count_nonzero(out[-1])) == 0


@pytest.mark.parametrize("D,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("build", [(1, False), (2, False), (2, True)])
def test_nan_in_places_that_a_row_does_not_see_stays_there(D, dtype, build, monkeypatch):
    """A key and a value that are NaN, each in one block of a token, over rows some of which see the token: causal, behind a window, and alone."""
    monkeypatch.setattr(paged, "cached_build", lambda *a: build)
    paged._host.clear()
    for mask, window in (("causal", 0), ("sliding", 20)):
        for bad in (3, 30, 58, 61):
            pools, table, n, offsets, positions = batch([64], [8], 16, 1, D, dtype, bad)
            q, plan = rnd((8, 2, D), 4, dtype), AttnPlan(mask, window, D ** -0.5, None, True, True)
            want = oracle(q, pools, plan, table, n, offsets, positions, dtype)
            sees = [bad <= p and (mask == "causal" or p - bad < window) for p in range(56, 64)]
            slot = int(table[0, bad // 16]) * 16 + bad % 16
            k, v = paged.read_kv(*pools, i32([slot]))
            for which in ("v", "k"):
                bk, bv = k.clone(), v.clone()
                (bv if which == "v" else bk)[0, 0, 37] = math.inf
                paged.store_kv(bk, bv, *pools, i32([slot]))
                out = paged.attention_cached(q, *pools, plan, table, n, offsets, positions)
                for r in range(8):
                    block = out[r, :, 32:64]
                    if which == "k":
                        block = out[r]
                    rest = torch.cat((out[r, :, :32], out[r, :, 64:]), -1) if which == "v" else out[r, :, :0]
                    assert bool(torch.isnan(block).all()) == sees[r] and not torch.isnan(rest).any()
                    if not sees[r]:
                        assert ((out[r].double() - want[0][r]).abs() <= want[1][r]).all()
                paged.store_kv(k, v, *pools, i32([slot]))
    paged._host.clear()


def test_queries_that_are_infinite_or_nan_stay_with_their_rows():
    pools, table, n, offsets, positions = batch([40, 50], [3, 1], 16, 2, 128, BF, 1)
    q, plan = rnd((4, 4, 128), 4), AttnPlan("causal", 0, 0.1, None, True, True)
    want = paged.attention_cached(q, *pools, plan, table, n, offsets, positions)
    bad = q.clone()
    bad[1, 2, 5], bad[3, 0, 70] = math.nan, math.inf
    got = paged.attention_cached(bad, *pools, plan, table, n, offsets, positions)
    hit = torch.zeros((4, 4), dtype=torch.bool, device=DEV)
    hit[1, 2] = hit[3, 0] = True
    assert bool(torch.isnan(got[hit]).all()) and torch.equal(got[~hit], want[~hit])


def test_peaked_rows_and_keys_with_a_few_large_columns():
    """Scores far apart, and sums of large terms that cancel: what is cut off a sum would show here."""
    for dtype, D in ((BF, 128), (HF, 64)):
        pools, table, n, offsets, positions = batch([600, 90], [2, 1], 16, 2, D, dtype, 5)
        slots = torch.cat([(table[b].long()[torch.arange(m, device=DEV) // 16] * 16 + torch.arange(m, device=DEV) % 16) for b, m in enumerate(n.tolist())]).to(torch.int32)
        k, v = paged.read_kv(*pools, slots)
        k[:, :, 3] = 200 + k[:, :, 3]
        k[:, :, 40] = 200 + k[:, :, 40]
        paged.store_kv(k, v, *pools, slots)
        q = rnd((3, 8, D), 6, dtype)
        q[:, :, 40] = -q[:, :, 3]
        for scale in (D ** -0.5, 4.0):
            plan = AttnPlan("causal", 0, scale, None, True, True)
            check(paged.attention_cached(q, *pools, plan, table, n, offsets, positions), oracle(q, pools, plan, table, n, offsets, positions, dtype))


def test_pools_beyond_32_bits():
    """Pages whose codes and scales lie more than 4 GiB behind the pool's first."""
    page, Hkv, D = 64, 8, 128
    pages = (9 << 29) // (Hkv * page * D // 2)                   # 4.5 GiB of codes
    kp, vp = (Pool4(torch.empty((pages, Hkv, page // 16, 8 * D), dtype=torch.uint8, device=DEV), torch.empty((pages, Hkv, page // 16, D // 2), dtype=torch.uint8, device=DEV), BF) for _ in range(2))
    last = [pages - 1, 3, pages - 7, pages // 2]
    table, n = i32([last]), i32([250])
    slots = torch.cat([torch.arange(page, device=DEV) + p * page for p in last])[:250].to(torch.int32)
    k, v = rnd((250, Hkv, D), 1), rnd((250, Hkv, D), 2)
    table_of, positions = rotary.rotary_table(300, D, device=DEV), torch.arange(250, dtype=torch.int32, device=DEV)
    q = paged.append_kv(rnd((250, 16, D), 3), k, v, kp, vp, slots, positions, table_of)
    small = [paged.pool4(4, page, Hkv, D, BF, DEV) for _ in range(2)]
    low = torch.arange(250, dtype=torch.int32, device=DEV)
    paged.append_kv(q, k, v, *small, low, positions, table_of)
    assert all(torch.equal(a, b) for a, b in zip(paged.read_kv(kp, vp, slots), paged.read_kv(*small, low)))
    plan = AttnPlan("causal", 0, D ** -0.5, None, True, True)
    got = paged.attention_cached(q[-1:], kp, vp, plan, table, n)
    assert torch.equal(got, paged.attention_cached(q[-1:], *small, plan, i32([[0, 1, 2, 3]]), n))
    offsets = i32([0, 250])
    got = paged.attention_cached(q, kp, vp, plan, table, n, offsets, positions)
    assert torch.equal(got, paged.attention_cached(q, *small, plan, i32([[0, 1, 2, 3]]), n, offsets, positions))


def serve(kind, steps, plan, table_of, norm, prompts, Hq, Hkv, D, page, streams=None):
    """Prompts and then single and several tokens at a time through extend_tables, append_kv and attention_cached: [(rows, positions, request of each row, output)], the cache."""
    B = len(prompts)
    pools = [paged.pool4(64, page, Hkv, D, BF, DEV) for _ in range(2)]
    free = torch.randperm(64, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(DEV)
    table, cached, out = torch.full((B, 12), -1, dtype=torch.int32, device=DEV), i32([0] * B), []
    for i in range(steps):
        new = i32(prompts) if i == 0 else i32([1 + (b + i) % 3 if kind == "several" else 1 for b in range(B)])
        total = int(new.sum()) + 3                  # a padded step
        step = paged.extend_tables(cached, new, table, free, page, total)
        qkv = rnd((total, Hq + 2 * Hkv, D), 100 + i)
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        q = paged.append_kv(q, k, v, *pools, step.slots, step.positions, table_of, **norm)
        o = paged.attention_cached(q, *pools, plan, table, step.lengths, step.offsets, step.positions)
        out.append((qkv, step, o, q))
        free, cached = free[int(step.pages):], step.lengths
    return out, pools, table, cached


@pytest.mark.parametrize("kind", ["one", "several"])
def test_a_serving_loop_is_attention_over_the_whole_history(kind):
    Hq, Hkv, D, page = 8, 2, 128, 16
    prompts = [40, 0, 1, 100, 16]
    table_of = rotary.rotary_table(400, D, device=DEV)
    norm = {"eps": 1e-6, "q_weight": 1 + 0.2 * rnd((D,), 1, F32), "k_weight": 1 + 0.2 * rnd((D,), 2, F32)}
    plan = AttnPlan("causal", 0, D ** -0.5, None, True, True)
    out, pools, table, cached = serve(kind, 12, plan, table_of, norm, prompts, Hq, Hkv, D, page)
    history = [[] for _ in prompts]
    for qkv, step, o, q in out:
        ends, places = step.offsets.tolist(), step.positions.tolist()
        for b in range(len(prompts)):
            lo, hi = ends[b], ends[b + 1]
            assert places[lo:hi] == list(range(len(history[b]), len(history[b]) + hi - lo))
            for t in range(lo, hi):
                history[b].append((qkv[t, Hq:Hq + Hkv], qkv[t, Hq + Hkv:], step.positions[t:t + 1]))
        # the queries are those of rotate_heads, the output the formula over what the cache holds
        want_q, _ = rotary.rotate_heads(qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], step.positions, table_of, **norm)
        assert torch.equal(q, want_q)
        want = oracle(q, pools, plan, table, step.lengths, step.offsets, step.positions, BF)      # (later keys are hidden by the mask)
        check(o, want)
        assert int(torch.count_nonzero(o[ends[-1]:])) == 0
    # the cache holds each request's keys and values, rotated by their positions, in 4 bits
    for b, rows in enumerate(history):
        if not rows:
            continue
        k, v, p = (torch.cat([r[i][None] if i < 2 else r[i] for r in rows]) for i in range(3))
        _, k = rotary.rotate_heads(k, k, p, table_of, **norm)
        pair = [paged.pool4(-(-len(rows) // 16), 16, Hkv, D, BF, DEV) for _ in range(2)]
        at = torch.arange(len(rows), dtype=torch.int32, device=DEV)
        paged.store_kv(k, v, *pair, at)
        slots = (table[b].long()[at.long() // page] * page + at % page).to(torch.int32)
        assert all(torch.equal(x, y) for x, y in zip(paged.read_kv(*pools, slots), paged.read_kv(*pair, at)))


def test_a_captured_step_replays_with_other_lengths():
    """One graph over extend_tables, append_kv and attention_cached of a padded batch; between replays the program's own eager work."""
    Hq, Hkv, D, page, B, total = 8, 2, 64, 16, 4, 12
    plan, table_of = AttnPlan("sliding", 60, D ** -0.5, 20.0, True, True), rotary.rotary_table(5000, D, device=DEV)
    pools = [paged.pool4(300, page, Hkv, D, BF, DEV) for _ in range(2)]
    cached, new, table, free = i32([0] * B), i32([0] * B), torch.full((B, 40), -1, dtype=torch.int32, device=DEV), i32(range(300))
    qkv = rnd((total, Hq + 2 * Hkv, D), 1)

    def step(to):
        s = paged.extend_tables(cached, new, table, free, page, total)
        q = paged.append_kv(qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], *to, s.slots, s.positions, table_of, eps=1e-6)
        return paged.attention_cached(q, *to, plan, table, s.lengths, s.offsets, s.positions), s

    step(pools)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, s = step(pools)
    lengths = [0] * B
    for i in range(8):
        fresh = [(i + b) % 5 if i % 3 else 3 for b in range(B)]
        fresh = [min(f, 3) for f in fresh]
        cached.copy_(i32(lengths))
        new.copy_(i32(fresh))
        free.copy_(torch.roll(free, -int(s.pages)) if i else free)
        qkv.copy_(rnd(qkv.shape, 50 + i))
        got.zero_()
        copy = [Pool4(p.codes.clone(), p.scales.clone(), p.dtype) for p in pools]
        old = table.clone()
        graph.replay()
        torch.cuda.synchronize()
        done = table.clone()
        table.copy_(old)
        want, ws = step(copy)
        assert torch.equal(got, want) and torch.equal(done, table) and all(torch.equal(a, b) for a, b in zip(s, ws))
        assert all(torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) for a, b in zip(pools, copy))
        lengths = ws.lengths.tolist()


def test_two_graphs_and_a_larger_eager_call_do_not_share_room():
    plan = AttnPlan("causal", 0, 0.1, None, True, True)
    sets = []
    for seed, lengths in ((1, [5000, 300]), (2, [4000, 2500, 1]), (3, [6000] * 5)):
        pools, table, n, offsets, positions = batch(lengths, [2] * (len(lengths) - 1) + [1], 16, 2, 64, HF, seed)
        sets.append((rnd((len(positions), 8, 64), seed, HF), *pools, plan, table, n, offsets, positions))
    want = [paged.attention_cached(*a) for a in sets]
    torch.cuda.synchronize()
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g, a in zip(graphs, sets):
        with torch.cuda.graph(g):
            got.append(paged.attention_cached(*a))
    side = torch.cuda.Stream()
    for _ in range(4):
        for t in got:
            t.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        eager = paged.attention_cached(*sets[2])
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(eager, want[2])


def test_threads_on_one_stream_and_on_streams_of_their_own():
    plan, sets = AttnPlan("causal", 0, 0.1, None, True, True), []
    for seed in range(4):
        pools, table, n, offsets, positions = batch([4000, 2500 - seed], [1, 2], 16, 2, 128, BF, seed)
        sets.append((rnd((3, 8, 128), seed), *pools, plan, table, n, offsets, positions))
    want = [paged.attention_cached(*a) for a in sets]
    torch.cuda.synchronize()
    wrong = []

    def run(a, w, own):
        with torch.cuda.stream(torch.cuda.Stream() if own else torch.cuda.default_stream()):
            got = [paged.attention_cached(*a) for _ in range(30)]
            torch.cuda.current_stream().synchronize()
        wrong.extend(1 for x in got if not torch.equal(x, w))

    for own in (False, True):
        threads = [threading.Thread(target=run, args=(*x, own)) for x in zip(sets, want)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert not wrong


def test_repeated_calls_are_taken_by_the_host_module(monkeypatch):
    pools, table, n, offsets, positions = batch([300, 200], [1, 2], 16, 2, 128, BF, 1)
    rows = [torch.randn((2, 2, 128), device=DEV).to(BF) for _ in range(2)]
    plan, a = AttnPlan("causal", 0, 0.1, None, True, True), rnd((3, 8, 128), 1)
    kp, vp = rnd((4, 16, 2, 128), 1), rnd((4, 16, 2, 128), 2)
    table_of = rotary.rotary_table(100, 128, device=DEV)
    calls = [lambda: paged.attention_cached(a, *pools, plan, table, n, offsets, positions), lambda: paged.read_kv(*pools, positions), lambda: paged.read_kv(kp, vp, positions),
             lambda: paged.append_kv(a, a[:, :2], a[:, 2:4], kp, vp, positions, positions, table_of), lambda: paged.store_kv(*rows, *pools, n),
             lambda: rotary.rotate_heads(a, a, positions, table_of)]
    first = [c() for c in calls]

    def refuse(*a, **kw):
        raise AssertionError("the general path")

    for module, name in ((paged, "_cached"), (paged, "_read"), (paged, "_append"), (rotary, "_general")):
        monkeypatch.setattr(module, name, refuse)
    for c, f in zip(calls, first):
        again = c()
        for x, y in zip(again if isinstance(again, tuple) else (again,), f if isinstance(f, tuple) else (f,)):
            assert (x is None and y is None) or x.shape == y.shape
    # a pool of the other type is another call
    half = Pool4(pools[0].codes, pools[0].scales, HF)
    with pytest.raises(AssertionError, match="general"):
        paged.attention_cached(a, half, pools[1], plan, table, n, offsets, positions)
    with pytest.raises(AssertionError, match="general"):
        paged.store_kv(*rows, half, pools[1], n)
    monkeypatch.setenv("LOOPFUSE_CHECK_TABLES", "1")
    for c in calls:
        with pytest.raises(AssertionError, match="general"):
            c()


def test_checked_tables(monkeypatch):
    monkeypatch.setenv("LOOPFUSE_CHECK_TABLES", "1")
    pools, table, n, offsets, positions = batch([300, 200], [1, 2], 16, 2, 128, BF, 1)
    plan, q = AttnPlan("causal", 0, 0.1, None, True, True), rnd((3, 8, 128), 1)
    want = oracle(q, pools, plan, table, n, offsets, positions, BF)
    check(paged.attention_cached(q, *pools, plan, table, n, offsets, positions), want)
    for bad in (dict(lengths=n + 500), dict(table=table - 1), dict(offsets=offsets.flip(0))):
        a = {**dict(table=table, lengths=n, offsets=offsets, positions=positions), **bad}
        with pytest.raises(ValueError):
            paged.attention_cached(q, *pools, plan, **a)
    with pytest.raises(ValueError):
        paged.store_kv(q[:, :2], q[:, 2:4], *pools, i32([1, 1, 2]))
    with pytest.raises(ValueError):
        rotary.rotate_heads(q, q, i32([1, 2, 100]), rotary.rotary_table(100, 128, device=DEV))


def test_a_prompt_behind_a_cached_prefix():
    """A prompt's next part over the cache's values, read back, by attention over packed rows: as attention_cached gives it."""
    pools, table, n, offsets, positions = batch([200], [60], 16, 2, 128, BF, 4)
    q, plan = rnd((60, 8, 128), 1), AttnPlan("causal", 0, 128 ** -0.5, None, True, True)
    got = paged.attention_cached(q, *pools, plan, table, n, offsets, positions)
    t = torch.arange(200, device=DEV)
    k, v = paged.read_kv(*pools, (table[0].long()[t // 16] * 16 + t % 16).to(torch.int32))
    layout = packed.packed_layout(i32([0, 200]), 200)
    whole = packed.attention_packed(torch.cat((q.new_zeros(140, 8, 128), q)), k, v, AttnPlan("causal", 0, 128 ** -0.5), layout)[140:]
    # two results, each off by 2^-8 of its size and as much of the probabilities' rounding
    assert (got.double() - whole.double()).norm() <= 4 * 2.0 ** -8 * whole.double().norm()


def test_inside_a_compiled_function():
    pools, table, n, offsets, positions = batch([30, 20], [1, 2], 16, 2, 64, BF, 1)
    plan, q = AttnPlan("causal", 0, 0.1, None, True, True), rnd((3, 4, 64), 1)
    want = paged.attention_cached(q * 2, *pools, plan, table, n, offsets, positions)
    got = torch.compile(lambda q: paged.attention_cached(q * 2, *pools, plan, table, n, offsets, positions), backend="eager")(q)
    assert torch.equal(got, want)


@pytest.mark.parametrize("scale,cap", [(1e-44, None), (1e-30, 1e30), (1.0, 1e-30)])
def test_scales_close_to_the_least_number(scale, cap):
    """Scores that differ by nothing: rows are means of the values that they see."""
    pools, table, n, offsets, positions = batch([70, 33], [9, 1], 16, 2, 64, BF, 1)
    plan, q = AttnPlan("causal", 0, scale, cap, True, True), rnd((10, 8, 64), 2)
    out = paged.attention_cached(q, *pools, plan, table, n, offsets, positions)
    check(out, oracle(q, pools, plan, table, n, offsets, positions, BF))
