"""What the page pools in 4 bits and the operators over them refuse, and how ``attention_cached`` deals its work to workgroups; no GPU."""
import math
import random

import pytest
import torch
from torch.autograd import forward_ad

from loopfuse_amd import lowering, paged, rotary
from loopfuse_amd.lowering import AttnPlan, UnsupportedPlan
from loopfuse_amd.paged import Pool4
from test_ragged import OnGpu, fake, nothing_is_launched  # noqa: F401  (a fixture that every test here uses)

BF, HF, F32, I32, U8 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.uint8


def pool(pages=3, page=16, heads=2, D=64, dtype=BF):
    p = paged.pool4(pages, page, heads, D, dtype)
    return Pool4(p.codes.as_subclass(OnGpu), p.scales.as_subclass(OnGpu), dtype)


# ---- pool4 ---------------------------------------------------------------------------------------------------

def test_a_pool_has_17_bytes_for_32_elements():
    p = paged.pool4(5, 32, 3, 128, HF)
    assert p.shape == (5, 32, 3, 128) and p.codes.numel() == 5 * 32 * 3 * 64 and p.scales.numel() == 5 * 32 * 3 * 4
    assert p.dtype is HF and p.device.type == "cpu" and int(torch.count_nonzero(p.codes)) == 0


@pytest.mark.parametrize("args", [(3, 8, 2, 64, BF), (3, 24, 2, 64, BF), (3, 16, 2, 96, BF), (3, 16, 0, 64, BF), (-1, 16, 2, 64, BF), (3, 16, 2, 64, F32), (3, 16.0, 2, 64, BF), (3, 0, 2, 64, BF)])
def test_pools_that_are_refused(args):
    with pytest.raises(UnsupportedPlan):
        paged.pool4(*args)


def broken(**kw):
    p = pool()
    return Pool4(kw.get("codes", p.codes), kw.get("scales", p.scales), kw.get("dtype", p.dtype))


POOLS = {
    "type": broken(dtype=HF), "codes of another type": broken(codes=pool().codes.char()), "dims": broken(codes=pool().codes[0]), "codes of 96": broken(codes=fake((3, 2, 1, 768), U8)),
    "scales of fewer heads": broken(scales=pool().scales[:, :1]), "scales of fewer pages": broken(scales=pool().scales[:2]),
    "pages of 48 tokens": broken(codes=fake((3, 2, 3, 512), U8), scales=fake((3, 2, 3, 32), U8)), "heads apart": broken(codes=fake((3, 4, 1, 512), U8)[:, ::2]),
    "one page": broken(codes=fake((1, 2, 1, 512), U8).expand(3, 2, 1, 512)), "off its border": broken(codes=fake((3 * 1024 + 1,), U8)[1:].view(3, 2, 1, 512)),
    "a pool of rows": fake((3, 16, 2, 64)),
}


@pytest.mark.parametrize("which", ["k_pool", "v_pool"])
@pytest.mark.parametrize("case", POOLS)
def test_calls_refuse_pools_that_are_none(case, which):
    a = dict(k_pool=pool(), v_pool=pool())
    a[which] = POOLS[case]
    rows, slots = fake((10, 2, 64)), fake((10,), I32)
    for call in (lambda: paged.store_kv(rows, rows, a["k_pool"], a["v_pool"], slots), lambda: paged.read_kv(a["k_pool"], a["v_pool"], slots),
                 lambda: paged.append_kv(fake((10, 4, 64)), rows, rows, a["k_pool"], a["v_pool"], slots, slots, fake((50, 64), F32)),
                 lambda: paged.attention_cached(fake((3, 4, 64)), a["k_pool"], a["v_pool"], PLAN, fake((3, 4), I32), fake((3,), I32))):
        with pytest.raises(UnsupportedPlan):
            call()


def test_attention_over_a_prefix_refuses_pools_in_4_bits():
    with pytest.raises(UnsupportedPlan, match="4 bits"):
        paged.attention_shared(fake((3, 4, 1, 64)), pool(), pool(), AttnPlan(scale=0.1, k_paged=True, v_paged=True), fake((3, 4), I32), fake((3,), I32))


def test_pools_on_the_cpu_are_refused():
    p, rows, i = paged.pool4(3, 16, 2, 64, BF), fake((10, 2, 64)), fake((10,), I32)
    for call in (lambda: paged.store_kv(rows, rows, p, p, i), lambda: paged.read_kv(p, p, i), lambda: paged.read_kv(rows.as_subclass(torch.Tensor)[None], rows[None], i),
                 lambda: paged.attention_cached(fake((3, 4, 64)), p, p, PLAN, fake((3, 4), I32), fake((3,), I32))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


# ---- append_kv, read_kv ---------------------------------------------------------------------------------------

def append(**change):
    a = dict(q=fake((10, 4, 64)), k=fake((10, 2, 64)), v=fake((10, 2, 64)), k_pool=fake((3, 4, 2, 64)), v_pool=fake((3, 4, 2, 64)), slots=fake((10,), I32),
             positions=fake((10,), I32), table=fake((50, 64), F32))
    a.update(change)
    return a


APPEND = {
    "rows of v": dict(v=fake((9, 2, 64))), "heads of v": dict(v=fake((10, 1, 64))), "type of v": dict(v=fake((10, 2, 64), HF)), "slots": dict(slots=fake((9,), I32)),
    "slots in 64 bits": dict(slots=fake((10,), torch.int64)), "positions": dict(positions=fake((9,), I32)), "no positions": dict(positions=None),
    "pool heads": dict(k_pool=fake((3, 4, 1, 64)), v_pool=fake((3, 4, 1, 64))), "pools of two sizes": dict(v_pool=fake((6, 2, 2, 64))), "page size": dict(k_pool=fake((3, 6, 2, 64)), v_pool=fake((3, 6, 2, 64))),
    "pool type": dict(k_pool=fake((3, 4, 2, 64), HF)), "a pool of one page": dict(k_pool=fake((1, 4, 2, 64)).expand(3, 4, 2, 64)), "head dim": dict(q=fake((10, 4, 128))),
    "weights without eps": dict(q_weight=fake((64,))), "weights without eps or a table": dict(q_weight=fake((64,)), table=None), "a pool in 4 bits of other heads": dict(k_pool=pool(heads=1), v_pool=pool(heads=1)),
    "a pool in 4 bits of another head dim": dict(k_pool=pool(D=128), v_pool=pool(D=128)),
}


@pytest.mark.parametrize("case", APPEND)
def test_appends_that_are_refused(case):
    with pytest.raises(UnsupportedPlan):
        paged.append_kv(**append(**APPEND[case]))


def test_appends_that_are_served_reach_a_launch():
    for a in (append(), append(table=None), append(table=None, eps=1e-6), append(eps=0.0, q_weight=fake((64,))), append(k_pool=pool(), v_pool=pool()),
              append(k_pool=fake((12, 2, 64)), v_pool=fake((12, 2, 64)))):
        with pytest.raises(AssertionError, match="a launch"):
            paged.append_kv(**a)
    with pytest.raises(AssertionError, match="a launch"):
        paged.store_kv(fake((10, 2, 64)), fake((10, 2, 64)), pool(), pool(), fake((10,), I32))
    empty = append(q=fake((0, 4, 64)), k=fake((0, 2, 64)), v=fake((0, 2, 64)), slots=fake((0,), I32), positions=fake((0,), I32))
    assert paged.append_kv(**empty).shape == (0, 4, 64)


@pytest.mark.parametrize("name", ["q", "k", "v", "k_pool"])
def test_forward_mode_derivatives_are_refused(name):
    with forward_ad.dual_level():
        a = append()
        a[name] = forward_ad.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(UnsupportedPlan, match="tangents"):
            paged.append_kv(**a)


def test_reads_that_are_refused():
    i = fake((5,), I32)
    for a in ((fake((3, 4, 2, 64)), fake((3, 4, 1, 64)), i), (fake((3, 4, 2, 64)), fake((3, 4, 2, 64)), i.long()), (fake((3, 4, 2, 64), F32),) * 2 + (i,), (fake((3, 6, 2, 64)),) * 2 + (i,),
              (fake((3, 4, 2, 60)),) * 2 + (i,), (fake((64,)),) * 2 + (i,), (None, None, i), (pool(), pool(page=32), i), (pool(), pool(dtype=HF), i)):
        with pytest.raises(UnsupportedPlan):
            paged.read_kv(*a)
    assert [t.shape for t in paged.read_kv(pool(), pool(), fake((0,), I32))] == [(0, 2, 64)] * 2


def test_checked_slots_and_positions(monkeypatch):
    monkeypatch.setattr(lowering, "_checks_tables", lambda: True)
    i = fake((10,), I32)
    apart = torch.arange(10, dtype=I32).as_subclass(OnGpu)
    for a, served in ((append(slots=apart), True), (append(), False), (append(slots=apart + 3), False), (append(slots=apart - 20), True), (append(slots=apart, positions=i + 50), False)):
        with pytest.raises(AssertionError if served else ValueError):
            paged.append_kv(**a)


# ---- attention_cached: refusals --------------------------------------------------------------------------------

PLAN = AttnPlan("causal", scale=0.1, k_paged=True, v_paged=True)


def cached(**change):
    a = dict(q=fake((7, 4, 64)), k_pool=pool(9), v_pool=pool(9), plan=PLAN, table=fake((3, 5), I32), lengths=fake((3,), I32), offsets=fake((4,), I32), positions=fake((7,), I32))
    a.update(change)
    return a


HUGE = Pool4(*(torch.empty((1, 2, 1 << 21, n), dtype=U8).as_subclass(OnGpu) for n in (512, 32)), BF)       # (never touched: it takes no memory)
CACHED = {
    "fp32": dict(q=fake((7, 4, 64), F32)), "type": dict(q=fake((7, 4, 64), HF)), "dims": dict(q=fake((7, 4, 1, 64))), "head dim": dict(q=fake((7, 4, 96))), "another head dim": dict(q=fake((7, 4, 128))),
    "heads": dict(q=fake((7, 3, 64))), "mask": dict(plan=AttnPlan("other", scale=0.1)), "window": dict(plan=AttnPlan("sliding", scale=0.1)), "denominator": dict(plan=AttnPlan("causal", scale=0.1, denom_add=1.0)),
    "scale": dict(plan=AttnPlan("causal", scale=0.0)), "nan scale": dict(plan=AttnPlan("causal", scale=math.nan)), "softcap": dict(plan=AttnPlan("causal", scale=0.1, softcap=0.0)),
    "an infinite softcap": dict(plan=AttnPlan("causal", scale=0.1, softcap=math.inf)), "type of the table": dict(table=fake((3, 5), F32)), "dims of the table": dict(table=fake((5,), I32)),
    "requests": dict(lengths=fake((2,), I32)), "type of lengths": dict(lengths=fake((3,), torch.int64)), "offsets": dict(offsets=fake((3,), I32)), "offsets in 64 bits": dict(offsets=fake((4,), torch.int64)),
    "positions": dict(positions=fake((6,), I32)), "several rows without positions": dict(positions=None), "no offsets": dict(offsets=None), "out": dict(out=fake((7, 4, 128))),
    "out of one row": dict(out=fake((1, 4, 64)).expand(7, 4, 64)), "type of out": dict(out=fake((7, 4, 64), HF)), "strides": dict(q=fake((7, 4, 68))[..., :64]),
    "room beyond 2**30 keys": dict(table=fake((3, 1), I32).expand(3, (1 << 26) + 1)), "groups of 2**20 heads": dict(q=fake((1, 1, 64)).expand(7, 1 << 20, 64), k_pool=pool(9, heads=1), v_pool=pool(9, heads=1)),
    "pages of V further apart": dict(v_pool=Pool4(fake((9, 4, 1, 512), U8)[:, :2], fake((9, 4, 1, 32), U8)[:, :2], BF)),
    "pages of codes further apart": dict(k_pool=Pool4(fake((9, 4, 1, 512), U8)[:, :2], pool(9).scales, BF), v_pool=Pool4(fake((9, 4, 1, 512), U8)[:, :2], pool(9).scales, BF)),
    "a page of 2 GiB": dict(k_pool=HUGE, v_pool=HUGE, table=fake((3, 1), I32)),
    "more than can lie on a line": dict(q=fake((1, 4, 64)).expand(1 << 16, 4, 64), positions=fake((1,), I32).expand(1 << 16), table=fake((1, 1), I32).expand(1 << 16, 1 << 20), lengths=fake((1,), I32).expand(1 << 16), offsets=fake((1,), I32).expand((1 << 16) + 1)),
}


@pytest.mark.parametrize("case", CACHED)
def test_cached_calls_that_are_refused(case):
    with pytest.raises(UnsupportedPlan):
        paged.attention_cached(**cached(**CACHED[case]))


def test_cached_calls_that_are_served_reach_a_launch():
    parts = Pool4(fake((9, 4, 1, 512), U8)[:, :2], fake((9, 4, 1, 32), U8)[:, :2], BF)
    for a in (cached(), cached(k_pool=parts, v_pool=parts), cached(plan=AttnPlan(None, scale=0.1)), cached(plan=AttnPlan("sliding", 3, scale=0.1, softcap=-5.0)), cached(q=fake((3, 2, 64)), offsets=None, positions=None),
              cached(q=fake((2, 2, 64)), positions=None), cached(out=fake((7, 8, 64))[:, ::2]), cached(table=fake((3, 5), torch.int64))):
        with pytest.raises(AssertionError, match="a launch"):
            paged.attention_cached(**a)
    assert paged.attention_cached(**cached(q=fake((0, 4, 64)), positions=fake((0,), I32))).shape == (0, 4, 64)


def test_checked_tables(monkeypatch):
    monkeypatch.setattr(lowering, "_checks_tables", lambda: True)
    monkeypatch.setattr(paged.lowering, "get_kernel", lowering.get_kernel)
    some = fake((3,), I32) + 20
    for a, served in ((cached(lengths=some), True), (cached(lengths=some, table=fake((3, 5), I32) - 1), False), (cached(lengths=some, table=fake((3, 5), I32) + 9), False),
                      (cached(lengths=some + 100), False), (cached(offsets=torch.tensor([0, 3, 2, 5], dtype=I32).as_subclass(OnGpu)), False), (cached(offsets=fake((4,), I32) + 8), False),
                      (cached(table=fake((3, 5), I32) - 1), True)):
        with pytest.raises(AssertionError if served else ValueError):
            paged.attention_cached(**a)


# ---- attention_cached: who does what ----------------------------------------------------------------------------

def line_of(lengths, new, window, group, Hkv, rows, fixed):
    """(requests in order: chunks, pairs, size of a unit) as the kernel forms them."""
    res = []
    for n, m in zip(lengths, new):
        start = min(max(n - m - window + 1, 0), max(n - 1, 0)) & ~31 if window else 0
        pairs = max((n - start + 31) // 32, 1)
        res.append((-(-m * group // rows), pairs, 1 if fixed < 0 else pairs + fixed))
    return res


BATCHES = [([1000, 500], [1, 1], 0, 4, 8), ([0], [1], 0, 1, 1), ([0, 0, 0], [0, 0, 1], 0, 1, 2), ([5, 5], [0, 1], 0, 1, 2), ([8192 * (64 - i) // 64 for i in range(64)], [1] * 64, 0, 4, 8), ([100000, 1], [1, 5], 0, 8, 2),
           ([6000, 0, 33, 32, 31], [5, 0, 33, 1, 2], 1024, 4, 4), ([3000] * 200, [1] * 200, 0, 1, 1), ([6001, 4500, 3000, 1500], [1000] * 4, 0, 4, 8), ([70], [70], 7, 3, 3)]


@pytest.mark.parametrize("lengths,new,window,group,Hkv", BATCHES)
@pytest.mark.parametrize("choice", [None, (512, 16, 20), (7, 0, 1), (1024, 4, 8), (1, 3, 5), (64, 16, 400)])
def test_every_pair_has_one_workgroup_and_every_part_a_place(lengths, new, window, group, Hkv, choice):
    """The kernel's own arithmetic: the pairs of each unit are dealt once, parts lie in places of their own within the room for them, and the ones that lf_cached_combine looks
    for are those that were left."""
    B, T = len(lengths), sum(new)
    for blocks, rowwaves in ((1, False), (2, False), (2, True)):
        rows = 16 * blocks * (4 if rowwaves else 1)
        most = (T * group // rows + min(T, B)) * Hkv
        keys = max(lengths)
        workgroups, fixed, least = choice or paged.cached_shares(most, keys, T * group / B, (blocks, rowwaves), 128)
        requests = line_of(lengths, new, window, group, Hkv, rows, fixed)
        units = [(b, u) for b, (chunks, _, _) in enumerate(requests) for u in range(chunks * Hkv)]
        assert len(units) <= most
        line = sum(c * Hkv * s for c, _, s in requests)
        share = max(least, -(-line // workgroups))
        before = [0]
        for c, _, s in requests:
            before.append(before[-1] + c * Hkv * s)
        numbers = [0]
        for c, _, _ in requests:
            numbers.append(numbers[-1] + c * Hkv)
        done, parts, written = {u: [] for u in units}, {}, set()
        for w in range(workgroups):
            place, end = min(w * share, line), min((w + 1) * share, line)
            while place < end:
                b = next(i for i in range(B) if before[i + 1] > place)
                chunks, pairs, size = requests[b]
                unit = (place - before[b]) // size
                lo = place - before[b] - unit * size
                hi = min(size, lo + end - place)
                place += hi - lo
                if hi <= fixed:
                    continue
                p0, p1 = (0, pairs) if fixed < 0 else (max(lo - fixed, 0), hi - fixed)
                done[b, unit].append((p0, p1))
                if (p0, p1) == (0, pairs):
                    written.add((b, unit))
                    continue
                slot = numbers[b] + unit + w
                assert slot not in parts and slot < most + workgroups
                parts[slot] = (b, unit)
        for (b, unit), got in done.items():
            assert [x for p in sorted(got) for x in range(*p)] == list(range(requests[b][1]))
            if fixed < 0:
                assert (b, unit) in written
                continue
            size, at = requests[b][2], before[b] + unit * requests[b][2]
            first = (at + fixed) // share
            count = (at + size - 1) // share - first + 1
            assert (count == 1) == ((b, unit) in written)
            if count > 1:
                assert [parts.get(numbers[b] + unit + first + z) for z in range(count)] == [(b, unit)] * count


def test_rows_by_the_reciprocal_of_the_group():
    """row / group as the kernel forms it, the upper half of row times 2^32 / group rounded up, for the rows that a launch may have."""
    rng = random.Random(1)
    for group in [*range(2, 200), 1000, 4096]:
        per, most = -(-(1 << 32) // group), ((1 << 32) - 1) // group ** 2 * group       # (T * group ** 2 < 2^32)
        for row in [0, 1, group - 1, group, most - 1, most - group, most] + [rng.randrange(most + 1) for _ in range(300)]:
            assert row * per >> 32 == row // group


def test_builds_that_the_rules_choose_are_built_ahead():
    import __graft_entry__
    built = set(__graft_entry__.cache_specs())
    for dtype in (BF, HF):
        for D in (64, 128):
            for mask in (0, 1, 2):
                for cap in (False, True):
                    for rows in (1, 4, 16, 40, 64, 65, 500, 10000):
                        for keys in (500, 5000, 10 ** 6):
                            assert paged.cached_spec(dtype, D, mask, cap, False, *paged.cached_build(rows, 32 * rows, keys, D)) in built
        for D in (16, 48, 64, 96, 128, 256):
            assert rotary.kernel_spec(dtype, D) in built and rotary.kernel_spec(dtype, D, 1) in built
            assert D not in (64, 128) or rotary.kernel_spec(dtype, D, 2) in built


def test_checked_slots_are_those_of_tokens(monkeypatch):
    """A row of no token is left out of the pools whatever its slot, and so out of the check."""
    monkeypatch.setattr(lowering, "_checks_tables", lambda: True)
    apart, none = torch.arange(10, dtype=I32).as_subclass(OnGpu), fake((10,), I32)
    none[[2, 5, 9]] = -1
    twice, behind = apart.clone(), apart.clone()
    twice[[2, 5]] = 7
    behind[9] = 12
    # (the pools hold 12 tokens)
    for a, served in ((dict(slots=twice, positions=none), True), (dict(slots=behind, positions=none), True), (dict(slots=twice), False), (dict(slots=behind), False),
                      (dict(slots=fake((10,), I32), positions=none), False), (dict(slots=fake((10,), I32), positions=none.clamp(max=-1)), True)):
        for pools in ({}, dict(k_pool=pool(pages=1), v_pool=pool(pages=1))):
            if pools and a["slots"] is behind:
                continue       # (which hold 16)
            with pytest.raises(AssertionError if served else ValueError):
                paged.append_kv(**append(**pools, **a))
    with pytest.raises(ValueError):       # a store knows no positions
        paged.store_kv(fake((10, 2, 64)), fake((10, 2, 64)), pool(), pool(), twice)


def test_launches_of_a_unit_each_beyond_32_bits():
    """2^24 requests of one token and few keys: 17 / 16 * 2^24 workgroups of 256 threads at most."""
    def call(B):
        one = lambda *shape: fake((1,) * len(shape), I32).expand(*shape)
        return cached(q=fake((1, 1, 64)).expand(B, 1, 64), k_pool=pool(9, heads=1), v_pool=pool(9, heads=1), table=one(B, 1), lengths=one(B), offsets=None, positions=None)

    for B, served in ((1 << 24, False), (15_800_000, False), (15_700_000, True)):
        assert (B // 16 + B >= 1 << 24) != served
        with pytest.raises(AssertionError if served else UnsupportedPlan):
            paged.attention_cached(**call(B))


@pytest.mark.parametrize("scale,softcap", [(1e-46, None), (1e39, None), (0.1, 1e-46), (0.1, 1e39), (1.0, 1e-39), (1e-46, 1.0)])
def test_scales_that_are_no_numbers_in_32_bits_are_refused(scale, softcap):
    """The kernels multiply masked scores, -inf, with a scale that must not be 0, and divide by the cap."""
    with pytest.raises(UnsupportedPlan):
        paged.attention_cached(**cached(plan=AttnPlan("causal", scale=scale, softcap=softcap)))
    for plan in (AttnPlan("causal", scale=1e-44), AttnPlan("causal", scale=1e38), AttnPlan("causal", scale=1e-30, softcap=1e30), AttnPlan("causal", scale=1.0, softcap=-1e-38)):
        with pytest.raises(AssertionError, match="a launch"):
            paged.attention_cached(**cached(plan=plan))
