"""Page tables and slots from lengths, stores into page pools, and attention over a shared prefix and requests' own keys
(``loopfuse_amd.paged``) against plain implementations: Python loops, and the formulas in 64 bits.

Tolerance of an attention result, e the half step of the type (2^-8 bf16, 2^-11 fp16): e (P |V|) for the probabilities, which are rounded
for the second product, and e |O| for the result; besides, in 32 bits, a probability is off by 2^-17 scale |Q| |K| (128 products)
+ 2^-20 of itself, with a softcap by 2^-19 cap more (its tanh is off by 2^-22), and the sums by 2^-17 of the sizes of their terms.  fp16: half of the
least step, 2^-25, per probability relative to the largest."""
import math
import random

import pytest
import torch

from loopfuse_amd import paged
from loopfuse_amd.lowering import AttnPlan

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# ---- extend_tables -------------------------------------------------------------------------------------------

def plain_tables(cached, new, table, free, page, total):
    table, free = [list(r) for r in table], list(free)
    slots, positions, offsets, lengths, taken = [], [], [0], [], 0
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        for i in range(-(-c // page), -(-(c + n) // page)):
            if i < len(table[b]):
                table[b][i] = free[taken] if taken < len(free) else -1
            taken += 1
        length = c
        for t in range(c, c + n):
            positions.append(t)
            i = t // page
            slots.append(table[b][i] * page + t % page if i < len(table[b]) and table[b][i] >= 0 else -1)
            length += slots[-1] >= 0 and len(slots) <= total
        offsets.append(offsets[-1] + n)
        lengths.append(length)
    rest = [-1] * max(0, total - len(slots))
    return table, offsets, lengths, (slots + rest)[:total], (positions + rest)[:total], taken


TABLES = [
    # cached, new, page, width, free pages left out or beyond, total beyond the tokens
    ([0], [0], 16, 1, 0, 0),
    ([0], [1], 1, 1, 0, 3),
    ([5, 16, 17, 0, 31], [1, 1, 1, 1, 1], 16, 3, 0, 0),
    ([0, 0, 0], [100, 0, 33], 8, 20, 2, 700),
    ([3, 0, -7, 40], [-2, 300, 9, 0], 4, 90, 5, 13),
    ([10, 20, 30], [50, 50, 50], 16, 9, -4, 6),           # not enough free pages
    ([10, 20, 30], [50, 50, 500], 16, 9, 0, 6),           # a row too short
    ([1, 2, 3], [70, 80, 90], 64, 9, 0, -100),            # tokens behind the last row
    ([10, 20, 30, 64, 3], [50, 50, 0, 50, 5], 16, 3, -5, -40),      # all of it
    ([100, 5], [3, 3], 16, 2, 0, 0),                      # more in the cache than the table has room for
    ([i * 7 % 50 for i in range(700)], [i * 5 % 13 for i in range(700)], 2, 40, 0, 100),
    ([0], [20000], 16, 1250, 0, 0),
    ([], [], 16, 4, 3, 9),
]


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("cached,new,page,width,spare,beyond", TABLES)
def test_tables_slots_and_positions_are_the_plain_loops(cached, new, page, width, spare, beyond, dtype):
    rng = random.Random(len(cached) + page)
    need = sum(-(-(max(c, 0) + max(n, 0)) // page) - -(-max(c, 0) // page) for c, n in zip(cached, new))
    ids = rng.sample(range(1000000), len(cached) * width + max(0, need + spare))
    table = [ids[b * width:(b + 1) * width] for b in range(len(cached))]
    free = ids[len(cached) * width:]
    total = max(0, sum(max(n, 0) for n in new) + beyond)
    want = plain_tables(cached, new, table, free, page, total)
    # a table that is a part of a wider tensor: what lies beside it stays
    wide = torch.full((len(cached), width + 3), -5, dtype=dtype, device=DEV)
    dev_table = wide[:, 1:1 + width]
    dev_table.copy_(torch.tensor(table, dtype=dtype).view(len(cached), width))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    step = paged.extend_tables(i32(cached), i32(new), dev_table, torch.tensor(free, dtype=dtype, device=DEV), page, total)
    assert dev_table.tolist() == want[0]
    assert (wide[:, 0] == -5).all() and (wide[:, 1 + width:] == -5).all()
    assert step.offsets.tolist() == want[1] and step.lengths.tolist() == want[2]
    assert step.slots.tolist() == want[3] and step.positions.tolist() == want[4] and step.pages.tolist() == [want[5]]


def test_pages_whose_slots_pass_32_bits_are_none():
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    for dtype in (torch.int32, torch.int64):
        pages = [2 ** 27 - 1, 2 ** 27, 2 ** 28] + ([2 ** 33 + 1] if dtype == torch.int64 else [2 ** 31 - 1])
        step = paged.extend_tables(i32([0] * 4), i32([16] * 4), torch.zeros((4, 1), dtype=dtype, device=DEV), torch.tensor(pages, dtype=dtype, device=DEV), 16, 64)
        assert step.slots.tolist() == list(range(2 ** 31 - 16, 2 ** 31)) + [-1] * 48


def test_attention_after_pages_ran_out_reads_what_was_stored():
    # 3 free pages for the 5 that are asked for: the entries that got none are -1, and no key is looked for there
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(1)
    page, Hkv, D, new = 16, 2, 128, [20, 30, 10]
    kp, vp = (torch.full((4, page, Hkv, D), math.nan, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    k, v = (torch.randn((60, Hkv, D), generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2))
    table = torch.full((3, 4), -1, dtype=torch.int32, device=DEV)
    step = paged.extend_tables(i32([0, 0, 0]), i32(new), table, i32([2, 0, 3]), page, 60)
    assert step.lengths.tolist() == [20, 16, 0] and step.pages.tolist() == [5]
    assert table.tolist() == [[2, 0, -1, -1], [3, -1, -1, -1], [-1, -1, -1, -1]]
    paged.store_kv(k, v, kp, vp, step.slots)
    q = torch.randn((3, 4, 1, D), generator=gen, device=DEV).to(torch.bfloat16)
    plan = AttnPlan(scale=D ** -0.5, k_paged=True, v_paged=True)
    check(paged.attention_shared(q, kp, vp, plan, table, step.lengths), oracle(q, kp, vp, table, step.lengths, None, 0, D ** -0.5, None))


# ---- store_kv ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("T,Hkv,D,pages,page,dtype", [(1, 1, 64, 1, 1, torch.bfloat16), (37, 2, 64, 9, 8, torch.float16), (300, 8, 128, 40, 16, torch.bfloat16),
                                                      (65, 3, 40, 200, 1, torch.float16), (19, 32, 128, 2, 64, torch.bfloat16), (5, 48, 128, 3, 4, torch.float16)])
def test_rows_land_in_their_slots(T, Hkv, D, pages, page, dtype):
    gen = torch.Generator(device=DEV).manual_seed(T)
    qkv = torch.randn((T, 2 * Hkv + 1, D), generator=gen, device=DEV).to(dtype)       # views of a fused projection
    k, v = qkv[:, 1:1 + Hkv], qkv[:, 1 + Hkv:]
    pools = [torch.randn((pages, page, Hkv, D) if page > 1 else (pages, Hkv, D), generator=gen, device=DEV).to(dtype) for _ in range(2)]
    slots = torch.randperm(max(pages * page, T), generator=gen, device=DEV)[:T].to(torch.int32)       # some behind the last
    slots[::5] = -1
    slots[T // 2] = 2 ** 31 - 1
    want = [p.clone() for p in pools]
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            for rows, pool in ((k, want[0]), (v, want[1])):
                pool.view(-1, Hkv, D)[s] = rows[t]
    assert paged.store_kv(k, v, *pools, slots) is None
    assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1])


def test_stores_into_a_pool_of_head_major_pages():
    base = torch.zeros((6, 4, 8, 64), dtype=torch.bfloat16, device=DEV)               # [pages, heads, page, D]
    pool = base.transpose(1, 2)
    rows = torch.randn((11, 4, 64), device=DEV).to(torch.bfloat16)
    slots = torch.randperm(48, device=DEV)[:11].to(torch.int32)
    paged.store_kv(rows, rows, pool, torch.zeros_like(pool), slots)
    for t, s in enumerate(slots.tolist()):
        assert torch.equal(pool[s // 8, s % 8], rows[t])
    assert base.count_nonzero().item() == rows.count_nonzero().item()


# ---- attention_shared ------------------------------------------------------------------------------------------

def batch(B, lengths, prefix, page, Hkv, group, D, dtype, seed=0, width=None, table_dtype=torch.int32, spare=3, size=1.0):
    """Q, pools, table, lengths, prefix table; the pages of no one hold NaN, and so do tokens behind a request's (and the prefix's) last."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    pre = -(-prefix // page)
    width = max(1, -(-max(lengths, default=0) // page)) if width is None else width
    count = pre + sum(-(-n // page) for n in lengths) + spare
    ids = torch.randperm(count, generator=gen, device=DEV).tolist()
    pools = [torch.full((count, page, Hkv, D), math.nan, device=DEV) for _ in range(2)]
    prefix_table, ids = ids[:pre], ids[pre:]
    table = torch.full((B, width), -1, dtype=table_dtype)
    for i, p in enumerate(prefix_table):
        n = min(page, prefix - i * page)
        for pool in pools:
            pool[p, :n] = torch.randn((n, Hkv, D), generator=gen, device=DEV)
    for b, length in enumerate(lengths):
        for i in range(-(-length // page)):
            p, n = ids.pop(), min(page, length - i * page)
            table[b, i] = p
            for pool in pools:
                pool[p, :n] = torch.randn((n, Hkv, D), generator=gen, device=DEV) * size
    q = torch.randn((B, Hkv * group, 1, D), generator=gen, device=DEV) * size
    return (q.to(dtype), pools[0].to(dtype), pools[1].to(dtype), table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV),
            torch.tensor(prefix_table, dtype=table_dtype, device=DEV))


def oracle(q, k_pool, v_pool, table, lengths, prefix_table, prefix, scale, cap):
    B, Hq, _, D = q.shape
    page, Hkv = k_pool.shape[1:3]
    g, e = Hq // Hkv, torch.finfo(q.dtype).eps / 2
    least = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    for b, n in enumerate(lengths.tolist()):
        rows = [(int(prefix_table[t // page]), t % page) for t in range(prefix)] + [(int(table[b, t // page]), t % page) for t in range(n)]
        if not rows:
            continue
        pg, at = (torch.tensor(x, device=q.device) for x in zip(*rows))
        for h in range(Hkv):
            k, v = k_pool[pg, at, h].double(), v_pool[pg, at, h].double()
            qh = q[b, h * g:(h + 1) * g, 0].double()
            s = qh @ k.t() * scale
            if cap:
                s = cap * torch.tanh(s / cap)
            p = torch.softmax(s, dim=-1)
            er = e + 2.0 ** -17 * scale * (qh.abs() @ k.abs().t()) + 2.0 ** -20 + (2.0 ** -19 * cap if cap else 0.0)
            o = p @ v
            out[b, h * g:(h + 1) * g, 0] = o
            bound[b, h * g:(h + 1) * g, 0] = (p * (2 * er - e + 2.0 ** -17) + least) @ v.abs() + e * o.abs() + least
    return out, bound * 1.01


def check(got, want, what="out"):
    value, bound = want
    assert not torch.isnan(got).any(), f"{what}: NaN"
    err = (got.double() - value).abs()
    worst = (err - bound).max().item()
    assert worst <= 0, f"{what}: {worst} beyond its bound, at an error of {err.max().item()}"


SHARED = [
    # lengths of the own keys, prefix, page, Hkv, group, D, dtype, softcap
    ([1], 0, 16, 1, 1, 64, torch.bfloat16, None),
    ([0], 0, 16, 2, 2, 128, torch.float16, None),
    ([0, 0, 0], 5, 16, 8, 4, 128, torch.bfloat16, None),
    ([3, 0, 17, 16], 0, 16, 8, 4, 128, torch.bfloat16, None),
    ([40, 20], 1000, 16, 8, 4, 128, torch.bfloat16, None),
    ([700, 1, 0, 333, 64], 130, 8, 4, 2, 64, torch.float16, 30.0),
    ([2000, 1, 900], 17, 1, 4, 8, 128, torch.bfloat16, None),
    ([5, 9], 257, 2, 3, 3, 64, torch.float16, None),
    ([100] * 70, 200, 16, 2, 1, 64, torch.bfloat16, None),
    ([33, 4000], 1, 64, 8, 2, 64, torch.bfloat16, 20.0),
    ([10 * i for i in range(40)], 513, 16, 1, 40, 128, torch.float16, None),
    ([60, 61, 62], 4100, 16, 16, 1, 128, torch.float16, None),
]


@pytest.mark.parametrize("lengths,prefix,page,Hkv,group,D,dtype,cap", SHARED)
def test_attention_over_a_shared_prefix_is_the_formula(lengths, prefix, page, Hkv, group, D, dtype, cap):
    q, kp, vp, table, n, pre = batch(len(lengths), lengths, prefix, page, Hkv, group, D, dtype, seed=prefix + page)
    plan = AttnPlan(scale=D ** -0.5, softcap=cap, k_paged=True, v_paged=True)
    out = paged.attention_shared(q, kp, vp, plan, table, n, prefix_table=pre, prefix_len=prefix)
    check(out, oracle(q, kp, vp, table, n, pre, prefix, D ** -0.5, cap))
    if prefix:       # the other form of the prefix, other splits and pieces
        for choice in ({"prefix": "tiles", "splits": 3}, {"prefix": "tiles", "near": False}, {"prefix": "stream", "splits": 2, "least": 32, "target_log2": 12}):
            other = paged.attention_shared(q, kp, vp, plan, table, n, prefix_table=pre, prefix_len=prefix, choice=choice)
            check(other, oracle(q, kp, vp, table, n, pre, prefix, D ** -0.5, cap), str(choice))
    given = torch.full((len(lengths), 2 * Hkv * group, 1, D), 9.0, dtype=dtype, device=DEV)
    assert paged.attention_shared(q, kp, vp, plan, table, n, prefix_table=pre, prefix_len=prefix, out=given[:, ::2]) is not None
    assert torch.equal(given[:, ::2], out) and (given[:, 1::2] == 9).all()


def test_tables_in_64_bits_and_pools_of_one_token_pages():
    q, kp, vp, table, n, pre = batch(3, [5, 0, 77], 40, 1, 8, 2, 128, torch.bfloat16, table_dtype=torch.int64)
    plan = AttnPlan(scale=0.1, k_paged=True, v_paged=True)
    want = oracle(q, kp, vp, table, n, pre, 40, 0.1, None)
    check(paged.attention_shared(q, kp, vp, plan, table, n, prefix_table=pre, prefix_len=40), want)
    check(paged.attention_shared(q, kp[:, 0], vp[:, 0], plan, table, n, prefix_table=pre, prefix_len=40), want)
