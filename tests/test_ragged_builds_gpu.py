"""Every build that the rules of the operators for different lengths can choose against the formulas in 64 bits: on small batches with the rules
overridden, and on batches large enough that the rules choose the builds of real sizes by themselves, which is asserted.  Tolerances: those derived in
test_packed_gpu.py and test_paged_gpu.py."""
import pytest
import torch

import test_paged_gpu as paged_tests
from loopfuse_amd import lowering, packed, paged
from loopfuse_amd.lowering import AttnPlan
from test_packed_gpu import check, inputs, layout_of, oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HALF = torch.bfloat16, torch.float16


@pytest.fixture
def specs(monkeypatch):
    """The builds that calls launch from now on, none of them kept from before or for later tests."""
    seen, get = [], lowering.get_kernel

    def record(spec, *a):
        seen.append(spec)
        return get(spec, *a)

    monkeypatch.setattr(lowering, "get_kernel", record)
    paged._host.clear()
    yield seen
    paged._host.clear()


def options(specs, family):
    """The -D options of the one build of a family among ``specs``."""
    found = {s for s in specs if s.family in family}
    assert len(found) == 1, found
    return set(found.pop().options())


# ---- packed: small batches, every build -----------------------------------------------------------------------------------------

LENGTHS = [513, 1, 257, 0, 300, 64, 256]        # tails of one row behind tiles of 32 ... 256
MASKS = [("causal", 0, None), (None, 0, None), ("sliding", 100, None), ("causal", 0, 20.0), ("sliding", 65, 30.0), (None, 0, 5.0)]


@pytest.mark.parametrize("D,dtype", [(128, BF), (128, HALF), (64, BF), (64, HALF)])
@pytest.mark.parametrize("mask,window,cap", MASKS)
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (4, 2), (4, 1)])
def test_builds_of_the_forward(D, dtype, mask, window, cap, Hq, Hkv, monkeypatch, specs):
    """Key tiles of 64 and 32, plain and whole-row stores, 1, 2 and 4 heads per workgroup; with what rounding takes from O beside it."""
    q, k, v, g, bounds = inputs(LENGTHS, Hq, Hkv, D, dtype, D + Hq, 3, 70)
    plan, layout, T = AttnPlan(mask, window=window, scale=D ** -0.5, softcap=cap), layout_of(bounds, len(q)), len(q)
    want = oracle(q, k, v, g, bounds, mask, window, D ** -0.5, cap)[0]["out"]
    results = []
    for bn in (0, 32) if D == 128 else (0,):
        for stay in (False, True):
            monkeypatch.setattr(lowering, "prefill_kv_tile", lambda *a: bn)
            monkeypatch.setattr(lowering, "prefill_out_stays", lambda n: stay)
            paged._host.clear()
            specs.clear()
            out = packed.attention_packed(q, k, v, plan, layout)
            got = options(specs, ("prefill_swp",))
            assert ("-DLF_STAY=1" in got) == stay and ("-DLF_BN=32" in got) == (bn == 32) and (f"-DLF_GQAPACK={Hq // Hkv}" in got) == (Hq > Hkv)
            check(out, want, f"out {bn} {stay}")
            lse, low = torch.empty(Hq, T, device=DEV), torch.zeros_like(q)
            assert torch.equal(packed._forward(q, k, v, plan, layout, None, lse, low), out)
            results.append((bn, out, low, lse))
            into = torch.full((T, 2 * Hq, D), 3.0, dtype=dtype, device=DEV)
            packed.attention_packed(q, k, v, plan, layout, out=into[:, ::2])
            lo, hi = bounds[0], bounds[-1]
            assert torch.equal(into[lo:hi, ::2], out[lo:hi]) and (into[:, 1::2] == 3).all() and (into[:lo] == 3).all() and (into[hi:] == 3).all()
    # the stores move the same bits
    for bn, out, low, lse in results:
        first = next(r for r in results if r[0] == bn)
        rows = slice(bounds[0], bounds[-1])
        assert torch.equal(out, first[1]) and torch.equal(low, first[2]) and torch.equal(lse[:, rows], first[3][:, rows])


@pytest.mark.parametrize("D,dtype", [(128, BF), (128, HALF), (64, BF), (64, HALF)])
@pytest.mark.parametrize("mask,window,cap", MASKS)
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (4, 1)])
def test_builds_of_the_backward(D, dtype, mask, window, cap, Hq, Hkv, monkeypatch, specs):
    """Whole keys, two blocks of them and queries shared by two waves, dQ of 256 and 512 threads, dS kept and formed again, whole-row and plain stores."""
    q, k, v, g, bounds = inputs(LENGTHS, Hq, Hkv, D, dtype, D + Hq, 3, 70)
    plan, layout, T = AttnPlan(mask, window=window, scale=D ** -0.5, softcap=cap), layout_of(bounds, len(q)), len(q)
    want = oracle(q, k, v, g, bounds, mask, window, D ** -0.5, cap)[0]
    lse, low = torch.empty(Hq, T, device=DEV), torch.zeros_like(q)
    o = packed._forward(q, k, v, plan, layout, None, lse, low)
    code = lowering._MASK_NAMES[mask]
    for keys, q_split in ((1, False), (1, True)) + (((2, False),) if lowering.bwd_two_key_blocks(D, code, cap is not None) else ()):
        for threads in (256, 512) if D == 128 else (256,):
            for ds in (False, True) if D == 128 or cap else (False,):
                for stay in (False, True):
                    monkeypatch.setattr(lowering, "bwd_key_blocks", lambda *a: keys)
                    monkeypatch.setattr(packed, "bwd_q_split", lambda *a: q_split)
                    monkeypatch.setattr(packed, "bwd_dq_threads", lambda *a: threads)
                    monkeypatch.setattr(packed, "bwd_keep_ds", lambda *a: ds)
                    monkeypatch.setattr(lowering, "bwd_grads_stay", lambda n: stay)
                    what = f"{keys} blocks, split {q_split}, {threads} threads, dS {ds}, stay {stay}"
                    paged._host.clear()
                    specs.clear()
                    for with_low in (low, None):
                        grads = packed._backward(q, k, v, o, lse, g, plan, layout, with_low)
                        for name, t in zip(("dq", "dk", "dv"), grads):
                            check(t, want[name], f"{name}: {what}")
                    got = options(specs, ("bwd", "bwd_both"))
                    assert {f"-DLF_BW_W={keys}", f"-DLF_BW_DQ_NT={threads}"} <= got
                    assert ("-DLF_BW_QSPLIT=1" in got, "-DLF_BW_DS=1" in got, "-DLF_STAY=1" in got) == (q_split, ds, stay)
                    assert ("-DLF_BW_BOTH=1" in got) == (D == 64 and not ds)


@pytest.mark.parametrize("mask", ["causal", None, "sliding"])
@pytest.mark.parametrize("threads,q_split", [(256, False), (512, False), (256, True)])
def test_kept_ds_of_a_sequence_of_nan_stays_apart(mask, threads, q_split, monkeypatch):
    """Sequences of odd numbers of 32-row blocks, whose dS lie beside each other."""
    monkeypatch.setattr(packed, "bwd_dq_threads", lambda *a: threads)
    monkeypatch.setattr(packed, "bwd_q_split", lambda *a: q_split)
    q, k, v, g, bounds = inputs([90, 33, 65, 1, 300], 2, 2, 128, BF)
    plan, layout, lse = AttnPlan(mask, window=40, scale=0.1), layout_of(bounds, len(q)), torch.empty((2, len(q)), device=DEV)
    res = []
    for bad in (None, 1, 3):
        a = [t.clone() for t in (q, k, v, g)]
        if bad is not None:
            for t in a:
                t[bounds[bad]:bounds[bad + 1]] = float("nan")
        paged._host.clear()
        o = packed.attention_packed(*a[:3], plan, layout, lse=lse)
        grads = packed.attention_packed_backward(*a[:3], o, lse, a[3], plan, layout)
        assert "lf_attn_bwd_delta" in lowering._last_launch["kernels"]
        res.append((bad, (o, *grads)))
    paged._host.clear()
    for bad, tensors in res[1:]:
        keep = torch.ones(len(q), dtype=torch.bool, device=DEV)
        keep[bounds[bad]:bounds[bad + 1]] = False
        assert all(torch.equal(x[keep], y[keep]) for x, y in zip(tensors, res[0][1]))


# masks, and the builds that there are: head dim 64 has small workgroups, and keeps dS with a softcap only
ONE_KEY = [(D, *mask, *build) for D in (64, 128) for mask in (("causal", 0, None), (None, 0, None), ("sliding", 1, None), ("sliding", 9, 20.0), (None, 0, 5.0))
           for build in ((256, True, True), (512, False, True), (256, False, False), (512, True, False)) if D == 128 or (build[0] == 256 and (mask[2] or not build[2]))]


@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("D,mask,window,cap,threads,q_split,ds", ONE_KEY)
def test_rows_that_see_one_key_have_no_gradient_of_scores(D, dtype, mask, window, cap, threads, q_split, ds, monkeypatch):
    """Their softmax is 1 whatever Q and K are: dQ is zero, and dK of keys that nothing else sees; dV is dO."""
    monkeypatch.setattr(packed, "bwd_dq_threads", lambda *a: threads)
    monkeypatch.setattr(packed, "bwd_q_split", lambda *a: q_split)
    monkeypatch.setattr(packed, "bwd_keep_ds", lambda *a: ds)
    plan = AttnPlan(mask, window=window, scale=D ** -0.5, softcap=cap)
    for lengths in ([1] * 50, [1, 0, 0, 1], [1, 70, 1, 300]):
        q, k, v, g, bounds = inputs(lengths, 4, 2, D, dtype, len(lengths))
        layout = layout_of(bounds, len(q))
        paged._host.clear()
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        dq, dk, dv = torch.autograd.grad(packed.attention_packed(*leaves, plan, layout), leaves, g)
        want = oracle(q, k, v, g, bounds, mask, window, plan.scale, cap)[0]
        for name, t in (("dq", dq), ("dk", dk), ("dv", dv)):
            check(t, want[name], name)
        for lo, hi in zip(bounds[:-1], bounds[1:]):
            if hi - lo == 1 or (mask == "sliding" and window == 1):
                assert not dq[lo:hi].any() and not dk[lo:hi].any()
            elif hi > lo and mask is not None:
                assert not dq[lo].any() and dq[lo + 1:hi].any()
    paged._host.clear()


@pytest.mark.parametrize("D", [64, 128])
def test_windows_beyond_all_rows_and_batches_of_no_sequence(D):
    q, k, v, g, bounds = inputs([200, 1, 90], 4, 2, D, BF, 0, 5, 3)
    layout, T = layout_of(bounds, len(q)), len(q)
    for window in (200, 1 << 20, 1 << 40):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out = packed.attention_packed(*leaves, AttnPlan("sliding", window=window, scale=0.1), layout)
        want = oracle(q, k, v, g, bounds, "causal", 0, 0.1, None)[0]
        for name, t in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, g))):
            check(t, want[name], f"{name} {window}")
    none = packed.packed_layout(torch.tensor([7], dtype=torch.int32, device=DEV), T)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = packed.attention_packed(*leaves, AttnPlan("causal", scale=0.1), none)
    assert not out.any() and not any(t.any() for t in torch.autograd.grad(out, leaves, g))


@pytest.mark.parametrize("D,mask,cap", [(128, "causal", None), (64, None, None), (128, "sliding", 30.0)])
def test_peaked_rows(D, mask, cap):
    """Scores of +-100 and more: rows whose weight lies on one key, far from the first tile's maximum."""
    q, k, v, g, bounds = inputs([400, 65, 130], 4, 2, D, BF, 2)
    q, k = q * 4, k * 4
    plan, layout = AttnPlan(mask, window=150, scale=0.5, softcap=cap), layout_of(bounds, len(q))
    want = oracle(q, k, v, g, bounds, mask, 150, 0.5, cap)[0]
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = packed.attention_packed(*leaves, plan, layout)
    for name, t in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, g))):
        check(t, want[name], name)


# ---- packed: batches of real sizes, by the rules ------------------------------------------------------------------------------------

LARGE = [
    # lengths, Hq, Hkv, D, dtype, mask, window, softcap, options of the forward and of the backward that the rules choose
    ([1048, 700, 900, 1500, 300, 333, 1, 1024, 257, 999], 32, 32, 128, HALF, "causal", 0, None, {"-DLF_BN=32"}, {"-DLF_BW_W=1", "-DLF_BW_DQ_NT=512", "-DLF_BW_DS=1"}),
    ([2048, 1100, 900, 1500, 700, 333, 2000, 1025], 32, 32, 128, BF, "causal", 0, None, {"-DLF_BN=32"}, {"-DLF_BW_W=2", "-DLF_BW_DQ_NT=512", "-DLF_BW_DS=1"}),
    ([2048, 1000, 37, 1500, 600, 1, 800, 2000, 99, 257, 1200, 500], 32, 8, 128, BF, "causal", 0, None, {"-DLF_BN=32", "-DLF_GQAPACK=4"}, {"-DLF_BW_DQ_NT=512", "-DLF_BW_DS=1"}),
    ([4001, 1000, 2500, 333, 1], 32, 8, 128, HALF, "sliding", 256, 50.0, {"-DLF_BN=32", "-DLF_GQAPACK=4"}, {"-DLF_BW_W=1", "-DLF_BW_DQ_NT=512", "-DLF_BW_DS=1"}),
    ([1025, 1500, 700, 2000], 32, 32, 128, BF, None, 0, None, {"-DLF_BN=32"}, {"-DLF_BW_W=2", "-DLF_BW_DQ_NT=512", "-DLF_BW_DS=1"}),
    ([1000, 37, 500, 800, 250, 64, 1, 900, 333, 700, 600, 450, 100, 200, 999, 512, 31, 33, 800, 700, 650, 128, 129, 255], 16, 4, 64, HALF, "causal", 0, None,
     {"-DLF_GQAPACK=4"}, {"-DLF_BW_BOTH=1", "-DLF_BW_DQ_NT=256", "-DLF_BW_QSPLIT=1"}),
    ([1000, 37, 1500, 800, 1250, 64, 1, 1900], 16, 16, 64, BF, "causal", 0, None, set(), {"-DLF_BW_BOTH=1", "-DLF_BW_DQ_NT=256"}),
]


@pytest.mark.parametrize("case", range(len(LARGE)))
def test_batches_of_real_sizes(case, specs):
    lengths, Hq, Hkv, D, dtype, mask, window, cap, forward, backward = LARGE[case]
    q, k, v, g, bounds = inputs(lengths, Hq, Hkv, D, dtype, case, 0, 5)
    plan, layout = AttnPlan(mask, window=window, scale=D ** -0.5, softcap=cap), layout_of(bounds, len(q))
    specs.clear()
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = packed.attention_packed(*leaves, plan, layout)
    grads = torch.autograd.grad(out, leaves, g)
    got = options(specs, ("prefill_swp",)), options(specs, ("bwd", "bwd_both"))
    # O, its residue and the gradients leave in whole rows at these sizes
    assert forward <= got[0] and backward <= got[1], got
    assert "-DLF_STAY=1" not in got[0] and "-DLF_STAY=1" not in got[1] and ("-DLF_BW_QSPLIT=1" in got[1]) == ("-DLF_BW_QSPLIT=1" in backward), got
    want = oracle(q, k, v, g, bounds, mask, window, D ** -0.5, cap)[0]
    for name, t in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
        check(t, want[name], name)
    again = packed.attention_packed(*leaves, plan, layout)
    assert torch.equal(again, out) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(again, leaves, g), grads))


@pytest.mark.parametrize("D,dtype", [(40, BF), (100, HALF), (8, HALF), (127, BF)])
@pytest.mark.parametrize("mask,window,cap", [("causal", 0, None), ("sliding", 30, 15.0)])
def test_gradients_of_other_head_dims(D, dtype, mask, window, cap):
    q, k, v, g, bounds = inputs([70, 1, 200, 33], 4, 2, D, dtype, D, 0, 4)
    plan, layout = AttnPlan(mask, window=window, scale=D ** -0.5, softcap=cap), layout_of(bounds, len(q))
    want = oracle(q, k, v, g, bounds, mask, window, D ** -0.5, cap)[0]
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = packed.attention_packed(*leaves, plan, layout)
    for name, t in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, g))):
        check(t, want[name], name)


# ---- a shared prefix and own keys: heads loaded together ------------------------------------------------------------------------------

def shared_oracle(q, kp, vp, table, n, pre, prefix, scale, cap):
    return paged_tests.oracle(q, kp, vp, table.cpu(), n.cpu(), pre.cpu(), prefix, scale, cap)


COOP = [
    # lengths, prefix, page, Hkv, group, D, dtype, softcap, choice
    ([300, 0, 1, 45, 16, 700], 0, 16, 8, 4, 128, BF, None, {"coop": 4}),
    ([300, 0, 1, 45, 16, 700], 0, 16, 8, 4, 128, HALF, 30.0, {"coop": 8}),
    ([300, 0, 1, 45, 16, 700], 130, 16, 4, 2, 128, HALF, None, {"coop": 4, "prefix": "tiles"}),
    ([300, 0, 1, 45, 16, 700], 130, 16, 8, 4, 128, BF, 20.0, {"coop": 4, "prefix": "tiles", "splits": 2}),
    ([300, 0, 1, 45, 16, 700], 130, 8, 4, 1, 128, BF, None, {"coop": 4, "prefix": "tiles", "near": False}),
    ([300, 0, 1, 45, 16, 700], 333, 16, 12, 2, 128, BF, None, {"coop": 4, "prefix": "stream", "splits": 3}),
    ([300, 0, 1, 45, 16, 700], 333, 64, 8, 5, 128, BF, None, {"coop": 8, "prefix": "stream"}),
    ([300, 0, 1, 45, 16, 700], 0, 1, 8, 4, 128, BF, None, {"coop": 4, "least": 32, "target_log2": 12}),
    ([300, 0, 1, 45, 16, 700], 0, 16, 8, 4, 64, HALF, None, {"coop": 8}),
    ([300, 0, 1, 45, 16, 700], 257, 8, 16, 1, 64, BF, 25.0, {"coop": 8, "prefix": "stream"}),
    ([300, 0, 1, 45, 16, 700], 257, 64, 8, 17, 64, BF, None, {"coop": 8, "prefix": "stream", "least": 64, "target_log2": 12}),
]


@pytest.mark.parametrize("case", range(len(COOP)))
def test_own_keys_whose_heads_are_loaded_together(case, specs):
    lengths, prefix, page, Hkv, group, D, dtype, cap, choice = COOP[case]
    q, kp, vp, table, n, pre = paged_tests.batch(len(lengths), lengths, prefix, page, Hkv, group, D, dtype, seed=case)
    plan = AttnPlan(scale=D ** -0.5, softcap=cap, k_paged=True, v_paged=True)
    want = shared_oracle(q, kp, vp, table, n, pre, prefix, D ** -0.5, cap)
    for more in ({}, {"least": 256, "target_log2": 6}):
        specs.clear()
        out = paged.attention_shared(q, kp, vp, plan, table, n, prefix_table=pre, prefix_len=prefix, choice={**choice, **more})
        got = options(specs, ("decode",))
        assert {"-DLF_COOP=1", "-DLF_SHARED=1", f"-DLF_DW={choice['coop']}"} <= got
        assert (f"-DLF_PREFIX={2 - choice.get('near', True)}" in got) == (choice.get("prefix") == "tiles")
        paged_tests.check(out, want, str(more))


SHARED_LARGE = [
    # requests, most own keys, prefix, Hkv, group, D, dtype, softcap, options that the rules choose
    (64, 1024, 2048, 8, 4, 128, BF, None, {"-DLF_COOP=1", "-DLF_DW=4", "-DLF_PREFIX=1"}),
    (128, 300, 8208, 8, 4, 128, HALF, None, {"-DLF_COOP=1", "-DLF_DW=4", "-DLF_PREFIX=1"}),
    (64, 900, 0, 8, 4, 128, BF, 30.0, {"-DLF_COOP=1", "-DLF_DW=4"}),
    (160, 400, 0, 8, 4, 64, BF, None, {"-DLF_COOP=1", "-DLF_DW=8"}),
    (120, 400, 100, 8, 1, 64, HALF, None, {"-DLF_PREFIX=1"}),
    (40, 1900, 0, 8, 8, 64, HALF, None, {"-DLF_COOP=1", "-DLF_DW=8"}),
]


@pytest.mark.parametrize("case", range(len(SHARED_LARGE)))
def test_requests_of_real_numbers(case, specs):
    B, most, prefix, Hkv, group, D, dtype, cap, chosen = SHARED_LARGE[case]
    lengths = torch.randint(0, most + 1, (B,), generator=torch.Generator().manual_seed(case)).tolist()
    lengths[:3] = [most, 0, 1]
    q, kp, vp, table, n, pre = paged_tests.batch(B, lengths, prefix, 16, Hkv, group, D, dtype, seed=case)
    plan = AttnPlan(scale=D ** -0.5, softcap=cap, k_paged=True, v_paged=True)
    specs.clear()
    out = paged.attention_shared(q, kp, vp, plan, table, n, prefix_table=pre, prefix_len=prefix)
    assert chosen <= options(specs, ("decode",)), options(specs, ("decode",))
    paged_tests.check(out, shared_oracle(q, kp, vp, table, n, pre, prefix, D ** -0.5, cap))
    for _ in range(3):
        assert torch.equal(paged.attention_shared(q, kp, vp, plan, table, n, prefix_table=pre, prefix_len=prefix), out)


@pytest.mark.parametrize("choice", [{"coop": 4, "prefix": "tiles"}, {"coop": 4, "prefix": "tiles", "near": False}, {"coop": 0, "prefix": "tiles", "near": False}, {"coop": 8, "prefix": "stream"}], ids=str)
def test_builds_with_tables_in_64_bits(choice):
    q, kp, vp, table, n, pre = paged_tests.batch(4, [90, 0, 300, 16], 150, 16, 8, 4, 128, BF, seed=3, table_dtype=torch.int64)
    plan = AttnPlan(scale=0.1, k_paged=True, v_paged=True)
    want = shared_oracle(q, kp, vp, table, n, pre, 150, 0.1, None)
    paged_tests.check(paged.attention_shared(q, kp, vp, plan, table, n, prefix_table=pre, prefix_len=150, choice=choice), want)


@pytest.mark.parametrize("page,D", [(2, 128), (4, 64), (32, 128), (128, 64), (512, 128)])
def test_other_page_sizes(page, D):
    q, kp, vp, table, n, pre = paged_tests.batch(4, [90, 0, 700, 33], 600, page, 8, 4, D, HALF, seed=page)
    plan = AttnPlan(scale=0.1, k_paged=True, v_paged=True)
    want = shared_oracle(q, kp, vp, table, n, pre, 600, 0.1, None)
    for choice in (None, {"prefix": "stream", "splits": 3}, {"prefix": "tiles", "near": False}) + (({"coop": 4},) if D == 128 else ({"coop": 8, "prefix": "stream"},)):
        paged_tests.check(paged.attention_shared(q, kp, vp, plan, table, n, prefix_table=pre, prefix_len=600, choice=choice), want, str(choice))


@pytest.mark.parametrize("prefix", [0, 70])
def test_thousands_of_requests(prefix):
    """The lengths are scanned 64 at a time."""
    lengths = [(i * 37) % 41 for i in range(3000)]
    q, kp, vp, table, n, pre = paged_tests.batch(3000, lengths, prefix, 16, 2, 2, 64, BF, seed=1)
    plan = AttnPlan(scale=0.1, k_paged=True, v_paged=True)
    out = paged.attention_shared(q, kp, vp, plan, table, n, prefix_table=pre, prefix_len=prefix)
    some = list(range(0, 3000, 43)) + [2998, 2999]
    at = torch.tensor(some, device=DEV)
    paged_tests.check(out[at], shared_oracle(q[at], kp, vp, table[at], n[at], pre, prefix, 0.1, None))
    assert torch.isfinite(out).all() and (prefix or not out[n == 0].any())
