"""The largest sizes, overridden choices and derivatives that the operators for different lengths refuse; how they lay out what they keep; no GPU."""
import pytest
import torch
from torch.autograd import forward_ad

from loopfuse_amd import lowering, packed, paged
from loopfuse_amd.lowering import UnsupportedPlan
from test_ragged import PLAN, fake, layout, nothing_is_launched, pools, qkv, shared  # noqa: F401  (a fixture that every test here uses)


@pytest.mark.parametrize("total", [(1 << 31) - 1, (1 << 31) - 256, packed.MAX_ROWS + 1])
def test_layouts_whose_tiles_do_not_fit_32_bits(total):
    with pytest.raises(UnsupportedPlan):
        packed.packed_layout(fake((3,), torch.int32), total)


def test_rows_up_to_the_most_fit_32_bits_when_rounded_up():
    # lf_packed_sort and lf_packed_plan add a tile's rows less one, the attention kernels walk three tiles of 64 behind the last one
    assert packed.MAX_ROWS + max(packed.TILE_HEIGHTS) + 4 * 64 < 1 << 31


def test_more_sequences_than_can_be_ranked():
    with pytest.raises(UnsupportedPlan):
        packed.packed_layout(fake((1,), torch.int32).expand(packed.MAX_SEQUENCES + 2), 1000)
    # [3 + 4 heights][sequences + 2] numbers, indexed in 32 bits
    assert 7 * (packed.MAX_SEQUENCES + 2) < 1 << 31


@pytest.mark.parametrize("T,heads,D", [((1 << 31) - 1, 1, 8), (1 << 31, 1, 8), ((1 << 31) - 255, 1, 8), (1 << 24, 32, 128)])
def test_stores_whose_rows_pass_32_bits(T, heads, D):
    k, pool = fake((1, heads, D)).expand(T, heads, D), fake((2, 4, heads, D))
    with pytest.raises(UnsupportedPlan):
        paged.store_kv(k, k, pool, pool, fake((1,), torch.int32).expand(T))


def test_more_requests_than_can_be_summed():
    many = fake((1,), torch.int32).expand(paged.MAX_REQUESTS + 1)
    with pytest.raises(UnsupportedPlan):
        paged.extend_tables(many, many, fake((paged.MAX_REQUESTS + 1, 1), torch.int32), fake((4,), torch.int32), 16, 10)


CHOICES = [{"prefix": "rows"}, {"splits": -1}, {"splits": 2.0}, {"target_log2": -1}, {"target_log2": 25}, {"least": -32}, {"least": 48}, {"least": (1 << 30) + 32},
           {"coop": 3}, {"coop": True}, {"near": 1}, {"other": 1}, {"coop": 8}, {"coop": 4, "prefix": "tiles"}]


@pytest.mark.parametrize("choice", CHOICES, ids=str)
def test_choices_that_are_refused(choice):
    # (2 heads of 64: no heads to load together)
    with pytest.raises(UnsupportedPlan, match="choice"):
        paged.attention_shared(**shared(choice=choice))


@pytest.mark.parametrize("Hkv,D,choice", [(8, 128, {"coop": 8, "prefix": "tiles"}), (4, 128, {"coop": 8}), (6, 128, {"coop": 4}), (4, 64, {"coop": 4}), (4, 64, {"coop": 8})], ids=str)
def test_heads_that_are_not_loaded_together(Hkv, D, choice):
    kp, vp = pools(9, 4, Hkv, D)
    with pytest.raises(UnsupportedPlan, match="coop"):
        paged.attention_shared(**shared(q=fake((3, 2 * Hkv, 1, D)), k_pool=kp, v_pool=vp, choice=choice))


@pytest.mark.parametrize("Hkv,D,choice", [(8, 128, {"coop": 8, "prefix": "stream"}), (4, 128, {"coop": 4, "prefix": "tiles"}), (8, 64, {"coop": 8, "prefix": "stream"}), (8, 128, {"coop": 0})], ids=str)
def test_heads_that_are_loaded_together(Hkv, D, choice):
    kp, vp = pools(9, 4, Hkv, D)
    with pytest.raises(AssertionError, match="a launch"):
        paged.attention_shared(**shared(q=fake((3, 2 * Hkv, 1, D)), k_pool=kp, v_pool=vp, choice=choice))


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(which, grad):
    with forward_ad.dual_level():
        a = list(qkv())
        a[which] = forward_ad.make_dual(a[which], torch.ones_like(a[which]))
        if grad:
            a[0] = a[0].requires_grad_()
        with pytest.raises(UnsupportedPlan, match="tangents"), pytest.MonkeyPatch.context() as m:
            m.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
            packed.attention_packed(*a, PLAN, layout(10))
        kp, vp = pools()
        with pytest.raises(UnsupportedPlan, match="tangents"):
            paged.store_kv(forward_ad.make_dual(fake((10, 2, 64)), fake((10, 2, 64))), fake((10, 2, 64)), kp, vp, fake((10,), torch.int32))
        with pytest.raises(UnsupportedPlan, match="tangents"):
            paged.attention_shared(**shared(q=forward_ad.make_dual(fake((3, 4, 1, 64)), fake((3, 4, 1, 64)))))


@pytest.mark.parametrize("own,pre", [(513, 9), (0, 4), (171 * 3, 5 * 3), (1, 0), (7, 7)])
@pytest.mark.parametrize("D", [64, 128])
def test_partial_results_lie_on_the_borders_they_are_read_at(own, pre, D):
    floats, ml, pre_acc, pre_ml = paged.scratch_parts(own, pre, D)
    spans = sorted([(0, 4 * own * D), (ml, 8 * own), (pre_acc, 4 * pre * D), (pre_ml, 8 * pre)])
    assert all(a + n <= b for (a, n), (b, _) in zip(spans, spans[1:])) and spans[-1][0] + spans[-1][1] <= 4 * floats
    assert pre_acc % 16 == 0 and ml % 8 == 0 and pre_ml % 8 == 0


@pytest.mark.parametrize("which", ["table", "prefix_table"])
def test_checked_tables_look_at_the_pool_that_they_name_pages_of(which, monkeypatch):
    """A V pool of fewer pages than K's: ids that K has and V has not."""
    monkeypatch.setattr(lowering, "_checks_tables", lambda: True)
    kp, vp = pools(9, 4, 2, 64)[0], pools(5, 4, 2, 64)[1]
    a = shared(k_pool=kp, v_pool=vp, lengths=fake((3,), torch.int32) + 5)
    with pytest.raises(AssertionError, match="a launch"):
        paged.attention_shared(**a)
    a[which] = a[which] + 7
    with pytest.raises(ValueError, match="page ids"):
        paged.attention_shared(**a)
    with pytest.raises(AssertionError, match="a launch"):
        paged.attention_shared(**a, **{{"table": "v_table", "prefix_table": "prefix_v_table"}[which]: a[which] - 7})


@pytest.mark.parametrize("stride,served", [(10_631_104, True), (10_631_112, False)])
def test_rows_of_k_and_v_lie_within_32_bits(stride, served, monkeypatch):
    """10 rows and three tiles behind them, 2 bytes per element: below 2**32 bytes in all."""
    monkeypatch.setattr(lowering, "_check_tensor", lambda *a: None)
    monkeypatch.setattr(packed, "_rows", lambda *a: None)
    q, k, v = qkv()
    far = torch.empty_strided((10, 2, 64), (stride, 64, 1), dtype=k.dtype, device="meta")
    assert (2 * 202 * stride + 128 < 1 << 32) == served
    for a in ((q, far, v), (q, k, far)):
        with pytest.raises(AssertionError if served else UnsupportedPlan, match="a launch" if served else "reach"):
            packed.attention_packed(*a, PLAN, layout(10))


def test_one_row_may_have_any_stride(monkeypatch):
    monkeypatch.setattr(lowering, "_kernels_of", lambda spec: None)
    q, k, v = qkv(T=1)
    far = [t.as_strided(t.shape, (1 << 40, 64, 1)) for t in (q, k, v)]
    with pytest.raises(AssertionError, match="a launch"):
        packed.attention_packed(*far, PLAN, layout(1))
    with pytest.raises(AssertionError, match="a launch"):
        packed.attention_packed_backward(*far, q, fake((4, 1), torch.float32), far[0], PLAN, layout(1))
