"""The operators for different lengths over operands whose rows lie together or that name what is not there: gradients without memory of their own,
pages that are none, the largest sizes."""
import pytest
import torch

from loopfuse_amd import packed
from loopfuse_amd.lowering import AttnPlan
from test_packed_gpu import check, inputs, layout_of, oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def formulas(q, k, v, g, bounds, plan):
    return oracle(q, k, v, g, bounds, plan.mask, plan.window, plan.scale, plan.softcap)[0]


# ---- rows that lie together: their reads behind a sequence's last row are not zeros ---------------------------------------------

@pytest.mark.parametrize("lengths,Hq,Hkv,D,mask,cap", [([50, 1, 97, 33], 4, 2, 64, "causal", None), ([70, 131, 5], 4, 2, 128, None, None), ([45, 300], 2, 1, 128, "sliding", 20.0),
                                                       ([1], 2, 2, 128, "causal", None), ([1], 2, 2, 64, "causal", None)])
def test_output_gradients_whose_rows_are_one(lengths, Hq, Hkv, D, mask, cap):
    """The gradient of a sum over rows and an expanded one have a row stride of 0."""
    q, k, v, g, bounds = inputs(lengths, Hq, Hkv, D, torch.bfloat16, 3)
    plan, layout = AttnPlan(mask, window=60, scale=D ** -0.5, softcap=cap), layout_of(bounds, len(q))
    w = g[0].clone()
    want = formulas(q, k, v, w.expand_as(q), bounds, plan)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    for _ in range(2):
        out = packed.attention_packed(*leaves, plan, layout)
        summed = torch.autograd.grad((out.sum(0) * w).sum(), leaves)
        expanded = torch.autograd.grad(packed.attention_packed(*leaves, plan, layout), leaves, w.expand_as(q))
        lse = torch.empty((Hq, len(q)), device=DEV)
        o = packed.attention_packed(q, k, v, plan, layout, lse=lse)
        direct = packed.attention_packed_backward(q, k, v, o, lse, w.expand_as(q), plan, layout)
        for how, grads in (("sum", summed), ("expanded", expanded)):
            for name, t in zip(("dq", "dk", "dv"), grads):
                check(t, want[name], f"{how} {name}")
        check(direct[2], want["dv"], "direct dv")


@pytest.mark.parametrize("D,mask", [(64, "causal"), (128, None)])
def test_operands_whose_rows_are_one(D, mask):
    """Q, K or V of one row expanded over all rows, and rows that overlap: as their copies."""
    q, k, v, g, bounds = inputs([50, 1, 97], 4, 2, D, torch.bfloat16, 5)
    T = len(q)
    plan, layout = AttnPlan(mask, scale=D ** -0.5), layout_of(bounds, T)
    over = torch.randn(8 * T + 4 * D, generator=torch.Generator(DEV).manual_seed(6), device=DEV).to(torch.bfloat16)
    for i in range(3):
        heads = (q, k, v)[i].shape[1]
        for t in ((q, k, v)[i][:1].expand(T, -1, -1), over.as_strided((T, heads, D), (8, D, 1))):
            views = [t if j == i else x for j, x in enumerate((q, k, v))]
            copies = [x.clone(memory_format=torch.contiguous_format) for x in views]
            lse = torch.empty((4, T), device=DEV)
            o = packed.attention_packed(*copies, plan, layout, lse=lse)
            assert torch.equal(packed.attention_packed(*views, plan, layout), o)
            want = packed.attention_packed_backward(*copies, o, lse, g, plan, layout)
            for _ in range(2):
                got = packed.attention_packed_backward(*views, o, lse, g, plan, layout)
                assert all(torch.equal(a, b) for a, b in zip(got, want)), (i, t.stride())
            a, b = ([x.detach().requires_grad_(True) for x in y] for y in (views, copies))
            a, b = (torch.autograd.grad(packed.attention_packed(*y, plan, layout), y, g) for y in (a, b))
            assert all(torch.equal(x, y) for x, y in zip(a, b)), (i, t.stride())
