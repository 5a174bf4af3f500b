"""Attention over packed sequences (``packed.attention_packed``, forward and backward) against the formulas in 64 bits, sequence
by sequence.

Tolerances.  With e the half step of the operands' type (2^-8 bf16, 2^-11 fp16) a result may be off by
  O  : e (P |V|)   the probabilities are rounded for the second product, + e |O| for the result,
  dV : e (P^T |dO|) + e |dV|,
  dK : scale (|E|^T |Q|) + e |dK|,  dQ : scale (|E| |K|) + e |dQ|,  where E = e |dS| + P (|dO| . e (P |V| + |O|)): dS is rounded for
       the products, and delta is formed of the rounded O,
each with what the sums in 32 bits add: a probability is off by 2^-17 scale |Q| |K| (128 products) + 2^-20 of itself, and with a
softcap by 1e-4 (its polynomial); dP and delta by 2^-17 of the sums of their terms' sizes.  fp16 operands have a least step of 2^-24:
half of one per element of P (relative to a row's maximum) and of dS."""
import math

import pytest
import torch

from loopfuse_amd import lowering, packed
from loopfuse_amd.lowering import AttnPlan

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def oracle(q, k, v, dout, bounds, mask, window, scale, cap):
    """{name: (value, bound)} for out, lse, dq, dk, dv of the packed sequences; rows of none are zero with bound zero."""
    e = torch.finfo(q.dtype).eps / 2
    least = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    Hq, Hkv = q.shape[1], k.shape[1]
    names = {"out": q, "dq": q, "dk": k, "dv": v}
    res = {n: tuple(torch.zeros(t.shape, dtype=torch.float64, device=q.device) for _ in range(2)) for n, t in names.items()}
    lse = torch.zeros((Hq, q.shape[0]), dtype=torch.float64, device=q.device)
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        n = hi - lo
        if n == 0:
            continue
        i = torch.arange(n, device=q.device)
        rel = i[:, None] - i[None, :]
        keep = torch.ones_like(rel, dtype=torch.bool) if mask is None else rel >= 0
        if mask == "sliding":
            keep &= rel < window
        for h in range(Hq):
            a = h // (Hq // Hkv)
            qh, kh, vh, gh = q[lo:hi, h].double(), k[lo:hi, a].double(), v[lo:hi, a].double(), dout[lo:hi, h].double()
            s = qh @ kh.t() * scale
            th = torch.tanh(s / cap) if cap else None
            x = (cap * th if cap else s).masked_fill(~keep, -math.inf)
            L = torch.logsumexp(x, dim=-1, keepdim=True)
            p = torch.exp(x - L)
            o = p @ vh
            er = e + 2.0 ** -17 * scale * (qh.abs() @ kh.abs().t()) + 2.0 ** -20 + (1e-4 if cap else 0.0)      # of a probability, relative
            ep = p * er + least * keep
            av = ep @ vh.abs()
            eo = av + e * o.abs() + (p * (er - e)) @ vh.abs()
            dp, d = gh @ vh.t(), (gh * o).sum(-1, keepdim=True)
            ds = p * (dp - d)
            sums = 2.0 ** -17 * (gh.abs() @ vh.abs().t() + (gh.abs() * o.abs()).sum(-1, keepdim=True))
            es = ds.abs() * er + least * keep + p * ((gh.abs() * eo).sum(-1, keepdim=True) + sums)
            if cap:
                ds, es = ds * (1 - th * th), es * (1 - th * th) + 1e-4 * p * (dp - d).abs()
            res["out"][0][lo:hi, h], res["out"][1][lo:hi, h] = o, eo
            res["dq"][0][lo:hi, h], res["dq"][1][lo:hi, h] = scale * (ds @ kh), scale * (es @ kh.abs())
            res["dk"][0][lo:hi, a] += scale * (ds.t() @ qh)
            res["dk"][1][lo:hi, a] += scale * (es.t() @ qh.abs())
            res["dv"][0][lo:hi, a] += p.t() @ gh
            res["dv"][1][lo:hi, a] += ep.t() @ gh.abs()
            lse[h, lo:hi] = L[:, 0] / math.log(2.0)
    for n in ("dq", "dk", "dv"):
        res[n][1].add_(e * res[n][0].abs())
    # the results' own least step, and the sums' (2^-17 of the sizes is in the bounds already where e is)
    return {n: (x, b * 1.01 + (least if least else 1e-30)) for n, (x, b) in res.items()}, lse


def check(got, want, what):
    value, bound = want
    err = (got.double() - value).abs()
    assert not torch.isnan(got).any(), f"{what}: NaN"
    worst = (err - bound).max().item()
    assert worst <= 0, f"{what}: {worst} beyond its bound, at an error of {err.max().item()}"


def inputs(lengths, Hq, Hkv, D, dtype, seed=1, head=0, tail=0, scale=1.0):
    """Q, K, V, dO and the bounds; ``head`` / ``tail`` rows of no sequence hold NaN."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    T = head + sum(lengths) + tail
    q, k, v, g = (torch.randn((T, h, D), generator=gen, device=DEV).mul(scale).to(dtype) for h in (Hq, Hkv, Hkv, Hq))
    for t in (q, k, v, g):
        t[:head] = math.nan
        t[T - tail:] = math.nan
    bounds = [head]
    for n in lengths:
        bounds.append(bounds[-1] + n)
    return q, k, v, g, bounds


def layout_of(bounds, T, dtype=torch.int32):
    return packed.packed_layout(torch.tensor(bounds, dtype=dtype, device=DEV), T)


CASES = [
    # lengths, Hq, Hkv, D, dtype, mask, window, softcap, rows of no sequence in front and behind
    ([1], 1, 1, 64, torch.bfloat16, "causal", 0, None, 0, 0),
    ([1, 0, 2, 31, 32, 33, 0], 2, 2, 128, torch.bfloat16, "causal", 0, None, 0, 5),
    ([127, 128, 129, 300], 4, 4, 128, torch.float16, None, 0, None, 3, 0),
    ([0, 0, 0], 2, 1, 64, torch.float16, "causal", 0, None, 0, 70),
    ([500, 1, 257, 64], 8, 2, 128, torch.bfloat16, "causal", 0, None, 0, 130),
    ([500, 1, 257, 64], 8, 4, 64, torch.float16, "causal", 0, None, 0, 0),
    ([700, 90, 5], 6, 2, 128, torch.float16, "sliding", 100, None, 0, 0),
    ([700, 90, 5], 6, 6, 64, torch.bfloat16, "sliding", 1, None, 1, 1),
    ([333, 200], 4, 1, 128, torch.bfloat16, "sliding", 65, 30.0, 0, 0),
    ([333, 200], 3, 3, 64, torch.float16, "causal", 0, 20.0, 0, 9),
    ([260, 515], 16, 2, 128, torch.float16, None, 0, 5.0, 0, 0),
    ([2100, 1030], 2, 1, 128, torch.bfloat16, "causal", 0, None, 0, 0),
    ([40] * 70, 2, 2, 64, torch.bfloat16, "causal", 0, None, 0, 0),
]


@pytest.mark.parametrize("lengths,Hq,Hkv,D,dtype,mask,window,cap,head,tail", CASES)
def test_forward_and_gradients_are_the_formulas(lengths, Hq, Hkv, D, dtype, mask, window, cap, head, tail):
    q, k, v, g, bounds = inputs(lengths, Hq, Hkv, D, dtype, len(lengths) + D, head, tail)
    plan = AttnPlan(mask, window=window, scale=D ** -0.5, softcap=cap)
    layout = layout_of(bounds, q.shape[0])
    want, lse_ref = oracle(q, k, v, g, bounds, mask, window, D ** -0.5, cap)
    out = packed.attention_packed(q, k, v, plan, layout)
    check(out, want["out"], "out")
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out2 = packed.attention_packed(*leaves, plan, layout)
    assert torch.equal(out2, out)
    grads = torch.autograd.grad(out2, leaves, g)
    for name, t in zip(("dq", "dk", "dv"), grads):
        check(t, want[name], name)
    again = torch.autograd.grad(packed.attention_packed(*leaves, plan, layout), leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    # into a given tensor: rows of no sequence stay as they were; the log-sum-exp
    given, lse = torch.full_like(q, 7.0), torch.full((Hq, q.shape[0]), 5.0, device=DEV)
    assert packed.attention_packed(q, k, v, plan, layout, out=given, lse=lse) is given
    lo, hi = bounds[0], bounds[-1]
    assert torch.equal(given[lo:hi], out[lo:hi]) and (given[:lo] == 7).all() and (given[hi:] == 7).all()
    assert (lse[:, :lo] == 5).all() and (lse[:, hi:] == 5).all()
    assert (lse[:, lo:hi].double() - lse_ref[:, lo:hi]).abs().max().item() <= 2e-3 if hi > lo else True


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D,mask", [(2, 2, 64, "causal"), (8, 2, 128, "causal"), (4, 2, 128, None), (8, 1, 64, "sliding")])
def test_what_rounding_takes_from_the_result_is_kept_for_the_backward(Hq, Hkv, D, mask, dtype):
    # Q = 0: every probability is 1 / (number of keys), exact before the sum, so that O in 32 bits is the mean of V but for what its n
    # sums, the reciprocal and one product round, and O + low is off by that and by half a step of low
    lengths, lead = [1, 2, 0, 31, 130, 257], 3
    bounds = [lead]
    for n in lengths:
        bounds.append(bounds[-1] + n)
    T = bounds[-1] + 5
    g = torch.Generator(DEV).manual_seed(4)
    q = torch.zeros(T, Hq, D, dtype=dtype, device=DEV)
    k, v = ((2 * torch.rand(T, Hkv, D, generator=g, device=DEV) - 1).to(dtype) for _ in range(2))
    layout = packed.packed_layout(torch.tensor(bounds, dtype=torch.int32, device=DEV), T)
    plan = AttnPlan(mask, window=40, scale=1.0)
    lse, low = torch.empty(Hq, T, device=DEV), torch.full_like(q, math.nan)
    out = packed._forward(q, k, v, plan, layout, None, lse, low)
    want, _ = oracle(q, k, v, torch.zeros_like(q), bounds, mask, 40, 1.0, None)
    rows = slice(lead, bounds[-1])
    value, l64 = want["out"][0][rows], low[rows].double()
    off = (out[rows].double() + l64 - value).abs()
    bound = (257 + 4) * 2.0 ** -24 + torch.finfo(dtype).eps / 2 * l64.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert (off <= bound).all(), (off - bound).max()
    assert (out[rows].double() - value).abs().max() > 8 * bound.max()      # (what O alone is off by)
    assert torch.isnan(low[:lead]).all() and torch.isnan(low[bounds[-1]:]).all()
    dout = torch.randn(q.shape, generator=g, device=DEV).to(dtype)
    for name, t in zip(("dq", "dk", "dv"), packed._backward(q, k, v, out, lse, dout, plan, layout, low)):
        assert torch.isfinite(t).all(), name
