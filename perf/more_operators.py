"""Operators between a layer's projections and its attention over a cache, and the sizes that their speed is measured at.

Four operators, each with its plain form in elementary torch operations:

* ``rotate``  -- norms of queries and keys for each head and the rotation by their positions (``rotary.rotate_heads``), inference and
  training (gradients of Q, K and the norms' weights).
* ``append``  -- the same for new tokens, whose keys and values go into their slots of the page pools (``paged.append_kv``).
* ``append4`` -- the same into pools held in 4 bits; what the pools stand for is read back (``paged.read_kv``).
* ``cached``  -- attention of the new tokens of requests of different lengths over their keys and values in such pools, one token per request
  or several (``paged.attention_cached``).

Values in 4 bits are those of a sign, two bits of exponent and one of mantissa, 0 0.5 1 1.5 2 3 4 6, times a power of two that 32 neighbours of a row
share: the least one of which their largest size is below the 7-fold.

A case is a dict of plain values.  Lengths follow from the case alone (the seed shuffles which request has which): request i of n has
``longest * (1 - i / n) ** spread`` tokens.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def _rotate(name, T, longest, pad, Hq, Hkv, D, R, dtype, wtype, pairs, grad):
    return {"name": name, "op": "rotate", "T": T, "longest": longest, "pad": pad, "Hq": Hq, "Hkv": Hkv, "D": D, "R": R, "dtype": dtype, "wtype": wtype,
            "pairs": pairs, "grad": grad}


def _append(name, T, skipped, pages, page, Hq, Hkv, D, R, dtype, wtype, pairs):
    return {"name": name, "op": "append", "T": T, "skipped": skipped, "pages": pages, "page": page, "Hq": Hq, "Hkv": Hkv, "D": D, "R": R, "dtype": dtype,
            "wtype": wtype, "pairs": pairs}


def _append4(name, T, skipped, pages, page, Hq, Hkv, D, R, dtype, pairs):
    return {"name": name, "op": "append4", "T": T, "skipped": skipped, "pages": pages, "page": page, "Hq": Hq, "Hkv": Hkv, "D": D, "R": R, "dtype": dtype,
            "wtype": "", "pairs": pairs}


def _cached(name, B, longest, spread, new, pad, page, Hq, Hkv, D, dtype, mask, window, softcap):
    return {"name": name, "op": "cached", "B": B, "longest": longest, "spread": spread, "new": new, "pad": pad, "page": page, "Hq": Hq, "Hkv": Hkv, "D": D,
            "dtype": dtype, "mask": mask, "window": window, "softcap": softcap}


def listed():
    return [
        # a short prompt of a small model without norms: launches and host work are what a user waits for
        _rotate("rotate_small", 48, 48, 0, 8, 8, 64, 64, "bf16", "", False, False),
        # a training step of documents packed into one tensor, normed heads, weights kept in 32 bits
        _rotate("rotate_train", 8192, 2048, 0, 32, 32, 128, 128, "bf16", "fp32", False, True),
        # a smaller model's, neighbours as pairs, half of each head rotated, grouped heads, a padded end
        _rotate("rotate_train_d64", 6001, 1000, 77, 16, 4, 64, 32, "fp16", "fp16", True, True),
        # the new tokens of one decode step
        _append("append_step", 64, 3, 4096, 16, 32, 8, 128, 128, "bf16", "bf16", False),
        # those of a batch of prompts
        _append("append_prompts", 16384, 100, 2048, 16, 32, 8, 128, 128, "bf16", "", False),
        # one decode step into a cache in 4 bits
        _append4("append4_step", 64, 3, 16, 16, 32, 8, 128, 128, "bf16", False),
        # prompts into such a cache, longer pages
        _append4("append4_prompts", 8192, 50, 160, 64, 32, 8, 128, 64, "fp16", False),
        # two users of a model with grouped heads: latency counts
        _cached("cached_small", 2, 1000, 1, 1, 0, 16, 32, 8, 128, "bf16", "causal", 0, 0.0),
        # a batch of conversations, a token each
        _cached("cached_batch", 64, 8192, 1, 1, 0, 16, 32, 8, 128, "bf16", "causal", 0, 0.0),
        # a few long documents, for which a cache in 4 bits is kept
        _cached("cached_long", 4, 100000, 1, 1, 0, 64, 32, 8, 128, "bf16", "causal", 0, 0.0),
        # drafts of a small model to be looked over, under a window and a softcap, a padded end
        _cached("cached_drafts", 48, 6000, 1, 5, 9, 16, 16, 4, 64, "fp16", "sliding", 1024, 30.0),
        # the next parts of a few prompts, behind what the cache has of them
        _cached("cached_prompts", 4, 6001, 1, 1000, 0, 16, 32, 8, 128, "bf16", "causal", 0, 0.0),
    ]


def _lengths(n, longest, spread):
    return [int(longest * (1 - i / n) ** spread) for i in range(n)]


def _new(case):
    """New tokens of each request: all of them alike, as far as they have so many."""
    return [min(case["new"], n) for n in _lengths(case["B"], case["longest"], case["spread"])]


def work(case):
    op, Hq, Hkv, D = case["op"], case["Hq"], case["Hkv"], case["D"]
    if op == "cached":
        lengths, new = _lengths(case["B"], case["longest"], case["spread"]), _new(case)
        w = case["window"] if case["mask"] == "sliding" else 1 << 40
        pairs = keys = 0
        for n, m in zip(lengths, new):
            if case["mask"] == "none":
                pairs, keys = pairs + n * m, keys + n * (m > 0)
                continue
            pairs += sum(min(p + 1, w) for p in range(n - m, n))
            keys += min(n, w + m - 1) if m else 0
        pages = sum(-(-n // case["page"]) for n in lengths)
        return {"bytes": 2 * keys * Hkv * (D // 2 + D // 32) + 4 * sum(new) * Hq * D + 4 * (pages + 2 * case["B"] + sum(new)), "flops": 4 * Hq * D * pairs}
    T, row = case["T"] - (case["pad"] if op == "rotate" else 0), 2 * D
    table = 4 * case["R"] * min(T, _places(case))
    turned = 2 * T * (Hq + Hkv) * D * (2.0 if case["wtype"] else 1.0)
    if op == "rotate":
        both = (Hq + Hkv) * row * T
        # forward in and out; backward the gradient in, the inputs again where there is a norm, the gradients out
        return {"bytes": 2 * both + (3 if case["wtype"] else 2) * both * case["grad"] + table + 4 * T, "flops": turned * (3 if case["grad"] else 1)}
    kept = case["T"] - case["skipped"]
    bytes_in = (Hq + 2 * Hkv) * row * case["T"] + Hq * row * case["T"] + table + 8 * case["T"]
    if op == "append":
        return {"bytes": bytes_in + 2 * Hkv * row * kept, "flops": turned}
    place = Hkv * (D // 2 + D // 32)
    all_of = case["pages"] * case["page"]
    return {"bytes": bytes_in + 2 * place * kept + 2 * all_of * (place + Hkv * row), "flops": turned}


def _places(case):
    """Positions that the table of angles has."""
    return case["longest"] if case["op"] == "rotate" else 8192


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 6e14)


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("rotate", "rotate", "append", "append4", "cached", "cached", "cached"))
        dtype, D = rng.choice(("bf16", "bf16", "fp16")), rng.choice((64, 128, 128))
        Hkv, group, spread = rng.choice((1, 2, 3, 4, 8, 16, 32)), rng.choice((1, 1, 2, 3, 4, 8, 16)), rng.choice((0, 1, 1, 2, 3))
        wtype, pairs, page = rng.choice(("", dtype, dtype, "fp32")), rng.random() < 0.3, rng.choice((16, 16, 32, 64))
        if Hkv * group > 64:
            continue
        if op == "rotate":
            D = rng.choice((64, 128, 128, 80, 96, 256, 32))
            T = log(1, 16384)
            pad = rng.choice((0, rng.randrange(T)))
            case = _rotate("", T, log(1, 4096), pad, Hkv * group, Hkv, D, rng.choice((D, D, 16 * rng.randint(1, D // 16))), dtype, wtype, pairs, rng.random() < 0.6)
        elif op in ("append", "append4"):
            R = rng.choice((D, D, 16 * rng.randint(1, D // 16)))
            T = log(1, 32768) if op == "append" else log(1, 10000)
            skipped = rng.choice((0, rng.randrange(T)))
            if op == "append":
                page = rng.choice((1, 8, 16, 16, 64))
                case = _append("", T, skipped, -(-T // page) + log(1, 4096), page, Hkv * group, Hkv, D, R, dtype, wtype, pairs)
            else:
                case = _append4("", T, skipped, -(-T // page) + log(1, 64), page, Hkv * group, Hkv, D, R, dtype, pairs)
        else:
            mask = rng.choice(("causal", "causal", "causal", "sliding", "none"))
            new = rng.choice((1, 1, log(2, 16), log(2, 1500)))
            case = _cached("", log(1, 128), log(1, 60000), spread, new, rng.choice((0, 0, log(1, 100))), page, Hkv * group, Hkv, D, dtype, mask,
                           log(16, 4096) if mask == "sliding" else 0, rng.choice((0.0, 0.0, 30.0)))
            # scores and keys of the plain form
            if case["B"] * case["Hq"] * case["longest"] * min(new, case["longest"]) > 1 << 30 or case["B"] * case["longest"] * Hkv * D > 1 << 30:
                continue
        case.pop("name")
        if _cost(case) <= most:
            return case


# ---- what a user's program has in hand -------------------------------------------------------------------

def _angles(count, R, dev):
    """[count, R] in 32 bits: cosines, then sines, of position / 10000 ** (2 i / R)."""
    a = torch.arange(count, device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 / R * torch.arange(R // 2, device=dev, dtype=torch.float64))
    return torch.cat((torch.cos(a), torch.sin(a)), 1).float()


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    op, Hq, Hkv, D = (case[k] for k in ("op", "Hq", "Hkv", "D"))

    def normal(*shape):
        return torch.empty(shape, dtype=_DTYPES[case["dtype"]], device=dev).normal_(generator=gen)

    def channels(*shape):       # rows whose columns differ in size, as keys' do
        x = torch.randn(shape, generator=gen, device=dev)
        return (x * torch.exp(0.7 * torch.randn(shape[-2:], generator=gen, device=dev))).to(_DTYPES[case["dtype"]])

    if op == "cached":
        lengths = torch.tensor(_lengths(case["B"], case["longest"], case["spread"]), dtype=torch.int32, device=dev)
        new = torch.tensor(_new(case), dtype=torch.int32, device=dev)
        order = torch.randperm(case["B"], generator=gen, device=dev)
        lengths, new = lengths[order], new[order]
        page = case["page"]
        have = (lengths + page - 1) // page
        width, count = max(1, -(-case["longest"] // page)), sum(-(-n // page) for n in _lengths(case["B"], case["longest"], case["spread"])) + 3
        ids = torch.randperm(count, generator=gen, device=dev).to(torch.int32)
        first = have.cumsum(0) - have
        j = torch.arange(width, device=dev)
        # entries behind a request's last page hold nothing
        table = torch.where(j < have[:, None], ids[(first[:, None] + j).clamp(max=count - 1)], -1).to(torch.int32)
        offsets = torch.zeros(case["B"] + 1, dtype=torch.int32, device=dev)
        offsets[1:] = new.cumsum(0)
        T = sum(_new(case)) + case["pad"]
        row = torch.arange(T, device=dev)
        of = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
        real, of = of < case["B"], of.clamp(max=case["B"] - 1)
        positions = torch.where(real, lengths[of] - new[of] + row - offsets[of], -1).to(torch.int32)
        return {"case": case, "q": normal(T, Hq, D), "k": channels(count * page, Hkv, D), "v": normal(count * page, Hkv, D), "table": table,
                "lengths": lengths, "offsets": offsets, "positions": positions}
    T, places = case["T"], _places(case)
    state = {"case": case, "angles": _angles(places, case["R"], dev)}
    if op == "rotate":      # documents one behind the other
        at = torch.arange(T, device=dev)
        state["positions"] = torch.where(at < T - case["pad"], at % places, -1).to(torch.int32)
        if case["grad"]:
            state["dq"], state["dk"] = normal(T, Hq, D), normal(T, Hkv, D)
    else:
        state["positions"] = torch.randint(places, (T,), generator=gen, device=dev).to(torch.int32)
        state["slots"] = torch.randperm(case["pages"] * case["page"], generator=gen, device=dev)[:T].to(torch.int32)
        none = torch.randperm(T, generator=gen, device=dev)[:case["skipped"]]
        state["slots"][none] = -1
        state["positions"][none] = -1
        state["v"] = normal(T, Hkv, D)
    state["q"], state["k"] = normal(T, Hq, D), channels(T, Hkv, D)
    if case["wtype"]:
        state["q_weight"], state["k_weight"] = ((1 + 0.3 * torch.randn(D, generator=gen, device=dev)).to(_DTYPES[case["wtype"]]) for _ in range(2))
    if op == "append":
        state["k_pool"], state["v_pool"] = (normal(case["pages"], case["page"], Hkv, D) for _ in range(2))
    if op == "append4":      # what the pools hold of other requests, one of a few rows in each slot
        state["k_old"], state["v_old"] = channels(case["pages"] * case["page"], Hkv, D), normal(case["pages"] * case["page"], Hkv, D)
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if case["op"] == "rotate" and case["grad"]:
        for n in ("q", "k", "q_weight", "k_weight"):
            if n in state:
                state[n].requires_grad_(True)
    if case["op"] in ("append4", "cached"):
        k, v = (state.pop(n) for n in (("k_old", "v_old") if case["op"] == "append4" else ("k", "v")))
        if own:
            from loopfuse_amd.paged import pool4, store_kv
            every = torch.arange(len(k), dtype=torch.int32, device=k.device)
            state["k_pool"], state["v_pool"] = (pool4(len(k) // case["page"], case["page"], case["Hkv"], case["D"], k.dtype, k.device) for _ in range(2))
            store_kv(k, v, state["k_pool"], state["v_pool"], every)
            if case["op"] == "append4":
                state["every"] = every
        else:
            state["k_pool"], state["v_pool"] = _plain_in_4_bits(k), _plain_in_4_bits(v)
    return state


# ---- the operators ---------------------------------------------------------------------------------------

def run(state):
    return (_RUN_OWN if own else _RUN_PLAIN)[state["case"]["op"]](state)


def _norms(state):
    if not state["case"]["wtype"]:
        return {}
    return {"q_weight": state["q_weight"], "k_weight": state["k_weight"], "eps": EPS}


def _own_rotate(state):
    from loopfuse_amd.rotary import rotate_heads
    case = state["case"]
    q, k = rotate_heads(state["q"], state["k"], state["positions"], state["angles"], pairs=case["pairs"], **_norms(state))
    if not case["grad"]:
        return {"q": q, "k": k}
    names = [n for n in ("q", "k", "q_weight", "k_weight") if n in state]
    grads = torch.autograd.grad((q, k), [state[n] for n in names], (state["dq"], state["dk"]))
    return {"q": q, "k": k, **{"d" + n: g for n, g in zip(names, grads)}}


def _own_append(state):
    from loopfuse_amd.paged import append_kv
    q = append_kv(state["q"], state["k"], state["v"], state["k_pool"], state["v_pool"], state["slots"], state["positions"], state["angles"],
                  pairs=state["case"]["pairs"], **_norms(state))
    return {"q": q, "k_pool": state["k_pool"], "v_pool": state["v_pool"]}


def _own_append4(state):
    from loopfuse_amd.paged import append_kv, read_kv
    q = append_kv(state["q"], state["k"], state["v"], state["k_pool"], state["v_pool"], state["slots"], state["positions"], state["angles"],
                  pairs=state["case"]["pairs"])
    k, v = read_kv(state["k_pool"], state["v_pool"], state["every"])
    return {"q": q, "k_pool": k, "v_pool": v}


def _own_cached(state):
    from loopfuse_amd.lowering import AttnPlan
    from loopfuse_amd.paged import attention_cached
    case = state["case"]
    plan = AttnPlan(mask=None if case["mask"] == "none" else case["mask"], window=case["window"], scale=case["D"] ** -0.5, softcap=case["softcap"] or None,
                    k_paged=True, v_paged=True)
    return {"out": attention_cached(state["q"], state["k_pool"], state["v_pool"], plan, state["table"], state["lengths"], state["offsets"], state["positions"])}


def _plain_turn(x, state, weight):
    """The norm of each head and the rotation, in 32 bits."""
    case, R, x = state["case"], state["case"]["R"], x.float()
    live = state["positions"] >= 0
    a = state["angles"][state["positions"].clamp(min=0).long()][:, None]
    cos, sin = a[..., :R // 2], a[..., R // 2:]
    if case["wtype"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    turned, rest = x[..., :R], x[..., R:]
    if case["pairs"]:
        x0, x1 = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1).flatten(-2)
    else:
        x0, x1 = turned[..., :R // 2], turned[..., R // 2:]
        turned = torch.cat((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1)
    return torch.where(live[:, None, None], torch.cat((turned, rest), -1), 0.0)


def _plain_both(state):
    return tuple(_plain_turn(state[n], state, state.get(n + "_weight")).to(state[n].dtype) for n in ("q", "k"))


def _plain_rotate(state):
    q, k = _plain_both(state)
    if not state["case"]["grad"]:
        return {"q": q, "k": k}
    names = [n for n in ("q", "k", "q_weight", "k_weight") if n in state]
    grads = torch.autograd.grad((q, k), [state[n] for n in names], (state["dq"], state["dk"]))
    return {"q": q, "k": k, **{"d" + n: g for n, g in zip(names, grads)}}


def _plain_append(state):
    q, k = _plain_both(state)
    slots = state["slots"].long()
    kept = slots >= 0
    for rows, pool in ((k, state["k_pool"]), (state["v"], state["v_pool"])):
        pool.view(-1, *pool.shape[2:])[slots[kept]] = rows[kept]
    return {"q": q, "k_pool": state["k_pool"], "v_pool": state["v_pool"]}


def _plain_in_4_bits(rows):
    """[rows, heads, D] as codes, two to a byte, and the exponents of the blocks of 32, a byte each."""
    x = rows.float().reshape(*rows.shape[:-1], -1, 32)
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m < 0.875, e - 3, e - 2).clamp(-127, 13 if rows.dtype == torch.float16 else 125)
    a = torch.ldexp(x.abs(), -e[..., None]).clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    a = torch.round(a / step) * step
    code = torch.where(a < 2.0, 2 * a, torch.where(a < 4.0, a + 2, a / 2 + 4)).to(torch.uint8) + 8 * (x < 0).to(torch.uint8)
    code = code.reshape(rows.shape)
    return code[..., 0::2] | code[..., 1::2] << 4, (e + 127).to(torch.uint8)


def _plain_of_4_bits(codes, exponents):
    values = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    values = torch.cat((values, -values))
    x = values[torch.stack((codes & 15, codes >> 4), -1).long()].flatten(-2)
    return torch.ldexp(x.reshape(*exponents.shape, 32), exponents[..., None].int() - 127).flatten(-2)


def _plain_append4(state):
    q, k = _plain_both(state)
    slots = state["slots"].long()
    kept = slots >= 0
    out = {"q": q}
    for name, rows in (("k_pool", k), ("v_pool", state["v"])):
        for held, part in zip(state[name], _plain_in_4_bits(rows[kept])):
            held[slots[kept]] = part
        out[name] = _plain_of_4_bits(*state[name]).to(rows.dtype)
    return out


def _plain_cached(state):
    case, lengths, offsets = state["case"], state["lengths"].long(), state["offsets"].long()
    B, Hq, Hkv, D, page = (case[k] for k in ("B", "Hq", "Hkv", "D", "page"))
    table = state["table"].long().clamp(min=0)
    W, N, T, dev = table.shape[1] * page, max(_new(case)), state["q"].shape[0], table.device

    def keys(pool):      # [B, Hkv, W, D]
        codes, exponents = (t.view(-1, page, *t.shape[1:])[table] for t in pool)
        return _plain_of_4_bits(codes, exponents).reshape(B, W, Hkv, D).permute(0, 2, 1, 3).contiguous()

    if N == 0 or T == 0:
        return {"out": torch.zeros_like(state["q"])}
    i, j = torch.arange(N, device=dev), torch.arange(W, device=dev)
    live = i < (offsets[1:] - offsets[:-1])[:, None]                          # [B, N]
    rows = (offsets[:-1, None] + i).clamp(max=T - 1)
    q = state["q"][rows].float().reshape(B, N, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    k = keys(state["k_pool"])
    s = torch.matmul(q, k.transpose(-2, -1).contiguous()).reshape(B, Hkv, -1, N, W) * D ** -0.5
    del k
    if case["softcap"]:
        s = torch.tanh(s / case["softcap"]) * case["softcap"]
    p = torch.where(live, state["positions"].long()[rows], -1)[..., None]     # [B, N, 1]
    keep = (j < lengths[:, None, None]) & live[..., None]
    if case["mask"] != "none":
        keep = keep & (j <= p)
    if case["mask"] == "sliding":
        keep = keep & (p - j < case["window"])
    s = s.masked_fill(~keep[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    del s
    e = e / e.sum(-1, keepdim=True).clamp(min=1e-30)                          # a row without a key: zeros
    o = torch.matmul(e.reshape(B, Hkv, -1, W), keys(state["v_pool"])).reshape(B, Hkv, -1, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, Hq, D)
    out = torch.zeros(state["q"].shape, device=dev)
    out[rows[live]] = o[live]
    return {"out": out.to(state["q"].dtype)}


_RUN_OWN = {"rotate": _own_rotate, "append": _own_append, "append4": _own_append4, "cached": _own_cached}
_RUN_PLAIN = {"rotate": _plain_rotate, "append": _plain_append, "append4": _plain_append4, "cached": _plain_cached}


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------

def exact(case, seed):
    state = _inputs(case, seed)
    if case["op"] == "cached":
        return _exact_cached(case, state)
    q, k = _exact_turn(case, state, "q"), _exact_turn(case, state, "k")
    if case["op"] == "rotate":
        out = {"q": q[0], "k": k[0]}
        if case["grad"]:
            for n, made in (("q", q), ("k", k)):
                x, w = made[1](state["d" + n].double())
                out["d" + n] = x
                if case["wtype"]:
                    out[f"d{n}_weight"] = w
        return out
    held = {}
    for name, rows, old in (("k_pool", k[0], "k_old"), ("v_pool", state["v"].double(), "v_old")):
        if case["op"] == "append4":
            pool = _exact_4_bits(state[old].double(), case["dtype"])
            rows = _exact_4_bits(rows.to(_DTYPES[case["dtype"]]).double(), case["dtype"])
        else:
            pool = state[name].double().reshape(-1, case["Hkv"], case["D"])
        # which row a slot holds: the one that names it, or none
        holds = torch.full((pool.shape[0] + 1,), -1, dtype=torch.long, device=pool.device)
        holds[state["slots"].long()] = torch.arange(case["T"], device=pool.device)           # -1 names the one behind the last
        holds = holds[:-1]
        pool = torch.where((holds >= 0)[:, None, None], rows[holds.clamp(min=0)], pool)
        held[name] = pool if case["op"] == "append4" else pool.reshape(state[name].shape)
    return {"q": q[0], **held}


def _exact_turn(case, state, name):
    """(result, gradient -> (gradient of the rows, of the weight)): the rotation as a product of complex numbers."""
    R, D, x = case["R"], case["D"], state[name].double()
    dead = state["positions"] < 0
    turn = torch.complex(*state["angles"].double()[state["positions"].long().clamp(min=0)].split(R // 2, 1))[:, None]
    turn = torch.where(dead[:, None, None], 0.0, turn)

    def rotated(y, by):
        z = torch.complex(y[..., :R:2], y[..., 1:R:2]) if case["pairs"] else torch.complex(y[..., :R // 2], y[..., R // 2:R])
        z = z * by
        res = torch.where(dead[:, None, None], 0.0, y)
        if case["pairs"]:
            res[..., :R:2], res[..., 1:R:2] = z.real, z.imag
        else:
            res[..., :R // 2], res[..., R // 2:R] = z.real, z.imag
        return res

    if not case["wtype"]:
        return rotated(x, turn), lambda g: (rotated(g, turn.conj()), None)
    w = state[name + "_weight"].double()
    size = (x.square().sum(-1, keepdim=True) / D + EPS).sqrt()
    n = x / size

    def back(g):
        g = rotated(g, turn.conj())
        h = g * w
        return (h - n * (h * n).sum(-1, keepdim=True) / D) / size, (g * n).sum((0, 1))

    return rotated(n * w, turn), back


def _exact_4_bits(rows, dtype):
    """The values that rows in 4 bits stand for."""
    x = rows.unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=1e-300) / 7)) + 1
    e = torch.where(top >= 7 * 2.0 ** e, e + 1, torch.where(top < 7 * 2.0 ** (e - 1), e - 1, e)).clamp(-127, 13 if dtype == "fp16" else 125)
    y = x / 2.0 ** e
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    middles = (grid[1:] + grid[:-1]) / 2
    up, down = torch.bucketize(y.abs(), middles, right=True), torch.bucketize(y.abs(), middles)      # ties up, and down: to the even one
    return (torch.sign(y) * grid[torch.where(up % 2 == 0, up, down)] * 2.0 ** e).flatten(-2)


def _exact_cached(case, state):
    Hq, Hkv, D, page, c = (case[k] for k in ("Hq", "Hkv", "D", "page", "softcap"))
    g, out = Hq // Hkv, torch.zeros(state["q"].shape, dtype=torch.float64, device=state["q"].device)
    ends, places = state["offsets"].tolist(), state["positions"].long()
    for b, n in enumerate(state["lengths"].tolist()):
        lo, hi = ends[b], ends[b + 1]
        if n == 0 or lo == hi:
            continue
        at = torch.arange(n, device=out.device)
        at = state["table"][b].long()[at // page] * page + at % page
        k, v = (_exact_4_bits(state[name][at].double(), case["dtype"]).permute(1, 0, 2).contiguous() for name in ("k", "v"))
        j, p = torch.arange(n, device=out.device), places[lo:hi, None]
        hidden = torch.zeros((hi - lo, n), dtype=torch.bool, device=out.device) if case["mask"] == "none" else j > p
        if case["mask"] == "sliding":
            hidden = hidden | (p - j >= case["window"])
        for h in range(Hkv):
            q = state["q"][lo:hi, h * g:(h + 1) * g].double().permute(1, 0, 2).contiguous()
            x = (q.reshape(-1, D) @ k[h].t().contiguous()).reshape(g, hi - lo, n) * D ** -0.5
            if c:
                x = c * torch.tanh(x / c)
            x = torch.softmax(x.masked_fill(hidden, float("-inf")), -1)
            out[lo:hi, h * g:(h + 1) * g] = (x.reshape(-1, n) @ v[h]).reshape(g, hi - lo, D).permute(1, 0, 2)
    return {"out": out}
