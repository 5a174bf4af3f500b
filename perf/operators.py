"""Operators for batches of requests of different lengths, and the sizes that their speed is measured at.

Four operators, each with its plain form in elementary torch operations:

* ``packed`` -- attention over sequences of different lengths that stand one behind the other in one tensor (``packed.attention_packed``),
  inference and training (gradients of Q, K and V).
* ``shared`` -- one new token per request against keys in pages: a prefix that all requests share, and each request's own keys
  (``paged.attention_shared``).
* ``tables`` -- the pages that requests need for their new tokens, taken from a list of free ones, and the slot of every new token
  (``paged.extend_tables``).
* ``store``  -- the rows of new keys and values into their slots of the page pools (``paged.store_kv``).

A case is a dict of plain values.  Lengths follow from the case alone (the seed shuffles which request has which): request i of n has
``longest * (1 - i / n) ** spread`` tokens, so that 0 makes them equal, 1 spreads them evenly and 2 or 3 leave a few long ones among
many short and empty ones.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _packed(name, N, longest, spread, pad, Hq, Hkv, D, dtype, mask, window, softcap, grad):
    return {"name": name, "op": "packed", "N": N, "longest": longest, "spread": spread, "pad": pad, "Hq": Hq, "Hkv": Hkv, "D": D,
            "dtype": dtype, "mask": mask, "window": window, "softcap": softcap, "grad": grad}


def _shared(name, B, prefix, longest, spread, page, Hq, Hkv, D, dtype, softcap):
    return {"name": name, "op": "shared", "B": B, "prefix": prefix, "longest": longest, "spread": spread, "page": page,
            "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "softcap": softcap}


def _tables(name, B, cached, new, spread, page, pad):
    return {"name": name, "op": "tables", "B": B, "cached": cached, "new": new, "spread": spread, "page": page, "pad": pad}


def _store(name, T, skipped, pages, page, Hkv, D, dtype):
    return {"name": name, "op": "store", "T": T, "skipped": skipped, "pages": pages, "page": page, "Hkv": Hkv, "D": D, "dtype": dtype}


def listed():
    return [
        # three short prompts of a small model: launches and host work are what a user waits for
        _packed("packed_small", 3, 48, 1, 0, 8, 8, 64, "bf16", "causal", 0, 0.0, False),
        # the prompts that a serving step takes in, 2k tokens at most, grouped heads, a padded end
        _packed("packed_prompts", 12, 2048, 1, 100, 32, 8, 128, "bf16", "causal", 0, 0.0, False),
        # layers with local attention and a softcap over a few long documents of odd lengths
        _packed("packed_window_cap", 5, 4001, 1, 0, 32, 8, 128, "fp16", "sliding", 256, 30.0, False),
        # a training step's attention over documents packed into one row, all heads with K/V of their own
        _packed("packed_train", 8, 2048, 1, 0, 32, 32, 128, "bf16", "causal", 0, 0.0, True),
        # a smaller model's: head dim 64, grouped heads, many short documents and a padded end
        _packed("packed_train_d64", 24, 1000, 2, 77, 16, 4, 64, "fp16", "causal", 0, 0.0, True),
        # two users behind one system prompt: latency counts
        _shared("shared_small", 2, 1000, 40, 1, 16, 32, 8, 128, "bf16", 0.0),
        # a batch of conversations behind one system prompt
        _shared("shared_batch", 64, 2048, 1024, 1, 16, 32, 8, 128, "bf16", 0.0),
        # many short answers to one long document
        _shared("shared_long", 128, 8208, 300, 1, 16, 32, 8, 128, "fp16", 0.0),
        # one decode step of a batch: a token each, a new page now and then
        _tables("tables_step", 64, 2048, 1, 1, 16, 0),
        # the prompts of a full batch, whose pages are all new
        _tables("tables_prompts", 256, 0, 2048, 1, 16, 500),
        # the keys and values of one decode step
        _store("store_step", 64, 3, 4096, 16, 8, 128, "bf16"),
        # those of a batch of prompts
        _store("store_prompts", 16384, 100, 2048, 16, 8, 128, "bf16"),
    ]


def _lengths(n, longest, spread):
    return [int(longest * (1 - i / n) ** spread) for i in range(n)]


def _pairs(length, mask, window):
    """(query, key) pairs of one sequence."""
    if mask == "none":
        return length * length
    w = min(window, length) if mask == "sliding" else length
    return w * (w + 1) // 2 + (length - w) * w


def work(case):
    op = case["op"]
    if op == "packed":
        lengths = _lengths(case["N"], case["longest"], case["spread"])
        Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
        product = 2 * Hq * D * sum(_pairs(n, case["mask"], case["window"]) for n in lengths)
        q, kv = 2 * sum(lengths) * Hq * D, 2 * sum(lengths) * Hkv * D
        if case["grad"]:     # two products forward, five backward; Q, dO, K, V in, O, dQ, dK, dV out
            return {"bytes": 4 * q + 4 * kv, "flops": 7 * product}
        return {"bytes": 2 * q + 2 * kv, "flops": 2 * product}
    if op == "shared":
        lengths = _lengths(case["B"], case["longest"], case["spread"])
        B, L, Hq, Hkv, D = (case[k] for k in ("B", "prefix", "Hq", "Hkv", "D"))
        pages = -(-L // case["page"]) + sum(-(-n // case["page"]) for n in lengths)
        return {"bytes": 4 * (L + sum(lengths)) * Hkv * D + 4 * B * Hq * D + 4 * (pages + B), "flops": 4 * Hq * D * (B * L + sum(lengths))}
    if op == "tables":
        cached, new = _requests(case)
        need = sum(-(-(c + n) // case["page"]) - -(-c // case["page"]) for c, n in zip(cached, new))
        used = sum(-(-(c + n) // case["page"]) - c // case["page"] for c, n in zip(cached, new) if n)
        T = sum(new) + case["pad"]
        # lengths in and out, offsets, free pages read, entries of the table written (new ones) and read (a last page that was there), slots, positions
        return {"bytes": 4 * (4 * case["B"] + 2 * need + (used - need) + 2 * T), "flops": 0}
    row = case["Hkv"] * case["D"] * 2
    return {"bytes": 4 * row * (case["T"] - case["skipped"]) + 4 * case["T"], "flops": 0}


def _requests(case):
    """Tokens in the cache and new ones of each request: a decode step (``new`` 1) or prompts."""
    if case["new"] == 1:
        return _lengths(case["B"], case["cached"], case["spread"]), [1] * case["B"]
    new = _lengths(case["B"], case["new"], case["spread"])
    return [case["cached"] * (i % 3) // 2 for i in range(case["B"])], new


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 6e14)


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("packed", "packed", "packed", "shared", "shared", "tables", "store"))
        dtype, D = rng.choice(("bf16", "bf16", "fp16")), rng.choice((64, 128, 128))
        Hkv, group, spread = rng.choice((1, 2, 3, 4, 8, 16, 32)), rng.choice((1, 1, 2, 3, 4, 8)), rng.choice((0, 1, 1, 2, 3))
        page = rng.choice((1, 8, 16, 16, 64))
        if Hkv * group > 64:
            continue
        if op == "packed":
            mask = rng.choice(("causal", "causal", "causal", "sliding", "none"))
            case = _packed("", log(1, 64), log(1, 6000), spread, rng.choice((0, log(1, 300))), Hkv * group, Hkv, D, dtype, mask,
                           log(16, 2048) if mask == "sliding" else 0, rng.choice((0.0, 0.0, 30.0)), rng.random() < 0.5)
            if case["N"] * case["Hq"] * case["longest"] ** 2 > 1 << 30:       # scores of the plain form
                continue
        elif op == "shared":
            case = _shared("", log(1, 128), rng.choice((0, log(1, 16384), log(256, 16384))), log(1, 4096), spread, page, Hkv * group, Hkv, D, dtype,
                           rng.choice((0.0, 0.0, 30.0)))
            if case["B"] * case["Hq"] * (case["prefix"] + case["longest"]) > 1 << 28:
                continue
        elif op == "tables":
            step = rng.random() < 0.5
            case = _tables("", log(1, 1024), rng.choice((0, log(1, 8192))), 1 if step else log(2, 4096), spread, page, rng.choice((0, log(1, 300))))
        else:
            T = log(1, 32768)
            case = _store("", T, rng.choice((0, rng.randrange(T))), -(-T // page) + log(1, 4096), page, Hkv, D, dtype)
        case.pop("name")
        if _cost(case) <= most:
            return case


# ---- what a user's program has in hand -------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]

    def normal(*shape):
        return torch.empty(shape, dtype=_DTYPES[case["dtype"]], device=dev).normal_(generator=gen)

    def shuffled(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)[torch.randperm(len(values), generator=gen, device=dev)]

    def pages_of(count):
        return torch.randperm(count, generator=gen, device=dev).to(torch.int32)

    if op == "packed":
        lengths = shuffled(_lengths(case["N"], case["longest"], case["spread"]))
        offsets = torch.zeros(case["N"] + 1, dtype=torch.int32, device=dev)
        offsets[1:] = lengths.cumsum(0)
        T = sum(_lengths(case["N"], case["longest"], case["spread"])) + case["pad"]
        q, k, v = normal(T, case["Hq"], case["D"]), normal(T, case["Hkv"], case["D"]), normal(T, case["Hkv"], case["D"])
        state = {"case": case, "q": q, "k": k, "v": v, "offsets": offsets}
        if case["grad"]:
            for t in (q, k, v):
                t.requires_grad_(True)
            state["dout"] = normal(T, case["Hq"], case["D"])
        if own:        # the layout of a batch serves all layers of a model, forward and backward
            from loopfuse_amd.packed import packed_layout
            state["layout"] = packed_layout(offsets, T)
        return state
    if op == "shared":
        lengths = _lengths(case["B"], case["longest"], case["spread"])
        page, pre = case["page"], -(-case["prefix"] // case["page"])
        width = max(1, -(-max(lengths) // page))
        count = pre + case["B"] * width
        order = pages_of(count)
        lengths = shuffled(lengths)
        table = order[pre:].view(case["B"], width)
        # entries behind a request's last page hold nothing
        table = torch.where(torch.arange(width, device=dev) < ((lengths + page - 1) // page)[:, None], table, -1).contiguous()
        pool = (count, page, case["Hkv"], case["D"])
        return {"case": case, "q": normal(case["B"], case["Hq"], 1, case["D"]), "k_pool": normal(*pool), "v_pool": normal(*pool),
                "table": table, "lengths": lengths, "prefix_table": order[:pre].contiguous()}
    if op == "tables":
        cached, new = _requests(case)
        page, B = case["page"], case["B"]
        order = torch.randperm(B, generator=gen, device=dev)
        width = max(1, max(-(-(c + n) // page) for c, n in zip(cached, new)))
        cached = torch.tensor(cached, dtype=torch.int32, device=dev)[order]
        total = sum(new) + case["pad"]
        need = sum(-(-n // page) + 1 for n in new)
        new = torch.tensor(new, dtype=torch.int32, device=dev)[order]
        ids = pages_of(B * width + need)
        have = (cached + page - 1) // page
        table = torch.where(torch.arange(width, device=dev) < have[:, None], ids[:B * width].view(B, width), -1).contiguous()
        return {"case": case, "cached": cached, "new": new, "table": table, "free": ids[B * width:].contiguous(), "total": total}
    slots = torch.randperm(case["pages"] * case["page"], generator=gen, device=dev)[:case["T"]].to(torch.int32)
    slots[torch.randperm(case["T"], generator=gen, device=dev)[:case["skipped"]]] = -1
    pool = (case["pages"], case["page"], case["Hkv"], case["D"])
    return {"case": case, "k": normal(case["T"], case["Hkv"], case["D"]), "v": normal(case["T"], case["Hkv"], case["D"]),
            "k_pool": normal(*pool), "v_pool": normal(*pool), "slots": slots}


# ---- the operators ---------------------------------------------------------------------------------------

def run(state):
    return (_RUN_OWN if own else _RUN_PLAIN)[state["case"]["op"]](state)


def _plan(case, paged):
    from loopfuse_amd.lowering import AttnPlan
    mask = case.get("mask", "none")
    return AttnPlan(mask=None if mask == "none" else mask, window=case.get("window", 0), scale=case["D"] ** -0.5,
                    softcap=case["softcap"] or None, k_paged=paged, v_paged=paged)


def _own_packed(state):
    from loopfuse_amd.packed import attention_packed
    case, q, k, v = state["case"], state["q"], state["k"], state["v"]
    out = attention_packed(q, k, v, _plan(case, False), state["layout"])
    if not case["grad"]:
        return {"out": out}
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), state["dout"])
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _own_shared(state):
    from loopfuse_amd.paged import attention_shared
    return {"out": attention_shared(state["q"], state["k_pool"], state["v_pool"], _plan(state["case"], True), state["table"], state["lengths"],
                                    prefix_table=state["prefix_table"], prefix_len=state["case"]["prefix"])}


def _own_tables(state):
    from loopfuse_amd.paged import extend_tables
    step = extend_tables(state["cached"], state["new"], state["table"], state["free"], state["case"]["page"], state["total"])
    return {"table": state["table"], "offsets": step.offsets, "lengths": step.lengths, "slots": step.slots, "positions": step.positions,
            "pages": step.pages}


def _own_store(state):
    from loopfuse_amd.paged import store_kv
    store_kv(state["k"], state["v"], state["k_pool"], state["v_pool"], state["slots"])
    return {"k_pool": state["k_pool"], "v_pool": state["v_pool"]}


def _plain_packed(state):
    case, offsets = state["case"], state["offsets"].long()
    N, Hq, Hkv, D = case["N"], case["Hq"], case["Hkv"], case["D"]
    T, L, dev = state["q"].shape[0], max(case["longest"], 1), offsets.device
    length = offsets[1:] - offsets[:-1]
    at = torch.arange(L, device=dev)
    live = at < length[:, None]                                               # [N, L]
    rows = (offsets[:-1, None] + at).clamp(max=T - 1) * live

    def padded(t):      # [N, H, L, D] in 32 bits
        return t[rows].float().permute(0, 2, 1, 3)

    q = padded(state["q"]).reshape(N, Hkv, Hq // Hkv, L, D)
    k, v = padded(state["k"])[:, :, None], padded(state["v"])[:, :, None]
    s = torch.matmul(q, k.transpose(-2, -1).contiguous()) * D ** -0.5
    if case["softcap"]:
        s = torch.tanh(s / case["softcap"]) * case["softcap"]
    i, j = at[:, None], at[None, :]
    keep = (j < length[:, None, None]) & torch.ones_like(j <= i)
    if case["mask"] != "none":
        keep = keep & (j <= i)
    if case["mask"] == "sliding":
        keep = keep & (i - j < case["window"])
    keep = torch.where(live[:, :, None], keep, j == 0)                        # rows of no sequence: any key, so that they hold numbers
    s = s.masked_fill(~keep[:, None, None], float("-inf"))
    e = torch.exp(s - s.amax(-1, keepdim=True).detach())
    o = torch.matmul(e / e.sum(-1, keepdim=True), v.contiguous()).reshape(N, Hq, L, D).permute(0, 2, 1, 3)
    row = torch.arange(T, device=dev)
    seq = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    inside = seq < N
    seq = seq.clamp(max=N - 1)
    out = o[seq, torch.where(inside, row - offsets[seq], 0)]
    out = torch.where(inside[:, None, None], out, 0.0).to(state["q"].dtype)
    if not case["grad"]:
        return {"out": out}
    dq, dk, dv = torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["dout"])
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _plain_shared(state):
    case, lengths = state["case"], state["lengths"]
    B, Hq, Hkv, D, L = case["B"], case["Hq"], case["Hkv"], case["D"], case["prefix"]
    g = Hq // Hkv
    table = state["table"].long().clamp(min=0)
    width = table.shape[1] * case["page"]

    def keys(pool):      # the shared ones [Hkv, L, D] and the requests' own [B, Hkv, width, D], in 32 bits
        first = pool[state["prefix_table"].long()].reshape(-1, Hkv, D)[:L].float().permute(1, 0, 2).contiguous()
        return first, pool[table].reshape(B, width, Hkv, D).float().permute(0, 2, 1, 3).contiguous()

    (k0, k1), (v0, v1) = keys(state["k_pool"]), keys(state["v_pool"])
    q = state["q"].float().reshape(B, Hkv, g, D)
    by_head = q.permute(1, 0, 2, 3).reshape(Hkv, B * g, D)
    s0 = torch.matmul(by_head, k0.transpose(1, 2).contiguous()).reshape(Hkv, B, g, L).permute(1, 0, 2, 3)
    s = torch.cat((s0, torch.matmul(q, k1.transpose(2, 3).contiguous())), dim=-1) * D ** -0.5
    if case["softcap"]:
        s = torch.tanh(s / case["softcap"]) * case["softcap"]
    at = torch.arange(L + width, device=s.device)
    live = at < L + lengths[:, None]                                          # [B, keys]
    s = s.masked_fill(~live[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    e = e / e.sum(-1, keepdim=True).clamp(min=1e-30)                          # a request without a key: zeros
    o0 = torch.matmul(e[..., :L].permute(1, 0, 2, 3).reshape(Hkv, B * g, L), v0).reshape(Hkv, B, g, D).permute(1, 0, 2, 3)
    o = o0 + torch.matmul(e[..., L:].contiguous(), v1)
    return {"out": o.reshape(B, Hq, 1, D).to(state["q"].dtype)}


def _plain_tables(state):
    page, free, table = state["case"]["page"], state["free"].long(), state["table"]
    cached, new = state["cached"].long(), state["new"].long()
    B, W = table.shape
    have = (cached + page - 1) // page
    need = (cached + new + page - 1) // page - have
    first = need.cumsum(0) - need
    offsets = torch.zeros(B + 1, dtype=torch.long, device=table.device)
    offsets[1:] = new.cumsum(0)
    j = torch.arange(W, device=table.device) - have[:, None]                  # number of an entry among the request's new ones
    taken = (first[:, None] + j).clamp(0, len(free) - 1)
    table.copy_(torch.where((j >= 0) & (j < need[:, None]), free[taken].to(torch.int32), table))
    row = torch.arange(state["total"], device=table.device)
    of = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    real = of < B
    of = of.clamp(max=B - 1)
    position = torch.where(real, cached[of] + row - offsets[of], -1)
    at = position.clamp(min=0)
    slot = torch.where(real, table[of, at // page].long() * page + at % page, -1)
    return {"table": table, "offsets": offsets.to(torch.int32), "lengths": (cached + new).to(torch.int32), "slots": slot.to(torch.int32),
            "positions": position.to(torch.int32), "pages": need.sum().reshape(1).to(torch.int32)}


def _plain_store(state):
    slots = state["slots"].long()
    kept = slots >= 0
    for rows, pool in ((state["k"], state["k_pool"]), (state["v"], state["v_pool"])):
        pool.view(-1, *pool.shape[2:])[slots[kept]] = rows[kept]
    return {"k_pool": state["k_pool"], "v_pool": state["v_pool"]}


_RUN_OWN = {"packed": _own_packed, "shared": _own_shared, "tables": _own_tables, "store": _own_store}
_RUN_PLAIN = {"packed": _plain_packed, "shared": _plain_shared, "tables": _plain_tables, "store": _plain_store}


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "packed":
        return _exact_packed(case, {n: t.detach() if torch.is_tensor(t) else t for n, t in state.items()})
    if case["op"] == "shared":
        return _exact_shared(case, state)
    if case["op"] == "tables":
        return _exact_tables(case, state)
    out = {}
    for name, rows in (("k_pool", state["k"]), ("v_pool", state["v"])):
        pool = state[name].double()
        for at, row in zip(*(x.tolist() for x in (state["slots"], torch.arange(case["T"])))) if case["T"] <= 256 else ():
            if at >= 0:
                pool[at // case["page"], at % case["page"]] = rows[row].double()
        if case["T"] > 256:
            flat = pool.reshape(-1, case["Hkv"], case["D"])
            # which row a slot holds: the one that names it, or none
            holds = torch.full((flat.shape[0] + 1,), -1, dtype=torch.long, device=flat.device)
            holds[state["slots"].long()] = torch.arange(case["T"], device=flat.device)       # -1 names the one behind the last
            holds = holds[:-1]
            pool = torch.where((holds >= 0)[:, None, None], rows.double()[holds.clamp(min=0)], flat).reshape(pool.shape)
        out[name] = pool
    return out


def _exact_packed(case, state):
    Hq, Hkv, D, c = case["Hq"], case["Hkv"], case["D"], case["softcap"]
    g, scale = Hq // Hkv, case["D"] ** -0.5
    ends = state["offsets"].tolist()
    res = {n: torch.zeros(t.shape, dtype=torch.float64, device=t.device)
           for n, t in (("out", state["q"]),) + ((("dq", state["q"]), ("dk", state["k"]), ("dv", state["v"])) if case["grad"] else ())}
    for lo, hi in zip(ends[:-1], ends[1:]):
        if hi == lo:
            continue
        i = torch.arange(hi - lo, device=state["q"].device)
        t = i[:, None] - i[None, :]
        hidden = torch.zeros_like(t, dtype=torch.bool) if case["mask"] == "none" else t < 0
        if case["mask"] == "sliding":
            hidden = hidden | (t >= case["window"])
        for h in range(Hkv):
            q = state["q"][lo:hi, h * g:(h + 1) * g].double().permute(1, 0, 2).contiguous()
            k, v = state["k"][lo:hi, h].double(), state["v"][lo:hi, h].double()
            x = (q.reshape(-1, D) @ k.t().contiguous()).reshape(g, hi - lo, hi - lo) * scale
            th = torch.tanh(x / c) if c else None
            x = (c * th if c else x).masked_fill(hidden, float("-inf"))
            p = torch.exp(x - torch.logsumexp(x, dim=-1, keepdim=True))
            o = (p.reshape(-1, hi - lo) @ v).reshape(g, hi - lo, D)
            res["out"][lo:hi, h * g:(h + 1) * g] = o.permute(1, 0, 2)
            if case["grad"]:
                do = state["dout"][lo:hi, h * g:(h + 1) * g].double().permute(1, 0, 2).contiguous()
                dp = (do.reshape(-1, D) @ v.t().contiguous()).reshape(p.shape)
                ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
                if c:
                    ds = ds * (1 - th * th)
                res["dq"][lo:hi, h * g:(h + 1) * g] = (ds.reshape(-1, hi - lo) @ k).reshape(g, hi - lo, D).permute(1, 0, 2)
                for a in range(g):
                    res["dk"][lo:hi, h] += ds[a].t().contiguous() @ q[a]
                    res["dv"][lo:hi, h] += p[a].t().contiguous() @ do[a]
    return res


def _exact_shared(case, state):
    Hq, Hkv, D, L, c = case["Hq"], case["Hkv"], case["D"], case["prefix"], case["softcap"]
    g, out = Hq // Hkv, torch.zeros(state["q"].shape, dtype=torch.float64, device=state["q"].device)
    k_rows, v_rows = (state[n].reshape(-1, Hkv, D) for n in ("k_pool", "v_pool"))
    at = torch.arange(max(L, case["longest"]), device=out.device)

    def rows_of(table, n):      # where the first n tokens of a table's pages lie
        return table.long()[at[:n] // case["page"]] * case["page"] + at[:n] % case["page"]

    first = rows_of(state["prefix_table"], L)
    for b, n in enumerate(state["lengths"].tolist()):
        rows = torch.cat((first, rows_of(state["table"][b], n)))
        if len(rows) == 0:
            continue
        k, v = (r[rows].double().permute(1, 0, 2).contiguous() for r in (k_rows, v_rows))
        x = (k @ state["q"][b, :, 0].double().reshape(Hkv, g, D).transpose(1, 2).contiguous()) * D ** -0.5       # [Hkv, keys, g]
        if c:
            x = c * torch.tanh(x / c)
        p = torch.exp(x - torch.logsumexp(x, dim=1, keepdim=True))
        out[b, :, 0] = (p.transpose(1, 2).contiguous() @ v).reshape(Hq, D)
    return {"out": out}


def _exact_tables(case, state):
    page, free = case["page"], iter(state["free"].tolist())
    table, offsets, lengths, slots, positions, taken = state["table"].tolist(), [0], [], [], [], 0
    for b, (c, n) in enumerate(zip(state["cached"].tolist(), state["new"].tolist())):
        for t in range(c, c + n):
            if t % page == 0:
                table[b][t // page] = next(free)
                taken += 1
            slots.append(table[b][t // page] * page + t % page)
            positions.append(t)
        offsets.append(offsets[-1] + n)
        lengths.append(c + n)
    rest = [-1] * (state["total"] - len(slots))
    return {"table": torch.tensor(table), "offsets": torch.tensor(offsets), "lengths": torch.tensor(lengths), "slots": torch.tensor(slots + rest),
            "positions": torch.tensor(positions + rest), "pages": torch.tensor([taken])}
