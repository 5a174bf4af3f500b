"""What the operators for requests of different lengths (``packed``, ``paged``) refuse, the rules of their work splits, and their
parameter blocks; no GPU."""
import ctypes
import math
import os
import re
import subprocess

import pytest
import torch

from loopfuse_amd import lowering, packed, paged, runtime
from loopfuse_amd.lowering import AttnPlan, UnsupportedPlan
import test_kernel_codegen as codegen

BF = torch.bfloat16


class OnGpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: checks of arguments run, nothing is launched."""
    is_cuda = True


def fake(shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnGpu)


@pytest.fixture(autouse=True)
def nothing_is_launched(monkeypatch):
    def refuse(*a, **kw):
        raise AssertionError("a launch")
    monkeypatch.setattr(lowering, "get_kernel", refuse)
    monkeypatch.setattr(lowering, "_call_key", lambda *a: None)
    monkeypatch.setattr(runtime, "current_device", lambda: -1)


def layout(total, count=2):
    return packed.PackedLayout(fake((count + 1,), torch.int32), total, fake((8, 4), torch.int32), (1, 1, 1, 1))


def qkv(T=10, Hq=4, Hkv=2, D=64, dtype=BF):
    return fake((T, Hq, D), dtype), fake((T, Hkv, D), dtype), fake((T, Hkv, D), dtype)


@pytest.mark.parametrize("offsets,total", [(torch.zeros(3), 5), (torch.zeros((2, 2), dtype=torch.int32), 5), (torch.zeros(0, dtype=torch.int32), 5),
                                           (fake((3,), torch.int32), -1), (fake((3,), torch.int32), 1 << 31), ([0, 5], 5)])
def test_layouts_that_are_refused(offsets, total):
    with pytest.raises(UnsupportedPlan):
        packed.packed_layout(offsets, total)


def test_no_cpu_fallback():
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        packed.packed_layout(i32, 5)
    q, k, v = (t.as_subclass(torch.Tensor) for t in qkv())
    with pytest.raises(RuntimeError, match="GPU"):
        packed.attention_packed(q, k, v, AttnPlan(), layout(10))
    with pytest.raises(RuntimeError, match="GPU"):
        paged.extend_tables(i32, i32, torch.zeros((3, 2), dtype=torch.int32), i32, 16, 5)
    with pytest.raises(RuntimeError, match="GPU"):
        paged.store_kv(k, v, torch.zeros((2, 4, 2, 64), dtype=BF), torch.zeros((2, 4, 2, 64), dtype=BF), torch.zeros(10, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="GPU"):
        paged.attention_shared(torch.zeros((3, 4, 1, 64), dtype=BF), torch.zeros((2, 4, 2, 64), dtype=BF), torch.zeros((2, 4, 2, 64), dtype=BF),
                               AttnPlan(), torch.zeros((3, 2), dtype=torch.int32), i32)


PLAN = AttnPlan("causal", scale=0.1)
PACKED = {
    "another number of rows": lambda q, k, v: ((q, k[:9], v), PLAN, layout(10), {}),
    "rows of the layout": lambda q, k, v: ((q, k, v), PLAN, layout(11), {}),
    "no layout": lambda q, k, v: ((q, k, v), PLAN, fake((3,), torch.int32), {}),
    "types": lambda q, k, v: ((q, k.half(), v), PLAN, layout(10), {}),
    "fp32": lambda q, k, v: ((q.float(), k.float(), v.float()), PLAN, layout(10), {}),
    "heads": lambda q, k, v: ((q[:, :3], k, v), PLAN, layout(10), {}),
    "kv heads": lambda q, k, v: ((q, k, v[:, :1]), PLAN, layout(10), {}),
    "head dim": lambda q, k, v: (qkv(D=192), PLAN, layout(10), {}),
    "head dims": lambda q, k, v: ((q, k, fake((10, 2, 128))), PLAN, layout(10), {}),
    "dims": lambda q, k, v: ((q[None], k[None], v[None]), PLAN, layout(10), {}),
    "strides": lambda q, k, v: ((q, fake((10, 2, 68))[..., :64], v), PLAN, layout(10), {}),
    "a stride of the last dim": lambda q, k, v: ((q, fake((10, 64, 2)).transpose(1, 2), v), PLAN, layout(10), {}),
    "alignment": lambda q, k, v: ((q, fake((10 * 2 * 64 + 1,))[1:].view(10, 2, 64), v), PLAN, layout(10), {}),
    "paging": lambda q, k, v: ((q, k, v), AttnPlan(k_paged=True), layout(10), {}),
    "denominator": lambda q, k, v: ((q, k, v), AttnPlan(denom_add=1.0), layout(10), {}),
    "mask": lambda q, k, v: ((q, k, v), AttnPlan("other"), layout(10), {}),
    "window": lambda q, k, v: ((q, k, v), AttnPlan("sliding"), layout(10), {}),
    "scale": lambda q, k, v: ((q, k, v), AttnPlan(scale=0.0), layout(10), {}),
    "nan scale": lambda q, k, v: ((q, k, v), AttnPlan(scale=math.nan), layout(10), {}),
    "softcap": lambda q, k, v: ((q, k, v), AttnPlan(softcap=0.0), layout(10), {}),
    "out": lambda q, k, v: ((q, k, v), PLAN, layout(10), {"out": fake((10, 2, 64))}),
    "out of one row": lambda q, k, v: ((q, k, v), PLAN, layout(10), {"out": fake((1, 4, 64)).expand(10, 4, 64)}),
    "lse": lambda q, k, v: ((q, k, v), PLAN, layout(10), {"lse": fake((10, 4), torch.float32)}),
    "out with gradients": lambda q, k, v: ((q.requires_grad_(), k, v), PLAN, layout(10), {"out": fake((10, 4, 64))}),
    "out of a padded head dim": lambda q, k, v: (qkv(D=40), PLAN, layout(10), {"out": fake((10, 4, 40))}),
    "rows beyond 32 bits": lambda q, k, v: ((q, torch.empty_strided((10, 2, 64), (1 << 28, 64, 1), dtype=BF, device="meta"), v), PLAN, layout(10), {}),
}


@pytest.mark.parametrize("case", PACKED)
def test_packed_calls_that_are_refused(case, monkeypatch):
    if "32 bits" in case:
        monkeypatch.setattr(lowering, "_check_tensor", lambda *a: None)
        monkeypatch.setattr(packed, "_rows", lambda *a: None)
    args, plan, lay, kw = PACKED[case](*qkv())
    with pytest.raises(UnsupportedPlan):
        packed.attention_packed(*args, plan, lay, **kw)


@pytest.mark.parametrize("case", [c for c in PACKED if "32 bits" not in c])
def test_packed_calls_with_gradients_that_are_refused(case, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    args, plan, lay, kw = PACKED[case](*qkv())
    with pytest.raises(UnsupportedPlan):
        packed.attention_packed(*(t.detach().as_subclass(OnGpu).requires_grad_() for t in args), plan, lay, **kw)
    with pytest.raises(UnsupportedPlan):
        packed.attention_packed(args[0].detach()[0, 0].as_subclass(OnGpu).requires_grad_(), *args[1:], plan, lay, **kw)


def test_packed_backward_calls_that_are_refused():
    q, k, v = qkv()
    lse = fake((4, 10), torch.float32)
    for o, l, g in ((q[:, :2], lse, q), (q, lse, q[:, :2]), (q, lse.t(), q), (q, lse.half(), q), (q.float(), lse, q), (q, lse, q[..., ::2])):
        with pytest.raises(UnsupportedPlan):
            packed.attention_packed_backward(q, k, v, o, l, g, PLAN, layout(10))


def tables(B=3, W=4, F=5, dtype=torch.int32):
    return fake((B,), torch.int32), fake((B,), torch.int32), fake((B, W), dtype), fake((F,), dtype)


TABLES = {
    "types of lengths": lambda c, n, t, f: (c.long(), n, t, f, 16, 10),
    "types of pages": lambda c, n, t, f: (c, n, t, f.long(), 16, 10),
    "type of the table": lambda c, n, t, f: (c, n, t.short(), f.short(), 16, 10),
    "requests": lambda c, n, t, f: (c, n[:2], t, f, 16, 10),
    "rows": lambda c, n, t, f: (c, n, t[:2], f, 16, 10),
    "dims": lambda c, n, t, f: (c, n, t[0], f, 16, 10),
    "page size": lambda c, n, t, f: (c, n, t, f, 12, 10),
    "no page": lambda c, n, t, f: (c, n, t, f, 0, 10),
    "pages beyond 32 bits": lambda c, n, t, f: (c, n, t, f, 1 << 31, 10),
    "total": lambda c, n, t, f: (c, n, t, f, 16, -1),
    "columns apart": lambda c, n, t, f: (c, n, fake((3, 8), torch.int32)[:, ::2], f, 16, 10),
    "rows of one": lambda c, n, t, f: (c, n, fake((1, 4), torch.int32).expand(3, 4), f, 16, 10),
    "a page size that is no number": lambda c, n, t, f: (c, n, t, f, 16.0, 10),
}


@pytest.mark.parametrize("case", TABLES)
def test_table_calls_that_are_refused(case):
    with pytest.raises(UnsupportedPlan):
        paged.extend_tables(*TABLES[case](*tables()))


def pools(pages=3, page=4, Hkv=2, D=64, dtype=BF):
    return fake((pages, page, Hkv, D), dtype), fake((pages, page, Hkv, D), dtype)


STORES = {
    "slots": lambda k, v, p, s: (k, v, *p, s[:9]),
    "type of slots": lambda k, v, p, s: (k, v, *p, s.long()),
    "heads": lambda k, v, p, s: (k[:, :1], v[:, :1], *p, s),
    "head dim": lambda k, v, p, s: (fake((10, 2, 128)), fake((10, 2, 128)), *p, s),
    "rows": lambda k, v, p, s: (k, v[:9], *p, s),
    "types": lambda k, v, p, s: (k, v.half(), *p, s),
    "fp32": lambda k, v, p, s: (k.float(), v.float(), *(t.float() for t in p), s),
    "a pool of another size": lambda k, v, p, s: (k, v, p[0], fake((6, 2, 2, 64)), s),
    "page size": lambda k, v, p, s: (k, v, *pools(page=3), s),
    "a pool of one page": lambda k, v, p, s: (k, v, p[0], fake((1, 4, 2, 64)).expand(3, 4, 2, 64), s),
    "an odd head dim": lambda k, v, p, s: (fake((10, 2, 68))[..., :60], v[..., :60], p[0][..., :60], p[1][..., :60], s),
    "dims of a pool": lambda k, v, p, s: (k, v, p[0][0, 0], p[1][0, 0], s),
}


@pytest.mark.parametrize("case", STORES)
def test_stores_that_are_refused(case):
    with pytest.raises(UnsupportedPlan):
        paged.store_kv(*STORES[case](fake((10, 2, 64)), fake((10, 2, 64)), pools(), fake((10,), torch.int32)))


def shared(**change):
    kp, vp = pools(9, 4, 2, 64)
    a = dict(q=fake((3, 4, 1, 64)), k_pool=kp, v_pool=vp, plan=AttnPlan(scale=0.1, k_paged=True, v_paged=True), table=fake((3, 5), torch.int32),
             lengths=fake((3,), torch.int32), prefix_table=fake((2,), torch.int32), prefix_len=7)
    a.update(change)
    return a


SHARED = {
    "mask": dict(plan=AttnPlan("causal", scale=0.1)), "denominator": dict(plan=AttnPlan(denom_add=1.0)), "scale": dict(plan=AttnPlan(scale=-1.0)),
    "softcap": dict(plan=AttnPlan(softcap=math.inf)), "two tokens": dict(q=fake((3, 4, 2, 64))), "head dim": dict(q=fake((3, 4, 1, 32))),
    "heads": dict(q=fake((3, 3, 1, 64))), "fp32": dict(q=fake((3, 4, 1, 64), torch.float32)), "types": dict(q=fake((3, 4, 1, 64), torch.float16)),
    "requests": dict(lengths=fake((2,), torch.int32)), "table": dict(table=fake((2, 5), torch.int32)), "type of lengths": dict(lengths=fake((3,), torch.int64)),
    "type of the table": dict(table=fake((3, 5), torch.float32)), "no prefix table": dict(prefix_table=None), "a short prefix table": dict(prefix_len=9),
    "type of the prefix table": dict(prefix_table=fake((2,), torch.int64)), "a negative prefix": dict(prefix_len=-1),
    "V table": dict(v_table=fake((3, 4), torch.int32)), "page sizes": dict(v_pool=fake((18, 2, 2, 64))), "page size": dict(k_pool=fake((9, 6, 2, 64)), v_pool=fake((9, 6, 2, 64))),
    "out": dict(out=fake((3, 4, 64))), "out of one row": dict(out=fake((1, 4, 1, 64)).expand(3, 4, 1, 64)), "kv heads": dict(v_pool=fake((9, 4, 1, 64))),
    "room beyond 2**30 keys": dict(table=fake((3, 1), torch.int32).expand(3, (1 << 28) + 1)),
    "a prefix beyond 2**30 keys": dict(prefix_table=fake((1,), torch.int32).expand((1 << 28) + 1), prefix_len=(1 << 30) + 1),
    "a prefix length that is no number": dict(prefix_len=torch.tensor(7)),
}


@pytest.mark.parametrize("case", SHARED)
def test_shared_calls_that_are_refused(case):
    with pytest.raises(UnsupportedPlan):
        paged.attention_shared(**shared(**SHARED[case]))


def test_the_host_module_leaves_other_operands_to_the_general_path():
    host = runtime.host()
    q, k, v = qkv()
    lay = layout(10)
    for a in ((q, k, v), tuple(t.as_subclass(torch.Tensor) for t in (q, k, v)), (None, 3, "x")):
        assert host.attention_packed(*a, None, None, lay.tiles, PLAN, 10, 1, False) is None
        assert host.key("p", a, (lay.tiles,), PLAN, (10,)) is None
        assert host.store_kv(*a, v, None) is None
    assert host.attention_packed(q, k, v, None, None, lay.tiles, object(), 10, 1, False) is None
    for call in (lambda: host.store_kv(q), lambda: host.key("p", q), lambda: host.keep(b"", b"", b"", {}, None, ()[:0] + (1.5,)), lambda: host.keep(b"", b"x" * 2000, b"", {}, None, ())):
        with pytest.raises(TypeError):
            call()


def test_a_leaf_of_a_living_graph_is_known():
    q = torch.randn(3, requires_grad=True)
    assert not packed.in_a_graph(q)
    out = q * 2
    assert packed.in_a_graph(q) and packed.in_a_graph(q)
    out.sum().backward()
    assert packed.in_a_graph(q)
    del out
    assert not packed.in_a_graph(q)


def _both_builds():
    import __graft_entry__
    return sorted({s for s in __graft_entry__.ragged_specs() if s.family == "bwd_both"}, key=lambda s: s.name())


@pytest.mark.parametrize("spec", _both_builds(), ids=lambda s: s.name()[12:])
def test_the_launch_of_all_gradients_keeps_its_accumulators(spec):
    """As for the other backward builds: no spill, results of MFMAs left alone until they are there, and in each of the two parts no other
    instruction on an AGPR between its first and its last MFMA."""
    if not os.path.exists(codegen.OBJDUMP):
        pytest.skip("needs the ROCm LLVM tools")
    lines = codegen._kernels(spec)["lf_attn_bwd_both"]
    codegen._check("both", lines)
    codegen._check_settled("both", lines)
    mfma = [i for i, ln in enumerate(lines) if ln.startswith("v_mfma")]
    cut = max(range(1, len(mfma)), key=lambda j: mfma[j] - mfma[j - 1])
    assert mfma[cut] - mfma[cut - 1] > 200          # (the end of one part and the begin of the other)
    for part in (mfma[:cut], mfma[cut:]):
        for ln in lines[part[0]:part[-1]]:
            assert ln.startswith("v_mfma") or not re.search(r"\ba(\d+|\[\d+:\d+\])", ln), ln
    for ln in lines:
        m = re.match(r"v_mfma_\S+ (a\[\d+:\d+\]),.*, (\S+)$", ln)
        assert m is None or m.group(1) == m.group(2), ln


# ---- parameter blocks and rules --------------------------------------------------------------------------------

KERNELS = os.path.join(runtime.KERNEL_DIR)


@pytest.mark.parametrize("mirror,device,source", [
    (packed._PlanParams, "LfPackedPlanParams", "lf_packed_plan.hip"), (packed.PackedAttnParams, "LfPackedAttnParams", "lf_packed.hip.h"),
    (packed.PackedBwdParams, "LfPackedBwdParams", "lf_attn_bwd.hip"), (paged._TablesParams, "LfTablesParams", "lf_paged_tables.hip"),
    (paged._StoreParams, "LfStoreParams", "lf_store_kv.hip"), (paged.SharedParams, "LfSharedParams", "lf_shared.hip.h")])
def test_parameter_blocks_list_the_fields_of_their_kernels(mirror, device, source):
    text = open(os.path.join(KERNELS, source)).read()
    body = text[re.search(r"struct %s\b[^;{]*\{" % device, text).end():]
    body = re.sub(r"//[^\n]*", "", body[:body.index("};")])
    fields = []
    for decl in body.split(";"):
        if decl.strip():
            fields += [re.sub(r"\[.*\]|[^A-Za-z0-9_]", "", x.split()[-1]) for x in decl.split(",")]
    assert fields == [n for n, *_ in mirror.__dict__["_fields_"]]
    # a derived block begins behind its base's last byte, at a multiple of 8 as the compiler places a pointer
    if mirror.__mro__[1] is not ctypes.Structure:
        assert getattr(mirror, fields[0]).offset == ctypes.sizeof(mirror.__mro__[1]) and ctypes.sizeof(mirror.__mro__[1]) % 8 == 0


@pytest.mark.parametrize("mirror,host,base", [
    (packed._PlanParams, "LfPackedPlanParamsHost", ""), (packed.PackedAttnParams, "LfPackedAttnParamsHost", "attn."),
    (packed.PackedBwdParams, "LfPackedBwdParamsHost", "bwd."), (paged._TablesParams, "LfTablesParamsHost", ""),
    (paged._StoreParams, "LfStoreParamsHost", ""), (paged.SharedParams, "LfSharedParamsHost", "attn.")])
def test_parameter_blocks_of_c_hosts_are_the_mirrors(tmp_path, mirror, host, base):
    own = [n for n, *_ in mirror.__dict__["_fields_"]]
    inherited = [n for n, *_ in mirror.__mro__[1].__dict__.get("_fields_", ())] if base else []
    prog = "#include <stdio.h>\n#include <stddef.h>\n#include \"lf_ragged_params.h\"\nint main(void) {\n"
    for n in own + inherited:
        prog += f'  printf("{n} %zu\\n", offsetof({host}, {base if n in inherited else ""}{n}));\n'
    prog += f'  printf("sizeof %zu\\n", sizeof({host}));\n  return 0;\n}}\n'
    (tmp_path / "off.c").write_text(prog)
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c11", "-I" + include, str(tmp_path / "off.c"), "-o", str(tmp_path / "off")], check=True)
    out = dict(line.split() for line in subprocess.run([str(tmp_path / "off")], capture_output=True, text=True, check=True).stdout.splitlines())
    for n in own + inherited:
        assert int(out[n]) == getattr(mirror, n).offset, n
    assert int(out["sizeof"]) == ctypes.sizeof(mirror)


def tiles_of(lengths, height, size, cap):
    """The list of a group size, by its definition: sequences by length, groups of neighbours, tiles by their work."""
    order = sorted(range(len(lengths)), key=lambda i: (-lengths[i], i))
    out = []
    for a in range(0, len(order), size):
        group = [(rank, i, -(-lengths[i] // height)) for rank, i in enumerate(order[a:a + size])]
        out += [(i, t) for _, _, i, t in sorted((-(n - t), rank, i, t) for rank, i, n in group for t in range(n))]
    assert len(out) <= cap
    return out


@pytest.mark.parametrize("lengths", [[1], [0, 0], [5, 100, 33, 64, 0, 33], [257] * 9 + [1000, 3]])
def test_a_place_formula_gives_that_order(lengths):
    """What lf_packed_plan computes for a tile, place = tiles in front of the group + sum max(0, n_j - c) + its member's number."""
    for height in packed.TILE_HEIGHTS:
        for size in packed.GROUP_SIZES:
            cap = sum(lengths) // height + len(lengths) + 2
            want, got = tiles_of(lengths, height, size, cap), {}
            order = sorted(range(len(lengths)), key=lambda i: (-lengths[i], i))
            n = [-(-lengths[i] // height) for i in order]
            for a in range(0, len(order), size):
                for g in range(a, min(a + size, len(order))):
                    for t in range(n[g]):
                        c = n[g] - t
                        got[sum(n[:a]) + g - a + sum(max(0, x - c) for x in n[a:a + size])] = (order[g], t)
            assert [got[i] for i in range(len(got))] == want


@pytest.mark.parametrize("mask,window", [(lowering.MASK_NONE, 0), (lowering.MASK_CAUSAL, 0), (lowering.MASK_SLIDING, 1), (lowering.MASK_SLIDING, 100)])
@pytest.mark.parametrize("lengths", [[1], [31, 33, 0, 1, 64], [300, 2, 2, 2, 2], [0, 0, 95]])
def test_kept_ds_of_sequences_does_not_overlap(mask, window, lengths):
    """lf_bw_ds_before and lf_bw_ds_row: blocks of one sequence end in front of the next one's, the last one's in front of ds_blocks."""
    T, spans, row0 = sum(lengths), [], 0
    n_all = -(-T // 32)
    per = n_all if mask == lowering.MASK_NONE else (n_all + 2) // 2 if mask == lowering.MASK_CAUSAL else (window + 30) // 32 + 1
    for seq, length in enumerate(lengths):
        base, n = (row0 // 32 + seq) * per, -(-length // 32)
        if n:
            if mask == lowering.MASK_NONE:
                end = n * n
            elif mask == lowering.MASK_CAUSAL:
                end = n * (n + 1) // 2
            else:
                before = (window + 30) // 32
                end = (n - 1) * (before + 1) - (n - 1 - before) + n - 1 + 1
            spans.append((base, base + end))
        row0 += length
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
    assert not spans or spans[-1][1] <= packed.ds_blocks(mask, window, T, len(lengths))


def test_pieces_of_own_keys_fit_the_launch():
    """lf_shared_split and the pieces it makes: never more than the grid, 2^target / units + B, has room for."""
    gen = torch.Generator().manual_seed(3)
    for _ in range(2000):
        B = int(torch.randint(1, 200, (), generator=gen))
        units, target, least = (int(torch.randint(1, n, (), generator=gen)) for n in (40, 12, 9))
        lengths = torch.randint(0, int(torch.randint(1, 20000, (), generator=gen)), (B,), generator=gen).tolist()
        split = max(32 * least, (((sum(lengths) * units) >> target) + 32) & ~31)
        assert sum(-(-n // split) for n in lengths) <= (1 << target) // units + B


def test_splits_of_a_prefix_are_whole_tiles_and_few():
    for units in (1, 3, 8, 32, 300):
        for keys in (1, 2, 16, 129, 4000):
            for own in (0, 1 << 40):
                for D in (64, 128):
                    n = paged.prefix_splits(units, keys, 128, D, keys << 17, own)
                    assert 1 <= n <= min(64, keys) and (own == 0 or n == 1)
