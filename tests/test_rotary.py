"""What ``rotary.rotate_heads`` refuses, its table of angles, its parameter blocks, and the formulas of its gradients against differences; no GPU."""
import ctypes
import math
import re
import os
import subprocess

import pytest
import torch
from torch.autograd import forward_ad

from loopfuse_amd import lowering, packed, paged, rotary, runtime
from loopfuse_amd.lowering import UnsupportedPlan
from test_ragged import fake, nothing_is_launched  # noqa: F401  (a fixture that every test here uses)

F32, I32 = torch.float32, torch.int32


# ---- the table -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("length,dim,base", [(1, 2, 10000.0), (0, 16, 10000.0), (70, 64, 10000.0), (300, 128, 500000.0)])
def test_the_table_holds_cosines_and_sines(length, dim, base):
    table = rotary.rotary_table(length, dim, base)
    assert table.shape == (length, dim) and table.dtype == F32
    for pos in range(0, length, 23):
        for i in range(0, dim // 2, 5):
            angle = pos * base ** (-2 * i / dim)
            # (an angle below 300 is off by 2^-44 in 64 bits, the value by that and half a step of 32 bits)
            assert abs(table[pos, i].item() - math.cos(angle)) <= 2.0 ** -25 + 2.0 ** -40
            assert abs(table[pos, dim // 2 + i].item() - math.sin(angle)) <= 2.0 ** -25 + 2.0 ** -40


def test_angles_of_far_positions_keep_their_digits():
    # 10^6 * f has 20 bits in front of the point: 32 bits would leave 4 behind it
    f = torch.tensor([1.0, 0.123456789], dtype=torch.float64)
    table = rotary.rotary_table(1_000_001, 4, frequencies=f)
    for i in range(2):
        angle = 1_000_000 * f[i].item()
        assert abs(table[-1, i].item() - math.cos(angle)) < 1e-7 and abs(table[-1, 2 + i].item() - math.sin(angle)) < 1e-7


@pytest.mark.parametrize("args,kw", [((-1, 4), {}), ((4, 3), {}), ((4, 0), {}), ((4, 4), {"frequencies": torch.ones(3)})])
def test_tables_that_are_refused(args, kw):
    with pytest.raises(UnsupportedPlan):
        rotary.rotary_table(*args, **kw)


# ---- refusals ------------------------------------------------------------------------------------------------

def operands(T=10, Hq=4, Hkv=2, D=64, R=64, dtype=torch.bfloat16):
    return dict(q=fake((T, Hq, D), dtype), k=fake((T, Hkv, D), dtype), positions=fake((T,), I32), table=fake((50, R), F32))


ROTATE = {
    "fp32": dict(q=fake((10, 4, 64), F32), k=fake((10, 2, 64), F32)), "types": dict(k=fake((10, 2, 64), torch.float16)), "rows": dict(k=fake((9, 2, 64))),
    "dims": dict(q=fake((10, 64))), "dims of k": dict(k=fake((10, 1, 2, 64))), "head dims": dict(k=fake((10, 2, 128))),
    "an odd head dim": dict(q=fake((10, 4, 72)), k=fake((10, 2, 72))), "a head dim beyond 256": dict(q=fake((10, 1, 272)), k=fake((10, 1, 272))),
    "no heads": dict(k=fake((10, 0, 64))), "positions in 64 bits": dict(positions=fake((10,), torch.int64)), "positions": dict(positions=fake((9,), I32)),
    "no positions": dict(positions=None), "table in 16 bits": dict(table=fake((50, 64))), "dims of the table": dict(table=fake((64,), F32)),
    "more rotated than there are": dict(table=fake((50, 80), F32)), "rotated by eights": dict(table=fake((50, 24), F32)),
    "a table of columns": dict(table=fake((64, 50), F32).t()), "a table of one row": dict(table=fake((1, 64), F32).expand(50, 64)),
    "a table off its border": dict(table=fake((50 * 64 + 1,), F32)[1:].view(50, 64)), "nothing to do": dict(table=None),
    "weights without eps": dict(q_weight=fake((64,))), "a weight's size": dict(q_weight=fake((32,)), eps=1e-6), "a weight's type": dict(k_weight=fake((64,), torch.float16), eps=1e-6),
    "weights of two types": dict(q_weight=fake((64,)), k_weight=fake((64,), F32), eps=1e-6), "eps": dict(eps=-1.0), "no eps": dict(eps=math.nan),
    "an infinite eps": dict(eps=math.inf), "strides": dict(q=fake((10, 4, 68))[..., :64]), "a stride of the last dim": dict(q=fake((10, 64, 4)).transpose(1, 2)),
    "alignment": dict(q=fake((10 * 4 * 64 + 1,))[1:].view(10, 4, 64)),
}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("case", ROTATE)
def test_rotations_that_are_refused(case, grad, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    a = {**operands(), **ROTATE[case]}
    if grad:
        a["q"] = a["q"].detach().as_subclass(type(a["k"])).requires_grad_()
    with pytest.raises(UnsupportedPlan):
        rotary.rotate_heads(**a)


def test_the_table_gets_no_gradient(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    a = operands()
    a["q"].requires_grad_()
    a["table"].requires_grad_()
    with pytest.raises(UnsupportedPlan, match="table"):
        rotary.rotate_heads(**a)


def test_rotations_that_are_served_reach_a_launch():
    for a in (operands(), operands(D=16, R=16), operands(D=256, R=48, dtype=torch.float16), operands(T=1), {**operands(), "table": None, "eps": 1e-5},
              {**operands(), "eps": 0.0, "q_weight": fake((64,), F32)}, {**operands(), "pairs": True}):
        with pytest.raises(AssertionError, match="a launch"):
            rotary.rotate_heads(**a)
    q, k = rotary.rotate_heads(**operands(T=0))
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)


def test_no_cpu_fallback():
    a = {n: t.as_subclass(torch.Tensor) for n, t in operands().items()}
    with pytest.raises(RuntimeError, match="GPU"):
        rotary.rotate_heads(**a)
    for name in ("positions", "table"):
        with pytest.raises(RuntimeError, match="GPU"):
            rotary.rotate_heads(**{**operands(), name: a[name]})
    with pytest.raises(RuntimeError, match="GPU"):
        rotary.rotate_heads(**operands(), q_weight=torch.ones(64, dtype=torch.bfloat16), eps=1e-6)


@pytest.mark.parametrize("name", ["q", "k", "q_weight"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(name, grad, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    with forward_ad.dual_level():
        a = {**operands(), "q_weight": fake((64,), F32), "eps": 1e-6}
        if grad:
            a["k" if name == "q" else "q"].requires_grad_()
        a[name] = forward_ad.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(UnsupportedPlan, match="tangents"):
            rotary.rotate_heads(**a)


def test_launches_beyond_32_bits(monkeypatch):
    monkeypatch.setattr(lowering, "_check_tensor", lambda *a: None)
    q, k = (fake((1, h, 256)).expand(1 << 28, h, 256) for h in (32, 8))
    with pytest.raises(UnsupportedPlan, match="too large"):
        rotary.rotate_heads(q, k, fake((1,), I32).expand(1 << 28), fake((4, 256), F32))


def test_gradients_refuse_saved_tensors_that_are_others():
    """What hooks of saved tensors give back in their place."""
    a = operands()
    right = dict(dq_out=fake((10, 4, 64)), dk_out=fake((10, 2, 64)), **a, q_weight=None, k_weight=None, eps=1e-6, pairs=False, sums=(False, False))
    elsewhere = torch.zeros((10, 4, 64), dtype=torch.bfloat16)
    for change in (dict(q=fake((10, 4, 64), F32)), dict(q=fake((9, 4, 64))), dict(k=fake((10, 3, 64))), dict(q=elsewhere), dict(q=fake((10, 4, 128)), k=fake((10, 2, 128))), dict(positions=fake((9,), I32)),
                   dict(positions=fake((10,), torch.int64)), dict(table=fake((50, 64))), dict(table=torch.zeros(50, 64)), dict(q_weight=fake((32,))), dict(dq_out=fake((10, 4, 64), torch.float16)),
                   dict(dq_out=fake((10, 5, 64))), dict(eps=None, dk_out=fake((9, 2, 64)))):
        with pytest.raises((UnsupportedPlan, RuntimeError)):
            rotary._backward(**{**right, **change})
    with pytest.raises(AssertionError, match="a launch"):
        rotary._backward(**right)


def test_threads_of_a_row_and_groups_of_heads():
    for D in range(16, 257, 16):
        n = rotary.slots_of(D)
        assert n in (1, 2, 4, 8, 16) and 16 * n >= D > 8 * n or D == 16
    for T in (1, 7, 1000, 20000):
        for H in (1, 3, 32):
            for D in (16, 80, 128, 256):
                chunks, blocks = rotary.grid(T, H, D)
                groups = 256 // rotary.slots_of(D)
                assert 2 * chunks >= H > 2 * (chunks - 1) and blocks * groups >= T * chunks > (blocks - 1) * groups


def test_the_host_module_leaves_other_operands_to_the_general_path():
    host, a = runtime.host(), operands()
    assert host.rotate_heads(a["q"], a["k"], a["table"], None, None, a["positions"], None, False) is None
    assert host.rotate_heads(None, 3, "x", None, None, None, None, False) is None
    assert host.rotate_backward(a["q"], a["k"], None, None, a["table"], None, None, a["positions"], None, False, False, False) is None
    for call in (host.rotate_heads, host.rotate_backward, host.append_kv, host.read_kv, host.attention_cached):
        with pytest.raises(TypeError):
            call(a["q"])


# ---- the formulas of the gradients ---------------------------------------------------------------------------

def turned(x, table, positions, R, pairs, w, eps):
    """The operator by its definition."""
    live = (positions >= 0) & (positions < table.shape[0])
    a = table[torch.where(live, positions, 0)][:, None]
    c, s = a[..., :R // 2], a[..., R // 2:]
    if eps is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    t, rest = x[..., :R], x[..., R:]
    x0, x1 = (t[..., 0::2], t[..., 1::2]) if pairs else (t[..., :R // 2], t[..., R // 2:])
    y0, y1 = x0 * c - x1 * s, x1 * c + x0 * s
    t = torch.stack((y0, y1), -1).flatten(-2) if pairs else torch.cat((y0, y1), -1)
    return torch.where(live[:, None, None], torch.cat((t, rest), -1), torch.zeros((), dtype=x.dtype))


def gradients(x, g, table, positions, R, pairs, w, eps):
    """(dx, dw) by the formulas that the kernel uses."""
    live = ((positions >= 0) & (positions < table.shape[0]))[:, None, None]
    a = table[torch.where(live[:, 0, 0], positions, 0)][:, None]
    c, s = a[..., :R // 2], a[..., R // 2:]
    t, rest = g[..., :R], g[..., R:]
    g0, g1 = (t[..., 0::2], t[..., 1::2]) if pairs else (t[..., :R // 2], t[..., R // 2:])
    z0, z1 = g0 * c + g1 * s, g1 * c - g0 * s
    dz = torch.cat((torch.stack((z0, z1), -1).flatten(-2) if pairs else torch.cat((z0, z1), -1), rest), -1) * live
    if eps is None:
        return dz, None
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n, h = x * r, dz * w
    return (h - n * (h * n).mean(-1, keepdim=True)) * r * live, (dz * n).sum((0, 1))


@pytest.mark.parametrize("eps", [None, 0.1])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("D,R", [(16, 16), (32, 16)])
def test_the_formulas_gradients_are_those_of_differences(D, R, pairs, eps):
    gen = torch.Generator().manual_seed(D + R)
    rnd = lambda *shape: torch.randn(shape, generator=gen, dtype=torch.float64)
    table, positions = rotary.rotary_table(9, R, 10.0).double(), torch.tensor([3, -1, 0, 8, 9])
    x, w, g = rnd(5, 2, D).requires_grad_(), rnd(D).requires_grad_(), rnd(5, 2, D)
    f = lambda x, w: turned(x, table, positions, R, pairs, w, eps)
    assert torch.autograd.gradcheck(f, (x, w), eps=1e-6, atol=1e-6)
    dx, dw = gradients(x.detach(), g, table, positions, R, pairs, w.detach(), eps)
    want = torch.autograd.grad(f(x, w), (x, w), g, allow_unused=True)
    assert torch.allclose(dx, want[0], atol=1e-12) and (eps is None or torch.allclose(dw, want[1], atol=1e-12))


# ---- parameter blocks ------------------------------------------------------------------------------------------

BLOCKS = [(rotary.RotateParams, "LfRotateParams", "lf_rotate.hip"), (rotary.RotateBwdParams, "LfRotateBwdParams", "lf_rotate.hip"),
          (packed._PositionsParams, "LfPackedPositionsParams", "lf_packed_positions.hip"), (paged._ReadParams, "LfReadParams", "lf_read_kv.hip"), (paged.CachedParams, "LfCachedParams", "lf_cached.hip")]


@pytest.mark.parametrize("mirror,device,source", BLOCKS, ids=lambda x: x if isinstance(x, str) else "")
def test_parameter_blocks_list_the_fields_of_their_kernels(mirror, device, source):
    text = open(os.path.join(runtime.KERNEL_DIR, source)).read()
    body = text[text.index("struct %s {" % device):]
    body = re.sub(r"//[^\n]*", "", body[body.index("{") + 1:body.index("};")])
    fields = []
    for decl in body.split(";"):
        if decl.strip():
            fields += [re.sub(r"[^A-Za-z0-9_]", "", x.split()[-1]) for x in decl.split(",")]
    assert fields == [n for n, *_ in mirror._fields_]


@pytest.mark.parametrize("mirror,device,source", BLOCKS, ids=lambda x: x if isinstance(x, str) else "")
def test_parameter_blocks_of_c_hosts_are_the_mirrors(tmp_path, mirror, device, source):
    own, host = [n for n, *_ in mirror._fields_], device + "Host"
    prog = "#include <stdio.h>\n#include <stddef.h>\n#include \"lf_ragged_params.h\"\nint main(void) {\n"
    for n in own:
        prog += f'  printf("{n} %zu\\n", offsetof({host}, {n}));\n'
    prog += f'  printf("sizeof %zu\\n", sizeof({host}));\n  return 0;\n}}\n'
    (tmp_path / "p.c").write_text(prog)
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I" + include, str(tmp_path / "p.c"), "-o", str(tmp_path / "p")], check=True)
    out = dict(line.split() for line in subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout.splitlines())
    assert {n: int(out[n]) for n in own} == {n: getattr(mirror, n).offset for n in own} and int(out["sizeof"]) == ctypes.sizeof(mirror)


def test_a_table_alone_gets_no_gradient_either(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    a = operands()
    a["table"].requires_grad_()
    with pytest.raises(UnsupportedPlan, match="table"):
        rotary.rotate_heads(**a)
    with torch.no_grad(), pytest.raises(AssertionError, match="a launch"):       # (nothing is asked for)
        rotary.rotate_heads(**a)


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_of_the_table_are_refused(grad, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    with forward_ad.dual_level():
        a = operands()
        if grad:
            a["q"].requires_grad_()
        a["table"] = forward_ad.make_dual(a["table"], torch.ones_like(a["table"]))
        with pytest.raises(UnsupportedPlan, match="tangents"):
            rotary.rotate_heads(**a)
        rows = fake((10, 2, 64))
        with pytest.raises(UnsupportedPlan, match="tangents"):
            paged.append_kv(a["q"].detach(), rows, rows, fake((3, 4, 2, 64)), fake((3, 4, 2, 64)), a["positions"], a["positions"], a["table"])


def test_launches_whose_queries_and_keys_together_are_beyond_32_bits(monkeypatch):
    """2^23 workgroups for the queries and as many for the keys, of 256 threads each."""
    monkeypatch.setattr(lowering, "_check_tensor", lambda *a: None)
    rows = fake((1, 1, 128)).expand(1 << 28, 1, 128)
    positions, table = fake((1,), I32).expand(1 << 28), fake((4, 128), F32)
    assert rotary.grid(1 << 28, 1, 128) == (1, 1 << 23)
    for call in (lambda: rotary.rotate_heads(rows, rows, positions, table),
                 lambda: rotary._backward(rows, rows, None, None, positions, table, None, None, None, False, (False, False))):
        with pytest.raises(UnsupportedPlan, match="too large"):
            call()
    less = slice((1 << 28) - 32)
    with pytest.raises(AssertionError, match="a launch"):
        rotary.rotate_heads(rows[less], rows[less], positions[less], table)


def test_the_table_is_where_its_frequencies_are():
    frequencies = torch.ones(4, device="meta")
    assert rotary.rotary_table(3, 8, frequencies=frequencies).device.type == "meta"
    assert rotary.rotary_table(3, 8, frequencies=torch.ones(4), device="meta").device.type == "meta"
    with torch.device("meta"):
        assert rotary.rotary_table(3, 8, frequencies=torch.ones(4, device="cpu")).device.type == "cpu"
        assert rotary.rotary_table(3, 8).device.type == "meta"
