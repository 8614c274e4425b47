"""The C entry points beside the optimizer, the router and the served layers: structs laid out alike, plans, and bad
arguments refused before a GPU is looked for."""
import ctypes as C
import os
import struct
import subprocess

import pytest

from conftest import ROOT, gpu_available, import_package

eps = import_package()
from eps_b200 import dense  # noqa: E402

LIB = eps.load_library()
A = 1 << 20      # an address that is only looked at, never read, by a call that is refused


def refused(fn, *args):
    st = eps.Status()
    rc = fn(*args, C.byref(st))
    assert rc == st.code and (rc == 0 or st.message)
    return rc


def test_struct_layouts_match_the_header(tmp_path):
    pairs = [("EpsB200Gradient", dense.Gradient), ("EpsB200GradientNorm", dense.GradientNormArgs), ("EpsB200BalanceLoss", dense.BalanceLossArgs),
             ("EpsB200LowRank", dense.LowRank)]
    lines = []
    for c, py in pairs:
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in py._fields_]
    lines.append('printf("%zu\\n", sizeof(EpsB200GradientResult));')
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "eps_b200_dense.h"\nint main(void){' + "".join(lines) + "return 0;}")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "s")]).split()]
    want = []
    for _, py in pairs:
        want += [C.sizeof(py)] + [getattr(py, f[0]).offset for f in py._fields_]
    assert got == [*want, 12]
    codes = {C.c_int32: "i", C.c_uint32: "I", C.c_uint64: "L", C.c_int64: "l", C.c_float: "f", C.c_double: "d", C.c_void_p: "P"}
    for packed, py in ((dense._GRADIENT_NORM, dense.GradientNormArgs), (dense._BALANCE, dense.BalanceLossArgs), (dense._LOW_RANK, dense.LowRank)):
        plain = "".join(codes[f[1]] for f in py._fields_)
        assert struct.calcsize("@" + plain) == packed.size == C.sizeof(py) and len(packed.unpack(bytes(packed.size))) == len(py._fields_)


def plan_of(*tensors, room=None):
    t = (dense.Gradient * len(tensors))(*(dense.Gradient(a, n, ty, 0) for a, n, ty in tensors))
    size = LIB.eps_b200_gradient_norm_plan_bytes(t, len(tensors))
    plan, blocks = (C.c_uint8 * max(1, min(size, 1 << 20)))(), C.c_uint64()
    rc = refused(LIB.eps_b200_gradient_norm_plan, t, len(tensors), plan, size if room is None else room, C.byref(blocks))
    spans = [struct.unpack_from("@PIi", plan, 16 * i) for i in range(blocks.value)]
    return rc, size, spans


def test_gradient_plan():
    """Spans of 16 KB that cover every element once, all but a tensor's first beginning on 16 bytes."""
    tensors = [(A, 10000, 0), (A + (1 << 20) + 2, 50001, 1), (A + (2 << 20), 0, 2), (A + (3 << 20) + 4, 3, 0), (A + (4 << 20) + 14, 8192, 2)]
    rc, size, spans = plan_of(*tensors)
    assert rc == 0 and size == 16 * len(spans)
    left = list(spans)
    for at, n, kind in tensors:
        width, end = (4 if kind == 0 else 2), at + n * (4 if kind == 0 else 2)
        while at < end:
            a, count, ty = left.pop(0)
            assert a == at and ty == kind and 0 < count * width <= 16384 + 14
            at += count * width
            assert at == end or at % 16 == 0
        assert at == end
    assert not left
    assert plan_of(*tensors, room=size - 1)[0] == eps.INVALID_ARGUMENT
    for bad in ([(A, 10, 3)], [(A + 1, 10, 1)], [(None, 10, 0)], [(A, 10, 0), (A + 36, 1, 0)], [(A, 10, 0), (A + 8, 0, 0), (A, 10, 0)],
                [(A, 1 << 45, 0)], [((1 << 64) - 16, 8, 0)]):
        assert plan_of(*bad)[0] == eps.INVALID_ARGUMENT
    assert plan_of((A, 10, 0), (A + 40, 1, 0), (A + 8, 0, 0))[0] == 0
    assert refused(LIB.eps_b200_gradient_norm_plan, None, 1, None, 0, None) == eps.INVALID_ARGUMENT


def norm(**change):
    fields = dict(device=0, kind=0, clip=0, plan=A, blocks=1000, max_norm=1.0, result=A, workspace=A, workspace_bytes=1 << 20)
    return bytes(dense.GradientNormArgs(**{**fields, **change}))


@pytest.mark.parametrize("change", [dict(kind=2), dict(clip=2), dict(plan=None), dict(plan=A + 8), dict(blocks=1 << 31), dict(max_norm=-1.0),
                                    dict(max_norm=float("nan")), dict(result=None), dict(workspace=None), dict(workspace=A + 4),
                                    dict(workspace_bytes=7992)])
def test_gradient_norm_refuses(change):
    assert refused(LIB.eps_b200_gradient_norm, norm(**change), None) == eps.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_gradient_norm, None, None) == eps.INVALID_ARGUMENT


def balance(**change):
    fields = dict(device=0, type=0, score=0, normalise=1, experts=16, top_k=2, tokens=8, weight=1.0, logits=A, logits_stride=16)
    return bytes(dense.BalanceLossArgs(**{**fields, **change}))


@pytest.mark.parametrize("change", [dict(type=3), dict(score=2), dict(experts=0), dict(experts=1025), dict(top_k=0), dict(top_k=33),
                                    dict(tokens=1 << 31), dict(tokens=1 << 30), dict(weight=float("inf")), dict(logits=None)])
def test_balance_loss_refuses(change):
    assert refused(LIB.eps_b200_balance_loss, balance(**change), A, A, A, A, A, A, 1 << 40, None) == eps.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_balance_loss_backward, balance(**change), A, A, A, A, 16, A, 16, None) == eps.INVALID_ARGUMENT


def test_balance_loss_refuses_missing_tensors():
    for i in range(5):
        args = [A] * 5
        args[i] = None
        assert refused(LIB.eps_b200_balance_loss, balance(), *args, None, 0, None) == eps.INVALID_ARGUMENT
    large = balance(tokens=100000)
    space = LIB.eps_b200_balance_loss_workspace(100000, 16)
    assert space and not LIB.eps_b200_balance_loss_workspace(8, 16)
    for room in ((A, space - 1), (None, space), (A + 2, space)):
        assert refused(LIB.eps_b200_balance_loss, large, A, A, A, A, A, *room, None) == eps.INVALID_ARGUMENT
    for counts, counted, out in ((None, A, A), (A, None, A), (A, A, None)):
        assert refused(LIB.eps_b200_balance_loss_backward, balance(), counts, counted, None, None, 0, out, 16, None) == eps.INVALID_ARGUMENT


def low_rank(**change):
    fields = dict(device=0, type=1, adapters=4, rank=16, inner=64, channels=32, rows=4, down=A, up=A, ids=A, x=A, base=A * 2, out=A * 3,
                  x_stride=64, base_stride=32, out_stride=32)
    return bytes(dense.LowRank(**{**fields, **change}))


@pytest.mark.parametrize("change", [dict(type=3), dict(adapters=0), dict(adapters=16385), dict(rank=0), dict(rank=129), dict(inner=0), dict(channels=0),
                                    dict(inner=1 << 30), dict(rows=1 << 31), dict(down=None), dict(up=None), dict(down=A + 8), dict(up=A + 2),
                                    dict(ids=None), dict(x=None), dict(out=None), dict(x_stride=-1), dict(base_stride=-1), dict(out_stride=31),
                                    dict(out=A), dict(out=A + 2 * 63), dict(out=A + 64 * 2 * 3), dict(out=A * 2 + 16), dict(out=A * 2, out_stride=40),
                                    dict(out=A * 2, base_stride=0), dict(rows=129), dict(rows=129, workspace=A + 8, workspace_bytes=1 << 20),
                                    dict(rows=129, workspace=A, workspace_bytes=100)])
def test_low_rank_refuses(change):
    assert refused(LIB.eps_b200_low_rank, low_rank(**change), None) == eps.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_low_rank, None, None) == eps.INVALID_ARGUMENT


def test_low_rank_layout():
    assert [LIB.eps_b200_low_rank_rank(r) for r in (1, 8, 9, 16, 17, 33, 64, 65, 128, 129)] == [8, 8, 16, 16, 32, 64, 64, 128, 128, 0]
    assert [LIB.eps_b200_low_rank_inner(k) for k in (1, 32, 33, 4096)] == [64, 64, 64, 4096]
    assert LIB.eps_b200_low_rank_workspace(128, 100) == 0
    for rows, n in ((129, 1), (1000, 16384), (100000, 3)):      # the units of the worst split, the rows' order, and a count
        assert LIB.eps_b200_low_rank_workspace(rows, n) >= 16 + 16 * (rows // 64 + min(rows, n + 1)) + 4 * rows


@pytest.mark.skipif(gpu_available(), reason="checks the no-GPU failure path")
def test_without_a_gpu_calls_fail_loudly():
    gone = (eps.UNAVAILABLE, eps.RUN_FAILED)
    assert refused(LIB.eps_b200_gradient_norm, norm(), None) in gone
    assert refused(LIB.eps_b200_balance_loss, balance(), A, A, A, A, A, None, 0, None) in gone
    assert refused(LIB.eps_b200_low_rank, low_rank(), None) in gone
    # what may share memory: base itself, and columns of one tensor
    assert refused(LIB.eps_b200_low_rank, low_rank(out=A * 2), None) in gone
    assert refused(LIB.eps_b200_low_rank, low_rank(x_stride=128, out_stride=128, out=A + 2 * 64), None) in gone
    assert refused(LIB.eps_b200_low_rank, low_rank(rows=0, x=None, out=None, ids=None), None) == 0


def test_host_tensors_are_refused():
    import torch
    x = torch.ones(4, 8)
    ids = torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: dense.GradientNorm([x]), lambda: dense.balance_loss(x, ids), lambda: dense.balance_loss_backward(x, ids, ids, 2),
                 lambda: dense.Adapters(x, x)):
        with pytest.raises(eps.EpsError) as e:
            call()
        assert e.value.code == eps.INVALID_ARGUMENT
