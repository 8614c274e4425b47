"""The dense operators' C entry points: declared, exported, bound, laid out alike, and refusing bad
arguments before they look for a GPU."""
import ctypes as C
import os
import re
import struct
import subprocess

import pytest

from conftest import ROOT, gpu_available, import_package

eps = import_package()
from eps_b200 import dense  # noqa: E402

HEADER = os.path.join(ROOT, "include", "eps_b200_dense.h")
LIB = eps.load_library()


def test_entry_points_are_declared_exported_and_bound():
    declared = set(re.findall(r"EPS_B200_EXPORT\s+[\w\s\*]+?\b(eps_b200_\w+)\s*\(", open(HEADER).read()))
    out = subprocess.run(["nm", "-D", "--defined-only", eps.library_path()], capture_output=True, text=True, check=True).stdout
    assert declared == set(dense.ENTRY_POINTS)
    assert declared <= set(re.findall(r"\bT\s+(eps_b200_\w+)", out))


def test_struct_layouts_match_the_header(tmp_path):
    pairs = [("EpsB200BlockNorm", dense.BlockNorm), ("EpsB200BlockNormGradients", dense.BlockNormGradientArgs),
             ("EpsB200RouteExperts", dense.RouteExperts), ("EpsB200Int8Product", dense.Int8Product),
             ("EpsB200AdamWTensor", dense.AdamWTensor), ("EpsB200AdamW", dense.AdamWArgs)]
    lines = []
    for c, py in pairs:
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in py._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "eps_b200_dense.h"\nint main(void){' + "".join(lines) + "return 0;}")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "s")]).split()]
    want = []
    for _, py in pairs:
        want += [C.sizeof(py)] + [getattr(py, f[0]).offset for f in py._fields_]
    assert got == want
    for packed, py in ((dense._BLOCK_NORM, dense.BlockNorm), (dense._BLOCK_NORM_GRADIENTS, dense.BlockNormGradientArgs),
                       (dense._ROUTE, dense.RouteExperts), (dense._INT8_PRODUCT, dense.Int8Product)):
        assert packed.size == C.sizeof(py)
        codes = {C.c_int32: "i", C.c_uint32: "I", C.c_uint64: "L", C.c_int64: "l", C.c_float: "f", C.c_void_p: "P"}
        plain = "".join(codes[f[1]] for f in py._fields_)
        assert struct.calcsize("@" + plain) == packed.size and len(packed.unpack(bytes(packed.size))) == len(py._fields_)


def refused(fn, *args):
    st = eps.Status()
    rc = fn(*args, C.byref(st))
    assert rc == st.code and (rc == 0 or st.message)
    return rc


A = 1 << 20      # an address that is only looked at, never read, by a call that is refused


def norm(**change):
    fields = dict(device=0, kind=0, gate_kind=2, activation=1, post_norm=1, pre_norm=1, type=1, residual_type=1, parameter_type=0,
                  columns=64, rows=4, epsilon=1e-6, scale=1.0, y=A, gate=A, y_stride=64, gate_stride=64)
    return bytes(dense.BlockNorm(**{**fields, **change}))


@pytest.mark.parametrize("change", [dict(kind=2), dict(gate_kind=3), dict(gate_kind=0), dict(activation=4), dict(type=3), dict(residual_type=2),
                                    dict(parameter_type=2), dict(columns=0), dict(columns=8193), dict(rows=1 << 40), dict(epsilon=0.0),
                                    dict(epsilon=float("nan")), dict(scale=float("nan")), dict(y=None)])
def test_block_norm_refuses(change):
    assert refused(LIB.eps_b200_block_norm, norm(**change), A, 64, A, 64, A, 64, None) == eps.INVALID_ARGUMENT
    g = dense.BlockNormGradientArgs(dz=A, h=A, dx=A)
    assert refused(LIB.eps_b200_block_norm_backward, norm(**change), bytes(g), None) == eps.INVALID_ARGUMENT


def test_block_norm_refuses_missing_tensors():
    call = lambda x, h, z: refused(LIB.eps_b200_block_norm, norm(), x, 64, h, 64, z, 64, None)  # noqa: E731
    assert call(None, A, A) == call(A, None, A) == call(A, A, None) == eps.INVALID_ARGUMENT
    back = lambda args, **g: refused(LIB.eps_b200_block_norm_backward, args, bytes(dense.BlockNormGradientArgs(**g)), None)  # noqa: E731
    assert back(norm(), dz=A) == eps.INVALID_ARGUMENT
    assert back(norm(pre_norm=0), dz=A, h=A) == eps.INVALID_ARGUMENT
    assert back(norm(y=None, gate=None, gate_kind=0), dh=A, dy=A) == eps.INVALID_ARGUMENT
    assert back(norm(post_norm=0), dh=A, dpost_weight=A) == eps.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_block_norm, None, A, 64, A, 64, A, 64, None) == eps.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_block_norm_backward, norm(), None, None) == eps.INVALID_ARGUMENT


def routing(**change):
    fields = dict(device=0, type=0, score=0, renormalise=1, experts=16, top_k=2, groups=4, top_groups=2, tokens=8, scale=1.0,
                  logits=A, logits_stride=16)
    return bytes(dense.RouteExperts(**{**fields, **change}))


@pytest.mark.parametrize("change", [dict(type=5), dict(score=2), dict(experts=0), dict(experts=1025), dict(groups=0), dict(groups=3),
                                    dict(top_groups=0), dict(top_groups=5), dict(top_k=0), dict(top_k=33), dict(top_k=9), dict(tokens=1 << 31),
                                    dict(scale=float("nan")), dict(logits=None)])
def test_routing_refuses(change):
    assert refused(LIB.eps_b200_route_experts, routing(**change), None, A, A, None, None, None, None, 0, None) == eps.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_route_experts_backward, routing(**change), A, A, A, 16, None) == eps.INVALID_ARGUMENT


def test_routing_refuses_missing_tensors():
    assert refused(LIB.eps_b200_route_experts, routing(), None, None, A, None, None, None, None, 0, None) == eps.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_route_experts, routing(), None, A, A, A, None, A, A, 1 << 20, None) == eps.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_route_experts_backward, routing(), A, None, A, 16, None) == eps.INVALID_ARGUMENT


def linear(**change):
    fields = dict(device=0, type=1, experts=2, channels=32, inner=64, rows_divisor=1, rows=4, weight=A, weight_scale=A, offsets=A, out=A,
                  workspace=A, workspace_bytes=1 << 20)
    return bytes(dense.Int8Product(**{**fields, **change}))


@pytest.mark.parametrize("change", [dict(type=7), dict(experts=0), dict(channels=0), dict(inner=0), dict(inner=131073), dict(rows=1 << 31),
                                    dict(offsets=None), dict(weight=None), dict(weight_scale=None), dict(out=None), dict(weight=A + 1),
                                    dict(out=A + 2), dict(workspace=A + 4)])
def test_int8_refuses(change):
    assert refused(LIB.eps_b200_int8_product, linear(**change), A, A, None) == eps.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_int8_linear, linear(**change), A, 64, 4, None, None) == eps.INVALID_ARGUMENT


def test_int8_refuses_missing_tensors():
    assert refused(LIB.eps_b200_int8_product, linear(), None, A, None) == eps.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_int8_product, linear(), A + 1, A, None) == eps.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_int8_linear, linear(rows=400, workspace_bytes=8), A, 64, 400, None, None) == eps.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_int8_linear, linear(), A, 64, 3, None, None) == eps.INVALID_ARGUMENT        # fewer rows than asked for
    assert refused(LIB.eps_b200_int8_linear, linear(rows_divisor=0), A, 64, 3, A, None) == eps.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_int8_quantize, 0, 0, A, 64, 4, 64, None, 1, 4, None, A, None) == eps.INVALID_ARGUMENT


def adamw(**change):
    fields = dict(device=0, parameter_type=1, gradient_type=1, state_bits=32, first=A, second=A, learning_rate=1e-3, beta1=0.9, beta2=0.999,
                  epsilon=1e-8, weight_decay=0.0, step=1)
    return C.byref(dense.AdamWArgs(**{**fields, **change}))


@pytest.mark.parametrize("change", [dict(parameter_type=4), dict(gradient_type=2), dict(state_bits=16), dict(state_bits=8), dict(first=None),
                                    dict(first=A + 4), dict(parameter_type=0, gradient_type=0, master=A), dict(step=0), dict(learning_rate=-1.0),
                                    dict(learning_rate=float("inf")), dict(beta1=1.0), dict(beta2=-1.0), dict(epsilon=0.0), dict(weight_decay=float("nan"))])
def test_adamw_refuses(change):
    assert refused(LIB.eps_b200_adamw, adamw(**change), A, 1, 1, None) == eps.INVALID_ARGUMENT


def test_adamw_plan():
    t = (dense.AdamWTensor * 3)(dense.AdamWTensor(A, A, 10000, 0), dense.AdamWTensor(A, A, 0, 10240), dense.AdamWTensor(A, A, 4096, 10240))
    size = LIB.eps_b200_adamw_plan_bytes(t, 3)
    plan, blocks = (C.c_uint8 * size)(), C.c_uint64()
    assert refused(LIB.eps_b200_adamw_plan, t, 3, plan, size, C.byref(blocks)) == 0
    chunks = (C.c_uint32 * (2 * blocks.value)).from_buffer(plan, 3 * C.sizeof(dense.AdamWTensor))
    elements = lambda c: 2048 * c[1]  # noqa: E731
    seen = [(chunks[2 * i], chunks[2 * i + 1]) for i in range(blocks.value)]
    assert size == 3 * C.sizeof(dense.AdamWTensor) + 8 * blocks.value
    for tensor, n in ((0, 10000), (1, 0), (2, 4096)):
        mine = [elements(c) for c in seen if c[0] == tensor]
        assert mine == list(range(0, n, 2048))
    assert refused(LIB.eps_b200_adamw_plan, t, 3, plan, size - 1, C.byref(blocks)) == eps.INVALID_ARGUMENT
    t[2].state_begin = 10241
    assert refused(LIB.eps_b200_adamw_plan, t, 3, plan, size, C.byref(blocks)) == eps.INVALID_ARGUMENT
    t[2].state_begin, t[2].gradient = 10240, None
    assert refused(LIB.eps_b200_adamw_plan, t, 3, plan, size, C.byref(blocks)) == eps.INVALID_ARGUMENT


@pytest.mark.skipif(gpu_available(), reason="checks the no-GPU failure path")
def test_without_a_gpu_calls_fail_loudly():
    assert refused(LIB.eps_b200_route_experts, routing(), None, A, A, None, None, None, None, 0, None) in (eps.UNAVAILABLE, eps.RUN_FAILED)
    assert refused(LIB.eps_b200_adamw, adamw(), A, 1, 1, None) in (eps.UNAVAILABLE, eps.RUN_FAILED)


def test_host_tensors_are_refused():
    import torch
    x = torch.ones(4, 8)
    for call in (lambda: dense.block_norm(x), lambda: dense.route(x, 2), lambda: dense.quantize_rows(x), lambda: dense.AdamW([x])):
        with pytest.raises(eps.EpsError) as e:
            call()
        assert e.value.code == eps.INVALID_ARGUMENT
