"""The dense block beside the embedding store: Python binding of include/eps_b200_dense.h.

    h, z = dense.block_norm(x, y, gate, post_weight=..., pre_weight=..., scale=0.5)
    routing = dense.route(logits, top_k=8, score="sigmoid", bias=balance)
    experts = dense.QuantizedExperts.from_weights(weight)          # [experts, channels, inner]
    out = experts.product(z, offsets=routing.offsets, rows=routing.order, rows_divisor=8)
    out = dense.Adapters(down, up).product(x, ids, base=layer.product(x))
    balance = dense.balance_loss(logits, routing.experts)
    clip = dense.GradientNorm(gradients).measure(max_norm=1.0)
    dense.AdamW(parameters, gradients, state_bits=8).step(gradient_scale=clip.scale, skip=clip.skip)

Every tensor is a torch CUDA tensor; work goes to torch's current stream of the
tensors' device and is asynchronous, results and workspaces come from torch's
allocator, and nothing is kept between calls but what the classes hold.  Calls
can be captured in a CUDA graph; a captured AdamW step counts its replays.  There is no CPU fallback; a refused call raises
``EpsError`` with ``code`` INVALID_ARGUMENT before anything is launched.

Results carry no autograd history, whether their inputs require gradients or not:
gradients come from the *_backward functions.

Leading axes of a tensor count as rows; the last axis must be contiguous, rows may
have any stride.  Element types are float32, bfloat16 and float16.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
import threading
from array import array
from typing import NamedTuple, Sequence

import torch

from . import EpsError, INVALID_ARGUMENT, Status, load_library

__all__ = ["block_norm", "block_norm_backward", "BlockNormGradients", "route", "route_backward",
           "Routing", "balance_loss", "balance_loss_backward", "BalanceLoss", "quantize_rows", "QuantizedExperts",
           "Adapters", "GradientNorm", "GradientMeasure", "AdamW", "ENTRY_POINTS"]

ENTRY_POINTS = ("eps_b200_block_norm", "eps_b200_block_norm_workspace",
                "eps_b200_block_norm_backward", "eps_b200_route_experts_workspace",
                "eps_b200_route_experts", "eps_b200_route_experts_backward",
                "eps_b200_int8_stride", "eps_b200_int8_quantize",
                "eps_b200_int8_product_workspace", "eps_b200_int8_product", "eps_b200_int8_linear",
                "eps_b200_adamw_plan_bytes", "eps_b200_adamw_plan", "eps_b200_adamw", "eps_b200_adamw_counted",
                "eps_b200_gradient_norm_plan_bytes", "eps_b200_gradient_norm_plan",
                "eps_b200_gradient_norm_workspace", "eps_b200_gradient_norm",
                "eps_b200_balance_loss_workspace", "eps_b200_balance_loss", "eps_b200_balance_loss_backward",
                "eps_b200_low_rank_rank", "eps_b200_low_rank_inner", "eps_b200_low_rank_workspace", "eps_b200_low_rank")

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_KINDS = {"rms": 0, "layer": 1}
_ACTIVATIONS = {"none": 0, "sigmoid": 1, "silu": 2, "tanh": 3}
_SCORES = {"softmax": 0, "sigmoid": 1}
_NORMS = {"l2": 0, "max": 1}
ADAMW_BLOCK = 256           # elements of a tensor that share a scale (EPS_B200_ADAMW_BLOCK)


# ------------------------------------------------------------------ C structs
class BlockNorm(C.Structure):
    _fields_ = [("device", C.c_int32), ("kind", C.c_int32), ("gate_kind", C.c_int32),
                ("activation", C.c_int32), ("post_norm", C.c_int32), ("pre_norm", C.c_int32),
                ("type", C.c_int32), ("residual_type", C.c_int32), ("parameter_type", C.c_int32),
                ("columns", C.c_uint32), ("rows", C.c_uint64), ("epsilon", C.c_float),
                ("scale", C.c_float), ("y", C.c_void_p), ("gate", C.c_void_p),
                ("y_stride", C.c_int64), ("gate_stride", C.c_int64), ("post_weight", C.c_void_p),
                ("post_bias", C.c_void_p), ("channel_scale", C.c_void_p),
                ("pre_weight", C.c_void_p), ("pre_bias", C.c_void_p)]


class BlockNormGradientArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("dh", "dz", "h")] + \
               [(n, C.c_int64) for n in ("dh_stride", "dz_stride", "h_stride")] + \
               [(n, C.c_void_p) for n in ("dx", "dy", "dgate")] + \
               [(n, C.c_int64) for n in ("dx_stride", "dy_stride", "dgate_stride")] + \
               [(n, C.c_void_p) for n in ("dpost_weight", "dpost_bias", "dchannel_scale",
                                          "dpre_weight", "dpre_bias", "workspace")] + \
               [("workspace_bytes", C.c_uint64)]


class RouteExperts(C.Structure):
    _fields_ = [("device", C.c_int32), ("type", C.c_int32), ("score", C.c_int32),
                ("renormalise", C.c_int32), ("experts", C.c_uint32), ("top_k", C.c_uint32),
                ("groups", C.c_uint32), ("top_groups", C.c_uint32), ("tokens", C.c_uint64),
                ("scale", C.c_float), ("reserved", C.c_int32), ("logits", C.c_void_p),
                ("logits_stride", C.c_int64)]


class Int8Product(C.Structure):
    _fields_ = [("device", C.c_int32), ("type", C.c_int32), ("experts", C.c_uint32),
                ("channels", C.c_uint32), ("inner", C.c_uint32), ("rows_divisor", C.c_uint32),
                ("rows", C.c_uint64), ("weight", C.c_void_p), ("weight_scale", C.c_void_p),
                ("bias", C.c_void_p), ("offsets", C.c_void_p), ("out", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64)]


class AdamWTensor(C.Structure):      # four words
    _fields_ = [("parameter", C.c_void_p), ("gradient", C.c_void_p), ("elements", C.c_uint64),
                ("state_begin", C.c_uint64)]


class AdamWArgs(C.Structure):
    _fields_ = [("device", C.c_int32), ("parameter_type", C.c_int32), ("gradient_type", C.c_int32),
                ("state_bits", C.c_int32), ("master", C.c_void_p), ("first", C.c_void_p),
                ("second", C.c_void_p), ("first_scale", C.c_void_p), ("second_scale", C.c_void_p),
                ("gradient_scale", C.c_void_p), ("skip", C.c_void_p), ("learning_rate", C.c_double),
                ("beta1", C.c_double), ("beta2", C.c_double), ("epsilon", C.c_double),
                ("weight_decay", C.c_double), ("step", C.c_uint64), ("seed", C.c_uint64)]


class AdamWClock(C.Structure):
    _fields_ = [("taken", C.c_int64), ("learning_rate", C.c_double), ("decay", C.c_float), ("rate", C.c_float),
                ("inverse_root", C.c_float), ("key", C.c_uint32)]


class Gradient(C.Structure):      # three words, of which the last is the type
    _fields_ = [("gradient", C.c_void_p), ("elements", C.c_uint64), ("type", C.c_int32), ("reserved", C.c_int32)]


class GradientNormArgs(C.Structure):
    _fields_ = [("device", C.c_int32), ("kind", C.c_int32), ("clip", C.c_int32), ("reserved", C.c_int32),
                ("plan", C.c_void_p), ("blocks", C.c_uint64), ("gradient_scale", C.c_void_p),
                ("max_norm", C.c_double), ("result", C.c_void_p), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_uint64)]


class BalanceLossArgs(C.Structure):
    _fields_ = [("device", C.c_int32), ("type", C.c_int32), ("score", C.c_int32),
                ("normalise", C.c_int32), ("experts", C.c_uint32), ("top_k", C.c_uint32),
                ("tokens", C.c_uint64), ("weight", C.c_float), ("reserved", C.c_int32),
                ("logits", C.c_void_p), ("logits_stride", C.c_int64), ("mask", C.c_void_p)]


class LowRank(C.Structure):
    _fields_ = [("device", C.c_int32), ("type", C.c_int32), ("adapters", C.c_uint32),
                ("rank", C.c_uint32), ("inner", C.c_uint32), ("channels", C.c_uint32),
                ("rows", C.c_uint64)] + \
               [(n, C.c_void_p) for n in ("down", "up", "scale", "ids", "x", "base", "out")] + \
               [(n, C.c_int64) for n in ("x_stride", "base_stride", "out_stride")] + \
               [("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64)]


def _bind():
    # the structs that are packed for each call go in as bytes of the same layout
    lib, P, vp, i64, u64, u32, i32 = (load_library(), C.POINTER, C.c_void_p, C.c_int64, C.c_uint64,
                                      C.c_uint32, C.c_int32)
    st = P(Status)
    lib.eps_b200_block_norm.argtypes = [C.c_char_p, vp, i64, vp, i64, vp, i64, vp, st]
    lib.eps_b200_block_norm_workspace.argtypes = [u64, u32]
    lib.eps_b200_block_norm_backward.argtypes = [C.c_char_p, C.c_char_p, vp, st]
    lib.eps_b200_route_experts_workspace.argtypes = [u64, u32, u32]
    lib.eps_b200_route_experts.argtypes = [C.c_char_p, vp, vp, vp, vp, vp, vp, vp, u64, vp, st]
    lib.eps_b200_route_experts_backward.argtypes = [C.c_char_p, vp, vp, vp, i64, vp, st]
    lib.eps_b200_int8_stride.argtypes = [u32]
    lib.eps_b200_int8_quantize.argtypes = [i32, i32, vp, i64, u64, u32, vp, u32, u64, vp, vp, vp, st]
    lib.eps_b200_int8_product_workspace.argtypes = [u64, u32, u32, u32]
    lib.eps_b200_int8_product.argtypes = [C.c_char_p, vp, vp, vp, st]
    lib.eps_b200_int8_linear.argtypes = [C.c_char_p, vp, i64, u64, vp, vp, st]
    lib.eps_b200_adamw_plan_bytes.argtypes = [P(AdamWTensor), u64]
    lib.eps_b200_adamw_plan.argtypes = [P(AdamWTensor), u64, vp, u64, P(u64), st]
    lib.eps_b200_adamw.argtypes = [P(AdamWArgs), vp, u64, u64, vp, st]
    lib.eps_b200_adamw_counted.argtypes = [P(AdamWArgs), vp, u64, u64, vp, vp, st]
    lib.eps_b200_gradient_norm_plan_bytes.argtypes = [P(Gradient), u64]
    lib.eps_b200_gradient_norm_plan.argtypes = [P(Gradient), u64, vp, u64, P(u64), st]
    lib.eps_b200_gradient_norm_workspace.argtypes = [u64]
    lib.eps_b200_gradient_norm.argtypes = [C.c_char_p, vp, st]
    lib.eps_b200_balance_loss_workspace.argtypes = [u64, u32]
    lib.eps_b200_balance_loss.argtypes = [C.c_char_p, vp, vp, vp, vp, vp, vp, u64, vp, st]
    lib.eps_b200_balance_loss_backward.argtypes = [C.c_char_p, vp, vp, vp, vp, i64, vp, i64, vp, st]
    lib.eps_b200_low_rank_rank.argtypes = [u32]
    lib.eps_b200_low_rank_inner.argtypes = [u32]
    lib.eps_b200_low_rank_workspace.argtypes = [u64, u32]
    lib.eps_b200_low_rank.argtypes = [C.c_char_p, vp, st]
    for name in ENTRY_POINTS:
        sized = name.endswith(("_workspace", "_bytes", "_stride", "_low_rank_rank", "_inner"))
        getattr(lib, name).restype = u64 if sized else C.c_int
    return lib


_lib = _bind()
_local = threading.local()


def _status():
    st = getattr(_local, "status", None)
    if st is None:
        st = _local.status = Status()
        _local.ref = C.byref(st)
    return st, _local.ref


def _call(fn, *args):
    st, ref = _status()
    rc = fn(*args, ref)
    if rc:
        raise EpsError(rc, st.message.decode(errors="replace"))


def _refuse(message):
    raise EpsError(INVALID_ARGUMENT, message)


def _choice(table, value, what):
    try:
        return table[value]
    except (KeyError, TypeError):
        _refuse(f"{what} is one of {', '.join(map(str, table))}: got {value!r}")


# A call of a small size takes the host longer than the GPU, so what follows is written
# for few and cheap steps: device indices instead of device objects, the stream's raw
# handle, and argument structs packed in one go.
_stream = torch._C._cuda_getCurrentRawStream      # of a device index


def _capturing(device):
    """Whether the current stream of a device index is being captured in a graph."""
    if torch._C._cuda_getDevice() != device:
        with torch.cuda.device(device):
            return torch._C._cuda_isCurrentStreamCapturing()
    return torch._C._cuda_isCurrentStreamCapturing()


def _tensor(t, what, device=None):
    """t's device index; refuses what is no CUDA tensor, or on another device."""
    index = t.get_device() if isinstance(t, torch.Tensor) else -1
    if index < 0:
        _refuse(f"{what} must be a CUDA tensor")
    if device is not None and index != device:
        _refuse(f"{what} is on cuda:{index}, not on cuda:{device}")
    return index


def _matrix(t, what, device=None, columns=None, rows=None):
    """(t as rows by columns, its row stride, rows, columns); its last axis contiguous."""
    _tensor(t, what, device)
    if t.dtype not in _TYPES:
        _refuse(f"{what} must be float32, bfloat16 or float16")
    if t.dim() != 2:
        if t.dim() < 1:
            _refuse(f"{what} must have a last axis")
        try:
            t = t.view(-1, t.shape[-1]) if t.numel() else t.reshape(0, t.shape[-1])
        except RuntimeError:
            _refuse(f"{what}: its leading axes cannot be seen as one")
    n, width = t.shape
    if columns is not None and width != columns:
        _refuse(f"{what} has {width} columns, not {columns}")
    if rows is not None and n != rows:
        _refuse(f"{what} has {n} rows, not {rows}")
    stride, inner = t.stride()
    if inner != 1 and width > 1:
        _refuse(f"the last axis of {what} must be contiguous")
    return t, stride, n, width


def _vector(t, what, device, n, dtype):
    """The address of a contiguous vector of n elements; 0 for None."""
    if t is None:
        return 0
    _tensor(t, what, device)
    if t.dtype != dtype or t.numel() != n or not t.is_contiguous():
        _refuse(f"{what} must be a contiguous {dtype} vector of {n}")
    return t.data_ptr()


def _ptr(t):
    return 0 if t is None else t.data_ptr()


class _Streams:
    """The streams on which tensors that the package holds are used.  torch's allocator hands
    freed memory out again in the order of the stream that it was made on; it has to hear of
    the others, or what is dropped here could be overwritten under a running kernel."""

    def __init__(self, device, *own, given=()):
        """own: made now, on the current stream; given: made by the caller, on streams that
        are not known here."""
        self.seen = set() if given else {_stream(device)}
        self.tensors = [t for t in (*own, *given) if t is not None]

    def use(self, stream, device):
        if stream not in self.seen:
            current = torch.cuda.current_stream(device)
            for t in self.tensors:
                t.record_stream(current)
            self.seen.add(stream)


def _pack(fields, *values):
    try:
        return fields.pack(*values)
    except (struct.error, TypeError, OverflowError) as e:
        _refuse(f"an argument is out of range: {e}")


# ------------------------------------------------------------ norms and gate
class BlockNormGradients(NamedTuple):
    """Gradients of block_norm's inputs; None for what was not given."""
    x: torch.Tensor
    y: torch.Tensor | None
    gate: torch.Tensor | None
    post_weight: torch.Tensor | None
    post_bias: torch.Tensor | None
    channel_scale: torch.Tensor | None
    pre_weight: torch.Tensor | None
    pre_bias: torch.Tensor | None


_BLOCK_NORM = struct.Struct("@9iIQ2f2P2q5P")           # BlockNorm
_BLOCK_NORM_GRADIENTS = struct.Struct("@3P3q3P3q6PQ")    # BlockNormGradientArgs


def _block_norm_args(device, rows, columns, rtype, y, gate, post_weight, post_bias, pre_weight, pre_bias,
                     channel_scale, scale, kind, activation, epsilon, post_norm, pre_norm, dtype):
    """The packed struct for a residual of rows by columns."""
    ptype = torch.float32
    for p in (post_weight, pre_weight, channel_scale, post_bias, pre_bias):
        if p is not None:
            ptype = p.dtype if isinstance(p, torch.Tensor) else None
            break
    if ptype != torch.float32 and ptype != dtype:
        _refuse("weights, biases and channel_scale have the block's type or float32, all the same")
    y_stride = gate_stride = gate_kind = 0
    if y is not None:
        y, y_stride, _, _ = _matrix(y, "y", device, columns, rows)
    if gate is not None:
        if y is None:
            _refuse("a gate needs a block output y")
        _tensor(gate, "gate", device)
        if gate.dtype != dtype:
            _refuse("the gate has the type of y")
        # one value a row: [rows] or [..., 1]; where D is 1 that is an element gate too, but not without its last axis
        if gate.numel() == rows and (columns > 1 or gate.dim() == 1):
            gate_kind = 1
            if not gate.is_contiguous():
                _refuse("a gate of one value a row must be contiguous")
        else:
            gate_kind = 2
            gate, gate_stride, _, _ = _matrix(gate, "gate", device, columns, rows)
    return _pack(_BLOCK_NORM, device, _choice(_KINDS, kind, "kind"), gate_kind,
                 _choice(_ACTIVATIONS, activation, "activation"), bool(post_norm), bool(pre_norm),
                 _TYPES[dtype], _TYPES[rtype], _TYPES[ptype], columns, rows, epsilon, scale,
                 _ptr(y), _ptr(gate), y_stride, gate_stride,
                 _vector(post_weight, "post_weight", device, columns, ptype),
                 _vector(post_bias, "post_bias", device, columns, ptype),
                 _vector(channel_scale, "channel_scale", device, columns, ptype),
                 _vector(pre_weight, "pre_weight", device, columns, ptype),
                 _vector(pre_bias, "pre_bias", device, columns, ptype))


def _block_type(residual, y, device):
    if y is None:
        return residual.dtype
    _tensor(y, "y", device)
    if y.dtype not in _TYPES:
        _refuse("y must be float32, bfloat16 or float16")
    return y.dtype


def block_norm(x, y=None, gate=None, *, post_weight=None, post_bias=None, pre_weight=None,
               pre_bias=None, channel_scale=None, scale: float = 1.0, kind: str = "rms",
               activation: str = "sigmoid", epsilon: float = 1e-6, post_norm: bool = True,
               pre_norm: bool = True):
    """The joint between two blocks of a residual network, in one pass.

        h = x + scale * channel_scale * activation(gate) * post_norm(y)
        z = pre_norm(h)

    x is the residual, y the output of the block before ([..., D]; None: h is x
    itself), gate its gate ([..., D] or one value a row), z the input of the block
    after.  x has the type of y, or is float32; z has the type of y.  kind "rms" or
    "layer"; activation "none", "sigmoid", "silu" or "tanh".  Weights, biases and
    channel_scale are vectors of D, all float32 or all of y's type.  D is at most
    8192.  Returns (h, z), z None without pre_norm."""
    residual, x_stride, rows, columns = _matrix(x, "x")
    device = residual.get_device()
    dtype = _block_type(residual, y, device)
    args = _block_norm_args(device, rows, columns, residual.dtype, y, gate, post_weight, post_bias, pre_weight,
                            pre_bias, channel_scale, scale, kind, activation, epsilon, post_norm, pre_norm, dtype)
    dense = torch.contiguous_format
    h = x if y is None else torch.empty_like(x, memory_format=dense)
    z = None
    if pre_norm:
        z = torch.empty_like(x, memory_format=dense) if dtype == x.dtype else torch.empty_like(x, dtype=dtype, memory_format=dense)
    _call(_lib.eps_b200_block_norm, args, residual.data_ptr(), x_stride, 0 if y is None else h.data_ptr(), columns,
          _ptr(z), columns, _stream(device))
    return h, z


def block_norm_backward(dh, dz, h, y=None, gate=None, *, post_weight=None, post_bias=None,
                        pre_weight=None, pre_bias=None, channel_scale=None, scale: float = 1.0,
                        kind: str = "rms", activation: str = "sigmoid", epsilon: float = 1e-6,
                        post_norm: bool = True, pre_norm: bool = True) -> BlockNormGradients:
    """Gradients of block_norm from those of its outputs, dh and dz (either may be
    None: no gradient comes that way).  h is the forward's output, the other
    arguments are the forward's inputs; x itself is not needed.  The statistics are
    computed again from h and y.  Gradients of x, y and gate have their types,
    gradients of weights, biases and channel_scale are float32.  Sums over rows are
    taken in a fixed order."""
    residual, h_stride, rows, columns = _matrix(h, "h")
    device = residual.get_device()
    dtype = _block_type(residual, y, device)
    args = _block_norm_args(device, rows, columns, residual.dtype, y, gate, post_weight, post_bias, pre_weight,
                            pre_bias, channel_scale, scale, kind, activation, epsilon, post_norm, pre_norm, dtype)
    if dz is not None and not pre_norm:
        _refuse("dz needs pre_norm")
    dh_stride = dz_stride = 0
    if dh is not None:
        dh, dh_stride, _, _ = _matrix(dh, "dh", device, columns, rows)
        if dh.dtype != residual.dtype:
            _refuse("dh has the type of h")
    if dz is not None:
        dz, dz_stride, _, _ = _matrix(dz, "dz", device, columns, rows)
        if dz.dtype != dtype:
            _refuse("dz has the type of y")
    dense = torch.contiguous_format
    dx = torch.empty_like(h, memory_format=dense)
    dy = None if y is None else torch.empty_like(y, memory_format=dense)
    dgate = None if gate is None else torch.empty_like(gate, memory_format=dense)
    post, pre = y is not None and post_norm, pre_norm
    wanted = (post and post_weight is not None, post and post_bias is not None,
              y is not None and channel_scale is not None, pre and pre_weight is not None,
              pre and pre_bias is not None)
    vectors, space, workspace = [None] * 5, 0, None
    if any(wanted):
        rest = iter(torch.empty((sum(wanted), columns), dtype=torch.float32, device=h.device).unbind())
        vectors = [next(rest) if w else None for w in wanted]
        space = _lib.eps_b200_block_norm_workspace(rows, columns)
        workspace = torch.empty(space, dtype=torch.uint8, device=h.device)
    grads = _pack(_BLOCK_NORM_GRADIENTS, _ptr(dh), _ptr(dz), residual.data_ptr(), dh_stride, dz_stride, h_stride,
                  dx.data_ptr(), _ptr(dy), _ptr(dgate), columns, columns, columns, *map(_ptr, vectors), _ptr(workspace), space)
    _call(_lib.eps_b200_block_norm_backward, args, grads, _stream(device))
    return BlockNormGradients(dx, dy, dgate, *vectors)


# ------------------------------------------------------------------- routing
class Routing(NamedTuple):
    """experts [tokens, top_k] int32, best first; weights [tokens, top_k] float32.
    Entry token * top_k + slot lies at position[token, slot] of `order`, the entries
    sorted by expert; expert e owns order[offsets[e]:offsets[e + 1]].  order, position
    and offsets are None if not asked for."""
    experts: torch.Tensor
    weights: torch.Tensor
    order: torch.Tensor | None
    position: torch.Tensor | None
    offsets: torch.Tensor | None


_ROUTE = struct.Struct("@4i4IQfiPq")          # RouteExperts


def _route_args(logits, stride, tokens, experts, top_k, score, renormalise, scale, groups, top_groups):
    return _pack(_ROUTE, logits.get_device(), _TYPES[logits.dtype], _choice(_SCORES, score, "score"),
                 bool(renormalise), experts, top_k, groups, top_groups, tokens, scale, 0, logits.data_ptr(), stride)


def route(logits, top_k: int, *, score: str = "softmax", bias=None, groups: int = 1,
          top_groups: int | None = None, renormalise: bool = True, scale: float = 1.0,
          sort: bool = True) -> Routing:
    """Routes tokens to their top_k experts.

    logits [tokens, experts].  Scores are softmax or sigmoid of the logits; `bias`
    (float32 [experts]) is added for the ranking alone.  With groups, only experts of
    the top_groups best of `groups` equal runs are eligible, a group counting the sum
    of its two best keys.  Weights are the chosen scores, divided by their sum if
    `renormalise`, times `scale`.  Equal keys go to the lower index; a masked logit
    is -inf, and ranks last whatever its bias.  At most 1024 experts and top_k 32.
    With `sort`, the entries sorted by expert come too."""
    logits, stride, tokens, experts = _matrix(logits, "logits")
    top_groups = groups if top_groups is None else top_groups
    if top_k <= 0 or groups <= 0 or top_groups <= 0:
        _refuse("top_k, groups and top_groups are positive")
    args = _route_args(logits, stride, tokens, experts, top_k, score, renormalise, scale, groups, top_groups)
    index, device = logits.get_device(), logits.device
    b = _vector(bias, "bias", index, experts, torch.float32)
    chosen = torch.empty((tokens, top_k), dtype=torch.int32, device=device)
    weights = torch.empty_like(chosen, dtype=torch.float32)
    if not sort:
        _call(_lib.eps_b200_route_experts, args, b, chosen.data_ptr(), weights.data_ptr(), 0, 0, 0, 0, 0, _stream(index))
        return Routing(chosen, weights, None, None, None)
    position = torch.empty_like(chosen)
    order = torch.empty_like(chosen).view(-1)
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=device)
    space = _lib.eps_b200_route_experts_workspace(tokens, experts, top_k)
    workspace = torch.empty(space, dtype=torch.uint8, device=device) if space else None
    # an empty tensor has no address, yet it is asked for
    _call(_lib.eps_b200_route_experts, args, b, chosen.data_ptr(), weights.data_ptr(),
          order.data_ptr() or offsets.data_ptr(), position.data_ptr() or offsets.data_ptr(), offsets.data_ptr(),
          _ptr(workspace), space, _stream(index))
    return Routing(chosen, weights, order, position, offsets)


def route_backward(logits, experts, dweights, *, score: str = "softmax", renormalise: bool = True,
                   scale: float = 1.0):
    """The logits' gradient from that of route's weights, for the experts it chose;
    the choice itself, the bias and the groups take none."""
    flat, stride, tokens, count = _matrix(logits, "logits")
    index = flat.get_device()
    _tensor(experts, "experts", index)
    _tensor(dweights, "dweights", index)
    if experts.dim() < 1 or experts.shape[-1] == 0 or experts.dtype != torch.int32 or not experts.is_contiguous():
        _refuse("experts must be a contiguous int32 tensor, as route gives it")
    top_k = experts.shape[-1]
    if experts.numel() != tokens * top_k:
        _refuse("experts and logits have different numbers of tokens")
    if dweights.dtype != torch.float32 or dweights.numel() != experts.numel() or not dweights.is_contiguous():
        _refuse("dweights must be contiguous float32, in the shape of experts")
    args = _route_args(flat, stride, tokens, count, top_k, score, renormalise, scale, 1, 1)
    out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    _call(_lib.eps_b200_route_experts_backward, args, experts.data_ptr(), dweights.data_ptr(), out.data_ptr(), count, _stream(index))
    return out


# -------------------------------------------------------------- balance loss
class BalanceLoss(NamedTuple):
    """loss, a float32 scalar; counts [experts] int32, each expert's entries; mass [experts]
    float32, the sum of its p over the tokens; tokens, an int32 scalar, how many were
    counted.  Of several ranks with a batch each, counts, mass and tokens add up to those
    of the joint batch."""
    loss: torch.Tensor
    counts: torch.Tensor
    mass: torch.Tensor
    tokens: torch.Tensor


_BALANCE = struct.Struct("@4i2IQfiPqP")          # BalanceLossArgs


def _balance_args(logits, stride, tokens, experts, top_k, score, normalise, mask, weight):
    index, at = logits.get_device(), 0
    if mask is not None:
        _tensor(mask, "mask", index)
        if mask.dtype != torch.bool or mask.numel() != tokens or not mask.is_contiguous():
            _refuse("mask must be contiguous bool, a value for each token")
        at = mask.data_ptr()
    return _pack(_BALANCE, index, _TYPES[logits.dtype], _choice(_SCORES, score, "score"), bool(normalise), experts, top_k,
                 tokens, weight, 0, logits.data_ptr(), stride, at)


def balance_loss(logits, experts, *, score: str = "softmax", normalise: bool = True, mask=None,
                 weight: float = 1.0) -> BalanceLoss:
    """The loss that balances a router's experts, and how many entries each has.

        p = softmax(logits) or sigmoid(logits), the latter divided by its sum if `normalise`
        loss = weight * E / (top_k * n^2) * sum_e counts[e] * mass[e],  mass[e] = sum_t p[t, e]

    logits [tokens, E]; experts [tokens, top_k] int32, as route gives them (entries outside
    [0, E) count for none).  mask [tokens] bool: only these n tokens count, the others'
    logits are not read.  A row of masked logits (-inf) alone has p = 0, and so has one of
    sigmoids of -88.71 and less, where float scores end; without a token the loss is 0.  At
    most 1024 experts and top_k 32."""
    logits, stride, tokens, count = _matrix(logits, "logits")
    index, device = logits.get_device(), logits.device
    _tensor(experts, "experts", index)
    if experts.dim() < 1 or experts.shape[-1] == 0 or experts.dtype != torch.int32 or not experts.is_contiguous():
        _refuse("experts must be a contiguous int32 tensor, as route gives it")
    top_k = experts.shape[-1]
    if experts.numel() != tokens * top_k:
        _refuse("experts and logits have different numbers of tokens")
    args = _balance_args(logits, stride, tokens, count, top_k, score, normalise, mask, weight)
    # one allocation: counts, mass, loss and tokens, 4 bytes each
    room = torch.empty(2 * count + 2, dtype=torch.int32, device=device)
    at = room.data_ptr()
    space = _lib.eps_b200_balance_loss_workspace(tokens, count)
    workspace = torch.empty(space, dtype=torch.uint8, device=device) if space else None
    _call(_lib.eps_b200_balance_loss, args, experts.data_ptr(), at + 8 * count, at, at + 4 * count, at + 8 * count + 4,
          _ptr(workspace), space, _stream(index))
    counts, mass, last = room.split_with_sizes((count, count, 2))
    loss, counted = last.unbind()
    return BalanceLoss(loss.view(torch.float32), counts, mass.view(torch.float32), counted)


def balance_loss_backward(logits, counts, tokens, top_k: int, *, score: str = "softmax", normalise: bool = True,
                          mask=None, weight: float = 1.0, dloss=None, add=None):
    """The logits' gradient from that of balance_loss (dloss, a float32 scalar on the GPU;
    None: 1), in the logits' type.  counts and tokens are the forward's, or their sums over
    ranks; the counts take no gradient.  `add`, a gradient of the logits that comes another
    way (route_backward's), is added before the one rounding; masked tokens get it alone."""
    flat, stride, rows, count = _matrix(logits, "logits")
    index = flat.get_device()
    if top_k <= 0:
        _refuse("top_k is positive")
    at = _vector(counts, "counts", index, count, torch.int32)
    n = _vector(tokens, "tokens", index, 1, torch.int32)
    d = _vector(dloss, "dloss", index, 1, torch.float32)
    add_stride = 0
    if add is not None:
        add, add_stride, _, _ = _matrix(add, "add", index, count, rows)
        if add.dtype != flat.dtype:
            _refuse("add has the type of the logits")
    args = _balance_args(flat, stride, rows, count, top_k, score, normalise, mask, weight)
    out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    _call(_lib.eps_b200_balance_loss_backward, args, at, n, d, _ptr(add), add_stride, out.data_ptr(), count, _stream(index))
    return out


# ------------------------------------------------------------- 8-bit products
def _row_index(rows, rows_divisor, device):
    if rows is None:
        return 0
    _tensor(rows, "rows", device)
    if rows.dtype != torch.int32 or rows.dim() != 1 or not rows.is_contiguous():
        _refuse("rows must be a contiguous int32 vector")
    if rows_divisor <= 0:
        _refuse("rows_divisor is positive")
    return rows.data_ptr()


def quantize_rows(x, rows=None, rows_divisor: int = 1):
    """x [..., inner] in 8-bit integers with one scale a row: (q, scale) with q
    [n, stride] int8, zeros behind `inner`, and scale [n] float32.  Row r is
    x[rows[r] // rows_divisor], or x[r] without `rows`."""
    x, stride, x_rows, inner = _matrix(x, "x")
    device = x.get_device()
    index = _row_index(rows, rows_divisor, device)
    n = x_rows if rows is None else rows.shape[0]
    padded = _lib.eps_b200_int8_stride(inner)
    q = torch.empty((n, padded), dtype=torch.int8, device=x.device)
    scale = torch.empty(n, dtype=torch.float32, device=x.device)
    _call(_lib.eps_b200_int8_quantize, device, _TYPES[x.dtype], x.data_ptr(), stride, x_rows, inner,
          index, rows_divisor, n, q.data_ptr(), scale.data_ptr(), _stream(device))
    return q, scale


_INT8_PRODUCT = struct.Struct("@2i4IQ6PQ")          # Int8Product


class QuantizedExperts:
    """The weights of one linear layer, or of one for each of several experts, held
    in 8-bit integers with a scale for each output channel; laid out once."""

    def __init__(self, weight, scale, bias=None):
        """weight int8 [experts, channels, inner] (or [channels, inner]), scale and
        bias float32 [experts, channels]."""
        _tensor(weight, "weight")
        if weight.dtype != torch.int8 or weight.dim() not in (2, 3) or 0 in weight.shape:
            _refuse("weight must be int8 [experts, channels, inner] or [channels, inner]")
        weight = weight if weight.dim() == 3 else weight[None]
        self.experts, self.channels, self.inner = weight.shape
        self.device = weight.device
        n = self.experts * self.channels
        for t, what in ((scale, "scale"), (bias, "bias")):
            _vector(t, what, weight.get_device(), n, torch.float32)
        if scale is None:
            _refuse("the weights need their scales")
        self.stride = _lib.eps_b200_int8_stride(self.inner)
        self.weight = torch.zeros((self.experts, self.channels, self.stride), dtype=torch.int8, device=self.device)
        self.weight[..., : self.inner] = weight
        self.scale = scale.reshape(self.experts, self.channels)
        self.bias = None if bias is None else bias.reshape(self.experts, self.channels)
        self._index, self._fixed = self.device.index, (self.weight.data_ptr(), self.scale.data_ptr(), _ptr(self.bias))
        self._streams = _Streams(self._index, self.weight, given=(self.scale, self.bias))

    @classmethod
    def from_weights(cls, weight, bias=None):
        """Quantizes weight [experts, channels, inner] (or [channels, inner])."""
        _tensor(weight, "weight")
        if weight.dim() not in (2, 3) or 0 in weight.shape:
            _refuse("weight must be [experts, channels, inner] or [channels, inner]")
        q, scale = quantize_rows(weight)
        q = q[:, : weight.shape[-1]].reshape(weight.shape)
        return cls(q, scale, None if bias is None else bias.float().contiguous())

    def product(self, x, offsets=None, rows=None, rows_divisor: int = 1):
        """Rows of x [..., inner], each quantized with its own scale, times the
        weights of their expert: [n, channels] in x's type.

        offsets int32 [experts + 1]: expert e takes rows offsets[e]:offsets[e + 1]
        (may be left out with one expert).  rows int32 [n]: row r of the product is
        made from x[rows[r] // rows_divisor] -- a Routing's `order` with rows_divisor
        = top_k; without it from x[r].  Rows in no expert's run are left unwritten."""
        device = self._index
        flat, x_stride, x_rows, _ = _matrix(x, "x", device, self.inner)
        index = _row_index(rows, rows_divisor, device)
        n = x_rows if rows is None else rows.shape[0]
        if offsets is not None:
            _tensor(offsets, "offsets", device)
            if offsets.dtype != torch.int32 or offsets.numel() != self.experts + 1 or not offsets.is_contiguous():
                _refuse("offsets must be a contiguous int32 vector of experts + 1")
        elif self.experts != 1:
            _refuse("several experts need offsets")
        shape = (*x.shape[:-1], self.channels) if rows is None else (n, self.channels)
        out = torch.empty(shape, dtype=flat.dtype, device=self.device)
        space = _lib.eps_b200_int8_product_workspace(n, self.experts, self.channels, self.inner)
        workspace = torch.empty(space, dtype=torch.uint8, device=self.device) if space else None
        args = _pack(_INT8_PRODUCT, device, _TYPES[flat.dtype], self.experts, self.channels, self.inner, rows_divisor, n,
                     *self._fixed, _ptr(offsets), out.data_ptr(),
                     _ptr(workspace), space)
        stream = _stream(device)
        self._streams.use(stream, device)
        _call(_lib.eps_b200_int8_linear, args, flat.data_ptr(), x_stride, x_rows, index, stream)
        return out


# ------------------------------------------------------------------ adapters
_LOW_RANK = struct.Struct("@2i4IQ7P3qPQ")          # LowRank


class Adapters:
    """Low-rank adapters beside a linear layer that many requests share, each row with its
    own: out[t] = base[t] + scale[a] * up[a] (down[a] x[t]) for a = ids[t].

    Laid out once; load() puts another adapter in the place of one.  A captured product reads
    what is held here, so the object has to outlive the graph."""

    def __init__(self, down, up, scale=None):
        """down [adapters, rank, inner] and up [adapters, channels, rank] of one type
        (float32, bfloat16 or float16), copied; scale float32 [adapters] (None: 1).
        Ranks are at most 128, adapters 16384."""
        index = _tensor(down, "down")
        _tensor(up, "up", index)
        if down.dim() != 3 or up.dim() != 3 or 0 in down.shape or 0 in up.shape:
            _refuse("down must be [adapters, rank, inner] and up [adapters, channels, rank]")
        self.adapters, self.rank, self.inner = down.shape
        self.channels = up.shape[1]
        if up.shape[0] != self.adapters or up.shape[2] != self.rank:
            _refuse("down and up have different numbers of adapters or ranks")
        if down.dtype not in _TYPES or up.dtype != down.dtype:
            _refuse("down and up must be float32, bfloat16 or float16, both the same")
        if self.rank > 128 or self.adapters > 16384:
            _refuse("ranks are at most 128, adapters 16384")
        _vector(scale, "scale", index, self.adapters, torch.float32)
        self.device, self.dtype = down.device, down.dtype
        rank, inner = _lib.eps_b200_low_rank_rank(self.rank), _lib.eps_b200_low_rank_inner(self.inner)
        self.down = torch.zeros((self.adapters, rank, inner), dtype=self.dtype, device=self.device)
        self.up = torch.zeros((self.adapters, self.channels, rank), dtype=self.dtype, device=self.device)
        self.down[:, : self.rank, : self.inner] = down.detach()
        self.up[..., : self.rank] = up.detach()
        self.scale = torch.ones(self.adapters, device=self.device) if scale is None else scale.detach().reshape(-1).clone()
        self._index, self._fixed = index, (self.down.data_ptr(), self.up.data_ptr(), self.scale.data_ptr())
        self._streams = _Streams(index, self.down, self.up, self.scale)

    def load(self, adapter: int, down, up, scale: float = 1.0):
        """Puts an adapter (down [rank, inner], up [channels, rank], of this rank or a lower
        one) in the place of number `adapter`, in the order of the current stream: what
        reads the old one on another stream has to be waited for."""
        if not 0 <= adapter < self.adapters:
            _refuse(f"adapters are 0 to {self.adapters - 1}")
        _tensor(down, "down", self._index)
        _tensor(up, "up", self._index)
        rank = down.shape[0] if down.dim() == 2 else 0
        if not 0 < rank <= self.rank or down.shape != (rank, self.inner) or up.shape != (self.channels, rank):
            _refuse(f"down must be [rank, {self.inner}] and up [{self.channels}, rank], with a rank of 1 to {self.rank}")
        if down.dtype != self.dtype or up.dtype != self.dtype:
            _refuse(f"down and up must be {self.dtype}")
        self._streams.use(_stream(self._index), self._index)
        self.down[adapter, :rank, : self.inner] = down.detach()
        self.down[adapter, rank:] = 0
        self.up[adapter, :, :rank] = up.detach()
        self.up[adapter, :, rank:] = 0
        self.scale[adapter] = scale
        return self

    def product(self, x, ids, base=None, out=None):
        """base + scale * up (down x) for x [..., inner], each row with the adapter that
        ids (int32, one a row) names: [..., channels] in x's type.  An id outside
        [0, adapters), such as -1, is no adapter: the row is base's.  base [..., channels]
        (None: 0), the shared layer's output; a row of stride 0 stands for all.  out: where
        the result goes, base itself for one; it may not overlap x, nor base otherwise.
        All have the adapters' type."""
        device = self._index
        flat, x_stride, rows, _ = _matrix(x, "x", device, self.inner)
        if flat.dtype != self.dtype:
            _refuse(f"x must be {self.dtype}, as the adapters are")
        _tensor(ids, "ids", device)
        if ids.dtype != torch.int32 or ids.numel() != rows or not ids.is_contiguous():
            _refuse("ids must be contiguous int32, one for each row of x")
        base_stride = 0
        if base is not None:
            base, base_stride, _, _ = _matrix(base, "base", device, self.channels, rows)
            if base.dtype != self.dtype:
                _refuse("base has the type of x")
        if out is None:
            result = out = torch.empty((*x.shape[:-1], self.channels), dtype=self.dtype, device=self.device)
            out_stride = self.channels
        else:
            result = out
            out, out_stride, _, _ = _matrix(out, "out", device, self.channels, rows)
            if out.dtype != self.dtype:
                _refuse("out has the type of x")
        space = _lib.eps_b200_low_rank_workspace(rows, self.adapters)
        workspace = torch.empty(space, dtype=torch.uint8, device=self.device) if space else None
        args = _pack(_LOW_RANK, device, _TYPES[self.dtype], self.adapters, self.rank, self.inner, self.channels, rows, *self._fixed,
                     ids.data_ptr(), flat.data_ptr(), _ptr(base), out.data_ptr(), x_stride, base_stride, out_stride,
                     _ptr(workspace), space)
        stream = _stream(device)
        self._streams.use(stream, device)
        _call(_lib.eps_b200_low_rank, args, stream)
        return result


# ------------------------------------------------------------- gradient norm
class GradientMeasure(NamedTuple):
    """norm and scale, float32 scalars on the GPU, and skip, an int32 one.  scale and skip
    are what AdamW.step takes: the factor that clips (times the given gradient_scale), and
    whether the norm is not finite (scale is 0 then)."""
    norm: torch.Tensor
    scale: torch.Tensor
    skip: torch.Tensor


_GRADIENT_NORM = struct.Struct("@4iPQPdPPQ")          # GradientNormArgs


class GradientNorm:
    """The norm over many gradients, and clipping by it.

        norm = |gradient_scale| * sqrt(sum g^2)                 kind "l2"; "max": max |g|
        scale = gradient_scale * min(1, max_norm / norm)

    `gradients` are contiguous float32, bfloat16 or float16 tensors of one device, each of
    its own type, no two of which overlap (the buffers of one AdamW or of several): their
    addresses go to the GPU now, their values are read by each call.  Sums are held in 64
    bits and taken in an order that sizes and alignment fix.  A captured call keeps its
    max_norm and the buffers it reads alive; the object has to outlive the graph."""

    def __init__(self, gradients: Sequence[torch.Tensor], *, kind: str = "l2"):
        self._kind, self._kept = _choice(_NORMS, kind, "kind"), []
        self.bind(gradients)

    def bind(self, gradients: Sequence[torch.Tensor]):
        """Makes these the buffers that are measured."""
        gradients = list(gradients)
        if not gradients:
            _refuse("no gradients")
        index = _tensor(gradients[0], "a gradient")
        if _capturing(index):
            _refuse("gradients are bound before a capture")
        words = array("Q")
        for g in gradients:
            _tensor(g, "a gradient", index)
            if g.dtype not in _TYPES or not g.is_contiguous():
                _refuse("gradients are contiguous, of float32, bfloat16 or float16")
            words.extend((g.data_ptr(), g.numel(), _TYPES[g.dtype]))
        tensors = (Gradient * len(gradients)).from_buffer(words)
        size = _lib.eps_b200_gradient_norm_plan_bytes(tensors, len(gradients))
        host = torch.empty(size, dtype=torch.uint8)
        blocks = C.c_uint64(0)
        _call(_lib.eps_b200_gradient_norm_plan, tensors, len(gradients), host.data_ptr(), size, C.byref(blocks))
        device = gradients[0].device
        plan = host.to(device)
        self.device, self.gradients = device, gradients
        self._bound = (gradients, plan, blocks.value, _lib.eps_b200_gradient_norm_workspace(blocks.value),
                       _Streams(index, plan, given=gradients))

    def _run(self, clip, max_norm, gradient_scale):
        _, plan, blocks, space, streams = self._bound
        device = self.device.index
        scale = _vector(gradient_scale, "gradient_scale", device, 1, torch.float32)
        result = torch.empty(3, dtype=torch.float32, device=self.device)
        workspace = torch.empty(space, dtype=torch.uint8, device=self.device) if space else None
        args = _pack(_GRADIENT_NORM, device, self._kind, clip, 0, plan.data_ptr(), blocks, scale, max_norm, result.data_ptr(),
                     _ptr(workspace), space)
        stream = _stream(device)
        streams.use(stream, device)
        _call(_lib.eps_b200_gradient_norm, args, stream)
        if _capturing(device) and not any(kept is self._bound for kept in self._kept):
            self._kept.append(self._bound)
        norm, factor, skip = result.unbind()
        return GradientMeasure(norm, factor, skip.view(torch.int32))

    def measure(self, max_norm: float = math.inf, *, gradient_scale=None) -> GradientMeasure:
        """The norm and the factor that brings it to max_norm at most; the gradients stay
        as they are.  gradient_scale: a float32 scalar on the GPU that the gradients are to
        be multiplied by anyway (one over a loss scale)."""
        return self._run(0, max_norm, gradient_scale)

    def clip(self, max_norm: float, *, gradient_scale=None) -> GradientMeasure:
        """measure(), and every gradient times that factor in place, in float and then
        rounded to its type; where the norm is not finite they stay as they are."""
        return self._run(1, max_norm, gradient_scale)


# --------------------------------------------------------------------- AdamW
class AdamW:
    """AdamW over many tensors, one launch a step.

        m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
        p -= learning_rate * (m_hat / (sqrt(v_hat) + epsilon) + weight_decay * p)

    The dense counterpart of the store's LazyAdam: every element moves at every
    step.  `gradients` are the buffers that step() reads; step(gradients) takes
    others.  state_bits 32 holds the moments in float32; 8 holds m and sqrt(v) as
    float8_e4m3fn with a scale for each 256 elements, m rounded to the nearest and
    sqrt(v) at random (a function of `seed`, the step and the element) so that small
    changes are right on average.  master=True keeps a float32 copy of 16-bit
    parameters, which is the one updated.

    The moments lie one tensor after the other in `first` and `second` (and `master`),
    tensor i from element starts[i] on; `first_scale` and `second_scale` hold the
    scales of 8-bit moments.

    A step that is captured in a CUDA graph counts itself: each replay is a step of its
    own.  From the first capture on, the number of steps is held on the GPU (`steps`
    waits for the current stream to read it), and learning_rate is set in the order of
    the current stream.  Gradients are bound before a capture; a captured step keeps
    those it reads alive, and the optimizer has to outlive the graph."""

    def __init__(self, parameters: Sequence[torch.Tensor], gradients: Sequence[torch.Tensor] | None = None, *,
                 learning_rate: float = 1e-3, beta1: float = 0.9, beta2: float = 0.999,
                 epsilon: float = 1e-8, weight_decay: float = 0.01, state_bits: int = 32,
                 master: bool = False, seed: int = 0):
        self.parameters = list(parameters)
        if not self.parameters:
            _refuse("no parameters")
        head = self.parameters[0]
        index = _tensor(head, "a parameter")
        if head.dtype not in _TYPES:
            _refuse("parameters are float32, bfloat16 or float16")
        for p in self.parameters:
            _tensor(p, "a parameter", index)
            if p.dtype != head.dtype or not p.is_contiguous():
                _refuse("parameters are contiguous and of one type")
        if state_bits not in (8, 32):
            _refuse("moments have 32 or 8 bits")
        if master and head.dtype == torch.float32:
            _refuse("float32 parameters take no master copy")
        self.device, self.state_bits, self._steps = head.device, state_bits, 0
        self.starts, total = [], 0
        for p in self.parameters:
            self.starts.append(total)
            total += -(-p.numel() // ADAMW_BLOCK) * ADAMW_BLOCK
        state = dict(dtype=torch.float32 if state_bits == 32 else torch.float8_e4m3fn, device=self.device)
        self.first, self.second = torch.zeros(total, **state), torch.zeros(total, **state)
        self.first_scale = self.second_scale = self.master = None
        if state_bits == 8:
            self.first_scale = torch.zeros(total // ADAMW_BLOCK, device=self.device)
            self.second_scale = torch.zeros(total // ADAMW_BLOCK, device=self.device)
        if master:
            self.master = torch.zeros(total, device=self.device)
            for p, a in zip(self.parameters, self.starts):
                self.master[a:a + p.numel()] = p.detach().reshape(-1)
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self._args = AdamWArgs(self.device.index, _TYPES[head.dtype], 0, state_bits, ptr(self.master),
                               ptr(self.first), ptr(self.second), ptr(self.first_scale), ptr(self.second_scale),
                               None, None, learning_rate, beta1, beta2, epsilon, weight_decay, 0, seed)
        # an AdamWClock: no step taken, no rate of its own; used from the first captured step on
        self._clock = torch.tensor(list(struct.unpack("@4q", bytes(AdamWClock(0, -1.0)))), device=self.device)
        self._counted, self._kept = False, []
        self._streams = _Streams(index, self.first, self.second, self.first_scale, self.second_scale, self.master, self._clock,
                                given=self.parameters)
        self._bound = None
        if gradients is not None:
            self.bind(gradients)

    @property
    def steps(self) -> int:
        """The number of steps taken."""
        return self._steps + (int(self._clock[0].item()) if self._counted else 0)

    @steps.setter
    def steps(self, value: int):
        if self._counted:
            self._clock[0] = value - self._steps     # graphs hold the sum's other part
        else:
            self._steps = value

    @property
    def learning_rate(self) -> float:
        return self._args.learning_rate

    @learning_rate.setter
    def learning_rate(self, value: float):
        if self._counted:
            if not 0 <= value < math.inf:
                _refuse("invalid learning rate")
            self._clock[1:2].view(torch.float64).fill_(value)
        self._args.learning_rate = value

    def bind(self, gradients: Sequence[torch.Tensor]):
        """Makes these the buffers that step() reads: their addresses go to the GPU
        now, their values are read at each step."""
        gradients = list(gradients)
        if len(gradients) != len(self.parameters):
            _refuse("a gradient for each parameter")
        if _capturing(self.device.index):
            _refuse("gradients are bound before a capture")
        dtype = gradients[0].dtype if isinstance(gradients[0], torch.Tensor) else None
        if dtype not in (self.parameters[0].dtype, torch.float32):
            _refuse("gradients have the parameters' type or float32")
        index, words = self.device.index, array("Q")
        for p, g, a in zip(self.parameters, gradients, self.starts):
            _tensor(g, "a gradient", index)
            if g.dtype != dtype or g.shape != p.shape or not g.is_contiguous():
                _refuse("gradients are contiguous, of one type and of the parameters' shapes")
            words.extend((p.data_ptr(), g.data_ptr(), p.numel(), a))
        tensors = (AdamWTensor * len(gradients)).from_buffer(words)
        size = _lib.eps_b200_adamw_plan_bytes(tensors, len(gradients))
        host = torch.empty(size, dtype=torch.uint8)
        blocks = C.c_uint64(0)
        _call(_lib.eps_b200_adamw_plan, tensors, len(gradients), host.data_ptr(), size, C.byref(blocks))
        plan = host.to(self.device)
        self._bound = (gradients, plan, blocks.value, _TYPES[dtype], _Streams(self.device.index, plan, given=gradients))

    def step(self, gradients: Sequence[torch.Tensor] | None = None, *, gradient_scale=None, skip=None):
        """One step.  gradient_scale: a float32 scalar on the GPU that multiplies
        every gradient (a clip factor, one over a loss scale).  skip: an int32 scalar
        on the GPU; where it is not 0 the step changes no parameter and no moment
        (it still counts as a step)."""
        if gradients is not None:
            self.bind(gradients)
        if self._bound is None:
            _refuse("no gradients: give them to AdamW, bind or step")
        _, plan, blocks, gtype, streams = self._bound
        a = self._args
        a.gradient_type = gtype
        device = self.device.index
        capturing = _capturing(device)
        a.gradient_scale = _vector(gradient_scale, "gradient_scale", device, 1, torch.float32)
        a.skip = _vector(skip, "skip", device, 1, torch.int32)
        a.step = self._steps + 1
        stream = _stream(device)
        streams.use(stream, device)
        self._streams.use(stream, device)
        if capturing or self._counted:
            _call(_lib.eps_b200_adamw_counted, C.byref(a), plan.data_ptr(), len(self.parameters), blocks,
                  self._clock.data_ptr(), stream)
            self._counted = True
            if capturing and not any(kept is self._bound for kept in self._kept):
                self._kept.append(self._bound)
        else:
            _call(_lib.eps_b200_adamw, C.byref(a), plan.data_ptr(), len(self.parameters), blocks, stream)
            self._steps += 1

    def state(self) -> dict:
        """What load_state takes, by reference."""
        held = {k: getattr(self, k) for k in ("first", "second", "first_scale", "second_scale", "master")}
        return {"steps": self.steps, **{k: v for k, v in held.items() if v is not None}}

    def load_state(self, steps: int, **tensors):
        """Copies moments (and scales, master parameters) of the same layout in, and
        sets the number of steps taken."""
        mine = self.state()
        mine.pop("steps")
        if steps < 0 or set(tensors) != set(mine):
            _refuse(f"a state has steps and {', '.join(mine)}")
        for k, t in tensors.items():
            if not isinstance(t, torch.Tensor) or t.shape != mine[k].shape or t.dtype != mine[k].dtype:
                _refuse(f"{k} must be {mine[k].dtype} of {tuple(mine[k].shape)}")
        for k, t in tensors.items():
            mine[k].copy_(t)
        self.steps = steps
        return self
