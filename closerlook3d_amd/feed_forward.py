"""Per-point feed-forward operators: csrc/gated_ffn.hip, point_norm.hip, dropout.hip.

    gated_feed_forward   (act(x Wg^T) * (x Wu^T)) Wd^T for every point, with its gradients
    point_norm           an rms or layer norm over the channels of a point: the entry of a block
    norm_gate_residual   the exit of a block -- norm, dropout, gate, scaled residual -- and the entry of the next, in one pass
    dropout              from a counter-based generator: the mask is formed again in the backward pass, never stored

and the modules on top of them: GatedFeedForward, CounterDropout, FeedForwardBlock (what backbones.Bottleneck appends when the
configuration asks for it).

Tensors are features (B, C, N), as everywhere in this package, or rows (R, C): pooled vectors, the input of nn.Linear.  (B, C, N)
features may lie channel-major (dense) or point-major (a transposed view of dense (B, N, C) rows); results lie as the first
input does.  The norms read channel-major features as they lie (up to 1024 channels, a multiple of four); otherwise the kernels work
on point-major rows and take and leave a transposed copy, so a chain of these operators is best kept point-major (to_point_major,
once, at its beginning; FeedForwardBlock does).  Types: float32, bfloat16, float16.  Everything is formed in f32 and rounded once, to
the type of the result (a gated feed-forward of 16-bit tensors: once more in front of its second products).

Points are independent of each other (only parameter gradients sum over them); padding points are computed like the others.  The
results of a point depend on no other point, and every gradient is summed in a fixed order: bit-identical run to run.  There is no
CPU fallback.  The operators can be captured into HIP graphs, forward and backward.  A forward-mode tangent, a derivative of a
gradient and a trace (torch.jit.trace, make_fx) are refused.
"""
import ctypes
import functools
import weakref

import torch
import torch.nn as nn
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # CL3D_F32 / _BF16 / _F16
_POINT, _CHANNEL = 0, 1                                             # CL3D_POINT_MAJOR / _CHANNEL_MAJOR
_ACTIVATIONS = {'silu': 0, 'gelu': 1, 'relu': 2}
_NORMS = {'none': 0, 'rms': 1, 'layer': 2}
_PRECISIONS = {'f32': 0, 'bf16': 1}
_OP_GATED_FFN, _OP_POINT_NORM = 17, 18
_MAX_NORM_CHANNELS, _WIDE_NORM_CHANNELS = 4096, 6144  # any number up to the first, multiples of 8 up to the second
_MAX_SIZE = 2 ** 31 - 1  # the C entries take 32-bit sizes
_MAX_GATES = 65535       # a grid's third axis


def _p(t):
    return None if t is None else t.data_ptr()


_is_tracing, _dispatch_modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack


def _check_trace(who):
    # (a trace holds the allocations of a call and nothing of what the launches put there)
    if _is_tracing() or (_dispatch_modes() and get_proxy_mode() is not None):
        raise RuntimeError(f"{who}: cannot be traced by torch.jit.trace or make_fx (capture a HIP graph instead)")


def _check_sizes(t, who, name):
    if t.numel() > _MAX_SIZE and max(t.shape) > _MAX_SIZE:  # (the first is the cheaper)
        raise ValueError(f"{who}: {name} has the shape {tuple(t.shape)}, no size is above {_MAX_SIZE}")


def _check_features(x, who, name='x'):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{who}: {name} is a tensor, got {type(x).__name__}")
    if not x.is_cuda:
        raise RuntimeError(f"{who}: CPU not supported")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{who}: {name} is float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() not in (2, 3):
        raise ValueError(f"{who}: {name} is (B, C, N) features or (R, C) rows, got {tuple(x.shape)}")
    _check_sizes(x, who, name)


def _sizes(x):
    """(B, C, N) of features; rows are clouds of one point."""
    return (x.shape[0], x.shape[1], 1) if x.dim() == 2 else tuple(x.shape)


def _check_param(t, shape, x, who, name, optional=True, f32=True):
    if t is None:
        if optional:
            return
        raise TypeError(f"{who}: {name} is missing")
    if isinstance(t, torch.Tensor) and t.shape == shape and t.dtype == x.dtype and t.device == x.device:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{who}: {name} is a tensor, got {type(t).__name__}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{who}: {name} has the shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.device != x.device:
        raise RuntimeError(f"{who}: {name} is on {t.device}, x on {x.device}")
    if t.dtype != x.dtype and not (f32 and t.dtype == torch.float32):
        raise TypeError(f"{who}: {name} is {t.dtype}, x is {x.dtype}")


def _point_major(t):
    if t.dim() == 2:
        return t.is_contiguous()
    (_, C, N), s = t.shape, t.stride()
    if s[1] == 1:
        return (s[2] == C and s[0] == C * N) or t.transpose(1, 2).is_contiguous()
    # (a stride other than 1 counts where there is more than one channel)
    return (C == 1 or t.numel() == 0) and t.transpose(1, 2).is_contiguous()


def _aligned(t):
    """Dense memory that starts on 16 bytes (what the kernels load)."""
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.preserve_format)


def _order(t):
    """(dense tensor, its memory order)."""
    if _point_major(t):
        return _aligned(t), _POINT
    return _aligned(t if t.is_contiguous() else t.contiguous()), _POINT if t.dim() == 2 else _CHANNEL


_raw_stream = torch._C._cuda_getCurrentRawStream  # (torch.cuda.current_stream() builds an object: 3.5 us a call)


def _stream(device):
    return _raw_stream(device.index)


_WORKSPACE = {}  # sizes of scratch, by what cl3d_workspace_bytes was asked


def _workspace(op, B, N, M, K, C, device):
    key = (op, B, N, M, K, C)
    nbytes = _WORKSPACE.get(key)
    if nbytes is None:
        if len(_WORKSPACE) > 4096:
            _WORKSPACE.clear()
        nbytes = _WORKSPACE[key] = _lib.lib().cl3d_workspace_bytes(*key)
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None, nbytes


def _empty(shape, order, dtype, device):
    if len(shape) == 3 and order == _POINT:
        B, C, N = shape
        return torch.empty_strided(shape, (N * C, 1, C), dtype=dtype, device=device)
    return torch.empty(shape, dtype=dtype, device=device)


def _swap(src, B, R, C, dst):
    """[B, R, C] -> [B, C, R], dense memory of the same type."""
    lib = _lib.lib()
    fn = lib.cl3d_transpose if src.dtype == torch.float32 else lib.cl3d_transpose16
    with _lib.on_device(src.device):
        _lib.check(fn(_p(src), B, R, C, _p(dst), _stream(src.device)))
    return dst


def _as_order(t, order):
    """t in the given memory order: itself, or a copy by the engine's transpose."""
    t, have = _order(t)
    if t.dim() == 2 or have == order or t.numel() == 0:
        return t
    if order == _CHANNEL and t.is_contiguous():
        return t
    B, C, N = t.shape
    out = _empty(t.shape, order, t.dtype, t.device)
    if order == _POINT:
        _swap(t, B, C, N, out)
    else:
        _swap(t, B, N, C, out)
    return out


class _Reorder(Function):
    @staticmethod
    def forward(ctx, x, order):
        ctx.back = _order(x)[1]
        _track(ctx, x)
        return _as_order(x, order).view_as(x)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        _check_capture(ctx, g.device)
        return _as_order(g, ctx.back), None


def to_point_major(features):
    """(B, C, N) features as a view of dense (B, N, C) rows, by the engine's transpose where they do not lie so already (up to 65535
    clouds of up to 4194240 points)."""
    _check_trace('to_point_major')
    _check_features(features, 'to_point_major', 'features')
    return features if _point_major(features) else _Reorder.apply(features, _POINT)


def to_channel_major(features):
    """(B, C, N) features as dense channel-major memory, what the other operators of this package read."""
    _check_trace('to_channel_major')
    _check_features(features, 'to_channel_major', 'features')
    return features if features.is_contiguous() else _Reorder.apply(features, _CHANNEL)


def _once(backward):
    """once_differentiable, also where the incoming gradient is a constant: that decorator takes the gradients it returns for constants
    then, and a second derivative through the saved tensors would silently be zero.  (ctx.linear: it is.)"""

    @functools.wraps(backward)
    def once(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled() or (ctx.linear and not any(g is not None and g.requires_grad for g in grads)):
            return out
        given = [t for t in out if t is not None]
        refuse = torch._C._functions.DelayedError(b"trying to differentiate twice a function that has one derivative", len(given))
        marked = refuse(*[t.detach().requires_grad_(True) for t in given])
        marked = iter(marked if isinstance(marked, tuple) else (marked,))
        return tuple(None if t is None else next(marked) for t in out)

    return once


def _recorded(*tensors):
    """Whether a call goes through its autograd function: a gradient is wanted, or a forward-mode level is open (the function refuses
    a tangent; the launches alone would lose it).  Other calls do without the node, which costs as much host time as the rest of a
    small call."""
    return forward_ad._current_level >= 0 or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors))


# Autograd runs a leaf's gradient on the stream that was current when the leaf's node was made, and keeps that node while any
# graph of the leaf lives.  A backward pass captured meanwhile, on another stream, is handed over to that stream, which no capture
# joins: ending it takes the process down.  Every eager graph of these operators is therefore known by its context while it lives
# (autograd frees the context with the graph), and a captured backward pass of the same leaves says so instead.
_LIVE = {}  # id -> weak reference.  Threads add and drop meanwhile: every use is one step of the interpreter (no walk in Python)


def _forget(ref, live=_LIVE):  # (bound: it may be called when the module's names are gone)
    if live.get(ref.key) is ref:
        live.pop(ref.key, None)


class _Ref(weakref.ref):
    __slots__ = ("key",)

    def __init__(self, ctx, callback):
        super().__init__(ctx, callback)
        self.key = id(ctx)


def _track(ctx, *inputs):
    """Called by a forward pass that autograd records, with the tensors it was given."""
    ctx.leaves = [weakref.ref(t) for t in inputs if t is not None and t.requires_grad and t.is_leaf]
    if ctx.leaves and not torch.cuda.is_current_stream_capturing():
        ctx.made_on = _raw_stream(inputs[0].device.index)
        _LIVE[id(ctx)] = _Ref(ctx, _forget)


def _check_capture(ctx, device):
    """Called by a backward pass."""
    if not _LIVE or not torch.cuda.is_current_stream_capturing():
        return
    mine = {id(t) for t in (r() for r in ctx.leaves) if t is not None}
    stream = _raw_stream(device.index)
    for other in [r() for r in list(_LIVE.values())]:
        if other is None or other is ctx or other.made_on == stream:
            continue
        if any(id(t) in mine for t in (r() for r in other.leaves) if t is not None):
            raise RuntimeError("a backward pass is being captured while an eager graph of the same leaves, made on another stream, is "
                               "alive: delete its outputs first, or warm up and capture on one stream (closerlook3d_amd.step_stream())")


# ------------------------------------------------------------------------------------------------- gated feed-forward
_FEW_POINTS, _HIDDEN = 64, 512  # CL3D_FFN_FEW, CL3D_FFN_HIDDEN


def _ffn_forward(x, w_gate, w_up, w_down, activation, precision, keep_hidden):
    """y and what a backward pass needs: the tensors as the kernels read them, the hidden activations if asked for, the sizes."""
    shape, dtype, device = x.shape, _DTYPES[x.dtype], x.device
    B, C, N = _sizes(x)
    x, order = _order(x)
    w_gate, w_up = _aligned(w_gate.contiguous()), _aligned(w_up.contiguous())
    w_down = None if w_down is None else _aligned(w_down.contiguous())
    H = w_gate.shape[0]
    # (empty_like: a dense tensor's memory order, at a third of the host time)
    y = torch.empty_like(x) if w_down is not None else _empty((shape[0], H) + tuple(shape[2:]), order, x.dtype, device)
    hidden = None
    if keep_hidden and w_down is not None and B * N > _FEW_POINTS:
        hidden = torch.empty((3 if dtype == 0 and precision == 0 else 1, B * N, (H + 7) // 8 * 8), dtype=torch.int16, device=device)
    if B * N:
        flags = dtype | order << 2 | precision << 3 | (w_down is not None) << 4 | (_HIDDEN if hidden is not None else 0)
        ws, nbytes = _workspace(_OP_GATED_FFN, B, N, H, flags, C, device)
        with _lib.on_device(device):
            _lib.check(_lib.lib().cl3d_gated_ffn_fwd(_p(x), _p(w_gate), _p(w_up), _p(w_down), dtype, order, B, C, N, H, activation,
                                                     precision, _p(y), _p(hidden), _p(ws), nbytes, _stream(device)))
    return y, (x, w_gate, w_up, w_down, hidden), (order, B, C, N, H, activation, precision)


class _GatedFeedForward(Function):
    """One C-ABI call per direction.  Kept for the backward pass: x, the weights and, if w_down has a gradient, the hidden
    activations; the two projections are formed again."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation, precision):
        _track(ctx, x, w_gate, w_up, w_down)
        y, kept, ctx.args = _ffn_forward(x, w_gate, w_up, w_down, activation, precision, ctx.needs_input_grad[3])
        ctx.save_for_backward(*kept)
        ctx.linear = False
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, w_gate, w_up, w_down, hidden = ctx.saved_tensors
        _check_capture(ctx, x.device)
        order, B, C, N, H, activation, precision = ctx.args
        need = ctx.needs_input_grad
        new = torch.empty_like if B * N else torch.zeros_like
        dx = torch.empty_like(x) if need[0] else None
        dwg = new(w_gate) if need[1] else None
        dwu = new(w_up) if need[2] else None
        dwd = new(w_down) if w_down is not None and need[3] else None
        if B * N:
            dy = _as_order(dy, order)
            dtype = _DTYPES[x.dtype]
            wants = (dx is not None) | (dwg is not None or dwu is not None) << 1 | (dwd is not None) << 2
            flags = (dtype | order << 2 | precision << 3 | (w_down is not None) << 4 | 32 | wants << 6
                     | (_HIDDEN if hidden is not None else 0))
            ws, nbytes = _workspace(_OP_GATED_FFN, B, N, H, flags, C, x.device)
            with _lib.on_device(x.device):
                _lib.check(_lib.lib().cl3d_gated_ffn_bwd(_p(x), _p(w_gate), _p(w_up), _p(w_down), _p(dy), _p(hidden), dtype, order, B,
                                                         C, N, H, activation, precision, _p(dx), _p(dwg), _p(dwu), _p(dwd), _p(ws),
                                                         nbytes, _stream(x.device)))
        return dx, dwg, dwu, dwd, None, None


def gated_feed_forward(x, w_gate, w_up, w_down=None, activation='silu', precision='f32'):
    """y = (act(x w_gate^T) * (x w_up^T)) w_down^T for every point of x, (B, C, N) features or (R, C) rows.

    w_gate, w_up (H, C) and w_down (C, H) have x's type; w_down None: the product of the two projections itself, with H channels.
    activation 'silu', 'gelu' (by the error function) or 'relu'.  precision, of float32 tensors: 'f32' multiplies at f32 accuracy,
    'bf16' rounds what enters a product to bfloat16, as in the other operators of this package; 16-bit tensors enter as they are.
    16-bit tensors: what enters a second product -- the hidden activations h, in the backward pass the gradients of the two
    projections -- is rounded to their type once more (f32 keeps its accuracy); in float16 it has that type's range too: above 65504 an
    infinity, below 2^-25 nothing.  Channel-major features: up to 65535 clouds of up to 4194240 points."""
    who = 'gated_feed_forward'
    _check_trace(who)
    _check_features(x, who)
    C = x.shape[1]
    _check_param(w_gate, (w_gate.shape[0] if isinstance(w_gate, torch.Tensor) and w_gate.dim() == 2 else 'H', C), x, who, 'w_gate',
                 optional=False, f32=False)
    H = w_gate.shape[0]
    _check_sizes(w_gate, who, 'w_gate')
    _check_param(w_up, (H, C), x, who, 'w_up', optional=False, f32=False)
    _check_param(w_down, (C, H), x, who, 'w_down', f32=False)
    if C == 0 or H == 0:
        raise ValueError(f"{who}: no channels")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{who}: activation is one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if precision not in _PRECISIONS:
        raise ValueError(f"{who}: precision is one of {sorted(_PRECISIONS)}, got {precision!r}")
    args = (x, w_gate, w_up, w_down, _ACTIVATIONS[activation], _PRECISIONS[precision])
    # (without a gradient: no autograd node)
    return _GatedFeedForward.apply(*args) if _recorded(x, w_gate, w_up, w_down) else _ffn_forward(*args, False)[0]


# ---------------------------------------------------------------------------------------------- norms around a block
def _norm_forward(x, y, weight, bias, gate, next_weight, next_bias, rng, opts, need_grad):
    """(out, next) in x's memory order, and what a backward pass needs."""
    kind, next_kind, eps, next_eps, scale, p = opts
    dtype, device = x.dtype, x.device
    B, C, N = _sizes(x)
    x, order = _order(x)
    y = None if y is None else _as_order(y, order)
    params = (weight, bias, gate, next_weight, next_bias)
    held, f32 = [], False
    for t in params:
        f32 = f32 or (t is not None and t.dtype == torch.float32)
    for t in params:  # (one type for all of them: a mixture goes to f32)
        if t is not None:
            t = (t if not f32 or t.dtype == torch.float32 else t.float()).contiguous()
            t = _aligned(t) if C > _MAX_NORM_CHANNELS else t
        held.append(t)
    out = torch.empty_like(x) if y is not None else None
    nxt = torch.empty_like(x) if next_kind else None
    stats = torch.empty((B * N, 4), dtype=torch.float32, device=device) if need_grad else None
    sizes = (B, N, C, _DTYPES[dtype], f32, kind, next_kind, gate is not None and gate.dim() == 2, scale, eps, next_eps, order, p)
    if B * N:
        # (the fields of cl3d_norm_residual in their order)
        block = _lib.NormResidual(*sizes, _p(rng), _p(x), _p(y), *map(_p, held), _p(out), _p(nxt), _p(stats))
        if order == _CHANNEL:
            copies = 1 + (y is not None) + (out is not None) + (nxt is not None)
            ws, block.ws_bytes = _workspace(_OP_POINT_NORM, B, N, 0, sizes[3] | order << 2 | copies << 3, C, device)
            block.ws = _p(ws)
        with _lib.on_device(device):
            _lib.check(_lib.lib().cl3d_norm_residual_fwd(ctypes.byref(block), _stream(device)))
    # (an exit alone: x is not looked at again)
    kept = (x if next_kind else None, y, *held, rng, stats)
    return out, nxt, kept, (order, sizes, [None if t is None else t.dtype for t in params])


class _NormResidual(Function):
    """cl3d_norm_residual_fwd / _bwd."""

    @staticmethod
    def forward(ctx, x, y, weight, bias, gate, next_weight, next_bias, rng, opts):
        _track(ctx, x, y, weight, bias, gate, next_weight, next_bias)
        out, nxt, kept, ctx.args = _norm_forward(x, y, weight, bias, gate, next_weight, next_bias, rng, opts, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*kept)
        ctx.linear = opts[0] == opts[1] == 0 and weight is None and gate is None  # (neither norm)
        return out, nxt

    @staticmethod
    @_once
    def backward(ctx, dout, dnext):
        x, y, weight, bias, gate, next_weight, next_bias, rng, stats = ctx.saved_tensors
        order, sizes, types = ctx.args
        B, N, C = sizes[:3]
        need, device = ctx.needs_input_grad, stats.device
        _check_capture(ctx, device)
        if dout is None and dnext is None:
            return (None,) * 9
        dout = None if dout is None else _as_order(dout, order)
        dnext = None if dnext is None else _as_order(dnext, order)
        like = x if y is None else y  # (one of them was kept, in this memory order)
        dx = torch.empty_like(like) if need[0] else None
        dy = torch.empty_like(like) if y is not None and need[1] else None
        new = torch.empty_like if B * N else torch.zeros_like
        grads = [new(t) if t is not None and n else None for t, n in zip((weight, bias, gate, next_weight, next_bias), need[2:7])]
        if B * N:
            sums = any(g is not None for g in grads)
            copies = 6 if order == _CHANNEL else 0
            ws, nbytes = None, 0
            if sums or copies:
                ws, nbytes = _workspace(_OP_POINT_NORM, B, N, 0, sizes[3] | order << 2 | copies << 3 | sums << 8, C, device)
            block = _lib.NormResidual(*sizes, _p(rng), _p(x), _p(y), _p(weight), _p(bias), _p(gate), _p(next_weight), _p(next_bias),
                                      None, None, _p(stats), _p(dout), _p(dnext), _p(dx), _p(dy), *map(_p, grads), _p(ws), nbytes)
            with _lib.on_device(device):
                _lib.check(_lib.lib().cl3d_norm_residual_bwd(ctypes.byref(block), _stream(device)))
        grads = [g if g is None or g.dtype == t else g.to(t) for g, t in zip(grads, types)]
        return (dx, dy, *grads, None, None)


def _check_channels(C, who):
    if not 0 < C <= _MAX_NORM_CHANNELS and not (0 < C <= _WIDE_NORM_CHANNELS and C % 8 == 0):
        raise ValueError(f"{who}: 1 to {_MAX_NORM_CHANNELS} channels, or a multiple of 8 up to {_WIDE_NORM_CHANNELS}, got {C}")


def _check_norm(x, kind, eps, who, none=False):
    if kind not in _NORMS or (kind == 'none' and not none):
        raise ValueError(f"{who}: a norm is one of {[k for k in _NORMS if none or k != 'none']}, got {kind!r}")
    if not eps >= 0:
        raise ValueError(f"{who}: eps is not negative, got {eps}")
    _check_channels(x.shape[1], who)


def point_norm(x, weight=None, bias=None, kind='rms', eps=1e-6):
    """norm(x) weight + bias over the channels of every point: the entry of a block.

    kind 'rms': x / sqrt(mean x^2 + eps); 'layer': (x - mean) / sqrt(var + eps), the variance over all C.  weight, bias (C,), of x's
    type or float32; None: 1 and 0.  Up to 4096 channels, or a multiple of 8 up to 6144."""
    who = 'point_norm'
    _check_trace(who)
    _check_features(x, who)
    _check_norm(x, kind, eps, who)
    C = x.shape[1]
    _check_param(weight, (C,), x, who, 'weight')
    _check_param(bias, (C,), x, who, 'bias')
    args = (x, None, None, None, None, weight, bias, None, (0, _NORMS[kind], 0.0, float(eps), 1.0, 0.0))
    return (_NormResidual.apply(*args) if _recorded(x, weight, bias) else _norm_forward(*args, False))[1]


def norm_gate_residual(x, y, weight=None, bias=None, gate=None, residual_scale=1.0, kind='rms', eps=1e-6, p=0.0, rng=None,
                       next_kind=None, next_weight=None, next_bias=None, next_eps=None):
    """The exit of a block, and with next_kind the entry of the one that follows, in one pass over the points:

        out = residual_scale * x + gate * dropout(norm(y) weight + bias, p)          next = norm(out) next_weight + next_bias

    x: the residual stream, y: the block's result, same shape and type.  kind 'rms', 'layer' or 'none' (y is added as it is).  gate
    (C,), or (B, C) for a gate of each cloud (for rows: of each row; up to 65535 of them), or None.  p, rng: as in dropout(); element
    (b, c, n) is number (b N + n) C + c of the draw.  next is formed from out before out is rounded.  Channels as in point_norm().
    Returns out, or (out, next) with next_kind."""
    who = 'norm_gate_residual'
    _check_trace(who)
    _check_features(x, who)
    _check_features(y, who, 'y')
    if y.shape != x.shape or y.dtype != x.dtype or y.device != x.device:
        raise ValueError(f"{who}: x and y have one shape, type and device, got {tuple(x.shape)} {x.dtype} and {tuple(y.shape)} {y.dtype}")
    _check_norm(x, kind, eps, who, none=True)
    B, C, _ = _sizes(x)
    _check_param(weight, (C,), x, who, 'weight')
    _check_param(bias, (C,), x, who, 'bias')
    per_cloud = isinstance(gate, torch.Tensor) and gate.dim() == 2
    _check_param(gate, (B, C) if per_cloud else (C,), x, who, 'gate')
    if per_cloud and B > _MAX_GATES:
        raise ValueError(f"{who}: a gate of each cloud for up to {_MAX_GATES} clouds, got {B}")
    if next_kind is None:
        if next_weight is not None or next_bias is not None:
            raise ValueError(f"{who}: a weight or bias of a norm that is not asked for (next_kind)")
        next_kind = 'none'
    else:
        _check_norm(x, next_kind, eps if next_eps is None else next_eps, who)
    _check_param(next_weight, (C,), x, who, 'next_weight')
    _check_param(next_bias, (C,), x, who, 'next_bias')
    if isinstance(residual_scale, torch.Tensor) and residual_scale.requires_grad and torch.is_grad_enabled():
        raise TypeError(f"{who}: residual_scale is a number (it has no gradient; a learned one: gate)")
    p = _check_p(p, who)
    if p > 0:
        _check_rng(rng, x, who)
    args = (x, y, weight, bias, gate, next_weight, next_bias, rng if p > 0 else None,
            (_NORMS[kind], _NORMS[next_kind], float(eps), float(eps if next_eps is None else next_eps), float(residual_scale), p))
    need = _recorded(x, y, weight, bias, gate, next_weight, next_bias)
    out, nxt = _NormResidual.apply(*args) if need else _norm_forward(*args, False)[:2]
    return out if next_kind == 'none' else (out, nxt)


# ---------------------------------------------------------------------------------------------------------- dropout
def _check_p(p, who):
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{who}: a probability is in [0, 1], got {p}")
    return p


def _check_rng(rng, x, who):
    if not isinstance(rng, torch.Tensor) or rng.dtype != torch.int64 or tuple(rng.shape) != (2,) or not rng.is_contiguous():
        raise TypeError(f"{who}: rng is a dense int64 tensor (seed, offset)")
    if rng.device != x.device:
        raise RuntimeError(f"{who}: rng is on {rng.device}, x on {x.device}")


class _Dropout(Function):
    @staticmethod
    def forward(ctx, x, p, rng):
        ctx.save_for_backward(rng)
        ctx.p = p
        _track(ctx, x)
        return _drop(x, p, rng)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        _check_capture(ctx, g.device)
        return _drop(g, ctx.p, ctx.saved_tensors[0]), None, None


def _drop(x, p, rng):
    lib, dtype = _lib.lib(), _DTYPES[x.dtype]
    if x.dim() == 3 and not x.is_contiguous() and _point_major(x):
        _check_sizes(x, 'dropout', 'x')
        out = torch.empty_like(x)
        with _lib.on_device(x.device):
            _lib.check(lib.cl3d_dropout_point_major(_p(x), dtype, *x.shape, p, _p(rng), _p(out), _stream(x.device)))
        return out
    x = x.contiguous()
    out = torch.empty_like(x)
    with _lib.on_device(x.device):
        _lib.check(lib.cl3d_dropout(_p(x), dtype, x.numel(), p, _p(rng), _p(out), _stream(x.device)))
    return out


def dropout(x, p, rng):
    """x / (1 - p) where word i of the draw is at least floor(p 2^32), else 0; i counts x's elements in the order of its dimensions.

    rng: int64 (2,) on x's device, (seed, offset).  Word i is number i % 4 of block offset + i / 4 of Philox 4x32-10 under the key
    `seed`: a draw of n elements uses ceil(n / 4) blocks (CounterRng hands out draws that do not overlap).  The numbers are read on
    the device, by the backward pass too: they must not be changed in between (autograd notices).  A dropped element is 0 whatever
    it was.  p = 0 returns x, p = 1 zeros.  x: any shape; float32, bfloat16 or float16.  The result lies as x does where x is dense or
    features in point-major memory, and is dense for other views; a gradient lies as the one that comes in."""
    who = 'dropout'
    _check_trace(who)
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{who}: x is a tensor, got {type(x).__name__}")
    if not x.is_cuda:
        raise RuntimeError(f"{who}: CPU not supported")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{who}: x is float32, bfloat16 or float16, got {x.dtype}")
    p = _check_p(p, who)
    if p == 0.0:
        return x
    _check_rng(rng, x, who)
    return _Dropout.apply(x, p, rng) if _recorded(x) else _drop(x, p, rng)


class CounterRng:
    """The state of a counter-based generator on one device: take(n) returns the (seed, offset) of a draw of n elements and moves
    on, by one small launch on the current stream -- a captured step draws anew in every replay."""

    def __init__(self, seed, device):
        seed = int(seed)
        if not -2 ** 63 <= seed < 2 ** 64:
            raise ValueError(f"CounterRng: a seed has 64 bits, got {seed}")
        self.state = torch.tensor([seed - 2 ** 64 if seed >= 2 ** 63 else seed, 0], dtype=torch.int64).to(device)
        if not self.state.is_cuda:
            raise RuntimeError("CounterRng: CPU not supported")

    def take(self, n):
        if n < 0:
            raise ValueError(f"CounterRng.take: {n} elements")
        _check_trace('CounterRng.take')
        out = torch.empty_like(self.state)
        with _lib.on_device(out.device):
            _lib.check(_lib.lib().cl3d_rng_take(_p(self.state), (n + 3) // 4, _p(out), _stream(out.device)))
        torch.autograd.graph.increment_version(self.state)  # (a draw from `state` itself, still waiting for its backward pass)
        return out


# ---------------------------------------------------------------------------------------------------------- modules
class _Draws:
    """A module's generators, one for each device it has seen, made on the first input there: from `seed` or, when that is None,
    from torch's CPU generator."""

    def __init__(self, seed):
        self.seed, self.rng, self.rngs = seed, None, {}  # rng: that of the last draw

    def take(self, x):
        if torch._C._current_graph_task_id() != -1:
            raise RuntimeError("dropout: a module draws its own numbers, which a backward pass that runs it again (activation "
                               "checkpointing) would not have a second time: draw outside of what is run twice and call dropout() there")
        rng = self.rngs.get(x.device)
        if rng is None:
            if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("dropout: run the module once before its step is captured (its generator is made on first use)")
            if self.seed is None:
                self.seed = int(torch.randint(0, 2 ** 62, (1,)).item())
            rng = self.rngs[x.device] = CounterRng(self.seed, x.device)
        self.rng = rng
        return rng.take(x.numel())


class CounterDropout(nn.Module):
    """nn.Dropout by dropout(): no mask in memory.  Every call in training mode is a draw of its own; one that activation checkpointing
    makes a second time is refused (draw outside of what is run twice and call dropout() there).  The generator's state is not part of
    the state dict."""

    def __init__(self, p=0.5, seed=None):
        super().__init__()
        self.p = _check_p(p, 'CounterDropout')
        self._draws = _Draws(seed)

    def forward(self, x):
        if not self.training or self.p == 0.0:
            return x
        return dropout(x, self.p, self._draws.take(x))

    def extra_repr(self):
        return f"p={self.p}"


class GatedFeedForward(nn.Module):
    """gated_feed_forward() with its weights, initialised as nn.Linear's."""

    def __init__(self, channels, hidden, activation='silu', precision='f32'):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"GatedFeedForward: activation is one of {sorted(_ACTIVATIONS)}, got {activation!r}")
        self.activation, self.precision = activation, precision
        self.w_gate = nn.Parameter(torch.empty(hidden, channels))
        self.w_up = nn.Parameter(torch.empty(hidden, channels))
        self.w_down = nn.Parameter(torch.empty(channels, hidden))
        for w in (self.w_gate, self.w_up, self.w_down):
            nn.init.kaiming_uniform_(w, a=5 ** 0.5)

    def forward(self, x):
        return gated_feed_forward(x, self.w_gate, self.w_up, self.w_down, self.activation, self.precision)


class FeedForwardBlock(nn.Module):
    """features -> residual_scale * features + gate * dropout(post_norm(gated_feed_forward(pre_norm(features)))).

    pre_norm and post_norm: 'rms', 'layer', or for post_norm 'none' (the default).  gate: a learned number per channel, from
    `gate_init`; None: none.  (B, C, N) features in either memory order, of the parameters' type; the result is channel-major when
    they are.  The dropout draws as CounterDropout does."""

    def __init__(self, channels, hidden, activation='silu', pre_norm='rms', post_norm='none', eps=1e-6, gate_init=1.0,
                 residual_scale=1.0, dropout=0.0, precision='f32', seed=None):
        super().__init__()
        if pre_norm not in ('rms', 'layer') or post_norm not in _NORMS:
            raise ValueError(f"FeedForwardBlock: norms are 'rms' or 'layer' (post_norm: or 'none'), got {pre_norm!r}, {post_norm!r}")
        _check_channels(channels, 'FeedForwardBlock')
        self.pre_norm, self.post_norm, self.eps, self.residual_scale = pre_norm, post_norm, eps, residual_scale
        self.p = _check_p(dropout, 'FeedForwardBlock')
        self._draws = _Draws(seed)

        def vector(value, present):
            return nn.Parameter(torch.full((channels,), float(value))) if present else None

        self.pre_weight, self.pre_bias = vector(1.0, True), vector(0.0, pre_norm == 'layer')
        self.post_weight, self.post_bias = vector(1.0, post_norm != 'none'), vector(0.0, post_norm == 'layer')
        self.gate = vector(0.0 if gate_init is None else gate_init, gate_init is not None)
        self.feed_forward = GatedFeedForward(channels, hidden, activation, precision)

    def forward(self, features):
        channel_major = features.dim() == 3 and not _point_major(features)
        x = to_point_major(features)
        y = self.feed_forward(point_norm(x, self.pre_weight, self.pre_bias, self.pre_norm, self.eps))
        p = self.p if self.training else 0.0
        out = norm_gate_residual(x, y, self.post_weight, self.post_bias, self.gate, self.residual_scale, self.post_norm, self.eps,
                                 p, self._draws.take(x) if p > 0 else None)
        return to_channel_major(out) if channel_major else out
