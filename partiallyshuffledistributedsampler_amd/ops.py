"""Batch-row operators: what the rows of a batch go through between the sampler and a model's
experts, on the GPU (libpss.so, include/pss.h "batch-row operators"), with their gradients.

    dropout(x, p, key, rows, residual)     keyed by (row id, column); the mask is never stored
    route(logits, k, ...)                  the k experts of every row, and the rows sorted by expert
    dispatch(x, routing)                   rows into expert order
    combine(y, routing, residual, p, ...)  experts' outputs summed back by weight

Dropout follows the sampler's counter order: its mask is a function of a key -- of a seed, an epoch,
a logical rank and a place in the model (`dropout_key`, `sampler.dropout_key`) -- and of the row's
id and column, not of a generator's state.  With a sample's position in its rank's stream as the
row's id a resumed run (state_dict) drops what the uninterrupted one would have dropped, whatever
the batch size and the number of GPUs.

Every call runs on the current stream of its tensors' device, allocates its outputs there and keeps
nothing; calls can be captured into a graph (capture a backward pass only while no eager autograd
graph of the same leaves is alive: torch ties a leaf's accumulation to the stream that it was first
used on, and waiting for that stream ends a capture).  fp32, bf16 and fp16 rows; sums and softmax statistics
are held in 32 bits or more and rounded once.  Rows may be strided, values of a row are adjacent
(any other layout is copied first).  CPU tensors: dropout alone (the CPU mode, the same bits);
routing needs a ROCm GPU.
"""
import ctypes
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .engine import require_gpu

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
SCORES = {"softmax": 0, "sigmoid": 1}
_MASK64 = (1 << 64) - 1


class Routing(NamedTuple):
    """What route() gives, for `T` rows of `k` slots:

    experts [T, k] int32    the slot's expert, -1 where there is none
    weights [T, k] float32  its weight (differentiable), 0 where there is none
    offsets [E + 1] int32   rows of the experts before e in expert order; the last: rows in all
    pos     [T, k] int32    the slot's place in expert order (slots without an expert come last)
    src     [T * k] int32   the slot t * k + j at each place: the inverse of pos
    """
    experts: torch.Tensor
    weights: torch.Tensor
    offsets: torch.Tensor
    pos: torch.Tensor
    src: torch.Tensor


def dropout_key(seed, epoch, rank=0, site=0):
    """The 64-bit dropout key of one logical rank's epoch at one place (`site`) of a model."""
    v = ctypes.c_uint64()
    _lib.call("pss_dropout_key", int(seed) & _MASK64, int(epoch), int(rank), int(site), ctypes.byref(v))
    return v.value


# ---- plumbing ------------------------------------------------------------------------------------
def _call(name, device, *args):
    """The C entry with the current stream of `device` (which it makes the current one) as the last
    argument."""
    fn = getattr(_lib.load(), name)
    i = device.index
    if i != torch.cuda.current_device():
        with torch.cuda.device(i):
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if rc:
        _lib.check(rc, name)


def _once(backward):
    """A backward pass that cannot be differentiated itself: torch's once_differentiable where a
    graph of it is asked for, the plain function (without its overhead) where not."""
    wrapped = once_differentiable(backward)

    def f(ctx, *grads):
        return (wrapped if torch.is_grad_enabled() else backward)(ctx, *grads)
    return staticmethod(f)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows2d(t):
    """t [..., D] as (tensor, rows, D, row stride): as it is where its rows lie at one distance and
    a row's values are adjacent, else a contiguous copy."""
    if t.dim() == 2 and (t.stride(1) == 1 or t.shape[1] <= 1) and t.stride(0) >= 0:
        return t, t.shape[0], t.shape[1], t.stride(0)
    t = t.contiguous()
    d = t.shape[-1] if t.dim() else 1
    return t, t.numel() // d if d else 0, d, d


def _check_rows(name, t, like=None, shape=None):
    if t.dtype not in DTYPES:
        raise TypeError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise TypeError("%s must have the dtype and device of the rows: %s on %s, got %s on %s"
                        % (name, like.dtype, like.device, t.dtype, t.device))
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError("%s must be %s, got %s" % (name, list(shape), list(t.shape)))


def _row_ids(rows, n, device):
    """(row0, ids tensor or None): an int, or an int64 tensor of one or n ids on the device."""
    if not isinstance(rows, torch.Tensor):
        rows = int(rows)
        if not -(1 << 63) <= rows < 1 << 63:
            raise ValueError("rows must fit 64 bits")
        return rows, None
    if rows.dtype != torch.int64 or rows.device != device:
        raise TypeError("rows must be an int, or an int64 tensor on the rows' device")
    if rows.numel() not in (1, n):
        raise ValueError("rows must hold one id (the first row's) or one per row (%d), got %d" % (n, rows.numel()))
    return 0, rows.reshape(-1).contiguous()


def _p(p):
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("p must be in [0, 1], got %r" % p)
    return p


def _n(ids):
    return 0 if ids is None else ids.numel()


# ---- dropout -------------------------------------------------------------------------------------
def _dropout(x, residual, p, key, row0, ids):
    x2, n, d, ld = _rows2d(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    ldr = 0
    if residual is not None:
        residual, _, _, ldr = _rows2d(residual)
    args = (x2.data_ptr(), ld, _ptr(residual), ldr, y.data_ptr(), n, d, DTYPES[x.dtype], p, key, row0, _ptr(ids), _n(ids))
    if x.device.type == "cpu":
        _lib.call("pss_dropout", *args, 1, None)
    else:
        _call("pss_dropout", x.device, *args, 0)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, key, row0, ids):
        ctx.args = p, key, row0
        ctx.save_for_backward(ids)
        return _dropout(x, residual, p, key, row0, ids)

    @_once
    def backward(ctx, dy):
        p, key, row0 = ctx.args
        dx = _dropout(dy, None, p, key, row0, *ctx.saved_tensors) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout(x, p, key, rows=0, residual=None):
    """Dropout of rows x [..., D] with the mask of (key, row id, column): kept values times
    1 / (1 - p), dropped ones 0 whatever they were; plus `residual` (same shape) before the one
    rounding.  p is taken to the nearest 1/65536.

    rows: the first row's id (an int, or a one-element int64 tensor, read on the device so that a
    captured call can be replayed with another), or an int64 tensor with every row's id.  All
    leading dimensions of x are rows, in order."""
    p = _p(p)
    _check_rows("x", x)
    if x.dim() == 0:
        raise ValueError("x must have rows [..., D]")
    if residual is not None:
        _check_rows("residual", residual, x, x.shape)
    if x.device.type != "cpu":
        require_gpu()
    row0, ids = _row_ids(rows, x.numel() // x.shape[-1] if x.shape[-1] else 0, x.device)
    key = int(key) & _MASK64
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, p, key, row0, ids)
    return _dropout(x, residual, p, key, row0, ids)


# ---- routing -------------------------------------------------------------------------------------
def _route(logits, k, score, bias, valid, groups, top_groups, group_sum, renormalise, scale):
    l2, n, e, ld = _rows2d(logits)
    dev = logits.device
    i32 = torch.int32
    experts = torch.empty((n, k), dtype=i32, device=dev)
    weights = torch.empty((n, k), dtype=torch.float32, device=dev)
    offsets = torch.empty(e + 1, dtype=i32, device=dev)
    pos = torch.empty((n, k), dtype=i32, device=dev)
    src = torch.empty(n * k, dtype=i32, device=dev)
    need = _lib.load().pss_route_workspace(n, e)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _call("pss_route", dev, l2.data_ptr(), ld, n, e, k, DTYPES[logits.dtype], score, _ptr(bias), _ptr(valid), groups,
          top_groups, group_sum, renormalise, scale, experts.data_ptr(), weights.data_ptr(), offsets.data_ptr(),
          pos.data_ptr(), src.data_ptr(), _ptr(ws), need)
    return experts, weights, offsets, pos, src


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, score, bias, valid, groups, top_groups, group_sum, renormalise, scale):
        out = _route(logits, k, score, bias, valid, groups, top_groups, group_sum, renormalise, scale)
        ctx.mark_non_differentiable(out[0], *out[2:])
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, out[0], out[1])
        ctx.args = k, score, renormalise, scale
        return out

    @_once
    def backward(ctx, _experts, dweights, *_plan):
        if dweights is None or not ctx.needs_input_grad[0]:
            return (None,) * 10
        logits, experts, weights = ctx.saved_tensors
        k, score, renormalise, scale = ctx.args
        l2, n, e, ld = _rows2d(logits)
        dweights = dweights.contiguous()
        dlogits = torch.empty((n, e), dtype=logits.dtype, device=logits.device)
        _call("pss_route_grad", logits.device, l2.data_ptr(), ld, n, e, k, DTYPES[logits.dtype], score, renormalise,
              scale, experts.data_ptr(), weights.data_ptr(), dweights.data_ptr(), dlogits.data_ptr())
        return (dlogits,) + (None,) * 9


def route(logits, k, *, score="softmax", bias=None, groups=1, top_groups=1, group_sum=1, renormalise=True, scale=1.0,
          valid=None):
    """Routing of every row of logits [T, E] to k of E experts -> Routing.

    score        "softmax" over the row or "sigmoid" of each logit
    bias         [E] float32, added to the scores for the choice alone (balance); no gradient
    groups       consecutive experts form this many equal groups, and only the top_groups groups of
                 the highest value -- the sum of their group_sum (1 or 2) best -- take part
    renormalise  a row's weights are divided by the sum of its chosen scores
    scale        factor of all weights
    valid        [T] bool: rows that are padding get no expert

    The best choice first, ties to the lower index.  A logit of -inf masks the expert; a row with
    fewer than k left has experts -1 and weights 0 in its last slots.  Gradients flow from
    Routing.weights to the logits.  E <= 1024, k <= 16, groups <= 64, T * k < 2^31."""
    _check_rows("logits", logits)
    if logits.dim() != 2:
        raise ValueError("logits must be [T, E], got %s" % list(logits.shape))
    if logits.device.type != "cuda":
        raise RuntimeError("route needs its logits on a ROCm GPU (no CPU fallback)")
    require_gpu()
    if score not in SCORES:
        raise ValueError("score must be 'softmax' or 'sigmoid', got %r" % (score,))
    n, e = logits.shape
    if bias is not None:
        if bias.dtype != torch.float32 or bias.device != logits.device or tuple(bias.shape) != (e,):
            raise ValueError("bias must be float32 [%d] on the logits' device" % e)
        bias = bias.detach().contiguous()
    if valid is not None:
        if valid.dtype != torch.bool or valid.device != logits.device or tuple(valid.shape) != (n,):
            raise ValueError("valid must be bool [%d] on the logits' device" % n)
        valid = valid.contiguous()
    args = (int(k), SCORES[score], bias, valid, int(groups), int(top_groups), int(group_sum), int(bool(renormalise)),
            float(scale))
    if torch.is_grad_enabled() and logits.requires_grad:
        return Routing(*_Route.apply(logits, *args))
    return Routing(*_route(logits, *args))


def _check_plan(r, device, n=None):
    """(T, k) of a Routing whose tensors are what route() makes."""
    if not isinstance(r, Routing):
        raise TypeError("routing must be a Routing (ops.route), got %s" % type(r).__name__)
    for name in ("experts", "pos"):
        t = getattr(r, name)
        if t.dtype != torch.int32 or t.dim() != 2 or t.device != device or not t.is_contiguous():
            raise ValueError("routing.%s must be contiguous int32 [T, k] on the rows' device" % name)
    if r.pos.shape != r.experts.shape:
        raise ValueError("routing.pos and routing.experts differ in shape")
    if n is not None and r.pos.shape[0] != n:
        raise ValueError("the routing is of %d rows, got %d" % (r.pos.shape[0], n))
    return r.pos.shape


# ---- dispatch and combine ------------------------------------------------------------------------
def _dispatch(x, experts, pos):
    x2, n, d, ld = _rows2d(x)
    k = pos.shape[1]
    xs = torch.empty((n * k, d), dtype=x.dtype, device=x.device)
    _call("pss_dispatch", x.device, x2.data_ptr(), ld, n, k, d, DTYPES[x.dtype], experts.data_ptr(), pos.data_ptr(),
          xs.data_ptr())
    return xs


def _combine(y, experts, pos, weights, residual, p, key, row0, ids):
    n, k = pos.shape
    y = y.contiguous()
    d = y.shape[1]
    out = torch.empty((n, d), dtype=y.dtype, device=y.device)
    ldr = 0
    if residual is not None:
        residual, _, _, ldr = _rows2d(residual)
    _call("pss_combine", y.device, y.data_ptr(), n, k, d, DTYPES[y.dtype], experts.data_ptr(), pos.data_ptr(),
          _ptr(weights), _ptr(residual), ldr, p, key, row0, _ptr(ids), _n(ids), out.data_ptr())
    return out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, experts, pos):
        ctx.save_for_backward(experts, pos)
        return _dispatch(x, experts, pos)

    @_once
    def backward(ctx, dxs):
        experts, pos = ctx.saved_tensors
        return _combine(dxs, experts, pos, None, None, 0.0, 0, 0, None), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, residual, experts, pos, p, key, row0, ids):
        ctx.save_for_backward(y, weights, experts, pos, ids)
        ctx.args = p, key, row0
        return _combine(y, experts, pos, weights, residual, p, key, row0, ids)

    @_once
    def backward(ctx, dout):
        want_y, want_w, want_r = ctx.needs_input_grad[:3]
        dy = dw = None
        if want_y or want_w:
            y, weights, experts, pos, ids = ctx.saved_tensors
            p, key, row0 = ctx.args
            n, k = pos.shape
            y = y.contiguous()
            d2, _, d, ld = _rows2d(dout)
            dy = torch.empty_like(y) if want_y else None
            dw = torch.empty((n, k), dtype=torch.float32, device=y.device) if want_w else None
            _call("pss_combine_grad", y.device, d2.data_ptr(), ld, y.data_ptr(), n, k, d, DTYPES[y.dtype],
                  experts.data_ptr(), pos.data_ptr(), weights.data_ptr(), p, key, row0, _ptr(ids), _n(ids), _ptr(dy),
                  _ptr(dw))
        return (dy, dw, dout if want_r else None) + (None,) * 6


def dispatch(x, routing):
    """The rows x [T, D] in expert order: [T * k, D], expert e's rows at
    [offsets[e], offsets[e + 1]) in the order of their tokens; rows of slots without an expert, the
    last ones, are 0."""
    _check_rows("x", x)
    if x.dim() != 2 or x.device.type != "cuda":
        raise ValueError("x must be [T, D] on a ROCm GPU")
    _check_plan(routing, x.device, x.shape[0])
    if torch.is_grad_enabled() and x.requires_grad:
        return _Dispatch.apply(x, routing.experts, routing.pos)
    return _dispatch(x, routing.experts, routing.pos)


def combine(y, routing, residual=None, p=0.0, key=0, rows=0):
    """The experts' outputs y [T * k, D] (in expert order) back to the rows' order, by weight:
    residual[t] + dropout(sum over t's slots with an expert of weight * y), [T, D].  p, key, rows: as
    dropout() has them.  Gradients for y, the routing's weights and the residual."""
    p = _p(p)
    _check_rows("y", y)
    if y.dim() != 2 or y.device.type != "cuda":
        raise ValueError("y must be [T * k, D] on a ROCm GPU")
    n, k = _check_plan(routing, y.device)
    if y.shape[0] != n * k:
        raise ValueError("y must have the routing's %d rows, got %d" % (n * k, y.shape[0]))
    w = routing.weights
    if w.dtype != torch.float32 or tuple(w.shape) != (n, k) or w.device != y.device:
        raise ValueError("routing.weights must be float32 [%d, %d] on the rows' device" % (n, k))
    w = w.contiguous()
    if residual is not None:
        _check_rows("residual", residual, y, (n, y.shape[1]))
    row0, ids = _row_ids(rows, n, y.device)
    key = int(key) & _MASK64
    if torch.is_grad_enabled() and (y.requires_grad or w.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        return _Combine.apply(y, w, residual, routing.experts, routing.pos, p, key, row0, ids)
    return _combine(y, routing.experts, routing.pos, w, residual, p, key, row0, ids)
