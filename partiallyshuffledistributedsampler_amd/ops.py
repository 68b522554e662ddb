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
nothing; the four calls above can be captured into a graph (capture a backward pass only while no
eager autograd graph of the same leaves is alive: torch ties a leaf's accumulation to the stream that
it was first used on, and waiting for that stream ends a capture).  They work on memory: torch.compile
runs them outside its graphs, and what records torch's own operations (jit.trace, make_fx, export,
fake tensors) is refused.  fp32, bf16 and fp16 rows; sums and softmax statistics are held in 32 bits
or more and rounded once.  Rows may be strided, values of a row are adjacent (any other layout is
copied first).  CPU tensors: dropout alone (the CPU mode, the same bits); routing needs a ROCm GPU.
"""
import ctypes
from typing import NamedTuple

import torch

from . import _lib

SCORES = {"softmax": 0, "sigmoid": 1}
_MASK64 = (1 << 64) - 1
_ENTRIES = ("pss_last_error", "pss_dropout", "pss_route_workspace", "pss_route", "pss_route_grad",
            "pss_dispatch", "pss_combine", "pss_combine_grad", "pss_gather_dropout")


def _load():
    """The torch binding (csrc/pss_torch.cpp) on the entries of the loaded libpss.so."""
    lib = _lib.load()
    try:
        from . import _pss_torch
    except ImportError as e:
        raise ImportError("_pss_torch.so is not built. Build it with `python -c 'import "
                          "__graft_entry__ as g; g.build()'` -- there is no fallback.") from e
    _pss_torch.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _ENTRIES})
    return _pss_torch


_c = _load()


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
    """The 64-bit dropout key of one logical rank's epoch at one place (`site`) of a model.  The seed is
    taken modulo 2^64; epoch fits 64 bits, rank and site 32, with a sign."""
    epoch, rank, site = int(epoch), int(rank), int(site)
    for name, n, bits in (("epoch", epoch, 63), ("rank", rank, 31), ("site", site, 31)):
        if not -(1 << bits) <= n < 1 << bits:
            raise ValueError("%s must fit %d bits, got %d" % (name, bits + 1, n))
    v = ctypes.c_uint64()
    _lib.call("pss_dropout_key", int(seed) & _MASK64, epoch, rank, site, ctypes.byref(v))
    return v.value


def _row_ids(rows):
    """(row0, ids tensor or None) of a row-id argument."""
    if isinstance(rows, torch.Tensor):
        return 0, rows
    rows = int(rows)
    if not -(1 << 63) <= rows < 1 << 63:
        raise ValueError("rows must fit 64 bits")
    return rows, None


def dropout(x, p, key, rows=0, residual=None):
    """Dropout of rows x [..., D] with the mask of (key, row id, column): kept values times
    1 / (1 - p), dropped ones 0 whatever they were; plus `residual` (same shape) before the one
    rounding.  p is taken to the nearest 1/65536.

    rows: the first row's id (an int, or a one-element int64 tensor, read on the device so that a
    captured call can be replayed with another), or an int64 tensor with every row's id.  All
    leading dimensions of x are rows, in order."""
    row0, ids = _row_ids(rows)
    return _c.dropout(x, p, int(key) & _MASK64, row0, ids, residual)


def gather(engine, data, base_rows, fpos, off, out=None, stream=None, p=0.0, key=0, rows=0):
    """IndexEngine.gather(..., p, key, rows): rows of device-resident files with dropout."""
    if stream is not None and not engine.cpu:
        with torch.cuda.stream(stream):     # (what the call allocates belongs to that stream, too)
            return gather(engine, data, base_rows, fpos, off, out, None, p, key, rows)
    row0, ids = _row_ids(rows)
    return _c.gather(engine._h.value if engine._h else 0, engine._dev(), engine.num_files, data, base_rows, fpos, off,
                     out, p, int(key) & _MASK64, row0, ids)


def route(logits, k, *, score="softmax", bias=None, groups=1, top_groups=1, group_sum=1, renormalise=True, scale=1.0,
          valid=None):
    """Routing of every row of logits [T, E] to k of E experts -> Routing.

    score        "softmax" over the row or "sigmoid" of each logit
    bias         [E] float32, added to the scores for the choice alone (balance); no gradient
    groups       consecutive experts form this many equal groups, and only the top_groups groups of
                 the highest value -- the sum of their group_sum (1 or 2) best -- take part
    renormalise  a row's weights are divided by the sum of its chosen scores
    scale        factor of all weights (1e-18 to 1e18 in magnitude)
    valid        [T] bool: rows that are padding get no expert

    The best choice first, ties to the lower index.  A logit or a bias of -inf masks the expert; a row
    with fewer than k left has experts -1 and weights 0 in its last slots.  A NaN is chosen last of all
    that are not masked, and makes the weights NaN if it is a logit's.  Gradients flow from
    Routing.weights to the logits.  E <= 1024, k <= 16, groups <= 64, T < 2^28, T * k < 2^31."""
    if score not in SCORES:
        raise ValueError("score must be 'softmax' or 'sigmoid', got %r" % (score,))
    return Routing(*_c.route(logits, k, SCORES[score], bias, valid, groups, top_groups, group_sum, bool(renormalise), scale))


def _plan(routing):
    if not isinstance(routing, Routing):
        raise TypeError("routing must be a Routing (ops.route), got %s" % type(routing).__name__)
    return routing


def dispatch(x, routing):
    """The rows x [T, D] in expert order: [T * k, D], expert e's rows at
    [offsets[e], offsets[e + 1]) in the order of their tokens; rows of slots without an expert, the
    last ones, are 0."""
    r = _plan(routing)
    return _c.dispatch(x, r.experts, r.pos)


def combine(y, routing, residual=None, p=0.0, key=0, rows=0):
    """The experts' outputs y [T * k, D] (in expert order) back to the rows' order, by weight:
    residual[t] + dropout(sum over t's slots with an expert of weight * y), [T, D].  p, key, rows: as
    dropout() has them.  Gradients for y, the routing's weights and the residual."""
    r = _plan(routing)
    row0, ids = _row_ids(rows)
    return _c.combine(y, r.weights, r.experts, r.pos, residual, p, int(key) & _MASK64, row0, ids)
