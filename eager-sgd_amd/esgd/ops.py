"""Operators of a language model's training step around its matrix products, on the device:
embedding lookup, tokens in their experts' order, and distillation from a teacher's top logits,
each with its gradient (C ABI: include/esgd_ops.h, which has the formulas).

They take torch tensors on a HIP device and run on the caller's current stream of that device;
nothing waits for the GPU, so all of them can be captured into a graph.  embedding,
expert_dispatch, expert_combine and distill_loss take part in autograd (once; their gradients
have no gradients, and a tensor with a forward-mode tangent is refused); the *_grad functions are
the same gradients called directly, for training steps that keep their own buckets --
embedding_grad can add into the one that the optimizer reduces.  float32, bfloat16 and float16;
sums are fp32, in a fixed order, so the same call gives the same bits every time.  Inputs
whose rows are contiguous are read where they lie, at any distance and alignment; others are
copied first.  There is no CPU path.
"""
from __future__ import annotations

import ctypes as C
import os

import torch

from . import _lib

HALF = 17        # ESGD_HALF
TOP_MAX = 1024   # ESGD_DISTILL_TOP_MAX


_names = []


def _bind(h):
    i, i64, f, sz, vp = C.c_int, C.c_int64, C.c_float, C.c_size_t, C.c_void_p
    psz = C.POINTER(sz)
    sig = {
        "esgd_embedding": [i, vp, i64, i64, i64, i, vp, i64, f, i, vp, i64, vp],
        "esgd_embedding_grad_work": [i64, i64, i64, psz],
        "esgd_embedding_grad": [i, vp, i64, i64, i64, i, vp, i64, f, i, vp, i64, i, vp, sz, vp],
        "esgd_expert_sort_work": [i64, i64, psz],
        "esgd_expert_sort": [i, vp, i64, i64, i64, vp, vp, vp, sz, vp],
        "esgd_expert_dispatch": [i, vp, i64, i64, i64, i64, vp, vp, vp],
        "esgd_expert_dispatch_grad": [i, vp, i64, i64, i64, i64, vp, vp, vp],
        "esgd_expert_combine": [i, vp, i64, i64, i64, i64, vp, vp, vp, vp],
        "esgd_expert_combine_grad": [i, vp, i64, vp, i64, i64, i64, i64, vp, vp, vp, vp, vp],
        "esgd_distill_work": [i64, i64, psz],
        "esgd_distill_loss": [i, vp, i64, i64, i64, i, vp, i, vp, i64, f, vp, vp, vp, sz, vp],
        "esgd_distill_grad": [i, vp, i64, i64, i64, i, vp, i, vp, i64, f, vp, vp, i64, vp, vp],
        "esgd_distill_loss_grad": [i, vp, i64, i64, i64, i, vp, i, vp, i64, f, vp, i64, vp, vp, vp, vp, sz, vp],
    }
    for name, args in sig.items():
        fn = getattr(h, name)
        fn.restype, fn.argtypes = i, args
    _names[:] = sig


_lib.register_signatures(_bind)


def _load():
    """esgd._ops, which checks tensors, allocates and makes the C calls (csrc/torch/ops_torch.cpp),
    with the entry points of the library that _lib has loaded."""
    h = _lib.lib()
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_ops.so")
    if not os.path.exists(path):
        raise _lib.EsgdError(_lib.ERROR, f"{path} not built (run `make ops` or __graft_entry__.build())")
    from . import _ops
    _ops.bind({name: C.cast(getattr(h, name), C.c_void_p).value for name in _names})
    return _ops


_ops = _load()


def _number(who: str, name: str, x):
    """Refuses a tensor where a number is taken: its gradient would be lost, and the call would
    wait for the GPU to read it."""
    if isinstance(x, torch.Tensor):
        raise ValueError(f"{who}: {name} is a tensor; a number is needed (no gradient goes there)")


# ---- embedding -----------------------------------------------------------------------------

def _padding(who: str, padding_index) -> int:
    """The row without gradient as the C calls take it, -1 for none."""
    if padding_index is None:
        return -1
    _number(who, "padding_index", padding_index)
    if padding_index < 0:
        raise ValueError(f"{who}: padding_index {padding_index} is negative (tokens outside the table need none)")
    return int(padding_index)


def embedding_grad(grad, tokens, num_rows: int, scale: float = 1.0, *, padding_index: int | None = None, dtype=None,
                   out=None, accumulate: bool = False):
    """The table's gradient, (num_rows, width): row v is scale * the sum of grad[t] over the
    tokens[t] == v, zeros where there is none.  Tokens outside [0, num_rows) and those equal to
    padding_index give nothing.  dtype: grad's own (default) or float32.  out: a contiguous
    tensor to write (its dtype counts then); accumulate=True adds to it instead, and reads and
    writes only the rows that the tokens name."""
    _number("embedding_grad", "num_rows", num_rows)
    _number("embedding_grad", "scale", scale)
    return _ops.embedding_grad(grad, tokens, num_rows, scale, _padding("embedding_grad", padding_index), dtype, out,
                               accumulate)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens, scale, padding_index, dtype):
        ctx.save_for_backward(tokens)
        ctx.rest = (weight.shape[0], scale, padding_index, weight.dtype)
        return _ops.embedding(weight, tokens, scale, dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        tokens, = ctx.saved_tensors
        rows, scale, padding_index, dtype = ctx.rest
        return (embedding_grad(grad, tokens, rows, scale, padding_index=padding_index, dtype=dtype),
                None, None, None, None)


def embedding(weight, tokens, scale: float = 1.0, *, padding_index: int | None = None, dtype=None):
    """weight[tokens] * scale, of shape (*tokens.shape, width).  A token outside the table --
    padding, say -1 -- reads as zeros and gives no gradient; padding_index is a row that is read
    as it is but gets no gradient either.  dtype: the result's, weight's own by default; a
    float32 table also gives bfloat16 or float16 rows.  The gradient is dense, of weight's dtype."""
    _number("embedding", "scale", scale)
    if padding_index is not None:
        _padding("embedding", padding_index)
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(weight, tokens, scale, padding_index, dtype)
    return _ops.embedding(weight, tokens, scale, dtype)


# ---- tokens by expert ------------------------------------------------------------------------

class ExpertOrder:
    """The (token, choice) pairs in their experts' order, made by expert_sort.

    offsets  (num_experts + 1,) int32: expert e has the places offsets[e] .. offsets[e + 1]
    slots    (tokens, choices) int32: the pair's place; -1 - place of a dropped pair, whose place
             lies behind every expert's
    """

    __slots__ = ("offsets", "slots", "num_experts")

    def __init__(self, offsets, slots, num_experts: int):
        self.offsets, self.slots, self.num_experts = offsets, slots, num_experts

    @property
    def tokens(self) -> int:
        return self.slots.shape[0]

    @property
    def choices(self) -> int:
        return self.slots.shape[1]


def expert_sort(experts, num_experts: int) -> ExpertOrder:
    """The order of the pairs of `experts` ((tokens, choices) or (tokens,), int32 or int64) by
    expert, equal experts by (token, choice).  Pairs whose expert is outside [0, num_experts)
    are dropped: they come last and take no part in dispatch and combine."""
    _number("expert_sort", "num_experts", num_experts)
    offsets, slots = _ops.expert_sort(experts, num_experts)
    return ExpertOrder(offsets, slots, num_experts)


def expert_dispatch_grad(grad_rows, order: ExpertOrder):
    """expert_dispatch's gradient: grad_x[t] = the sum of grad_rows over the token's places, in the order of its choices."""
    return _ops.expert_dispatch_grad(grad_rows, order.slots)


def expert_combine_grad(grad, rows, weights, order: ExpertOrder):
    """expert_combine's gradients (grad_rows, grad_weights): weights[t, j] * grad[t] at the pair's
    place, zeros at dropped pairs', and the products <grad[t], rows[place]> (float32)."""
    return _ops.expert_combine_grad(grad, rows, weights, order.slots)


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, slots):
        ctx.save_for_backward(slots)
        return _ops.expert_dispatch(x, slots)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return _ops.expert_dispatch_grad(grad, ctx.saved_tensors[0]), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, slots):
        ctx.save_for_backward(rows, weights, slots)
        return _ops.expert_combine(rows, weights, slots)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        rows, weights, slots = ctx.saved_tensors
        grad_rows, grad_weights = _ops.expert_combine_grad(grad, rows, weights, slots)
        return grad_rows, grad_weights.to(weights.dtype).view(weights.shape), None


def expert_dispatch(x, order: ExpertOrder):
    """The tokens' rows in their experts' order, (tokens * choices, width): x[t] at each place of
    token t, zeros at the places of dropped pairs (behind offsets[-1])."""
    if x.requires_grad and torch.is_grad_enabled():
        return _Dispatch.apply(x, order.slots)
    return _ops.expert_dispatch(x, order.slots)


def expert_combine(rows, weights, order: ExpertOrder):
    """out[t] = sum over j of weights[t, j] * rows[place of (t, j)], (tokens, width); dropped pairs
    (their rows and weights are not used) give nothing."""
    if (rows.requires_grad or weights.requires_grad) and torch.is_grad_enabled():
        return _Combine.apply(rows, weights, order.slots)
    return _ops.expert_combine(rows, weights, order.slots)


# ---- distillation ----------------------------------------------------------------------------

class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_logits, top_index, temperature):
        loss, stats = _ops.distill_loss(logits, top_logits, top_index, temperature)
        ctx.save_for_backward(logits, top_logits, top_index, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        logits, top_logits, top_index, stats = ctx.saved_tensors
        return (_ops.distill_grad(logits, top_logits, top_index, ctx.temperature, stats, grad), None, None, None)


def distill_loss(logits, top_logits, top_index, temperature: float = 1.0):
    """Per row, temperature^2 * KL(p || q) of the teacher's shares p = softmax(top_logits /
    temperature) over the entries of top_index in [0, vocab), and the student's
    q = softmax(logits / temperature): float32, of logits' shape without the last dimension.

    logits (..., vocab); top_logits and top_index (int32 or int64) (..., top), top <= 1024, in any
    order, the teacher a constant.  Entries outside the vocabulary (-1: none) and those of -inf
    take no part; an index that stands there twice counts twice.  A row left without any entry has
    loss and gradient 0 whatever its logits are.  logits of -inf have no share."""
    _number("distill_loss", "temperature", temperature)
    if logits.requires_grad and torch.is_grad_enabled():
        return _Distill.apply(logits, top_logits, top_index, temperature)
    return _ops.distill_loss(logits, top_logits, top_index, temperature)[0]


def distill_loss_grad(logits, top_logits, top_index, row_grad, temperature: float = 1.0):
    """(loss, grad_logits) of distill_loss at once, where the losses' gradients are known before:
    grad_logits = row_grad[r] * d loss[r] / d logits, contiguous, in logits' dtype.  row_grad: float32,
    of the loss's shape (1 / rows for the mean; an expanded scalar will do)."""
    _number("distill_loss_grad", "temperature", temperature)
    return _ops.distill_loss_grad(logits, top_logits, top_index, row_grad, temperature)
