"""The input-stage operators as differentiable functions: embed, dropout and rms_norm of hades_amd.ops
with their gradients for torch.autograd.

    x = functional.embed(weight, ids, scale=dim ** 0.5)               # weight.grad: dense, summed in float32
    x = functional.dropout(x, p, seed, offset, residual=stream)       # the mask is drawn again, not kept
    y, h = functional.rms_norm(x, gamma, residual=stream, dropout=(p, seed, offset))

`dropout` = (p, seed, offset) as in ops; an offset tensor must keep its value until the backward pass has
run (torch's version check raises otherwise).  The backward passes are not differentiable themselves, and
there are no forward-mode derivatives: a tensor that carries a tangent is refused, with gradients on or off.

Graph capture.  A leaf's gradient is accumulated on the stream of the first graph that used the leaf, for
as long as any graph of it lives.  If that graph was made eagerly on another stream (its output or loss is
still referenced), a backward pass under capture would pull that stream into the capture, which ends the
process on the default stream.  A graph that was itself captured on another stream would pull in that one.  The
functions here refuse both: under capture they raise if a graph of the same leaf, made through them on another
stream, is still alive.
"""
import weakref

import torch
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from . import ops

_graphs = {}      # id of a leaf -> (weak reference to it, weak set of the graphs that use it)


def _note(ctx, *leaves):
    """Records this call's graph with the leaves it uses; refuses a capture beside a graph of another stream."""
    capturing = ctx.captured = torch.cuda.is_current_stream_capturing()
    ctx.stream = torch.cuda.current_stream().cuda_stream
    for t in leaves:
        if t is None or not t.requires_grad or not t.is_leaf:
            continue
        key = id(t)
        entry = _graphs.get(key)
        if entry is None or entry[0]() is not t:
            entry = _graphs[key] = (weakref.ref(t, lambda r, key=key: _forget(key, r)), weakref.WeakSet())
        if capturing:
            for other in entry[1]:
                if other.stream == ctx.stream:
                    continue
                if other.captured:
                    raise RuntimeError("a graph of the same leaf that was captured on another stream is alive: capture "
                                       "on that stream, or drop its output and loss before capturing")
                raise RuntimeError("an eager graph of the same leaf lives on another stream: drop its output and loss "
                                   "before capturing (a backward pass under capture would end the process)")
        entry[1].add(ctx)


def _forget(key, ref):
    if key in _graphs and _graphs[key][0] is ref:
        del _graphs[key]


def _keep_drop(ctx, dropout, *saved):
    """Saves `saved` and an offset tensor for backward, the plain part of dropout on ctx."""
    ctx.drop = dropout
    if dropout is not None and isinstance(dropout[2], torch.Tensor):
        ctx.drop = (dropout[0], dropout[1], None)
        saved += (dropout[2],)
    ctx.save_for_backward(*saved)


def _kept(ctx):
    """(saved tensors, dropout) of _keep_drop"""
    saved, drop = ctx.saved_tensors, ctx.drop
    if drop is not None and drop[2] is None:
        return saved[:-1], (drop[0], drop[1], saved[-1])
    return saved, drop


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx, dropout):
        _note(ctx, weight)
        _keep_drop(ctx, dropout, ids)
        ctx.num_rows, ctx.scale, ctx.padding_idx = weight.size(0), scale, padding_idx
        return ops.embed(weight, ids, scale=scale, dropout=dropout)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (ids,), drop = _kept(ctx)
        grad = ops.embed_grad(grad.contiguous(), ids, ctx.num_rows, scale=ctx.scale, padding_idx=ctx.padding_idx,
                              dropout=drop)
        return grad, None, None, None, None


def _as_stream(x, residual):
    """x, widened where 16-bit rows go onto a float32 residual stream (ops.dropout takes rows of one type)."""
    if residual is not None and residual.dtype == torch.float32 and x.dtype in (torch.float16, torch.bfloat16):
        return x.float()
    return x


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, dropout):
        _note(ctx, x, residual)
        _keep_drop(ctx, dropout)
        ctx.x_dtype = x.dtype
        return ops.dropout(_as_stream(x, residual), *dropout, residual=residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _, drop = _kept(ctx)
        gx = ops.dropout_grad(grad.contiguous(), *drop).to(ctx.x_dtype) if ctx.needs_input_grad[0] else None
        return gx, grad if ctx.needs_input_grad[1] else None, None


class _RmsNorm(torch.autograd.Function):
    """Returns y, and h where it is not x."""

    @staticmethod
    def forward(ctx, x, weight, eps, residual, dropout):
        _note(ctx, x, weight, residual)
        ctx.set_materialize_grads(False)
        y, h, rstd = ops.rms_norm(x, weight, eps, residual=residual, dropout=dropout)
        _keep_drop(ctx, dropout, h, weight, rstd)
        ctx.x_dtype = x.dtype
        return y if h is x else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gh=None):
        (h, weight, rstd), drop = _kept(ctx)
        need_x, need_w, _, need_res, _ = ctx.needs_input_grad
        gh = None if gh is None else gh.contiguous()
        if gy is not None:
            gx, gres, gw = ops.rms_norm_grad(gy.contiguous(), h, weight, rstd, grad_h=gh, dropout=drop,
                                             weight_grad=need_w, residual_grad=need_res)
        elif gh is not None:          # only h was used
            gres, gw = gh, None
            gx = gh.to(ctx.x_dtype) if drop is None else ops.dropout_grad(gh, *drop).to(ctx.x_dtype)
        else:
            gx = gres = gw = None
        return gx if need_x else None, gw, None, gres if need_res else None, None


def _plain(*tensors):
    """Whether a call has no derivative to record: gradients are off and no tensor carries a forward-mode
    tangent (autograd.Function, which has no rule for tangents here, refuses those)."""
    if torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and unpack_dual(t).tangent is not None:
            return False
    return True


def embed(weight, ids, scale=1.0, padding_idx=None, dropout=None):
    """ops.embed; weight's gradient is ops.embed_grad (padding_idx gets none)."""
    if _plain(weight):      # no graph, and nothing that a capture could pull in
        return ops.embed(weight, ids, scale=scale, dropout=dropout)
    return _Embed.apply(weight, ids, scale, padding_idx, dropout)


def dropout(x, p, seed, offset, residual=None):
    """ops.dropout, and of 16-bit rows onto a float32 residual too, with a float32 sum; the gradients are the same mask
    on the output's gradient, and that gradient itself."""
    if _plain(x, residual):
        return ops.dropout(_as_stream(x, residual), p, seed, offset, residual=residual)
    return _Dropout.apply(x, residual, (p, seed, offset))


def rms_norm(x, weight=None, eps=1e-6, residual=None, dropout=None):
    """(y, h) of ops.rms_norm; h is x itself where there is neither residual nor dropout."""
    if _plain(x, weight, residual):
        return ops.rms_norm(x, weight, eps, residual=residual, dropout=dropout)[:2]
    out = _RmsNorm.apply(x, weight, eps, residual, dropout)
    return out if isinstance(out, tuple) else (out, x)
