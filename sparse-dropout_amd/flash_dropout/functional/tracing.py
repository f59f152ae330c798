"""The compiled functions under ``torch.jit.trace``.

A trace records operators and Python autograd functions.  The native functions are neither: of a call into them it would
record the allocation of the result and nothing that fills it, and the traced program would return uninitialised memory.
So while a trace is being taken their call is made inside a Python autograd function, which the trace records as one
operation on the call's tensors and runs again whenever the traced program runs.
"""
from __future__ import annotations

import functools
from collections.abc import Iterable

import torch

_is_tracing = torch._C._is_tracing  # what torch.jit.is_tracing asks outside of a script, in half of its time


class _Slot(int):
    """The place of a tensor among the operation's inputs."""


def _take(value, tensors: list):
    """``value`` with every tensor moved to ``tensors`` and a slot in its place."""
    if isinstance(value, torch.Tensor):
        tensors.append(value)
        return _Slot(len(tensors) - 1)
    if isinstance(value, Iterable) and not isinstance(value, str):
        return [_take(v, tensors) for v in value]
    return value


def _put(value, tensors):
    if isinstance(value, _Slot):
        return tensors[value]
    return [_put(v, tensors) for v in value] if isinstance(value, list) else value


class _RecordedCall(torch.autograd.Function):
    @staticmethod
    def forward(ctx, call, *tensors):
        ctx.leaves = [t.detach().requires_grad_(need) for t, need in zip(tensors, ctx.needs_input_grad[1:])]
        with torch.enable_grad(), torch.autocast("cuda", enabled=False):
            ctx.result = call(ctx.leaves)
        return ctx.result.detach()

    @staticmethod
    def backward(ctx, grad):
        ctx.saved_tensors  # (raises once the graph was freed)
        wanted = [t for t in ctx.leaves if t.requires_grad]
        # retained: whether there will be another backward is the outer graph's to say
        grads = iter(torch.autograd.grad(ctx.result, wanted, grad, retain_graph=True))
        return (None, *(next(grads) if t.requires_grad else None for t in ctx.leaves))


class _RecordedPlainCall(torch.autograd.Function):
    """Of a function without a gradient, which refuses inputs that want one: whether a trace's inputs do is only known when it is
    differentiated."""

    @staticmethod
    def forward(ctx, call, *tensors):
        with torch.autocast("cuda", enabled=False):
            return call([t.detach() for t in tensors])

    @staticmethod
    def backward(ctx, grad):
        raise NotImplementedError("the traced function has no gradient: call it under torch.no_grad()")


class _RecordedConstantCall(torch.autograd.Function):
    """Of a function whose results carry no gradient."""

    @staticmethod
    def forward(ctx, call, *tensors):
        results = call([t.detach() for t in tensors])
        ctx.mark_non_differentiable(*(results if isinstance(results, tuple) else (results,)))
        return results

    @staticmethod
    def backward(ctx, *grads):
        return (None,) * len(ctx.needs_input_grad)


def traceable(function=None, *, recorded=_RecordedCall, cast=True):
    """Makes a function of tensors that calls native code one recorded operation under ``torch.jit.trace``.  cast: under autocast it takes
    its operands in autocast's dtype."""

    if function is None:
        return functools.partial(traceable, recorded=recorded, cast=cast)

    @functools.wraps(function)
    def run(*args, **kwargs):
        if not _is_tracing():
            return function(*args, **kwargs)
        tensors: list[torch.Tensor] = []
        names, values = list(kwargs), _take([*args, *kwargs.values()], tensors)
        if cast and torch.is_autocast_enabled("cuda"):  # the casts are the trace's own
            dtype = torch.get_autocast_dtype("cuda")
            tensors = [t.to(dtype) if t.is_floating_point() and t.element_size() > 1 else t for t in tensors]  # (8-bit codes stay)

        def call(given):
            filled = _put(values, given)
            return function(*filled[:len(args)], **dict(zip(names, filled[len(args):])))

        return recorded.apply(call, *tensors)

    return run


def refused_under_trace(function):
    """Of a function that a trace would record none of: it writes its arguments, or lists of any length are what it takes and gives."""

    @functools.wraps(function)
    def run(*args, **kwargs):
        if _is_tracing():
            raise NotImplementedError(f"{function.__name__} cannot be traced")
        return function(*args, **kwargs)

    return run
