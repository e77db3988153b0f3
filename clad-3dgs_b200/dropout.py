"""Dropout from a counter-based generator, with a mask that is never stored.

`dropout(x, p, seed, offset)` keeps element e of x (counted in row-major
order) iff the e-th word that Philox4x32-10 gives for (seed, offset) is at
least floor(p * 2^32), scales what it keeps by 1 / (1 - p) and sets the rest
to zero. The same numbers always give the same decisions, whatever x's layout
or type, so the backward pass draws them again instead of reading a mask; a
program picks a new `offset` for every call (a step counter, say) under one
`seed`. `rows=True` decides once for each row (all of the last dimension):
Gaussians or tokens are dropped whole.

`offset` may be a one-element int64 CUDA tensor, read when the kernel runs: a
captured graph then draws anew at each replay once the program has advanced
it. It must not change between a forward pass and its backward pass (autograd
checks the tensor's version).

float32, float16 and bfloat16; inputs may have any layout, outputs are
contiguous. Kernels launch on the current stream of x's device and may be
captured into a graph. (Torch cannot capture any backward pass while an eager
autograd graph over the same leaf is alive: drop its outputs first, or capture
`apply` on the gradient.) Bad arguments raise RuntimeError before anything is
written.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

import _native as native

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
WORD = 2 ** 64


def _require(condition, message):
    if not condition:
        raise RuntimeError(message)


def check_draw(p, seed, offset, device):
    """Checks a dropout's numbers; returns (offset as an int, address of the
    device offset or None)."""
    if not (isinstance(p, (int, float)) and 0.0 <= p <= 1.0):
        raise RuntimeError("p must lie in [0, 1]")
    if not (isinstance(seed, int) and 0 <= seed < WORD):
        raise RuntimeError("seed must be an integer in [0, 2^64)")
    if isinstance(offset, torch.Tensor):
        _require(offset.device == device and offset.dtype == torch.int64
                 and offset.numel() == 1, "a tensor offset must be one int64 on the input's device")
        return 0, offset.data_ptr()
    if not (isinstance(offset, int) and 0 <= offset < WORD):
        raise RuntimeError("offset must be an integer in [0, 2^64) or a CUDA tensor")
    return offset, None


def parts_of(x):
    """(x without its tangent, the tangent) of a dual tensor, None of another. Only
    within a dual level there are any (forward_ad._current_level, -1 outside);
    callers look at that first, for asking torch takes 0.5 us."""
    primal, tangent = forward_ad.unpack_dual(x)
    return None if tangent is None else (primal, tangent)


def row_layout(x):
    """x as rows of its last dimension: (x, rows, width, row stride), packed
    first unless it is contiguous or a 2-D tensor with unit column stride."""
    width = x.shape[-1] if x.dim() else 1
    if x.numel() == 0:
        return x, 0, width, width
    if not x.is_contiguous():
        if x.dim() == 2 and x.stride(1) == 1:
            return x, x.shape[0], width, x.stride(0)
        x = x.contiguous()
    return x, x.numel() // width, width, width


def launch(device, what, entry, *arguments):
    """Calls a C entry on the current stream of `device`, with it current."""
    index = device.index
    if index == native.current_device():
        status = entry(*arguments, native.raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = entry(*arguments, native.raw_stream(index))
    if status:
        native.check(status, what)


def _run(x, p, seed, number, address, rows, out=None):
    """The launch, on checked arguments."""
    x, count, width, stride = row_layout(x)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    if count:
        launch(x.device, "dropout", native.library().clad3dgs_dropout, TYPES[x.dtype], count,
               width, x.data_ptr(), stride, out.data_ptr(), width, p, seed, number, address, rows)
    return out


def _check(x, p, seed, offset):
    _require(x.is_cuda, "dropout needs a CUDA tensor")
    _require(x.dtype in TYPES, "dropout takes float32, float16 or bfloat16")
    return check_draw(p, seed, offset, x.device)


def apply(x, p, seed, offset=0, *, rows=False, out=None):
    """The dropout without autograd. `out`: a contiguous tensor like x to write
    into; x itself (contiguous) for a call in place. Its autograd version is
    counted up, so a backward pass that needs its old values is refused."""
    number, address = _check(x, p, seed, offset)
    if out is not None:
        _require(out.device == x.device and out.dtype == x.dtype and out.shape == x.shape
                 and out.is_contiguous(), "out must be a contiguous tensor like x")
        same = out.data_ptr() == x.data_ptr() and x.is_contiguous()
        _require(same or not overlap(x, out), "out may be x itself, but not overlap it otherwise")
    y = _run(x.detach(), p, seed, number, address, bool(rows), out)
    if out is not None and not out.is_inference():
        torch.autograd.graph.increment_version(out)
    return y


def overlap(x, y):
    """Whether the memory between the first and the last element of x meets y's."""
    if x.numel() == 0 or y.numel() == 0:
        return False
    spans = []
    for t in (x, y):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        spans.append((t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()))
    return spans[0][0] < spans[1][1] and spans[1][0] < spans[0][1]


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset, rows):
        number, address = _check(x, p, seed, offset)
        ctx.numbers = p, seed, offset if address is None else None, rows
        if address is not None:
            ctx.save_for_backward(offset)
        return _run(x, p, seed, number, address, rows)

    @staticmethod
    def backward(ctx, grad):
        p, seed, offset, rows = ctx.numbers
        if offset is None:
            offset = ctx.saved_tensors[0]
        elif not torch.is_grad_enabled() and forward_ad._current_level < 0:
            return _run(grad, p, seed, offset, None, rows), None, None, None, None
        return dropout(grad, p, seed, offset, rows=rows), None, None, None, None


def dropout(x, p, seed, offset=0, *, rows=False):
    """x with a share p of its elements (rows=True: of its rows) set to zero and
    the others scaled by 1 / (1 - p); differentiable any number of times, in
    reverse and in forward mode."""
    if forward_ad._current_level >= 0 and (parts := parts_of(x)):  # the map is linear
        return forward_ad.make_dual(*(dropout(t, p, seed, offset, rows=rows) for t in parts))
    if x.requires_grad and torch.is_grad_enabled():
        return _Dropout.apply(x, p, seed, offset, bool(rows))
    number, address = _check(x, p, seed, offset)
    return _run(x, p, seed, number, address, bool(rows))
