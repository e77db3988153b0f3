"""Tables whose rows many Gaussians (or tokens) share: lookup with scaling, the
table's gradient by sorted tokens, and that gradient handed to Adam.

A codebook of SH coefficients, per-view or per-token embeddings: an index per
token names a row of `table` [rows, width].

* `lookup(table, index, scale=..., p=..., seed=..., offset=...)`: the rows, times
  `scale`, with the dropout of `dropout.dropout(out, p, seed, offset)` in the
  same pass; differentiable in the table, once in reverse mode and in forward
  mode.
* `lookup_gradient(grad, index, rows, ...)`: the adjoint, a dense [rows, width].
* `consume_torch_adam(table, first, second, grad, index, ...)`: the adjoint and
  torch-fused Adam on the table in one call, like the SH consume entries; of
  the gradient only the rows that tokens name exist, in a workspace.
* `token_order(index, rows)`: the tokens sorted by row. The two calls above sort
  for themselves unless they are given it; a program whose assignments stay
  the same over many steps sorts once.

Indices are int32 or int64, of any shape. A token equal to `padding_index`
names no row: its output is zero and it gives no gradient. An index outside
[0, rows) is treated the same and sets bit 256 of `_native.fault_status()` on
the tensors' device (the calls do not synchronise to look; the reader, with
that device current, does). Sums run in 32-bit floats in a fixed order (in 64
bits where the parts of a very long row meet): equal inputs give equal bits.

Kernels launch on the current stream of the tensors' device and may be captured
into a graph. (Torch cannot capture any backward pass while an eager autograd
graph over the same leaf is alive: drop its outputs first, or capture
`lookup_gradient`.) Bad arguments raise RuntimeError before anything is
written.
"""

from __future__ import annotations

import math
from functools import lru_cache
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

import _native as native
from dropout import TYPES, check_draw, launch, parts_of

MOST = 2 ** 31 - 1
_BITS = {torch.int32: 32, torch.int64: 64}
_LARGEST = torch.finfo(torch.float32).max


def _require(condition, message):
    if not condition:
        raise RuntimeError(message)


class TokenOrder(NamedTuple):
    """Tokens sorted by the row they name; see `token_order`."""
    pairs: torch.Tensor   # int32 [tokens, 2]: row (`rows` for none), position
    rows: int


def _index(index, device):
    """The checked index: (tensor, bits)."""
    if not (isinstance(index, torch.Tensor) and index.is_cuda
            and (device is None or index.device == device)):
        raise RuntimeError("index must be a tensor on the others' CUDA device")
    bits = _BITS.get(index.dtype)
    if bits is None:
        raise RuntimeError("index must be int32 or int64")
    if index.numel() > MOST:
        raise RuntimeError("at most 2^31 - 1 tokens")
    return index if index.is_contiguous() else index.contiguous(), bits


def _padding(padding_index):
    if padding_index is None:
        return 0, 0
    _require(isinstance(padding_index, int) and -2 ** 63 <= padding_index < 2 ** 63,
             "padding_index must be an integer")
    return 1, padding_index


def _check_scale(scale, p):
    """p as `check_draw` leaves it."""
    if not (isinstance(scale, (int, float)) and abs(scale) <= 1e38
            and (p == 1 or abs(scale) / (1 - p) <= _LARGEST)):
        raise RuntimeError("scale and scale / (1 - p) must be finite in 32 bits")


def _check_rows(rows):
    _require(isinstance(rows, int) and 0 <= rows <= MOST, "rows must be in [0, 2^31)")


def _matrix(t, name):
    """t as a matrix with unit column stride: (tensor, type, rows, width, row
    stride)."""
    kind = TYPES.get(t.dtype)
    if not (t.is_cuda and kind is not None and t.dim() == 2):
        raise RuntimeError(f"{name} must be a CUDA matrix of float32, float16 or bfloat16")
    rows, width = t.shape
    if t.is_contiguous():
        return t, kind, rows, width, width
    if t.stride(1) != 1 and width > 1:
        t = t.contiguous()
    return t, kind, rows, width, t.stride(0)


def _gradient_matrix(grad):
    """Output gradients [*, width] as a matrix, one row per token."""
    _require(grad.dim() >= 1, "grad must have one row per token")
    if grad.dim() != 2:
        rows = math.prod(grad.shape[:-1])
        grad = grad.reshape(rows, grad.shape[-1])
    return _matrix(grad, "grad")


def token_order(index, rows, *, padding_index=None):
    """The tokens of `index` (row-major) sorted by row, for `lookup_gradient` and
    `consume_torch_adam` on a table of `rows` rows."""
    index, bits = _index(index, None)
    _check_rows(rows)
    padded, padding = _padding(padding_index)
    n = index.numel()
    pairs = index.new_empty((n, 2), dtype=torch.int32)
    if n:
        lib = native.library()
        need = lib.clad3dgs_token_order_workspace(n, rows)
        workspace = index.new_empty(need, dtype=torch.uint8) if need else None
        launch(index.device, "token order", lib.clad3dgs_token_order, n, rows, index.data_ptr(),
               bits, padded, padding, pairs.data_ptr(), native.ptr(workspace), need)
    return TokenOrder(pairs, rows)


def _tokens(index, rows, padding_index, order, count, device):
    """The tokens as the C entries take them (index, bits, has padding, padding,
    order), and the tensor that has to live until the launch."""
    if order is None:
        index, bits = _index(index, device)
        _require(index.numel() == count, "grad must have one row per token")
        return (native.ptr(index), bits, *_padding(padding_index), None), index
    pairs = order.pairs if isinstance(order, TokenOrder) else None
    _require(pairs is not None and order.rows == rows and pairs.shape == (count, 2)
             and pairs.device == device and pairs.dtype == torch.int32 and pairs.is_contiguous(),
             "the token order belongs to another table, device or number of tokens")
    return (None, 0, 0, 0, native.ptr(pairs)), pairs


@lru_cache(maxsize=4096)
def _workspace_bytes(count, rows, width, consume, ordered):
    return native.library().clad3dgs_embedding_workspace(count, rows, width, consume, ordered)


def _workspace(count, rows, width, consume, ordered, like):
    """A call's workspace: (tensor or None, address or None, bytes)."""
    need = _workspace_bytes(count, rows, width, consume, ordered)
    if need == 0:
        return None, None, 0
    workspace = like.new_empty(need, dtype=torch.uint8)
    return workspace, workspace.data_ptr(), need


def _lookup(table, index, scale, padding_index, p, seed, offset):
    table, kind, rows, width, stride = _matrix(table, "table")
    device = table.device
    index, bits = _index(index, device)
    shape = (*index.shape, width)
    _check_rows(rows)
    padded, padding = _padding(padding_index)
    number, address = check_draw(p, seed, offset, device)
    _check_scale(scale, p)
    out = table.new_empty(shape)
    if out.numel():
        launch(device, "embedding lookup", native.library().clad3dgs_embedding_lookup, kind,
               index.numel(), rows, width, table.data_ptr(), stride, index.data_ptr(), bits,
               padded, padding, scale, p, seed, number, address, out.data_ptr())
    return out


def lookup_gradient(grad, index, rows, *, scale=1.0, padding_index=None, p=0.0, seed=0,
                    offset=0, order=None):
    """The table's gradient [rows, width] (grad's type) of a `lookup` with these
    arguments whose output has the gradient `grad` [*index.shape, width]. With
    `order` (from `token_order`), index and padding_index are not read. Not
    recorded for reverse mode (its result does not require grad); a tangent in
    forward mode goes through."""
    if forward_ad._current_level >= 0 and (parts := parts_of(grad)):  # as in lookup
        how = dict(scale=scale, padding_index=padding_index, p=p, seed=seed, offset=offset,
                   order=order)
        return forward_ad.make_dual(*(lookup_gradient(t, index, rows, **how) for t in parts))
    grad, kind, count, width, stride = _gradient_matrix(grad)
    device = grad.device
    _check_rows(rows)
    number, address = check_draw(p, seed, offset, device)
    _check_scale(scale, p)
    tokens, alive = _tokens(index, rows, padding_index, order, count, device)
    out = grad.new_empty((rows, width))
    if out.numel():
        space = _workspace(count, rows, width, 0, order is not None, out)
        launch(device, "embedding gradient", native.library().clad3dgs_embedding_gradient, kind,
               count, rows, width, grad.data_ptr(), stride, *tokens, scale, p, seed, number,
               address, out.data_ptr(), space[1], space[2])
    return out


def consume_torch_adam(table, first, second, grad, index, *, rate, bias1, bias2_sqrt,
                       scale=1.0, padding_index=None, p=0.0, seed=0, offset=0, order=None):
    """Torch-fused Adam (bias1 = 1 - 0.9^t, bias2_sqrt = sqrt(1 - 0.999^t), eps
    1e-15) on `table` and its moments, float32 [rows, width], in place, with the
    gradient that `lookup_gradient` would give in 32 bits. Rows without tokens
    are updated with a zero gradient. Like the other consume entries it does
    not touch step counters or autograd versions."""
    grad, kind, count, width, stride = _gradient_matrix(grad)
    device = grad.device
    _require(table.dim() == 2, "table must be a matrix")
    state = (table, first, second)
    shape = table.shape
    rows = shape[0]
    for t in state:
        _require(t.dtype == torch.float32 and t.device == device and t.shape == shape
                 and t.is_contiguous(), "table and moments must be contiguous CUDA float32 "
                 "[rows, width] on grad's device")
    _require(shape[1] == width, "table and grad must have the same width")
    _check_rows(rows)
    config = native.TorchAdamConfig(bias1, bias2_sqrt)  # (rounds to 32 bits)
    _require(math.isfinite(rate) and rate >= 0 and bias1 <= 1 and bias2_sqrt <= 1
             and config.bias1 > 0 and config.bias2_sqrt > 0, "invalid Adam configuration")
    number, address = check_draw(p, seed, offset, device)
    _check_scale(scale, p)
    tokens, alive = _tokens(index, rows, padding_index, order, count, device)
    size = 4 * rows * width
    spans = [(t.data_ptr(), t.data_ptr() + size) for t in state]
    read = [(grad.data_ptr(), grad.data_ptr()
             + ((count - 1) * stride + width) * grad.element_size()),
            (alive.data_ptr(), alive.data_ptr() + alive.numel() * alive.element_size())
            ] if count else []
    _require(not size or not any(
        a < d and c < b for k, (a, b) in enumerate(spans) for c, d in spans[k + 1:] + read),
        "table, moments, gradient and indices must be disjoint")
    if size:
        space = _workspace(count, rows, width, 1, order is not None, table)
        launch(device, "embedding consume", native.library().clad3dgs_embedding_consume_torch_adam,
               kind, count, rows, width, grad.data_ptr(), stride, *tokens, scale, p, seed, number,
               address, spans[0][0], spans[1][0], spans[2][0], rate,
               config, space[1], space[2])


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index, scale, padding_index, p, seed, offset, order):
        out = _lookup(table, index, scale, padding_index, p, seed, offset)
        tensor = isinstance(offset, torch.Tensor)
        ctx.numbers = (table.shape[0], scale, padding_index, p, seed, None if tensor else offset,
                       order)
        # An order's pairs are only saved to have their version checked (inference
        # tensors have none).
        ctx.save_for_backward(index, offset if tensor else None, None if order is None
                              or order.pairs.is_inference() else order.pairs)
        return out

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled():
            raise RuntimeError("embedding lookup supports first-order backward only")
        rows, scale, padding_index, p, seed, offset, order = ctx.numbers
        index, tensor, _ = ctx.saved_tensors
        return (lookup_gradient(grad, index, rows, scale=scale, padding_index=padding_index, p=p,
                                seed=seed, offset=offset if tensor is None else tensor, order=order),
                None, None, None, None, None, None, None)


def lookup(table, index, *, scale=1.0, padding_index=None, p=0.0, seed=0, offset=0, order=None):
    """scale * table[index], of the table's type, shaped [*index.shape, width]; with
    p > 0 through the dropout of (p, seed, offset). `order` (from `token_order`
    of the same index, rows and padding) spares the backward pass its sort."""
    if forward_ad._current_level >= 0 and (parts := parts_of(table)):  # linear in the table
        how = dict(scale=scale, padding_index=padding_index, p=p, seed=seed, offset=offset,
                   order=order)
        return forward_ad.make_dual(*(lookup(t, index, **how) for t in parts))
    if table.requires_grad and torch.is_grad_enabled():
        if order is not None:
            _require(table.dim() == 2 and isinstance(index, torch.Tensor),
                     "table must be a matrix and index a tensor")
            _tokens(None, table.shape[0], None, order, index.numel(), table.device)
        return _Lookup.apply(table, index, scale, padding_index, p, seed, offset, order)
    return _lookup(table, index, scale, padding_index, p, seed, offset)
