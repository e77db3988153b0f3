"""Tables whose rows many Gaussians (or tokens) share: lookup with scaling, the
table's gradient by sorted tokens, and that gradient handed to Adam.

A codebook of SH coefficients, per-view or per-token embeddings: an index per
token names a row of `table` [rows, width].

* `lookup(table, index, scale=..., p=..., seed=..., offset=...)`: the rows, times
  `scale`, with the dropout of `dropout.dropout(out, p, seed, offset)` in the
  same pass; differentiable once in the table.
* `lookup_gradient(grad, index, rows, ...)`: the adjoint, a dense [rows, width].
* `consume_torch_adam(table, first, second, grad, index, ...)`: the adjoint and
  torch-fused Adam on the table in one call, like the SH consume entries; of
  the gradient only the rows that tokens name exist, in a workspace.
* `token_order(index, rows)`: the tokens sorted by row. The two calls above sort
  for themselves unless they are given it; a program whose assignments stay
  the same over many steps sorts once.

Indices are int32 or int64, of any shape. A token equal to `padding_index`
names no row: its output is zero and it gives no gradient. An index outside
[0, rows) is treated the same and sets bit 256 of `_native.fault_status()`
(the calls do not synchronise to look). Sums run in 32-bit floats in a fixed
order: equal inputs give equal bits.

Kernels launch on the current stream of the tensors' device and may be captured
into a graph. (Torch cannot capture any backward pass while an eager autograd
graph over the same leaf is alive: drop its outputs first, or capture
`lookup_gradient`.) Bad arguments raise RuntimeError before anything is
written.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

import _native as native
from consume import check_disjoint
from dropout import TYPES, check_draw, on_device

MOST = 2 ** 31 - 1
_BITS = {torch.int32: 32, torch.int64: 64}


def _require(condition, message):
    if not condition:
        raise RuntimeError(message)


class TokenOrder(NamedTuple):
    """Tokens sorted by the row they name; see `token_order`."""
    pairs: torch.Tensor   # int32 [tokens, 2]: row (`rows` for none), position
    rows: int


def _check_index(index, device):
    _require(index.is_cuda and (device is None or index.device == device),
             "index must be on the tensors' CUDA device")
    _require(index.dtype in _BITS, "index must be int32 or int64")
    _require(index.numel() <= MOST, "at most 2^31 - 1 tokens")
    return index if index.is_contiguous() else index.contiguous()


def _check_padding(padding_index):
    if padding_index is None:
        return 0, 0
    _require(isinstance(padding_index, int) and -2 ** 63 <= padding_index < 2 ** 63,
             "padding_index must be an integer")
    return 1, padding_index


def _check_scale(scale):
    _require(isinstance(scale, (int, float)) and math.isfinite(scale), "scale must be finite")


def _matrix(t, name):
    """t as a matrix with unit column stride: (tensor, rows, width, row stride)."""
    _require(t.is_cuda and t.dtype in TYPES, f"{name} must be CUDA float32, float16 or bfloat16")
    _require(t.dim() == 2, f"{name} must be a matrix")
    if t.stride(1) != 1 and t.shape[1] > 1:
        t = t.contiguous()
    return t, t.shape[0], t.shape[1], t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _bytes(count, device):
    return torch.empty(max(count, 1), dtype=torch.uint8, device=device)


def token_order(index, rows, *, padding_index=None):
    """The tokens of `index` (row-major) sorted by row, for `lookup_gradient` and
    `consume_torch_adam` on a table of `rows` rows."""
    index = _check_index(index, None)
    _require(isinstance(rows, int) and 0 <= rows <= MOST, "rows must be in [0, 2^31)")
    padded, padding = _check_padding(padding_index)
    n, device = index.numel(), index.device
    pairs = torch.empty((n, 2), dtype=torch.int32, device=device)
    if n == 0:
        return TokenOrder(pairs, rows)
    lib = native.library()
    workspace = _bytes(lib.clad3dgs_token_order_workspace(n, rows), device)
    on_device(device, lambda: native.check(lib.clad3dgs_token_order(
        n, rows, index.data_ptr(), _BITS[index.dtype], padded, padding, pairs.data_ptr(),
        workspace.data_ptr(), workspace.numel(), native.stream_handle()), "token order"))
    return TokenOrder(pairs, rows)


def _order_of(index, rows, padding_index, order, tokens, device):
    """The checked order of `tokens` tokens, sorted here if it is not given."""
    if order is None:
        _require(index.numel() == tokens, "grad must have one row per token")
        _require(index.device == device, "index must be on the tensors' CUDA device")
        return token_order(index, rows, padding_index=padding_index)
    _require(isinstance(order, TokenOrder) and order.rows == rows
             and order.pairs.shape[0] == tokens and order.pairs.device == device,
             "the token order belongs to another table, device or number of tokens")
    return order


def _lookup(table, index, scale, padding_index, p, seed, offset):
    table, rows, width, stride = _matrix(table, "table")
    shape = (*index.shape, width)
    index = _check_index(index, table.device)
    _require(rows <= MOST, "at most 2^31 - 1 rows")
    _check_scale(scale)
    padded, padding = _check_padding(padding_index)
    number, address = check_draw(p, seed, offset, table.device)
    out = torch.empty(shape, dtype=table.dtype, device=table.device)
    if out.numel():
        on_device(table.device, lambda: native.check(
            native.library().clad3dgs_embedding_lookup(
                TYPES[table.dtype], index.numel(), rows, width, native.ptr(table), stride,
                index.data_ptr(), _BITS[index.dtype], padded, padding, scale, p, seed, number,
                address, out.data_ptr(), native.stream_handle()), "embedding lookup"))
    return out


def lookup_gradient(grad, index, rows, *, scale=1.0, padding_index=None, p=0.0, seed=0,
                    offset=0, order=None):
    """The table's gradient [rows, width] (grad's type) of a `lookup` with these
    arguments whose output has the gradient `grad` [*index.shape, width]. With
    `order` (from `token_order`), index and padding_index are not read."""
    _require(grad.dim() >= 1, "grad must have one row per token")
    grad, tokens, width, stride = _matrix(grad if grad.dim() == 2
                                          else grad.reshape(-1, grad.shape[-1])
                                          if grad.numel() else
                                          grad.new_empty(0, grad.shape[-1]), "grad")
    _check_scale(scale)
    device = grad.device
    number, address = check_draw(p, seed, offset, device)
    order = _order_of(index, rows, padding_index, order, tokens, device)
    out = torch.empty((rows, width), dtype=grad.dtype, device=device)
    if out.numel() == 0:
        return out
    lib = native.library()
    workspace = _bytes(lib.clad3dgs_embedding_workspace(tokens, rows, width, 0), device)
    on_device(device, lambda: native.check(lib.clad3dgs_embedding_gradient(
        TYPES[grad.dtype], tokens, rows, width, native.ptr(grad), stride,
        native.ptr(order.pairs), scale, p, seed, number, address, out.data_ptr(),
        workspace.data_ptr(), workspace.numel(), native.stream_handle()), "embedding gradient"))
    return out


def consume_torch_adam(table, first, second, grad, index, *, rate, bias1, bias2_sqrt,
                       scale=1.0, padding_index=None, p=0.0, seed=0, offset=0, order=None):
    """Torch-fused Adam (bias1 = 1 - 0.9^t, bias2_sqrt = sqrt(1 - 0.999^t), eps
    1e-15) on `table` and its moments, float32 [rows, width], in place, with the
    gradient that `lookup_gradient` would give in 32 bits. Rows without tokens
    are updated with a zero gradient. Like the other consume entries it does
    not touch step counters or autograd versions."""
    _require(grad.dim() >= 1, "grad must have one row per token")
    grad, tokens, width, stride = _matrix(grad if grad.dim() == 2
                                          else grad.reshape(-1, grad.shape[-1])
                                          if grad.numel() else
                                          grad.new_empty(0, grad.shape[-1]), "grad")
    device = grad.device
    for name, t in (("table", table), ("first", first), ("second", second)):
        _require(t.is_cuda and t.device == device and t.dtype == torch.float32
                 and t.dim() == 2 and t.shape == table.shape and t.is_contiguous(),
                 f"{name} must be contiguous CUDA float32 [rows, width] on grad's device")
    rows = table.shape[0]
    _require(table.shape[1] == width, "grad and table must have the same width")
    _check_scale(scale)
    _require(math.isfinite(rate) and rate >= 0 and 0 < bias1 <= 1 and 0 < bias2_sqrt <= 1,
             "invalid Adam configuration")
    number, address = check_draw(p, seed, offset, device)
    check_disjoint([table, first, second], [grad] if order is None else [grad, order.pairs],
                   "table, moments and gradient must be disjoint")
    order = _order_of(index, rows, padding_index, order, tokens, device)
    if table.numel() == 0:
        return
    lib = native.library()
    workspace = _bytes(lib.clad3dgs_embedding_workspace(tokens, rows, width, 1), device)
    on_device(device, lambda: native.check(lib.clad3dgs_embedding_consume_torch_adam(
        TYPES[grad.dtype], tokens, rows, width, native.ptr(grad), stride,
        native.ptr(order.pairs), scale, p, seed, number, address, table.data_ptr(),
        first.data_ptr(), second.data_ptr(), rate, native.TorchAdamConfig(bias1, bias2_sqrt),
        workspace.data_ptr(), workspace.numel(), native.stream_handle()), "embedding consume"))


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index, scale, padding_index, p, seed, offset, order):
        ctx.numbers = table.shape[0], scale, padding_index, p, seed, order
        tensor = isinstance(offset, torch.Tensor)
        ctx.offset = None if tensor else offset
        ctx.save_for_backward(index, *([offset] if tensor else []))
        return _lookup(table, index, scale, padding_index, p, seed, offset)

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled():
            raise RuntimeError("embedding lookup supports first-order backward only")
        rows, scale, padding_index, p, seed, order = ctx.numbers
        index, *tensor = ctx.saved_tensors
        offset = tensor[0] if tensor else ctx.offset
        return (lookup_gradient(grad, index, rows, scale=scale, padding_index=padding_index,
                                p=p, seed=seed, offset=offset, order=order),
                None, None, None, None, None, None, None)


def lookup(table, index, *, scale=1.0, padding_index=None, p=0.0, seed=0, offset=0, order=None):
    """scale * table[index], of the table's type, shaped [*index.shape, width]; with
    p > 0 through the dropout of (p, seed, offset). `order` (from `token_order`
    of the same index, rows and padding) spares the backward pass its sort."""
    if table.requires_grad and torch.is_grad_enabled():
        if order is not None:
            _order_of(index, table.shape[0], padding_index, order, index.numel(), table.device)
        return _Lookup.apply(table, index, scale, padding_index, p, seed, offset, order)
    return _lookup(table, index, scale, padding_index, p, seed, offset)
