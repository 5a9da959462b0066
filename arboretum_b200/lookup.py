# coding: utf-8
"""Rows of a learned table by token: the lookup with scaling and its gradient.

A forest of T trees with L leaves each is a table of T * L rows; a row of the data set is a bag
of T tokens (``Garden.leaf_tokens``) and its prediction the scaled sum of the rows they name.
With one token a bag and wide rows this is the embedding of category codes or of leaves.

The functions take torch CUDA tensors, work on the current stream of the tensors' device and only
enqueue work: no synchronisation, so they can be captured into a CUDA graph.  They are not recorded
by autograd: ``embedding_grad`` is the backward pass.
"""
import ctypes
import functools

import torch

from .core import _LIB, _call_and_throw_if_error

__all__ = ["embedding", "embedding_grad", "token_order", "TokenOrder"]

_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_TOKEN_BYTES = {torch.int32: 4, torch.int64: 8}


def _tensor(x, name):
    if not isinstance(x, torch.Tensor):
        raise TypeError("%s must be a torch tensor" % name)
    return x


def _float_type(x, name):
    code = _TYPE.get(x.dtype)
    if code is None:
        raise TypeError("%s must be float32, bfloat16 or float16, not %s" % (name, x.dtype))
    return code


def _no_grad(x, name):
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s requires grad, which is not recorded here: pass it detached and use "
                         "embedding_grad for the backward pass" % name)


def _one_device(first, **others):
    """The device index all tensors share."""
    if first.device.type != "cuda":
        raise ValueError("the tensors must be CUDA tensors")
    for name, x in others.items():
        if x is not None and x.device != first.device:
            raise ValueError("%s is on %s, the others are on %s" % (name, x.device, first.device))
    return first.device.index


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _extent(x):
    """[first, last) byte a tensor may touch."""
    if x.numel() == 0:
        return 0, 0
    at = x.data_ptr()
    return at, at + (sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1) * x.element_size()


def _apart(out, name, x):
    """Refuses an output that shares memory with an input."""
    a, b = _extent(out), _extent(x)
    if a[0] < b[1] and b[0] < a[1]:
        raise ValueError("out shares memory with %s" % name)


def _bags(tokens, pooled):
    """(tokens, bags, tokens a bag, bag stride, token stride)"""
    _tensor(tokens, "tokens")
    if tokens.dtype not in _TOKEN_BYTES:
        raise TypeError("tokens must be int32 or int64, not %s" % tokens.dtype)
    if pooled:
        if tokens.dim() != 2:
            raise ValueError("pooled tokens must have two dimensions: bags x tokens")
        return tokens, tokens.shape[0], tokens.shape[1], tokens.stride(0), tokens.stride(1)
    flat = tokens if tokens.dim() == 1 else tokens.reshape(-1)
    return flat, flat.shape[0], 1, flat.stride(0), 0


def _out(out, shape, dtype, out_dtype, device):
    """The output tensor as a matrix of rows, and what the caller gets."""
    if out is None:
        out = torch.empty(shape, dtype=out_dtype or dtype, device=device)
        rows = out
    else:
        _tensor(out, "out")
        if tuple(out.shape) != tuple(shape):
            raise ValueError("out must have shape %s, not %s" % (tuple(shape), tuple(out.shape)))
        if out_dtype is not None and out.dtype != out_dtype:
            raise TypeError("out is %s, out_dtype is %s" % (out.dtype, out_dtype))
        _no_grad(out, "out")
        rows = out
    if rows.dim() != 2:
        if not rows.is_contiguous():
            raise ValueError("an out of more than two dimensions must be contiguous")
        rows = rows.view(-1, shape[-1]) if rows.numel() else rows.reshape(0, shape[-1])
    if rows.numel() and rows.shape[1] > 1 and rows.stride(1) != 1:
        raise ValueError("the last dimension of out must be contiguous")
    if rows.dtype != dtype and rows.dtype != torch.float32 or rows.dtype not in _TYPE:
        raise TypeError("out must be %s or float32, not %s" % (dtype, rows.dtype))
    return rows, out


def embedding(tokens, table, scale=1.0, pooled=False, out=None, out_dtype=None):
    """Rows of ``table`` named by ``tokens``, times ``scale``.

    tokens: int32 or int64.  ``pooled=False``: any shape, the result has that shape and one more
    dimension; ``pooled=True``: bags x tokens with any strides, the rows of a bag are summed.
    table: rows x columns, float32 / bfloat16 / float16, columns contiguous, rows any distance
    apart.  A token outside [0, rows) (-1, say) is an empty slot: it adds nothing, and a bag of
    empty slots gives zeros.  Sums are held in float32 and rounded once, to the table's type or
    float32 (``out`` / ``out_dtype``).
    """
    _tensor(table, "table")
    kind = _float_type(table, "table")
    if table.dim() != 2:
        raise ValueError("table must have two dimensions: rows x columns")
    if table.numel() and table.shape[1] > 1 and table.stride(1) != 1:
        raise ValueError("the columns of table must be contiguous")
    _no_grad(table, "table")
    flat, bags, per_bag, bag_stride, token_stride = _bags(tokens, pooled)
    device = _one_device(table, tokens=tokens, out=out)
    rows, dim = table.shape
    given = out is not None
    matrix, out = _out(out, (bags, dim) if pooled else tokens.shape + (dim,), table.dtype, out_dtype, table.device)
    if given:
        _apart(out, "table", table)
        _apart(out, "tokens", tokens)
    _call_and_throw_if_error(_LIB.AEmbedding(
        table.data_ptr(), kind, rows, dim, table.stride(0), flat.data_ptr(), _TOKEN_BYTES[flat.dtype], bags, per_bag,
        bag_stride, token_stride, scale, matrix.data_ptr(), _TYPE[matrix.dtype], matrix.stride(0), device,
        _stream(device)))
    return out


@functools.lru_cache(maxsize=1024)
def _order_bytes(bags, per_bag, rows):
    order, scratch = ctypes.c_int64(0), ctypes.c_int64(0)
    _call_and_throw_if_error(_LIB.ATokenOrderBytes(bags, per_bag, rows, ctypes.byref(order), ctypes.byref(scratch)))
    return order.value, scratch.value


@functools.lru_cache(maxsize=1024)
def _grad_bytes(bags, per_bag, rows, dim, device):
    scratch = ctypes.c_int64(0)
    _call_and_throw_if_error(_LIB.AEmbeddingGradBytes(bags, per_bag, rows, dim, device, ctypes.byref(scratch)))
    return scratch.value


def _memory(size, device):
    return torch.empty(max(256, size), dtype=torch.uint8, device=device)


class TokenOrder(object):
    """The bags sorted by the tokens that name them (``token_order``): what ``embedding_grad``
    sorts anew in every call that is given tokens."""

    def __init__(self, tokens, rows, pooled=False):
        flat, self.bags, self.per_bag, bag_stride, token_stride = _bags(tokens, pooled)
        self.rows = int(rows)
        self.pooled = bool(pooled)
        self.shape = tuple(tokens.shape)
        order_bytes, scratch_bytes = _order_bytes(self.bags, self.per_bag, self.rows)
        device = _one_device(tokens)
        self.device = tokens.device
        self._stream = _stream(device)
        self._data = _memory(order_bytes, self.device)
        scratch = _memory(scratch_bytes, self.device)
        _call_and_throw_if_error(_LIB.ATokenOrder(
            flat.data_ptr(), _TOKEN_BYTES[flat.dtype], self.bags, self.per_bag, bag_stride, token_stride, self.rows,
            self._data.data_ptr(), scratch.data_ptr(), device, self._stream))

    def _use(self, stream):
        """Address of the order for a call on ``stream``."""
        if stream != self._stream:  # its memory must not be handed out again before that stream is done
            self._data.record_stream(torch.cuda.current_stream(self.device))
        return self._data.data_ptr()


def token_order(tokens, rows, pooled=False):
    """Sorts ``tokens`` once for several ``embedding_grad`` calls: tokens that stay the same from
    step to step, like the leaves a forest assigns.  ``rows``: of the table the tokens index."""
    return TokenOrder(tokens, rows, pooled)


def embedding_grad(grad, tokens, rows, scale=1.0, pooled=False, out=None, out_dtype=None, accumulate=False):
    """Gradient of ``embedding`` with respect to its table: rows x columns.

    grad: the gradient of its result (float32 / bfloat16 / float16; broadcast rows are read in
    place, other layouts whose columns are not contiguous are copied).  tokens: the same tokens, or
    a ``TokenOrder`` of them.  The result has grad's type or float32 (``out`` / ``out_dtype``);
    rows that no token names are zero, or stay as they are with ``accumulate=True``, which adds to
    ``out``.  Sums are held in float32, in an order that only the tokens decide: equal inputs give
    equal bits.
    """
    _tensor(grad, "grad")
    kind = _float_type(grad, "grad")
    _no_grad(grad, "grad")
    order = tokens if isinstance(tokens, TokenOrder) else None
    if order is None:
        flat, bags, per_bag, bag_stride, token_stride = _bags(tokens, pooled)
        shape = tuple(tokens.shape)
    else:
        if order.rows != rows:
            raise ValueError("the order was made for %d rows, not %d" % (order.rows, rows))
        shape, per_bag, bags, pooled = order.shape, order.per_bag, order.bags, order.pooled
    if grad.dim() < 1 or tuple(grad.shape[:-1]) != ((bags,) if pooled else shape):
        raise ValueError("grad must have shape %s x columns, not %s" % ((bags,) if pooled else shape, tuple(grad.shape)))
    dim = grad.shape[-1]
    if accumulate and out is None:
        raise ValueError("accumulate needs the gradient to add to: out")
    # bytes first: a size out of range is refused before anything is allocated
    order_bytes, sort_bytes = _order_bytes(bags, per_bag, rows)
    device = _one_device(grad, tokens=tokens, out=out)
    scratch_bytes = _grad_bytes(bags, per_bag, rows, dim, device)
    if grad.dim() != 2:
        grad = grad.reshape(-1, dim) if grad.numel() else grad.reshape(bags, dim)
    if grad.numel() and dim > 1 and grad.stride(1) != 1:
        grad = grad.contiguous()
    given = out is not None
    matrix, out = _out(out, (rows, dim), grad.dtype, out_dtype, grad.device)
    if given:
        _apart(out, "grad", grad)
        if order is None:
            _apart(out, "tokens", tokens)
    stream = _stream(device)
    if order is None:
        memory = _memory(order_bytes + max(sort_bytes, scratch_bytes), grad.device)
        order_at = memory.data_ptr()
        scratch_at = order_at + order_bytes
        _call_and_throw_if_error(_LIB.ATokenOrder(
            flat.data_ptr(), _TOKEN_BYTES[flat.dtype], bags, per_bag, bag_stride, token_stride, rows, order_at,
            scratch_at, device, stream))
    else:
        memory = _memory(scratch_bytes, grad.device)
        order_at, scratch_at = order._use(stream), memory.data_ptr()
    _call_and_throw_if_error(_LIB.AEmbeddingGrad(
        grad.data_ptr(), kind, bags, dim, grad.stride(0), order_at, per_bag, rows, scale, matrix.data_ptr(),
        _TYPE[matrix.dtype], matrix.stride(0), int(accumulate), scratch_at, device, stream))
    return out
