# coding: utf-8
"""Rows of a learned table by token: the lookup with scaling and its gradient.

A forest of T trees with L leaves each is a table of T * L rows; a row of the data set is a bag
of T tokens (``Garden.leaf_tokens``) and its prediction the scaled sum of the rows they name.
With one token a bag and wide rows this is the embedding of category codes or of leaves.

The functions take torch CUDA tensors, work on the current stream of the tensors' device and only
enqueue work: no synchronisation, so they can be captured into a CUDA graph.  They are not recorded
by autograd: ``embedding_grad`` is the backward pass; tensors that require grad or carry a forward-mode
tangent are refused, and so are calls while torch traces them.
"""
import torch  # noqa: F401  (_tensors.so needs its libraries)

from .core import ArboretumError

try:
    from . import _tensors
except ImportError as e:
    raise ImportError("arboretum_b200/_tensors.so does not load (%s): build it with `python arboretum_b200/build.py`" % e)

_tensors.set_error(ArboretumError)

__all__ = ["embedding", "embedding_grad", "token_order", "TokenOrder"]


def embedding(tokens, table, scale=1.0, pooled=False, out=None, out_dtype=None):
    """Rows of ``table`` named by ``tokens``, times ``scale`` (finite).

    tokens: int32 or int64.  ``pooled=False``: any shape, the result has that shape and one more
    dimension; ``pooled=True``: bags x tokens with any strides, the rows of a bag are summed.
    table: rows x columns, float32 / bfloat16 / float16, columns contiguous, rows any distance
    apart.  A token outside [0, rows) (-1, say) is an empty slot: it adds nothing, and a bag of
    empty slots gives zeros.  Sums are held in float32 and rounded once, to the table's type or
    float32 (``out`` / ``out_dtype``).
    """
    return _tensors.embedding(tokens, table, scale, pooled, out, out_dtype)


class TokenOrder(object):
    """The bags sorted by the tokens that name them (``token_order``): what ``embedding_grad``
    sorts anew in every call that is given tokens."""

    def __init__(self, tokens, rows, pooled=False):
        self._order = _tensors.token_order(tokens, rows, pooled)
        self.rows = int(rows)
        self.pooled = bool(pooled)
        self.shape = tuple(tokens.shape)


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
    ``out``.  Sums are held in float32 or more, in an order that only the tokens decide: equal inputs
    give equal bits.  Tokens are sorted in every call, which takes many times as long as the sums where
    bags are long (128 tokens for each of a million bags: 6.9 ms, the sums 0.1): tokens that come again
    are worth a ``token_order``.
    """
    if isinstance(tokens, TokenOrder):
        if tokens.rows != rows:
            raise ValueError("the order was made for %d rows, not %d" % (tokens.rows, rows))
        return _tensors.embedding_grad(grad, tokens.shape, rows, scale, tokens.pooled, out, out_dtype, accumulate,
                                       tokens._order)
    return _tensors.embedding_grad(grad, tokens, rows, scale, pooled, out, out_dtype, accumulate, None)
