"""Rows of a table by id (element, element pair, bond type), with a scale and a gradient by sorted ids.

``out = scale table[ids]``; an id outside the table (a padded atom's -1) gives a zero row and receives no
gradient. The table's gradient sums the rows of each id in the order of a stable sort, so it is the same
from run to run and needs no atomics: with a handful of elements in a batch nearly all rows meet in a
few table rows, and its error does not grow with their number. The two functions are each other's adjoints and differentiate to any order (reverse mode). CUDA tensors
(float32, float64) run ``csrc/embedding.cu``, others PyTorch's indexing.
"""
from __future__ import annotations

import torch
from torch import Tensor, nn
from torch.autograd import Function

from .. import _ext


_KERNEL = None


def _kernel():
    global _KERNEL
    if _KERNEL is None:
        mod = _ext.ops()
        if not hasattr(mod, "embedding_lookup"):
            raise RuntimeError("xnn_b200 extension without the lookup kernels: rebuild it (xnn_b200.build)")
        _KERNEL = mod.embedding_lookup
    return _KERNEL


class _Lookup(Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale = table.shape[0], scale
        if table.shape[0] == 0:
            return table.new_zeros(tuple(ids.shape) + (table.shape[1],))
        on = (ids >= 0) & (ids < table.shape[0])
        return torch.where(on[..., None], scale * table[torch.where(on, ids, 0)], 0.0)

    @staticmethod
    def backward(ctx, g):
        return _LookupGrad.apply(g, ctx.saved_tensors[0], ctx.rows, ctx.scale), None, None


class _LookupGrad(Function):
    @staticmethod
    def forward(ctx, g, ids, rows, scale):
        ctx.save_for_backward(ids)
        ctx.scale = scale
        on = (ids >= 0) & (ids < rows)
        total = g.new_zeros(rows, g.shape[-1], dtype=torch.float64).index_add_(0, ids[on].long(), g[on].double())
        return (scale * total).to(g.dtype)

    @staticmethod
    def backward(ctx, t):
        return _Lookup.apply(t, ctx.saved_tensors[0], ctx.scale), None, None, None


def embedding_lookup(table: Tensor, ids: Tensor, scale: float = 1.0) -> Tensor:
    """``scale * table[ids]``, ``(*ids.shape, width)``, with zero rows for ids outside ``0 .. rows - 1``."""
    if table.is_cuda:                            # the arguments are checked there
        return _kernel()(table, ids, scale)
    if table.dim() != 2 or table.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"table must be (rows, width) float32 or float64, got {table.dtype} {tuple(table.shape)}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"ids must be int64 or int32, got {ids.dtype}")
    if ids.device != table.device:
        raise ValueError(f"table on {table.device}, ids on {ids.device}")
    return _Lookup.apply(table, ids, float(scale))


class ScaledEmbedding(nn.Embedding):
    """``nn.Embedding`` (same parameter and initialisation) through :func:`embedding_lookup`, times ``scale``."""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: float = 1.0, **kwargs):
        for name in ("padding_idx", "max_norm", "sparse", "scale_grad_by_freq"):
            if kwargs.get(name) is not None and kwargs[name] is not False:      # padding_idx=0 is a request too
                raise ValueError(f"ScaledEmbedding does not take {name}")
        super().__init__(num_embeddings, embedding_dim, **kwargs)
        self.scale = float(scale)

    def forward(self, ids: Tensor) -> Tensor:
        return embedding_lookup(self.weight, ids, self.scale)
