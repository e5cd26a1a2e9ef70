"""Dropout whose mask is a function of a counter and is never stored.

Element ``e`` of the mask is kept when word ``e % 4`` of Philox4x32-10 (Salmon et al., SC 2011) at counter
``(e // 4, offset)`` under key ``seed`` is at least ``floor(p 2^32)``; what is kept is divided by ``1 - p``, what
is dropped is zero whatever it was. The backward pass forms the mask again from the same two numbers,
so the result is the same on every device, and a recomputed forward pass repeats its mask.
``shared`` dimensions share one mask entry (all coefficients of a node's channel, say), in one pass
over ``x``. CUDA tensors (float32, float64) run ``csrc/dropout.cu``, others the formula.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch
from torch import Tensor, nn
from torch.autograd import Function

from .. import _ext

Rng = Union[Tensor, Tuple[int, int]]
_LOW = 0xFFFFFFFF


def _multiply(m: int, x: Tensor) -> Tuple[Tensor, Tensor]:
    """High and low word of ``m x`` (both below 2^32, held in int64)."""
    low = m * (x & 0xFFFF)
    high = m * (x >> 16) + (low >> 16)
    return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)


def philox(blocks: Tensor, rng: Tensor) -> Tensor:
    """``(len(blocks), 4)`` words (int64, below 2^32) of the counters ``(block, offset)``, ``rng = (seed, offset)``."""
    seed, offset = rng[0], rng[1]
    zero = torch.zeros_like(blocks)
    c = [blocks & _LOW, (blocks >> 32) & _LOW, zero + (offset & _LOW), zero + ((offset >> 32) & _LOW)]
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        h0, l0 = _multiply(0xD2511F53, c[0])
        h1, l1 = _multiply(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return torch.stack(c, 1)


def _split(shape: torch.Size, shared: Tuple[int, ...]) -> Tuple[int, int, int]:
    """``(outer, shared, inner)`` sizes around the shared dimensions, which must be neighbours."""
    outer = common = inner = 1
    stage = 0
    for d, size in enumerate(shape):
        if size == 1:
            continue
        if d in shared:
            if stage == 2:
                raise ValueError(f"the shared dimensions {shared} of shape {tuple(shape)} must be neighbours")
            stage, common = 1, common * size
        elif stage == 0:
            outer *= size
        else:
            stage, inner = 2, inner * size
    return (1, 1, outer) if common == 1 else (outer, common, inner)


def _formula(x: Tensor, p: float, rng: Tensor, sizes: Tuple[int, int, int]) -> Tensor:
    outer, common, inner = sizes
    n = outer * inner
    words = philox(torch.arange((n + 3) // 4, device=x.device), rng).reshape(-1)[:n]
    keep = (words >= int(p * 2.0 ** 32)).view(outer, 1, inner)
    factor = 1.0 / (1.0 - p) if p < 1.0 else 0.0
    return torch.where(keep, x.reshape(outer, common, inner) * factor, 0.0).view(x.shape)


class _Dropout(Function):
    """The formula with the mask formed again in the backward pass."""

    @staticmethod
    def forward(ctx, x, p, rng, sizes):
        ctx.save_for_backward(rng)
        ctx.p, ctx.sizes = p, sizes
        return _formula(x, p, rng, sizes)

    @staticmethod
    def backward(ctx, g):
        return _Dropout.apply(g, ctx.p, ctx.saved_tensors[0], ctx.sizes), None, None, None


_KERNEL = None


def _kernel():
    global _KERNEL
    if _KERNEL is None:
        mod = _ext.ops()
        if not hasattr(mod, "counter_dropout"):
            raise RuntimeError("xnn_b200 extension without the dropout kernel: rebuild it (xnn_b200.build)")
        _KERNEL = mod.counter_dropout
    return _KERNEL


def counter_dropout(x: Tensor, p: float, rng: Rng, shared: Sequence[int] = ()) -> Tensor:
    """``x`` with entries dropped with probability ``p``, the others divided by ``1 - p``; differentiable to any
    order in reverse mode. ``rng = (seed, offset)``: two integers, or an int64 tensor of them on ``x``'s device (it is read
    when the kernels run, and again in the backward pass: advance a copy, not the tensor itself).
    ``shared``: neighbouring dimensions over which the mask is the same."""
    if not isinstance(rng, Tensor):
        rng = torch.tensor([int(rng[0]), int(rng[1])], dtype=torch.int64, device=x.device)
    if x.is_cuda:                                # the arguments are checked there
        return _kernel()(x, p, rng, shared)
    if x.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"counter_dropout takes float32 or float64, got {x.dtype}")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"the dropout probability must be in [0, 1], got {p}")
    if any(not -x.dim() <= int(d) < x.dim() for d in shared):
        raise ValueError(f"shared dimensions {tuple(shared)} of a tensor with {x.dim()} dimensions")
    if rng.dtype != torch.int64 or rng.shape != (2,) or rng.device != x.device:
        raise ValueError(f"rng must be two int64 numbers (seed, offset) on {x.device}")
    sizes = _split(x.shape, tuple(int(d) % x.dim() for d in shared))
    return x.clone() if 0 in x.shape else _Dropout.apply(x, p, rng, sizes)


class CounterDropout(nn.Module):
    """:func:`counter_dropout` in training mode with its own seed (drawn from PyTorch's generator when
    omitted) and an offset that each call advances. The two numbers live on the module's device, so a
    captured training step draws a new mask at every replay. Processes that start from one seed draw the
    same masks, each for its own rows, unless :meth:`set_rank` tells them apart (the trainer does). The state dict
    does not hold the numbers: a run that starts again draws from its seed's first mask on. Inside an activation checkpoint it is refused: the recomputed pass
    would meet another offset."""

    def __init__(self, p: float, shared: Sequence[int] = (), seed: Optional[int] = None):
        super().__init__()
        if not 0.0 <= float(p) <= 1.0:
            raise ValueError(f"the dropout probability must be in [0, 1], got {p}")
        self.p, self.shared = float(p), tuple(int(d) for d in shared)
        seed = int(torch.randint(0, 2 ** 62, ())) if seed is None else int(seed)
        self.register_buffer("rng", torch.tensor([seed, 0], dtype=torch.int64), persistent=False)

    def set_rank(self, rank: int) -> None:
        """Masks of rank ``rank``'s own: the offset counts from ``rank * 2^40`` on (rank 0 as without ranks)."""
        self.rng[1] = (self.rng[1] & ((1 << 40) - 1)) | (int(rank) << 40)

    def forward(self, x: Tensor) -> Tensor:
        if not self.training or self.p == 0.0:
            return x
        if torch._C._current_graph_task_id() != -1:
            raise RuntimeError("CounterDropout in a forward pass that a backward pass runs again (activation checkpointing) "
                               "would draw another mask: call counter_dropout with the numbers of the first pass")
        now = self.rng.clone()
        self.rng[1] += 1
        return counter_dropout(x, self.p, now, self.shared)

    def extra_repr(self) -> str:
        return f"p={self.p}, shared={self.shared}"
