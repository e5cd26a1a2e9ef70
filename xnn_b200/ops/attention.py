"""Softmax attention over the atoms of each structure of a packed batch.

The atoms of a batch are rows of ``q (N, H, D)`` and ``k, v (N, Hk, D)`` (``Hk`` divides ``H``; consecutive
query heads share a key head), and ``ptr (B + 1)`` says where each structure starts. With
``S = scale q k^T`` over the structure's atoms that ``key_mask`` allows,

    ``O = softmax(S) V``

and nothing of the size of ``S`` is stored: the backward pass forms the probabilities again from one
number a row, and so does the backward pass of that, which training on forces needs (forces are a first
derivative, the loss takes a second one). A row without an allowed key gives zeros and no gradient, and
so do rows before the first and behind the last structure. What a mask hides (NaN included) reaches
neither outputs nor gradients, and no structure's values reach another's.

On CUDA tensors (float32, float64; ``D <= 128``) this package's sm_100a kernels run
(``csrc/attention.cu``), on the calling thread's current stream, without a host synchronisation, so
they can be captured into a CUDA graph; results do not depend on the launch (no atomics). float32 structures of
more than 32 atoms run as products of exact parts, so an infinite operand that no mask hides gives NaN. On the
CPU the padded formula runs, differentiable to any order.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from .. import _ext
from .gemm import _status

_TYPES = (torch.float32, torch.float64)


_KERNEL = None


def _kernel():
    global _KERNEL
    if _KERNEL is None:
        mod = _ext.ops()
        if not hasattr(mod, "structure_attention"):
            raise RuntimeError("xnn_b200 extension without the attention kernels: rebuild it (xnn_b200.build)")
        _KERNEL = mod.structure_attention
    return _KERNEL


def _formula(q: Tensor, k: Tensor, v: Tensor, ptr: Tensor, mask: Optional[Tensor], scale: float) -> Tensor:
    """The same over padded structures ``(B, H, L, D)``."""
    n, heads, _ = q.shape
    length = (ptr[1:] - ptr[:-1]).max() if ptr.numel() > 1 else 0
    if not torch.jit.is_tracing():              # a trace keeps the length of its own inputs' structures
        length = int(length)
    out = q.new_zeros(n, heads, q.shape[2])
    if n == 0 or length == 0:
        return out + (q[:0].sum() + k[:0].sum() + v[:0].sum())      # zero, with a graph
    slot = ptr[:-1, None] + torch.arange(length, device=q.device)
    on = slot < ptr[1:, None]
    row = slot.clamp(max=n - 1)
    keys = on if mask is None else on & mask[row]

    def pad(t, valid):
        return torch.where(valid[..., None, None], t[row], 0.0).transpose(1, 2)

    def widen(t):
        return t.repeat_interleave(heads // t.shape[1], 1)
    qp, kp, vp = pad(q, on), widen(pad(k, keys)), widen(pad(v, keys))
    allowed = keys[:, None, None, :]
    s = torch.where(allowed, scale * (qp @ kp.transpose(2, 3)), float("-inf"))
    top = s.detach().amax(-1, keepdim=True)
    e = torch.where(allowed, torch.exp(s - torch.where(torch.isneginf(top), 0.0, top)), 0.0)
    total = e.sum(-1, keepdim=True)
    o = (e / torch.where(total > 0, total, 1.0)) @ vp
    return out.index_put((slot[on],), o.transpose(1, 2)[on])


def structure_attention(q: Tensor, k: Tensor, v: Tensor, ptr: Tensor, max_len: Optional[int] = None,
                        scale: Optional[float] = None, key_mask: Optional[Tensor] = None) -> Tensor:
    """``softmax(scale q k^T) v`` within each structure, ``(N, H, D)``.

    ``ptr``: int64 ``(structures + 1)`` first rows of the structures (ascending; structures may be empty,
    rows outside ``ptr[0] .. ptr[-1]`` belong to none). ``max_len``: no structure has more atoms
    (``N`` when omitted; a smaller bound lets short structures take the kernels made for them; where a structure
    exceeds it, the CPU refuses and on CUDA its gradients are NaN unless they are right). ``scale``: ``D ** -0.5`` when omitted. ``key_mask``: bool ``(N)``, false
    for atoms that nobody attends to. Differentiable twice on CUDA, to any order (and in forward mode) on
    the CPU; what CUDA has no derivative for raises an error."""
    if q.is_cuda:                                # the arguments are checked there
        return _kernel()(q, k, v, ptr, max_len, scale, key_mask, _status(q.device))
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 3:
            raise ValueError(f"{name} must be (atoms, heads, width), got {tuple(t.shape)}")
        if t.dtype not in _TYPES or t.dtype != q.dtype or t.device != q.device:
            raise TypeError(f"q, k and v must all be float32 or all float64 on one device, {name} is {t.dtype} on {t.device}")
    n, h, d = q.shape
    if k.shape != v.shape or k.shape[0] != n or k.shape[2] != d:
        raise ValueError(f"k and v must be ({n}, key heads, {d}), got {tuple(k.shape)} and {tuple(v.shape)}")
    if h < 1 or d < 1 or k.shape[1] < 1 or h % k.shape[1]:
        raise ValueError(f"the {k.shape[1]} key heads must divide the {h} query heads")
    if ptr.dim() != 1 or ptr.numel() < 1 or ptr.dtype != torch.int64 or ptr.device != q.device:
        raise ValueError(f"ptr must be int64 (structures + 1) on {q.device}, got {ptr.dtype} {tuple(ptr.shape)} on {ptr.device}")
    if key_mask is not None and (key_mask.dtype != torch.bool or key_mask.shape != (n,) or key_mask.device != q.device):
        raise ValueError(f"key_mask must be bool ({n},) on {q.device}")
    if max_len is None:
        max_len = n
    max_len = int(max_len)
    if max_len < 0:
        raise ValueError(f"max_len must not be negative, got {max_len}")
    scale = d ** -0.5 if scale is None else float(scale)
    if int(ptr[0]) < 0 or int(ptr[-1]) > n or bool((ptr[1:] < ptr[:-1]).any()):
        raise ValueError(f"ptr must ascend within 0 .. {n}")
    if ptr.numel() > 1 and int((ptr[1:] - ptr[:-1]).max()) > max_len:
        raise ValueError(f"a structure has more than max_len={max_len} atoms")
    return _formula(q, k, v, ptr, key_mask, scale)
