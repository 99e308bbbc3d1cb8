"""The norm of many gradients taken as one vector, and clipping to it (``mdp_grad_norm`` / ``mdp_grad_clip``): float32,
bfloat16 and float16 tensors in one call, sums in 64 bits in an order that depends on the sizes and element types alone, no
synchronisation."""
from __future__ import annotations

from array import array

import torch

from .. import _lib as L

_DTYPES = L.DTYPES
_contiguous, _device = torch.Tensor.is_contiguous, torch.Tensor.get_device
_address, _count = torch.Tensor.data_ptr, torch.Tensor.numel
_KINDS = {2.0: 2, 1.0: 1, float("inf"): 0}


def _kind(norm_type) -> int:
    kind = _KINDS.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type must be 1, 2 or inf, got {norm_type}")
    return kind


def _is_dense(t: torch.Tensor) -> bool:
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _check(t: torch.Tensor, device, what: str):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a torch.Tensor, got {type(t)}")
    if t.layout != torch.strided or t.dtype not in L.DTYPES:
        raise ValueError(f"{what} must be a strided float32, bfloat16 or float16 tensor, got {t.layout} {t.dtype}")
    L.require_gpu(t, what)
    if t.device != device:
        raise ValueError(f"{what} lives on '{t.device}', the first gradient on '{device}'")
    if not _is_dense(t):
        raise ValueError(f"{what} must fill its memory without gaps or overlap, got shape {tuple(t.shape)} strides {t.stride()}")


def _as_list(tensors) -> list:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _table(grads: list, outs: list | None) -> tuple[array, int]:
    """(``mdp_grad_t`` table: two pointers, the count and the two element types of each, as 64-bit words; device index)."""
    try:
        index = grads[0].get_device()
        kinds = [_DTYPES[t.dtype] for t in grads]
        plain = index >= 0 and all(map(_contiguous, grads)) and set(map(_device, grads)) == {index}
        if outs is None:
            outs, to = grads, kinds
        else:
            to = [_DTYPES[t.dtype] for t in outs]
            plain = (plain and all(map(_contiguous, outs)) and [t.shape for t in outs] == [t.shape for t in grads]
                     and all([o == k or o == 0 for o, k in zip(to, kinds)]) and set(map(_device, outs)) == {index})
    except (AttributeError, KeyError, RuntimeError, TypeError):
        plain = False
    if not plain:                            # something to refuse, or strides that take a closer look
        _check_all(grads, outs or grads)
        index, outs = grads[0].get_device(), outs or grads
        kinds, to = [_DTYPES[t.dtype] for t in grads], [_DTYPES[t.dtype] for t in outs]
    table = array("q", bytes(32 * len(grads)))
    table[0::4] = array("q", map(_address, grads))
    table[1::4] = table[0::4] if outs is grads else array("q", map(_address, outs))
    table[2::4] = array("q", map(_count, grads))
    table[3::4] = array("q", [k | o << 32 for k, o in zip(kinds, to)])
    return table, index


def _check_all(grads: list, outs: list):
    device = grads[0].device if isinstance(grads[0], torch.Tensor) else None
    for g, o in zip(grads, outs):
        _check(g, device, "gradient")
        if o is g:
            continue
        _check(o, device, "out")
        if o.dtype != g.dtype and o.dtype != torch.float32:
            raise ValueError(f"out must be of its gradient's type or float32, got {o.dtype} for {g.dtype}")
        if o.shape != g.shape or (o.stride() != g.stride() and not (o.is_contiguous() and g.is_contiguous())):
            raise ValueError(f"out must have its gradient's shape and strides: {tuple(o.shape)} {o.stride()} for "
                             f"{tuple(g.shape)} {g.stride()}")


def _launch(grads: list, outs: list | None, kind: int, max_norm: float | None) -> torch.Tensor:
    if not grads:
        return torch.zeros((), dtype=torch.float32)
    table, index = _table(grads, outs)
    n, first = len(grads), grads[0]
    workspace = first.new_empty(L.lib.mdp_grad_workspace(n), dtype=torch.float64)
    norm = first.new_empty((), dtype=torch.float32)
    if max_norm is None:
        L.launch(L.lib.mdp_grad_norm, index, table.buffer_info()[0], n, kind, workspace.data_ptr(), norm.data_ptr())
    else:
        L.launch(L.lib.mdp_grad_clip, index, table.buffer_info()[0], n, kind, max_norm, workspace.data_ptr(), norm.data_ptr())
    return norm


def _bound(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return max_norm


def grad_norm(grads, norm_type: float = 2.0) -> torch.Tensor:
    """Norm (float32, on the device) of all elements of ``grads`` (a tensor or several) taken as one vector: ``norm_type`` 2,
    1 or inf.  A NaN or infinity anywhere shows in it."""
    return _launch(_as_list(grads), None, _kind(norm_type), None)


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """Scales the ``.grad`` of ``parameters`` (a tensor or several; those without one are left out, one that is given twice
    counts once) in place by ``min(1, max_norm / (norm + 1e-6))`` and returns the norm before (float32, on the device).

    The factor is rounded to 32 bits and every product once to its gradient's type.  A norm that is infinite makes the factor
    0, or NaN where ``max_norm`` is infinite too; one that is NaN makes every gradient NaN; nothing synchronises to look."""
    grads = [p.grad for p in dict.fromkeys(_as_list(parameters)) if p.grad is not None]
    norm = _launch(grads, None, _kind(norm_type), _bound(max_norm))
    if grads:
        torch.autograd.graph.increment_version(grads)
    return norm


def clip_grads(grads, max_norm: float, norm_type: float = 2.0, out=None) -> tuple[list[torch.Tensor], torch.Tensor]:
    """``(out, norm)``: like ``clip_grad_norm_`` on the tensors ``grads`` with the result in ``out``, one tensor for each
    gradient, of its type or float32 (16-bit gradients clipped into the 32-bit ones that an optimiser reads); new tensors of
    the gradients' types when omitted.  An ``out`` may be its gradient itself; otherwise outputs and gradients must not
    overlap.  Works on values, as every function here: nothing is recorded for autograd, whatever requires a gradient."""
    grads = _as_list(grads)
    if out is None:
        out = [torch.empty_like(_known(g)) for g in grads]
    else:
        out = _as_list(out)
        if len(out) != len(grads):
            raise ValueError(f"{len(out)} outputs for {len(grads)} gradients")
    norm = _launch(grads, out, _kind(norm_type), _bound(max_norm))
    if out:
        torch.autograd.graph.increment_version(out)
    return out, norm


def _known(t):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"gradient must be a torch.Tensor, got {type(t)}")
    return t
