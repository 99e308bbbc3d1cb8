"""Categorical actions: drawing them from a policy's logits, and evaluating stored ones with the gradient by the logits.

Both work on the last axis of ``logits`` (float32, bfloat16 or float16; any leading axes; rows may have any stride) with an
optional boolean ``mask`` of the allowed entries that broadcasts against it, and with settings that are numbers or tensors
that broadcast against the leading axes (one per row).  On the current stream of the logits' device, one launch each
(``mdp_categorical_*``), two for a draw of long rows that settings cut, one more where it draws from the generator; sums of a
draw are in 64 bits."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _lib as L
from ..utils import math as M


def _logit_rows(logits: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(rows, vocab) with unit stride inside a row, and the row stride; copies only what no row stride describes."""
    L.require_gpu(logits, "logits")
    if logits.dtype not in L.DTYPES:
        raise ValueError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f"logits need at least one entry in the last dimension, got shape {tuple(logits.shape)}")
    return _two_dims(logits)


def _two_dims(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _mask_rows(mask, logits: torch.Tensor) -> tuple[torch.Tensor | None, int]:
    if mask is None:
        return None, 0
    L.require_gpu(mask, "mask")
    if mask.dtype != torch.bool:
        raise ValueError(f"mask must be a bool tensor (True = allowed), got {mask.dtype}")
    if mask.device != logits.device:
        raise ValueError(f"mask lives on '{mask.device}', logits on '{logits.device}'")
    if mask.shape != logits.shape:
        try:
            mask = mask.expand(logits.shape)
        except RuntimeError:
            raise ValueError(f"mask of shape {tuple(mask.shape)} does not broadcast against logits {tuple(logits.shape)}") from None
    return _two_dims(mask)


def _setting(value, name: str, dtype: torch.dtype, logits: torch.Tensor, low: float, high: float) -> tuple[torch.Tensor | None, float]:
    """(per-row tensor, 0) or (None, number); numbers are checked, tensors are read by the launch as they are."""
    if not isinstance(value, torch.Tensor):
        value = float(value)
        if not low <= value <= high:
            raise ValueError(f"{name} must be between {low:g} and {high:g}, got {value}")
        return None, value
    if value.device != logits.device:
        raise ValueError(f"{name} lives on '{value.device}', logits on '{logits.device}'")
    if value.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} gets no gradient: pass it detached")
    lead = logits.shape[:-1]
    if dtype == torch.int32 and (value.is_floating_point() or value.is_complex()):
        raise ValueError(f"{name} must be of whole numbers, an integer tensor, got {value.dtype}")
    if dtype == torch.int32 and value.dtype != dtype:
        value = value.to(torch.int64).clamp(-1, 2147483647)            # the narrower types hold no such bounds
    try:
        return value.detach().to(dtype).expand(lead).contiguous(), 0.0
    except RuntimeError:
        raise ValueError(f"{name} of shape {tuple(value.shape)} does not broadcast against the rows {tuple(lead)}") from None


def _per_row(t: torch.Tensor, name: str, dtype: torch.dtype, logits: torch.Tensor) -> torch.Tensor:
    L.require_gpu(t, name)
    if t.dtype != dtype or t.shape != logits.shape[:-1] or t.device != logits.device:
        raise ValueError(f"{name} must be {dtype} of shape {tuple(logits.shape[:-1])} on '{logits.device}', got {t.dtype} "
                         f"{tuple(t.shape)} on '{t.device}'")
    return t.contiguous()


def _address(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


_MOST = 3.4028234663852886e38


def sample_categorical(logits: torch.Tensor, u: torch.Tensor | None = None, *, temperature=1.0, top_k=0, top_p=1.0,
                       min_p=0.0, mask: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """One entry of every row: ``(actions int64, log_prob float32)``, both of the logits' leading shape.

    ``u`` (float32, leading shape, in [0, 1)) makes the draw: the answer is the first kept entry, by index, up to which the
    kept entries hold more than a share ``u`` of their weight ``exp(logit / temperature)``.  Without it the numbers come from
    the device generator of ``isaaclab_amd.utils.math`` (``seed_samplers``; seeded, or drawn from, before a capture), fresh on
    every replay of a captured call; there is one for each device, so calls that draw from it on two streams have to be ordered.

    Kept are the ``top_k`` largest allowed logits (0: all; equal ones by lowest index; per row: an integer tensor, what is
    negative counts as 0), of these the fewest largest that hold a share ``top_p`` of their weight (one at least), of these the
    ones of at least ``min_p`` times the largest weight.  ``temperature`` 0 (or below the smallest normal float) takes the largest
    logit (the first of equal ones) with log_prob 0.  ``log_prob`` is that of the distribution drawn from: without ``top_k`` /
    ``top_p`` / ``min_p`` it is what ``evaluate_categorical`` says.

    A row in which nothing is allowed gives action -1 and log_prob 0; a row with a NaN or +inf among its allowed logits gives
    action -1 and log_prob NaN, and so does a per-row temperature that is negative or NaN.  A per-row ``top_p`` / ``min_p`` that is
    NaN sets no limit.  No gradient."""
    x, ld = _logit_rows(logits)
    m, ld_mask = _mask_rows(mask, logits)
    lead = logits.shape[:-1]
    t_t, t_s = _setting(temperature, "temperature", torch.float32, logits, 0.0, _MOST)
    k_t, k_s = _setting(top_k, "top_k", torch.int32, logits, 0, 2147483647)
    if k_s != int(k_s):
        raise ValueError(f"top_k must be a whole number, got {k_s}")
    p_t, p_s = _setting(top_p, "top_p", torch.float32, logits, 0.0, 1.0)
    q_t, q_s = _setting(min_p, "min_p", torch.float32, logits, 0.0, 1.0)
    state = None
    if u is not None:
        u = _per_row(u, "u", torch.float32, logits)
    else:
        state = M._state(logits.device)
    actions, log_prob = x.new_empty(lead, dtype=torch.int64), x.new_empty(lead, dtype=torch.float32)
    a = L.MdpCategoricalSample(
        x.data_ptr(), ld, x.shape[0], x.shape[1], L.DTYPES[x.dtype], 0, _address(m), ld_mask,
        _address(t_t), _address(k_t), _address(p_t), _address(q_t), t_s, int(k_s), p_s, q_s, _address(u), _address(state),
        actions.data_ptr(), log_prob.data_ptr())
    L.launch(L.lib.mdp_categorical_sample, x.get_device(), L.byref(a))
    return actions, log_prob


def _eval_args(x, ld, actions, mask, ld_mask, t_t, t_s, log_prob, entropy, stats) -> "L.MdpCategoricalEval":
    return L.MdpCategoricalEval(x.data_ptr(), ld, x.shape[0], x.shape[1], L.DTYPES[x.dtype], t_s,
                                _address(mask), ld_mask, actions.data_ptr(), _address(t_t),
                                _address(log_prob), _address(entropy), _address(stats))


def _forward(x, ld, actions, mask, ld_mask, t_t, t_s, lead):
    log_prob, entropy = x.new_empty(lead, dtype=torch.float32), x.new_empty(lead, dtype=torch.float32)
    stats = x.new_empty((x.shape[0], 3), dtype=torch.float32)
    a = _eval_args(x, ld, actions, mask, ld_mask, t_t, t_s, log_prob, entropy, stats)
    L.launch(L.lib.mdp_categorical_evaluate, x.get_device(), L.byref(a))
    return log_prob, entropy, stats


def _backward(x, ld, actions, mask, ld_mask, t_t, t_s, stats, grad_log_prob, grad_entropy, shape):
    grad = x.new_empty(shape)
    a = _eval_args(x, ld, actions, mask, ld_mask, t_t, t_s, None, None, stats)
    L.launch(L.lib.mdp_categorical_evaluate_grad, x.get_device(), L.byref(a), _address(grad_log_prob), _address(grad_entropy),
             grad.data_ptr(), x.shape[1])
    return grad


class _Evaluate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, mask, temperature):
        x, ld = _logit_rows(logits)
        m, ld_mask = _mask_rows(mask, logits)
        t_t, t_s = _temperature(temperature, logits)
        log_prob, entropy, stats = _forward(x, ld, actions, m, ld_mask, t_t, t_s, logits.shape[:-1])
        # the logits themselves where they were read in place: autograd then notices that somebody writes to them
        ctx.save_for_backward(logits if x.data_ptr() == logits.data_ptr() else x, actions, m, t_t, stats)
        ctx.rest = (ld_mask, t_s, logits.shape)
        ctx.set_materialize_grads(False)
        return log_prob, entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_log_prob, grad_entropy):
        if grad_log_prob is None and grad_entropy is None:
            return None, None, None, None
        logits, actions, mask, t_t, stats = ctx.saved_tensors
        ld_mask, t_s, shape = ctx.rest
        x, ld = _two_dims(logits)
        gl, ge = (None if g is None else g.contiguous() for g in (grad_log_prob, grad_entropy))
        return _backward(x, ld, actions, mask, ld_mask, t_t, t_s, stats, gl, ge, shape), None, None, None


def _temperature(value, logits):
    if not isinstance(value, torch.Tensor) and not float(value) >= 2.0 ** -126:
        raise ValueError(f"temperature must be positive, got {value}")
    return _setting(value, "temperature", torch.float32, logits, 0.0, _MOST)


def evaluate_categorical(logits: torch.Tensor, actions: torch.Tensor, *, temperature=1.0,
                         mask: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(log_prob, entropy)`` (float32, leading shape) of ``actions`` (int64, leading shape) under
    ``softmax(logits / temperature)`` over the allowed entries; differentiable once by ``logits``.

    Action -1 (what a row with nothing allowed was given) has log_prob 0 and no gradient through it, an action that is not
    allowed -inf, one outside [-1, vocab) NaN.  A row with nothing allowed has entropy 0 and gradient 0; entries that are not
    allowed have gradient 0.  A NaN or +inf among the allowed logits makes its row NaN, and so does a per-row temperature that
    is not a finite number of at least 2^-126, the smallest normal one (a temperature for all rows is refused below it).

    Inside a captured graph use ``evaluate_categorical_grad``, which does without autograd's own streams and graph nodes."""
    L.require_gpu(logits, "logits")
    actions = _per_row(actions, "actions", torch.int64, logits)
    if isinstance(temperature, torch.Tensor) and temperature.requires_grad and torch.is_grad_enabled():
        raise ValueError("temperature gets no gradient: pass it detached")
    return _Evaluate.apply(logits, actions, mask, temperature)


def evaluate_categorical_grad(logits: torch.Tensor, actions: torch.Tensor, grad_log_prob: torch.Tensor | None,
                              grad_entropy: torch.Tensor | None, *, temperature=1.0,
                              mask: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(log_prob, entropy, grad_logits)``: the evaluation and the gradient of ``sum(grad_log_prob * log_prob + grad_entropy
    * entropy)`` by the logits, in their type, without autograd (two launches that a graph may capture): what goes in may
    require a gradient, none of the results does or passes one on.  ``grad_*``: float32, leading shape, or None for zeros."""
    x, ld = _logit_rows(logits.detach() if isinstance(logits, torch.Tensor) else logits)
    actions = _per_row(actions, "actions", torch.int64, logits)
    m, ld_mask = _mask_rows(mask, logits)
    t_t, t_s = _temperature(temperature, logits)
    gl = None if grad_log_prob is None else _per_row(grad_log_prob, "grad_log_prob", torch.float32, logits)
    ge = None if grad_entropy is None else _per_row(grad_entropy, "grad_entropy", torch.float32, logits)
    log_prob, entropy, stats = _forward(x, ld, actions, m, ld_mask, t_t, t_s, logits.shape[:-1])
    return log_prob, entropy, _backward(x, ld, actions, m, ld_mask, t_t, t_s, stats, gl, ge, logits.shape)
