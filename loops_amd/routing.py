"""Tokens per expert and the balance loss of a router, with its gradient, over the C ABI (``loops_expert_counts``,
``loops_balance_loss*``): column sums of a routing matrix (tokens x experts, ``choices`` ones per row).

With p = softmax(logits), c the counts, n the number of tokens whose mask holds and k the choices per token::

    loss = coefficient * experts * sum_e c_e / (n k) * mean_t p_te

The order in which experts take their tokens is ``embedding.group_tokens(chosen, experts)``.  Logits are float32, float16 or bfloat16,
expert indices int32 or int64 (one outside [0, experts) is not counted).  Calls are asynchronous on the current stream of the tensors'
device and may be captured into a graph; there is no CPU path.  Arguments of a wrong type raise TypeError, of a wrong shape or layout
ValueError; what the library itself refuses (an output that overlaps an input, sizes beyond its range) LoopsError.

Autograd records none of these calls: ``balance_loss`` refuses logits that require a gradient (ValueError) where it does record.  Call it
under ``torch.no_grad()``, on ``logits.detach()``, or from a ``torch.autograd.Function`` whose backward calls ``balance_loss_backward``.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .embedding import c_int, index_type, launch, not_recorded, pitch_of, same_device, value_type, workspace


def _mask(mask: Optional[torch.Tensor], tokens: int):
    if mask is None:
        return None
    if mask.dtype not in (torch.bool, torch.uint8):
        raise TypeError("mask must be bool or uint8")
    if not mask.is_contiguous() or mask.numel() != tokens:
        raise ValueError("mask must be contiguous with an element for each token")
    return mask.data_ptr()


def expert_counts(chosen: torch.Tensor, experts: int, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int32 [experts]: how often each expert stands in ``chosen`` ([tokens, choices] or [tokens], contiguous), in the rows whose
    ``mask`` holds."""
    index = index_type(chosen, "chosen")
    if chosen.dim() not in (1, 2) or not chosen.is_contiguous():
        raise ValueError("chosen must be [tokens, choices], contiguous")
    tokens = chosen.shape[0]
    choices = chosen.shape[1] if chosen.dim() == 2 else 1
    device = same_device(chosen, mask)
    masked = _mask(mask, tokens)
    c_int("loops_expert_counts", tokens, choices, experts)
    _keep, ws, size = workspace(device, "loops_expert_counts_workspace", tokens, choices, experts)
    counts = torch.empty(experts, dtype=torch.int32, device=device)
    launch(device, "loops_expert_counts", index, tokens, choices, chosen.data_ptr(), masked, experts, counts.data_ptr(), ws, size)
    return counts


class BalanceLoss(NamedTuple):
    """What ``balance_loss`` found; ``balance_loss_backward`` takes it back."""
    loss: torch.Tensor         # float32 []
    counts: torch.Tensor       # int32 [experts]
    probability: torch.Tensor  # float32 [experts]: mean over the tokens that take part
    tokens: torch.Tensor       # int32 []: how many those are
    choices: int
    coefficient: float


def balance_loss(logits: torch.Tensor, chosen: torch.Tensor, coefficient: float = 1.0, mask: Optional[torch.Tensor] = None) -> BalanceLoss:
    """The balance loss of ``logits`` [tokens, experts] (any distance between rows) for the experts ``chosen`` [tokens, choices] (contiguous);
    ``mask`` [tokens]: the tokens that take part (all where it is None)."""
    value, index = value_type(logits, "logits"), index_type(chosen, "chosen")
    if logits.requires_grad:
        not_recorded("logits")
    pitch = pitch_of(logits, "logits")
    tokens, experts = logits.shape
    if chosen.dim() != 2 or chosen.shape[0] != tokens or not chosen.is_contiguous():
        raise ValueError("chosen must be [tokens, choices], contiguous")
    choices = chosen.shape[1]
    device = same_device(logits, chosen, mask)
    masked = _mask(mask, tokens)
    c_int("loops_balance_loss", tokens, experts, choices)
    _keep, ws, size = workspace(device, "loops_balance_loss_workspace", tokens, experts)
    loss = torch.empty((), dtype=torch.float32, device=device)
    counts = torch.empty(experts, dtype=torch.int32, device=device)
    probability = torch.empty(experts, dtype=torch.float32, device=device)
    counted = torch.empty((), dtype=torch.int32, device=device)
    launch(device, "loops_balance_loss", value, index, tokens, experts, choices, logits.data_ptr(), pitch, chosen.data_ptr(), masked, coefficient,
           loss.data_ptr(), counts.data_ptr(), probability.data_ptr(), counted.data_ptr(), ws, size)
    return BalanceLoss(loss, counts, probability, counted, choices, coefficient)


def balance_loss_backward(logits: torch.Tensor, forward: BalanceLoss, mask: Optional[torch.Tensor] = None, grad_loss: Optional[torch.Tensor] = None,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of ``grad_loss * loss`` (a float32 scalar on the device; 1 where it is None) with respect to ``logits``, in their type: [tokens,
    experts].  ``logits`` and ``mask`` as in the forward call, ``forward`` what it returned."""
    value = value_type(logits, "logits")
    if out is not None and out.requires_grad:
        not_recorded("out")
    pitch = pitch_of(logits, "logits")
    tokens, experts = logits.shape
    if forward.counts.shape != (experts,):
        raise ValueError("forward was made of another number of experts")
    if forward.counts.dtype is not torch.int32 or forward.tokens.dtype is not torch.int32:
        raise TypeError("forward must hold int32 counts")
    if not forward.counts.is_contiguous() or forward.tokens.numel() != 1:
        raise ValueError("forward must hold contiguous counts and one number of tokens")
    device = same_device(logits, forward.counts, forward.tokens, mask, grad_loss, out)
    masked = _mask(mask, tokens)
    c_int("loops_balance_loss_backward", tokens, experts, forward.choices)
    upstream = None
    if grad_loss is not None:
        if grad_loss.dtype is not torch.float32:
            raise TypeError("grad_loss must be float32")
        if grad_loss.numel() != 1:
            raise ValueError("grad_loss must be a scalar")
        upstream = grad_loss.data_ptr()
    if out is None:
        out = torch.empty(tokens, experts, dtype=logits.dtype, device=device)
        out_pitch = experts
    else:
        if out.dtype is not logits.dtype:
            raise TypeError("out must have the logits' type")
        if out.shape != logits.shape:
            raise ValueError("out must have the logits' shape")
        out_pitch = pitch_of(out, "out")
    launch(device, "loops_balance_loss_backward", value, tokens, experts, forward.choices, logits.data_ptr(), pitch, forward.counts.data_ptr(),
           forward.tokens.data_ptr(), masked, forward.coefficient, upstream, out.data_ptr(), out_pitch)
    return out
