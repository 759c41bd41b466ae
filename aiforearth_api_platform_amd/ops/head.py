"""Classifier head epilogue: softmax + top-k in one HIP kernel (``csrc/kernels/head.hip``).

``softmax_topk(logits, k)`` -> ``(idx int32 [N,k], prob fp32 [N,k])``, sorted by descending probability,
ties to the lower class index. Replaces cast + ``torch.softmax`` + ``torch.topk`` (+ sort + index cast):
five launches in the serving engine's graph tail. The PyTorch path is the reference.

``label_logprobs(logits, labels, k)`` (``csrc/kernels/logprobs.hip``): the log-probability of given labels, the entropy
and the k most likely classes, over any number of classes.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _ext, mx


def softmax_topk(logits: torch.Tensor, k: int = 5) -> Tuple[torch.Tensor, torch.Tensor]:
    n, c = logits.shape
    if _ext.backend_for(logits) != "hip" or logits.dtype != torch.bfloat16 or c > 2048 or logits.stride(1) != 1:
        p, i = torch.topk(torch.softmax(logits.float(), dim=1), k, dim=1)
        return i.to(torch.int32), p
    idx = torch.empty(n, k, device=logits.device, dtype=torch.int32)
    prob = torch.empty(n, k, device=logits.device, dtype=torch.float32)
    _ext.call("ai4e_softmax_topk", logits.data_ptr(), logits.stride(0), n, c, k, idx.data_ptr(), prob.data_ptr(),
              _ext.stream_ptr(logits.device))
    return idx, prob


class LabelLogprobs(NamedTuple):
    logp: Optional[torch.Tensor]  # fp32, labels' shape; None without labels
    entropy: torch.Tensor         # fp32 [...], in nats
    top_idx: torch.Tensor         # int32 [..., k]
    top_logp: torch.Tensor        # fp32 [..., k], descending


MAX_ALTERNATIVES = 64


def label_logprobs(logits: torch.Tensor, labels: Optional[torch.Tensor] = None, k: int = 5) -> LabelLogprobs:
    """``logits`` [..., C] (bf16, fp16 or fp32; rows may be strided), ``labels`` [...] or [..., L] (int64 or int32) and
    ``0 <= k <= 64`` alternatives, ties to the lower class.

    A masked class has the logit -inf: its log-probability is -inf, it adds nothing to the entropy and is no alternative
    (where fewer than k classes are left, the rest are class -1 at -inf). A row with nothing left has log-probabilities
    -inf and entropy 0. A row with a NaN or +inf has no distribution: NaN, classes -1. A negative label means that the
    row has none: 0, so that sums pass over it; one of C or more gives NaN. No backward pass."""
    c = logits.shape[-1] if logits.dim() else 0
    if logits.dtype not in mx.DTYPE_CODE or not 0 < c <= mx.MAX_WIDTH:
        raise ValueError("label_logprobs expects bfloat16, float16 or float32 logits of 1 to 2^30 classes")
    if not 0 <= k <= min(c, MAX_ALTERNATIVES):
        raise ValueError(f"label_logprobs: k is 0 to {min(c, MAX_ALTERNATIVES)}, not {k}")
    lead, index = logits.shape[:-1], logits.get_device()
    n_labels = 0
    if labels is not None:
        if labels.dtype not in (torch.int64, torch.int32) or labels.get_device() != index:
            raise ValueError("label_logprobs: labels are int64 or int32, on the logits' device")
        shape = labels.shape
        if shape != lead and (len(shape) == 0 or shape[:-1] != lead):
            raise ValueError(f"label_logprobs: labels {tuple(shape)} fit no logits {tuple(logits.shape)}")
        n_labels = 1 if shape == lead else shape[-1]
        if n_labels > mx.MAX_WIDTH:
            raise ValueError("label_logprobs: a row has up to 2^30 labels")
    _ext.refuse_grad("label_logprobs", logits)
    if _ext.backend_for(logits) != "hip":
        return _label_logprobs_reference(logits, labels, n_labels, k)
    dev = logits.device
    logp = None if labels is None else mx.new(labels.shape, torch.float32, dev)
    entropy = mx.new(lead, torch.float32, dev)
    top_idx = mx.new((*lead, k), torch.int32, dev)
    top_logp = mx.new((*lead, k), torch.float32, dev)
    x = mx.rows_2d(logits)
    rows = x.shape[0]
    if rows:
        labels = None if labels is None else labels.contiguous()
        _ext.call_on(index, "ai4e_label_logprobs", x.data_ptr(), max(x.stride(0), c), rows, c, mx.DTYPE_CODE[x.dtype],
                     _ext.ptr(labels) if n_labels else None, int(n_labels > 0 and labels.dtype == torch.int64), n_labels, k,
                     _ext.ptr(logp), entropy.data_ptr(), top_idx.data_ptr(), top_logp.data_ptr())
    return LabelLogprobs(logp, entropy, top_idx, top_logp)


def _label_logprobs_reference(logits, labels, n_labels, k) -> LabelLogprobs:
    c = logits.shape[-1]
    x = logits.float().reshape(-1, c)
    nan = torch.full((), float("nan"), device=x.device)
    bad = ~(x < float("inf")).all(1)
    none = torch.isneginf(x).all(1) & ~bad
    lp = torch.log_softmax(x.double(), 1)
    lp = torch.where(none[:, None], torch.full_like(lp, -float("inf")), torch.where(bad[:, None], nan.double(), lp))
    term = torch.where(torch.isneginf(lp), torch.zeros_like(lp), lp.exp() * lp)
    entropy = (0.0 - term.sum(1)).float()
    order = torch.sort(torch.where(bad[:, None], torch.zeros_like(x), x), dim=1, descending=True, stable=True).indices[:, :k]
    top = lp.gather(1, order)
    idx = torch.where(torch.isneginf(top) | bad[:, None], torch.full_like(order, -1), order).to(torch.int32)
    logp = None if labels is None else torch.empty(labels.shape, device=x.device)
    if n_labels:
        lab = labels.reshape(-1, n_labels).long()
        logp = lp.gather(1, lab.clamp(0, c - 1))
        logp = torch.where(lab < 0, torch.zeros_like(logp), torch.where(lab >= c, nan.double(), logp)).float().view(labels.shape)
    lead = logits.shape[:-1]
    return LabelLogprobs(logp, entropy.view(lead), idx.view(*lead, k), top.float().view(*lead, k))
