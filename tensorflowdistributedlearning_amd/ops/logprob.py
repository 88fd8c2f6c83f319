"""Log-probabilities of given labels, with the entropy and the most probable classes of every row.

``label_log_probs(logits, labels, top_k)`` is what scoring, calibration, active selection and top-k
evaluation read off a classifier's (or a per-pixel classifier's) logits:

    log p_j = x_j − log Σ_i e^{x_i}        H = −Σ_j p_j log p_j

One pass over the logits on the GPU (``csrc/kernels/logprob.hip``); the backward pass recomputes the
probabilities from three floats per row.  Nothing of the size of the logits is stored besides them
and their gradient.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .common import on_gpu, ext

MAX_TOP_K = 32  # csrc/kernels/kernels.h LOGPROB_MAX_K
MAX_CLASSES = 2 ** 31 - 2 ** 16  # LOGPROB_MAX_C: the kernels count inside a row in 32 bits


class LabelLogProbs(NamedTuple):
    log_prob: Optional[torch.Tensor]      # [...] log p of the label; None without labels
    entropy: torch.Tensor                 # [...]
    top_log_prob: Optional[torch.Tensor]  # [..., top_k], descending; None for top_k = 0
    top_index: Optional[torch.Tensor]     # [..., top_k] int64


def ref_label_log_probs(logits, labels=None, top_k=0, ignore_index=-100, dtype=torch.float32):
    """The same outputs from elementary operations (CPU path; the tests' oracle in 64 bits)."""
    x = logits.to(dtype)
    C = x.shape[-1]
    nan = torch.full_like(x[..., 0], float("nan"))
    bad = ~(x < float("inf")).all(-1)             # a NaN or +inf in the row
    m = x.detach().amax(-1, keepdim=True).clamp_min(torch.finfo(dtype).min)
    z = x - m
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    empty = (total == 0).squeeze(-1)              # every class masked with -inf
    lse = torch.where(total > 0, torch.log(total.clamp_min(torch.finfo(dtype).tiny)),
                      torch.full_like(total, float("inf")))
    lp = z - lse
    p = torch.exp(lp)
    ent = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(-1)
    ent = torch.where(bad, nan, ent)
    lp = torch.where(bad[..., None], nan[..., None], lp)
    logp = tlp = ti = None
    if labels is not None:
        ok = ((labels >= 0) & (labels < C)) | (labels == ignore_index)
        got = lp.gather(-1, labels.clamp(0, C - 1).unsqueeze(-1)).squeeze(-1)
        got = got + torch.where(ok, torch.zeros_like(got), nan)
        if got.requires_grad:  # a gradient through a label out of range is NaN (a selection would pass 0)
            got.register_hook(lambda g: None if g is None else torch.where(ok | (g == 0), g, nan))
        logp = torch.where(labels == ignore_index, torch.zeros_like(got), got)
    if top_k:
        keys = torch.where(bad[..., None], torch.zeros_like(x), x)
        ti = torch.sort(keys, dim=-1, descending=True, stable=True).indices[..., :top_k]
        tlp = lp.gather(-1, ti)
    if logits.requires_grad and bool(empty.any()):
        # nothing depends on the logits of an empty row
        def cut(t):
            if t is None:
                return None
            e2 = empty.reshape(empty.shape + (1,) * (t.dim() - empty.dim()))
            return torch.where(e2, t.detach(), t)
        logp, ent, tlp = cut(logp), cut(ent), cut(tlp)
    return LabelLogProbs(logp, ent, tlp, ti)


def flat_rows(logits, labels, top_k, who):
    """Check the arguments of the log-probability operators; ``(logits [N, C] as the kernels read
    them on the GPU, labels int64 [N] or None, leading shape)``."""
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{who}: logits [..., C] with C >= 1, got {tuple(logits.shape)}")
    C = logits.shape[-1]
    if C > MAX_CLASSES:
        raise ValueError(f"{who}: at most {MAX_CLASSES} classes, got {C}")
    if not 0 <= top_k <= min(C, MAX_TOP_K):
        raise ValueError(f"{who}: 0 <= top_k <= min(C, {MAX_TOP_K}), got {top_k} for {C} classes")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{who}: bf16 / fp32 logits, got {logits.dtype}")
    lead = logits.shape[:-1]
    if labels is not None:
        if labels.shape != lead:
            raise ValueError(f"{who}: labels {tuple(labels.shape)} for logits {tuple(logits.shape)}")
        if labels.dtype.is_floating_point or labels.dtype.is_complex or labels.dtype == torch.bool:
            raise TypeError(f"{who}: integer labels, got {labels.dtype}")
        if labels.device != logits.device:
            raise ValueError(f"{who}: labels on {labels.device}, logits on {logits.device}")
        labels = labels.long()
    if not on_gpu(logits):
        return logits, labels, lead
    x = logits if logits.dim() == 2 else logits.reshape(-1, C)
    if (C > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < C):
        x = x.contiguous()
    return x, None if labels is None else labels.reshape(-1).contiguous(), lead


def label_log_probs(logits, labels=None, top_k=0, ignore_index=-100):
    """Log-probability of each row's label, the entropy of its distribution and its ``top_k`` most
    probable classes.

    ``logits`` [..., C] bf16 / fp32 (rows may be strided; classes contiguous, else they are copied);
    ``labels`` integers [...] or None.  Returns :class:`LabelLogProbs` of fp32 tensors; the indices
    are int64, ordered by descending logit, equal logits by ascending index.  Differentiable in the
    logits through ``log_prob``, ``entropy`` and ``top_log_prob`` (once).

    A class is masked with −inf.  A row with every class masked gives log-probabilities of −inf,
    entropy 0 and no gradient.  A label equal to ``ignore_index`` (checked first) gives
    log-probability 0 and no gradient through it; any other label outside [0, C) gives NaN, and the
    row's gradient is NaN where one that is not zero arrives at that log-probability.  A row with a
    NaN or +inf gives NaN throughout and the indices 0 … top_k − 1.
    """
    x, lab, lead = flat_rows(logits, labels, top_k, "label_log_probs")
    if not on_gpu(logits):
        return ref_label_log_probs(x, lab, top_k, ignore_index)
    out = ext().label_log_probs(x, lab, int(top_k), int(ignore_index))  # with its autograd node
    if logits.dim() == 2:
        return LabelLogProbs(*out)
    return LabelLogProbs(*(None if t is None else t.reshape(lead + t.shape[1:]) for t in out))
