"""Inverted dropout whose mask is a function of a counter and is never stored.

``dropout(x, p, key)``: element i (in row-major order) keeps its value, scaled by 1 / (1 − p'), iff
its 16 bits of Philox4x32-10 (Salmon et al. 2011) at counter (i // 8, key[1]) under seed key[0] are
not below 65536·p', with p' = round(65536 p) / 65536.  The backward pass makes the mask again from
the key (``csrc/kernels/dropout.hip``).  ``key`` is an int64 [2] tensor on x's device: inside a
captured training step it is an input like any other, so replays draw new masks as long as the key
is drawn inside the graph (:class:`DropoutKeys`).
"""
from __future__ import annotations

import torch

from .common import on_gpu, ext

_M32 = 0xFFFFFFFF


def _cut(p):
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout: 0 <= p <= 1, got {p}")
    cut = round(65536 * float(p))
    if cut == 65536 and p < 1:
        raise ValueError(f"dropout: p is a multiple of 2^-16, and {p} rounds to 1, which keeps nothing")
    return cut


def check_layer_p(p):
    """``p`` as a layer takes it: below 1, also as rounded."""
    if p == 1:
        raise ValueError("dropout: 0 <= p < 1, got 1")
    _cut(p)
    return float(p)


def ref_philox4x32(c, k, rounds=10):
    """Philox4x32 on int64 tensors holding 32-bit words: counters ``c`` (4), key ``k`` (2)."""
    c0, c1, c2, c3 = c
    k0, k1 = k
    for _ in range(rounds):
        # the 64-bit products may wrap into the sign: their bits are right, the shifts are masked
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & _M32) ^ c1 ^ k0, b & _M32, ((a >> 32) & _M32) ^ c3 ^ k1, a & _M32
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return c0, c1, c2, c3


def ref_dropout_keep(numel, p, key):
    """The mask: a bool tensor [numel], True where the element is kept."""
    blk = torch.arange((numel + 7) // 8, device=key.device)
    call = key[1].expand(blk.shape)
    w = ref_philox4x32((blk & _M32, blk >> 32, call & _M32, (call >> 32) & _M32),
                       (key[0] & _M32, (key[0] >> 32) & _M32))
    bits = torch.stack([h for c in w for h in (c & 0xFFFF, c >> 16)], 1).reshape(-1)[:numel]
    return bits >= _cut(p)


def _ref_dropout(x, cut, key):
    x = x.contiguous()
    keep = ref_dropout_keep(x.numel(), cut / 65536, key).view(x.shape)
    scale = 65536.0 / (65536 - cut) if cut < 65536 else 0.0
    return torch.where(keep, x.float() * scale, torch.zeros((), device=x.device)).to(x.dtype)


class _DropoutFn(torch.autograd.Function):
    """The CPU path's autograd node (the GPU's is native, csrc/bindings.cpp DropoutFn)."""

    @staticmethod
    def forward(ctx, x, cut, key):
        ctx.cut = cut
        ctx.save_for_backward(key)
        return _ref_dropout(x, cut, key)

    @staticmethod
    def backward(ctx, dy):
        # linear in x: the same operator on dy (which also makes it differentiable again)
        (key,) = ctx.saved_tensors
        return _DropoutFn.apply(dy, ctx.cut, key), None, None


def dropout(x, p, key):
    """``x`` (bf16 / fp32, any shape) with each element zeroed with probability ``p`` (a multiple of
    2^-16, rounded) and the others scaled by 1 / (1 − p).  ``key``: int64 [2] on x's device, the seed
    and the call number; equal keys give equal masks.  Changing ``key`` in place between the forward
    and the backward pass is an error (autograd's version check).  A p that is or rounds to 0 returns
    ``x`` itself; p = 1 drops everything, a p that only rounds to it is refused."""
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"dropout: bf16 / fp32 input, got {x.dtype}")
    if key.dtype != torch.int64 or key.shape != (2,):
        raise ValueError(f"dropout: key int64 [2], got {key.dtype} {tuple(key.shape)}")
    if key.device != x.device:
        raise ValueError(f"dropout: key on {key.device}, input on {x.device}")
    cut = _cut(p)
    if cut == 0:
        return x
    key = key.contiguous()
    return ext().dropout(x, key, cut) if on_gpu(x) else _DropoutFn.apply(x, cut, key)


class DropoutKeys:
    """A stream of keys on a device: ``next()`` gives (seed, n) for n = first, first + 1, …  Each key
    is a new tensor (a backward pass may come later); on the GPU the call number is advanced by a
    kernel, so a captured step draws a new key at every replay, and calls on several streams draw
    distinct ones."""

    def __init__(self, seed, device, first=0):
        device = torch.device(device)
        if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            # a state made inside the graph would be made again by every replay: the same masks
            raise RuntimeError("DropoutKeys: make it (run one step) before capturing a graph")
        with torch.inference_mode(False):  # an ordinary tensor, whichever call comes first
            self.state = torch.tensor([seed, first], dtype=torch.int64).to(device)

    def start_at(self, first):
        """The next key is (seed, first), in steps captured with this stream too: the state is
        written where it is, behind every draw that is queued on the device."""
        cuda = self.state.device.type == "cuda"
        if cuda:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("DropoutKeys.start_at: not inside a graph capture")
            torch.cuda.synchronize(self.state.device)
        self.state[1] = first
        if cuda:
            torch.cuda.current_stream(self.state.device).synchronize()

    def next(self):
        if on_gpu(self.state):
            return ext().dropout_next_key(self.state)
        key = self.state.clone()
        self.state[1] += 1
        return key
