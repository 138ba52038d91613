"""What stands between a decoder's logits and its token (see ``csrc/ixb_logits.cuh``): penalties for tokens that were seen, biases,
grammar masks and the arg-max in one launch.  The reference leaves this to HuggingFace's logits processors
(ixrun/generate.py:39-70)."""
from __future__ import annotations

import torch

from . import _lib

__all__ = ["apply_rules"]

MAX_VOCAB, MAX_TOKENS, MAX_BIASES = 393216, 2**20 - 1, 2047        # of a row, as ixb_logits takes them


def _on(dev: int, t, dtypes, shape, what: str):
    """a tensor of one of these types and of this shape (None: any size) with contiguous rows, on this device; its row pitch"""
    if t.dtype not in dtypes or not t.is_cuda or t.dim() != len(shape) or any(s is not None and s != n for s, n in zip(shape, t.shape)):
        raise ValueError(f"{what}: a CUDA tensor {list(shape)} of {' or '.join(str(d).replace('torch.', '') for d in dtypes)} expected")
    if t.get_device() != dev:
        raise ValueError(f"{what} is on another device")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: contiguous rows expected")
    if t.dim() == 2:
        pitch = t.stride(0) if t.shape[0] > 1 else t.shape[1]
        if pitch < t.shape[1]:
            raise ValueError(f"{what}: rows must not overlap")
        return pitch
    return t.shape[0]


def apply_rules(logits, history=None, n_tokens=None, n_prompt=None, repetition=None, presence=None, frequency=None, bias_ids=None,
                bias_values=None, mask=None, mask_row=None, out=None, token=None):
    """logits [B, V], bf16 or fp32 (column slices of wider rows allowed).  Per row b, each step rounded to fp32, in this order:
      tokens among the first n_tokens[b] of history[b] (int32 [B, L]):  x > 0 ? x / repetition[b] : x * repetition[b]
      and c > 0 times among those behind the first n_prompt[b]:        x - frequency[b] * c, then - presence[b]
      tokens named by bias_ids[b] (int32 [B, K]):                      x + bias_values[b] (fp32 [B, K]; the last entry counts)
      tokens whose bit in the row's mask (int32 [M, ceil(V / 32)], bit v % 32 of word v / 32) is 0:  -inf
    Row b has mask mask_row[b] (int32 [B]; none if that is -1), or mask b without mask_row.  Numbers outside 0 .. V - 1 in history and
    bias_ids are passed over (-1 as padding).  n_prompt None: everything counts as generated; penalties None: 1, 0, 0 (fp32 [B]).
    Writes out (fp32 [B, V], may be the fp32 logits; allocated if None) and token (int64 [B], may be None): the lowest index
    of the largest value (of a row of -inf: 0).  V up to 393216, L up to 1048575, K up to 2047.  Returns out."""
    if out is None and logits.dim() == 2:
        out = torch.empty(logits.shape, dtype=torch.float32, device=logits.device)
    if out is not None and _lib.host().logits(logits, history, n_tokens, n_prompt, repetition, presence, frequency, bias_ids, bias_values, mask, mask_row, out, token):
        return out
    if logits.dim() != 2 or not logits.is_cuda:
        raise ValueError("logits: a CUDA tensor [B, V] expected")
    dev, (b, v) = logits.get_device(), logits.shape
    f32, i32 = (torch.float32,), (torch.int32,)
    pitch = _on(dev, logits, (torch.bfloat16, torch.float32), (b, v), "logits")
    if history is None:
        if any(t is not None for t in (n_tokens, n_prompt, repetition, presence, frequency)):
            raise ValueError("penalties need the history of tokens")
        hist_pitch = hist_len = 0
    else:
        hist_pitch, hist_len = _on(dev, history, i32, (b, None), "history"), history.shape[1]
        if n_tokens is None:
            raise ValueError("the history needs n_tokens")
        for t, what in ((n_tokens, "n_tokens"), (n_prompt, "n_prompt")):
            if t is not None:
                _on(dev, t, i32, (b,), what)
        for t, what in ((repetition, "repetition"), (presence, "presence"), (frequency, "frequency")):
            if t is not None:
                _on(dev, t, f32, (b,), what)
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("bias_ids and bias_values go together")
    n_bias = 0
    if bias_ids is not None:
        n_bias = bias_ids.shape[-1]
        for t, types, what in ((bias_ids, i32, "bias_ids"), (bias_values, f32, "bias_values")):
            if _on(dev, t, types, (b, n_bias), what) != n_bias:
                raise ValueError(f"{what}: a contiguous tensor expected")
    n_masks = mask_pitch = 0
    if mask is not None:
        n_masks, mask_pitch = mask.shape[0], _on(dev, mask, i32, (None, (v + 31) // 32), "mask")
        if mask_row is None and n_masks != b:
            raise ValueError("a mask for every row, or mask_row")
    if mask_row is not None:
        if mask is None:
            raise ValueError("mask_row without mask")
        _on(dev, mask_row, i32, (b,), "mask_row")
    out_pitch = _on(dev, out, f32, (b, v), "out")
    if token is not None:
        _on(dev, token, (torch.int64,), (b,), "token")
    if b == 0 or v == 0:
        raise ValueError("logits must not be empty")
    if n_masks == 0:
        mask = mask_row = None
    ptr = lambda t: None if t is None or t.numel() == 0 else t.data_ptr()  # noqa: E731
    with _lib.on_device(dev) as st:
        _lib.check(_lib.lib().ixb_logits(logits.data_ptr(), int(logits.dtype == torch.float32), pitch, ptr(history), hist_len, hist_pitch,
                                         ptr(n_tokens), ptr(n_prompt), ptr(repetition), ptr(presence), ptr(frequency), ptr(bias_ids),
                                         ptr(bias_values), n_bias, ptr(mask), n_masks, mask_pitch, ptr(mask_row), out.data_ptr(), out_pitch,
                                         ptr(token), b, v, st))
    return out
