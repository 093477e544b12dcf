"""Sampling a token of each row of logits on the device (qwc_op_sample)."""

from __future__ import annotations

import torch

from .paged import cuda_index, current_stream, elsewhere, format_of, refuse
from .runtime import check, lib


def sample(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature: torch.Tensor | None = None,
           top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
           min_p: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(tokens int32 [rows], log-probabilities f32 [rows]) of [rows, vocab] logits (rows may be a
    view of wider ones), from one number in [0, 1) for each row. Settings are one value for each row
    on the device (top_k int32, the others f32); None leaves a cut out, and the temperature 1."""
    call, device = "qwc_op_sample", logits.device
    away = elsewhere(cuda_index(device), call)
    if away is not None:
        with away:
            return sample(logits, uniforms, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    fmt = format_of(logits, call)
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        refuse("invalid_argument", call)
    rows, vocab = logits.shape
    pointers = []
    for t, dtype in ((temperature, torch.float32), (top_k, torch.int32), (top_p, torch.float32), (min_p, torch.float32),
                     (uniforms, torch.float32)):
        if t is None:
            pointers.append(None)
            continue
        if t.shape != (rows,):
            refuse("shape_mismatch", call)
        if t.dtype != dtype or t.device != device or not t.is_contiguous():
            refuse("invalid_argument", call)
        pointers.append(t.data_ptr())
    tokens = torch.empty(rows, dtype=torch.int32, device=device)
    logprobs = torch.empty(rows, dtype=torch.float32, device=device)
    check(lib().qwc_op_sample(fmt, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab, *pointers,
                              tokens.data_ptr(), logprobs.data_ptr(), current_stream(device)), call)
    return tokens, logprobs
