"""What logits go through before the next token is chosen: penalties for repeated
tokens, biases and grammar masks, with the greedy choice (libaria_q4.so).

The reference masks logits on the CPU after downloading them (lold3344/ARIA
src/tokenizer.rs `mask_logits`); here one launch adjusts every row on the GPU.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import BF16, F16, F32, LogitRulesStruct, call
from .paged import _stream, _want, _workspace

__all__ = ["adjust", "allowed_mask"]

_DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def allowed_mask(allowed: torch.Tensor) -> torch.Tensor:
    """bool [..., V] -> the int32 words [..., ceil(V / 32)] that `adjust` reads (bit
    v % 32 of word v / 32)."""
    V = allowed.shape[-1]
    pad = -V % 32
    b = torch.nn.functional.pad(allowed.to(torch.int64), (0, pad)).unflatten(-1, ((V + pad) // 32, 32))
    w = (b << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(w >= 2**31, w - 2**32, w).to(torch.int32)


def _matrix(t: torch.Tensor, name: str, dtype, M: int, dev):
    if t.dtype != dtype or t.device != dev or t.dim() != 2 or t.shape[0] != M or (
            t.stride(1) != 1 and t.shape[1] > 1):
        raise TypeError(f"{name} must be {dtype} [{M}][...] on {dev} with contiguous rows")
    return t.data_ptr(), t.stride(0) if M > 1 else t.shape[1]


def adjust(logits: torch.Tensor, *, out: torch.Tensor | None = None, history: torch.Tensor | None = None,
           history_lens: torch.Tensor | None = None, prompt_lens: torch.Tensor | None = None,
           repetition: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
           presence: torch.Tensor | None = None, bias_tokens: torch.Tensor | None = None,
           bias_values: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
           want_token: bool = False, token: torch.Tensor | None = None):
    """logits [M][V] (f32, f16 or bf16, rows contiguous).  In f32 and in this order:
    tokens of history[m][:history_lens[m]] (int32 [M][cap]) have x > 0 ? x / repetition[m]
    : x * repetition[m]; those at or after prompt_lens[m], generated c times, lose
    frequency[m] * c and presence[m]; bias_values f32 are added at bias_tokens int32 [M][n]
    (-1: unused; equal tokens add up); tokens whose bit of allowed (int32 words
    [M or 1][ceil(V / 32)], see allowed_mask) is 0 become -inf.

    Returns (out, token): out of the logits' type (logits itself for in place) or f32;
    token int32 [M] with want_token, else None: the lowest index of the largest f32
    result, -1 where nothing is left above -inf."""
    if not logits.is_cuda or logits.dim() != 2 or logits.dtype not in _DTYPES:
        raise TypeError("logits must be an f32, f16 or bf16 [M][V] CUDA tensor")
    M, V = logits.shape
    dev = logits.device
    xp, x_row = _matrix(logits, "logits", logits.dtype, M, dev)
    if out is None:
        out = torch.empty((M, V), dtype=logits.dtype, device=dev)
    if out.dtype not in (logits.dtype, torch.float32) or out.shape != logits.shape:
        raise TypeError("out must be [M][V] of the logits' type or f32")
    yp, y_row = _matrix(out, "out", out.dtype, M, dev)
    r = LogitRulesStruct()
    if history is not None:
        r.history, r.history_row = _matrix(history, "history", torch.int32, M, dev)
        r.history_cap = history.shape[1]
        if history_lens is None:
            raise ValueError("history needs history_lens")
        r.history_lens = _want(history_lens, "history_lens", torch.int32, (M,), dev)
        if prompt_lens is not None:
            r.prompt_lens = _want(prompt_lens, "prompt_lens", torch.int32, (M,), dev)
    elif repetition is not None or frequency is not None or presence is not None:
        raise ValueError("penalties need a history")
    if repetition is not None:
        r.repetition = _want(repetition, "repetition", torch.float32, (M,), dev)
    if frequency is not None:
        r.frequency = _want(frequency, "frequency", torch.float32, (M,), dev)
    if presence is not None:
        r.presence = _want(presence, "presence", torch.float32, (M,), dev)
    if (bias_tokens is None) != (bias_values is None):
        raise ValueError("bias_tokens and bias_values go together")
    if bias_tokens is not None and bias_tokens.numel() > 0:
        r.bias_tokens, r.bias_row = _matrix(bias_tokens, "bias_tokens", torch.int32, M, dev)
        r.bias_values, v_row = _matrix(bias_values, "bias_values", torch.float32, M, dev)
        if bias_values.shape != bias_tokens.shape or v_row != r.bias_row:
            raise ValueError("bias_values must match bias_tokens")
        r.biases = bias_tokens.shape[1]
    if allowed is not None:
        rows = allowed.shape[0] if allowed.dim() == 2 else 0
        if rows not in (1, M) or allowed.shape[1] != (V + 31) // 32:
            raise ValueError("allowed must be int32 [M or 1][ceil(V / 32)]")
        r.allowed, a_row = _matrix(allowed, "allowed", torch.int32, rows, dev)
        r.allowed_row = a_row if rows == M else 0
    stream = _stream(dev)
    tp = wp = None
    nbytes = 0
    if want_token or token is not None:
        if token is None:
            token = torch.empty(M, dtype=torch.int32, device=dev)
        tp = _want(token, "token", torch.int32, (M,), dev)
        ws = _workspace("logits", _lib.lib().aria_logits_workspace_bytes(M), dev, stream)
        wp, nbytes = ws.data_ptr(), ws.numel()
    call("aria_logits_adjust", ctypes.addressof(r), xp, _DTYPES[logits.dtype], x_row, M, V, yp, _DTYPES[out.dtype],
         y_row, tp, wp, nbytes, stream)
    return out, token
