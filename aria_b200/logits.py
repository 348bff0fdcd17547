"""What logits go through before the next token is chosen: penalties for repeated
tokens, biases and grammar masks, with the greedy choice (libaria_q4.so).

The reference masks logits on the CPU after downloading them (lold3344/ARIA
src/tokenizer.rs `mask_logits`); here one launch adjusts every row on the GPU.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import BF16, F16, F32, LogitRulesStruct, call, fastcall
from .paged import _current_device, _held, _stream, _want, _workspace

__all__ = ["adjust", "allowed_mask"]

_WS_BYTES: dict = {}
_DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def allowed_mask(allowed: torch.Tensor) -> torch.Tensor:
    """bool [..., V] -> the int32 words [..., ceil(V / 32)] that `adjust` reads (bit
    v % 32 of word v / 32)."""
    V = allowed.shape[-1]
    pad = -V % 32
    b = torch.nn.functional.pad(allowed.to(torch.int64), (0, pad)).unflatten(-1, ((V + pad) // 32, 32))
    w = (b << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(w >= 2**31, w - 2**32, w).to(torch.int32)


def _ws_bytes(M: int) -> int:
    n = _WS_BYTES.get(M)
    if n is None:
        n = _WS_BYTES[M] = _lib.lib().aria_logits_workspace_bytes(M)
    return n


def _matrix(t: torch.Tensor, name: str, dtype, M: int, dev: int) -> int:
    """Row stride of an [M][...] matrix with contiguous rows."""
    s = t.stride()
    if t.dtype is not dtype or t.get_device() != dev or len(s) != 2 or t.shape[0] != M or (
            s[1] != 1 and t.shape[1] > 1):
        raise TypeError(f"{name} must be {dtype} [{M}][...] on cuda:{dev} with contiguous rows")
    return s[0] if M > 1 else t.shape[1]


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
    dev = logits.get_device()  # -1 on the CPU
    if dev >= 0:
        stream = _stream(dev)
        ws = _held("logits", dev, stream)
        r = fastcall().logits(ws[0], ws[1], stream, want_token, logits, out, history, history_lens, prompt_lens,
                              repetition, frequency, presence, bias_tokens, bias_values, allowed, token)
        if r is not None:
            return r
        if _current_device() != dev:  # a launch goes to the current device
            with torch.cuda.device(dev):
                return adjust(logits, out=out, history=history, history_lens=history_lens, prompt_lens=prompt_lens,
                              repetition=repetition, frequency=frequency, presence=presence, bias_tokens=bias_tokens,
                              bias_values=bias_values, allowed=allowed, want_token=want_token, token=token)
    # another device is current, the first call on a stream, one that needs more scratch, or something to say
    if dev < 0 or logits.dim() != 2 or logits.dtype not in _DTYPES:
        raise TypeError("logits must be an f32, f16 or bf16 [M][V] CUDA tensor")
    M, V = logits.shape
    i32, f32, rows = torch.int32, torch.float32, (M,)
    x_row = _matrix(logits, "logits", logits.dtype, M, dev)
    if out is None:
        out = torch.empty((M, V), dtype=logits.dtype, device=logits.device)
    if (out.dtype is not logits.dtype and out.dtype is not f32) or out.shape != logits.shape:
        raise TypeError("out must be [M][V] of the logits' type or f32")
    y_row = _matrix(out, "out", out.dtype, M, dev)
    hp = hl = pl = rp = fp = ap = btp = bvp = mp = None
    h_row = cap = b_row = biases = m_row = 0
    if history is not None:
        h_row = _matrix(history, "history", i32, M, dev)
        if history_lens is None:
            raise ValueError("history needs history_lens")
        hp, cap = history.data_ptr(), history.shape[1]
        hl = _want(history_lens, "history_lens", i32, rows, dev)
        if prompt_lens is not None:
            pl = _want(prompt_lens, "prompt_lens", i32, rows, dev)
    elif repetition is not None or frequency is not None or presence is not None:
        raise ValueError("penalties need a history")
    if repetition is not None:
        rp = _want(repetition, "repetition", f32, rows, dev)
    if frequency is not None:
        fp = _want(frequency, "frequency", f32, rows, dev)
    if presence is not None:
        ap = _want(presence, "presence", f32, rows, dev)
    if bias_tokens is not None and bias_values is not None:
        b_row = _matrix(bias_tokens, "bias_tokens", i32, M, dev)
        if bias_values.shape != bias_tokens.shape or _matrix(bias_values, "bias_values", f32, M, dev) != b_row:
            raise ValueError("bias_values must match bias_tokens")
        biases = bias_tokens.shape[1]
        if biases > 0:
            btp, bvp = bias_tokens.data_ptr(), bias_values.data_ptr()
    elif bias_tokens is not None or bias_values is not None:
        raise ValueError("bias_tokens and bias_values go together")
    if allowed is not None:
        n = allowed.shape[0] if allowed.dim() == 2 else 0
        if n not in (1, M) or allowed.shape[1] != (V + 31) // 32:
            raise ValueError("allowed must be int32 [M or 1][ceil(V / 32)]")
        m_row = _matrix(allowed, "allowed", i32, n, dev)
        if n != M:
            m_row = 0  # one row for all
        mp = allowed.data_ptr()
    r = LogitRulesStruct(hp, h_row, cap, hl, pl, rp, fp, ap, btp, bvp, b_row, biases, mp, m_row)
    stream = _stream(dev)
    tp = None
    ws = (None, 0)
    if want_token or token is not None:
        if token is None:
            token = torch.empty(rows, dtype=i32, device=logits.device)
        tp = _want(token, "token", i32, rows, dev)
        ws = _workspace("logits", _ws_bytes(M), dev, stream, "all")
    call("aria_logits_adjust", ctypes.addressof(r), logits.data_ptr(), _DTYPES[logits.dtype], x_row, M, V,
         out.data_ptr(), _DTYPES[out.dtype], y_row, tp, ws[0], ws[1], stream)
    return out, token
