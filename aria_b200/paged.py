"""A paged, bounded KV cache: attention of one new token over it, the attention
weight its slots have received, and eviction by that weight (libaria_q4.so).

    kv = PagedKV(k_pages, v_pages, block_table, lens)     # one per layer, kept
    w  = prompt_weights(q, k, lse)                        # after the prompt's attention
    out, lse = attention_paged(q, kv, k_new=k, v_new=v, weights=w, slot_pos=p, positions=pos)
    evict(kv, w, p, next_pos, keep, recent=..., sinks=..., lens_out=...)

The reference's cache (KVCache, lold3344/ARIA src/transformer_cuda.rs:144-155) is
contiguous and grows with the sequence; paging and eviction have no counterpart
there.  No fallback: without the library or a B200 every call raises.  Calls run
on the current stream of the tensors' device, whichever device is current; what they
write in place, they write in the order of that stream.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import BF16, F16, PagedKVStruct, call, fastcall

__all__ = ["PagedKV", "attention_paged", "prompt_weights", "evict", "clear_workspaces"]

_DTYPES = {torch.float16: F16, torch.bfloat16: BF16}
# (operator, device, stream) -> (pointer, bytes, tensor): scratch of eager calls, and of the
# calls of the graph that was captured last on the stream (with the capture's id)
_WORKSPACES: dict = {}
_GRAPH_WORKSPACES: dict = {}
_NO_WORKSPACE = (0, 0, None)


# The device's current stream as an integer, without building a Stream object: the
# host's part of a call is a few microseconds in all.
_stream = torch._C._cuda_getCurrentRawStream
_capturing = torch._C._cuda_isCurrentStreamCapturing
_current_device = torch._C._cuda_getDevice


def _capture_id(stream: int) -> int:
    n = ctypes.c_ulonglong(0)
    call("aria_stream_capture_id", stream, ctypes.addressof(n))
    return n.value


def _held(kind: str, dev: int, stream: int) -> tuple:
    """The scratch of one operator that exists for a call made now, or _NO_WORKSPACE.

    A captured graph keeps the addresses of its calls, so it shares no scratch with eager
    calls (which replace theirs when they need more) nor with another graph."""
    if stream != 0 and _capturing():  # (the default stream cannot be captured)
        ws = _GRAPH_WORKSPACES.get((kind, dev, stream))
        return ws if ws is not None and ws[3] == _capture_id(stream) else _NO_WORKSPACE
    return _WORKSPACES.get((kind, dev, stream), _NO_WORKSPACE)


def _workspace(kind: str, nbytes: int, dev: int, stream: int, cleared: str = "counters") -> tuple:
    """(pointer, bytes, tensor) of scratch of one operator on this device and stream; when it
    is new its counters ("counters": those at the start; "all": every byte may be one) are
    zero.  Grown on demand, and left by every call as the next one, of any size, needs it.
    Within a capture it is allocated from the graph's pool, which lives as long as the
    graph, and cleared by the graph itself."""
    ws = _held(kind, dev, stream)
    if ws[2] is None or ws[1] < nbytes:
        t = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=torch.device("cuda", dev))
        t[:_lib.lib().aria_paged_workspace_counter_bytes() if cleared == "counters" else None].zero_()
        if _capturing():
            graph = _capture_id(stream)
            for key in [k for k, w in _GRAPH_WORKSPACES.items() if w[3] != graph]:
                del _GRAPH_WORKSPACES[key]  # of captures before this one: their graphs' pools hold the memory
            ws = _GRAPH_WORKSPACES[kind, dev, stream] = (t.data_ptr(), t.numel(), t, graph)
        else:
            ws = _WORKSPACES[kind, dev, stream] = (t.data_ptr(), t.numel(), t)
    return ws


def clear_workspaces() -> None:
    """Forget the scratch of the serving operators; their next calls start from new.  For use
    after a call during which a wait on the device expired (aria_q4_take_device_error() !=
    0): it may have left counters behind.  (A graph's scratch is cleared by the graph.)"""
    _WORKSPACES.clear()
    _GRAPH_WORKSPACES.clear()


def _want(t: torch.Tensor, name: str, dtype, shape, dev: int) -> int:
    """Pointer of a contiguous tensor of this type and shape on CUDA device `dev`."""
    if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
        raise TypeError(f"{name} must be a contiguous {dtype} tensor on cuda:{dev}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.data_ptr()


def _int32(**values) -> None:
    """The C ABI's counts are 32-bit; ctypes would cut larger ones off in silence."""
    for name, v in values.items():
        if not -2**31 <= v < 2**31:
            raise ValueError(f"{name} = {v} does not fit 32 bits")


class PagedKV:
    """One layer's cache.  k_pages, v_pages: f16 or bf16 [num_pages][page_size]
    [kv_heads][head_dim], any strides that are multiples of 8 with contiguous head
    rows (a transposed view of pages stored head by head is one); block_table: int32
    [M][max_pages], -1 (or any entry outside the pool) where a sequence has no page;
    lens: int32 [M], the slots in use.  The tensors are kept and read at every call:
    write them in place to change pages, table or lengths."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor):
        if not k_pages.is_cuda or k_pages.dim() != 4 or k_pages.dtype not in _DTYPES:
            raise TypeError("k_pages must be a 4-D f16 or bf16 CUDA tensor")
        dev = k_pages.device
        if (v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype or v_pages.device != dev
                or v_pages.stride() != k_pages.stride()):
            raise ValueError("v_pages must match k_pages in shape, type, device and strides")
        if k_pages.stride(3) != 1:
            raise ValueError("the head dimension of the pages must be contiguous")
        if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.device != dev or (
                block_table.stride(1) != 1 and block_table.shape[1] > 1):
            raise TypeError("block_table must be int32 [M][max_pages] on the pages' device, rows contiguous")
        M = block_table.shape[0]
        _want(lens, "lens", torch.int32, (M,), dev.index)
        n, ps, H, dh = k_pages.shape
        self.k_pages, self.v_pages, self.block_table, self.lens = k_pages, v_pages, block_table, lens
        self.M, self.kv_heads, self.head_dim, self.page_size = M, H, dh, ps
        self.slots = ps * block_table.shape[1]
        self.dtype, self.device, self.index = k_pages.dtype, dev, dev.index
        self._new_shape = (M, H, dh)
        self._scale = 1.0 / math.sqrt(dh)
        # strides of dimensions of one entry are never used: 8 keeps them valid
        st = [s if c > 1 else 8 for s, c in zip(k_pages.stride(), k_pages.shape)]
        self._c = PagedKVStruct(k_pages.data_ptr(), v_pages.data_ptr(), st[0], st[1], st[2], n, ps, H, dh,
                                _DTYPES[k_pages.dtype], block_table.data_ptr(),
                                block_table.stride(0) if M > 1 else block_table.shape[1], block_table.shape[1],
                                lens.data_ptr())
        self._ref, self._lens_ptr = ctypes.addressof(self._c), lens.data_ptr()
        self._ws_bytes: dict = {}

    def _workspace_bytes(self, heads: int, weights: bool) -> int:
        key = (heads, weights)
        n = self._ws_bytes.get(key)
        if n is None:
            n = _lib.lib().aria_attention_paged_workspace_bytes(self._ref, self.M, heads, weights)
            self._ws_bytes[key] = n
        return n

    def _evict_bytes(self, keep: int) -> int:
        n = self._ws_bytes.get(keep)
        if n is None:
            n = self._ws_bytes[keep] = _lib.lib().aria_cache_evict_workspace_bytes(self._ref, self.M, keep)
        return n

    @classmethod
    def contiguous(cls, k_cache: torch.Tensor, v_cache: torch.Tensor, kv_heads: int, lens: torch.Tensor,
                   page_size: int = 16) -> "PagedKV":
        """A [M][max_seq][d] cache (what attention_prefill fills) as pages in order;
        max_seq a multiple of page_size."""
        M, max_seq, d = k_cache.shape
        if max_seq % page_size or d % kv_heads:
            raise ValueError("max_seq must be a multiple of page_size and d of kv_heads")
        per = max_seq // page_size
        table = torch.arange(M * per, dtype=torch.int32, device=k_cache.device).view(M, per)
        shape = (M * per, page_size, kv_heads, d // kv_heads)
        return cls(k_cache.view(shape), v_cache.view(shape), table, lens)


def _rows(t: torch.Tensor, name: str, kv: PagedKV, shape) -> tuple:
    """Strides of a [M][heads][head_dim] tensor with contiguous rows."""
    s = t.stride()
    if t.dtype is not kv.dtype or t.get_device() != kv.index or len(s) != 3:
        raise TypeError(f"{name} must be a 3-D {kv.dtype} tensor on cuda:{kv.index}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if s[2] != 1:
        raise ValueError(f"the head dimension of {name} must be contiguous")
    if shape[0] > 1 and shape[1] > 1:
        return s
    return (s[0] if shape[0] > 1 else 8, s[1] if shape[1] > 1 else 8, 1)  # strides of one entry are not used


def attention_paged(q: torch.Tensor, kv: PagedKV, *, k_new: torch.Tensor | None = None,
                    v_new: torch.Tensor | None = None, scale: float | None = None, out: torch.Tensor | None = None,
                    want_lse: bool = False, weights: torch.Tensor | None = None,
                    weights_out: torch.Tensor | None = None, slot_pos: torch.Tensor | None = None,
                    positions: torch.Tensor | None = None):
    """q [M][heads][head_dim] (any strides that are multiples of 8): one new token per
    sequence.  k_new, v_new [M][kv_heads][head_dim]: its own rows, stored at slot
    lens[m] and part of the attention (lens is the caller's to advance); where the table
    has no page for that slot they are neither.  Returns (out
    [M][heads][head_dim], lse f32 [M][heads] or None); a sequence without slots gives
    zeros and -inf.  scale defaults to 1 / sqrt(head_dim).

    weights f32 [M][kv_heads][cap >= kv.slots]: the running sums of the attention
    weight, updated in place or into weights_out; the new token's slot starts from 0,
    and its entry of slot_pos (int32, the same shape) becomes positions[m]."""
    stream = _stream(kv.index)
    ws = _WORKSPACES.get(("attn", kv.index, 0), _NO_WORKSPACE) if stream == 0 else _held("attn", kv.index, stream)
    r = fastcall().attention(kv._ref, kv.M, kv.kv_heads, kv.head_dim, kv.index, kv._scale if scale is None else scale,
                             ws[0], ws[1], stream, want_lse, q, k_new, v_new, out, weights, weights_out, slot_pos,
                             positions)
    if r is not None:
        return r
    # another device is current, the first call on a stream, one that needs more scratch, or
    # something to say
    if _current_device() != kv.index:  # a launch goes to the current device
        with torch.cuda.device(kv.index):
            return attention_paged(q, kv, k_new=k_new, v_new=v_new, scale=scale, out=out, want_lse=want_lse,
                                   weights=weights, weights_out=weights_out, slot_pos=slot_pos, positions=positions)
    shape = q.shape
    if len(shape) != 3 or shape[0] != kv.M or shape[2] != kv.head_dim or shape[1] == 0 or shape[1] % kv.kv_heads:
        raise ValueError(f"q must be [{kv.M}][heads][{kv.head_dim}] with heads a multiple of {kv.kv_heads}")
    dev, heads = kv.index, shape[1]
    qs = _rows(q, "q", kv, shape)
    kp = vp = None
    ns = (0, 0)
    if k_new is not None and v_new is not None:
        ns = _rows(k_new, "k_new", kv, kv._new_shape)
        if _rows(v_new, "v_new", kv, kv._new_shape) != ns:
            raise ValueError("k_new and v_new must have the same strides")
        kp, vp = k_new.data_ptr(), v_new.data_ptr()
    elif k_new is not None or v_new is not None:
        raise ValueError("k_new and v_new go together")
    if out is None:
        out = torch.empty(shape, dtype=kv.dtype, device=kv.device)
    os_ = _rows(out, "out", kv, shape)
    lse = torch.empty((shape[0], heads), dtype=torch.float32, device=kv.device) if want_lse else None
    wi = wo = sp = pp = None
    cap = 0
    if weights is not None:
        wshape = weights.shape
        if len(wshape) != 3 or wshape[0] != kv.M or wshape[1] != kv.kv_heads:
            raise ValueError("weights must be [M][kv_heads][cap]")
        cap = wshape[2]
        wi = _want(weights, "weights", torch.float32, wshape, dev)
        wo = wi if weights_out is None else _want(weights_out, "weights_out", torch.float32, wshape, dev)
        if slot_pos is not None:
            if positions is None or k_new is None:
                raise ValueError("slot_pos needs positions and k_new")
            sp = _want(slot_pos, "slot_pos", torch.int32, wshape, dev)
            pp = _want(positions, "positions", torch.int32, (kv.M,), dev)
    elif weights_out is not None or slot_pos is not None:
        raise ValueError("weights_out and slot_pos need weights")
    ws = _workspace("attn", kv._workspace_bytes(heads, wi is not None), dev, stream)
    call("aria_attention_paged", kv._ref, kv.M, heads, q.data_ptr(), qs[0], qs[1], kp, vp, ns[0], ns[1],
         scale if scale is not None else kv._scale, out.data_ptr(), os_[0], os_[1],
         lse.data_ptr() if lse is not None else None, wi, wo, cap, sp, pp, ws[0], ws[1], stream)
    return out, lse


def prompt_weights(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor, *, out: torch.Tensor | None = None,
                   scale: float | None = None, first_query: int = 0) -> torch.Tensor:
    """The attention weight each position of a prompt received from the queries at
    positions >= first_query: q [B][T][heads][dh], k [B][T][kv_heads][dh] (strides
    multiples of 8; views of a packed QKV output serve), lse f32 [B][heads][T] as the
    prompt's causal attention returned it.  Writes out[:, :, :T] of an f32
    [B][kv_heads][>= T] tensor with contiguous rows (a new [B][kv_heads][T] one by
    default) and returns it.  head_dim 64 or 128."""
    dev = q.get_device()  # -1 on the CPU
    if out is not None and dev >= 0:
        stream = _stream(dev)
        ws = _held("prompt", dev, stream)
        if fastcall().prompt(q, k, lse, out, scale if scale is not None else 1.0 / math.sqrt(q.shape[-1]), first_query,
                             ws[0], ws[1], stream):
            return out
    if dev >= 0 and _current_device() != dev:
        with torch.cuda.device(dev):
            return prompt_weights(q, k, lse, out=out, scale=scale, first_query=first_query)
    _int32(first_query=first_query)
    if q.dim() != 4 or k.dim() != 4 or q.dtype not in _DTYPES or k.dtype is not q.dtype or not q.is_cuda:
        raise TypeError("q and k must be 4-D f16 or bf16 CUDA tensors of one type")
    B, T, heads, dh = q.shape
    kvh = k.shape[2]
    if k.shape != (B, T, kvh, dh) or k.get_device() != dev or kvh == 0 or heads % kvh:
        raise ValueError("k must be [B][T][kv_heads][dh] with heads a multiple of kv_heads")
    qs, ks = q.stride(), k.stride()
    if qs[3] != 1 or ks[3] != 1:
        raise ValueError("the head dimension of q and k must be contiguous")
    if B == 1 or T == 1 or heads == 1 or kvh == 1:  # strides of one entry are not used
        qs = [s if c > 1 else 8 for s, c in zip(qs, q.shape)]
        ks = [s if c > 1 else 8 for s, c in zip(ks, k.shape)]
    lp = _want(lse, "lse", torch.float32, (B, heads, T), dev)
    if out is None:
        out = torch.empty((B, kvh, T), dtype=torch.float32, device=q.device)
    if out.dtype is not torch.float32 or out.get_device() != dev or out.dim() != 3 or out.shape[:2] != (B, kvh) or \
            out.shape[2] < T or (out.stride(2) != 1 and out.shape[2] > 1):
        raise ValueError("out must be f32 [B][kv_heads][>= T] with contiguous rows")
    stream = _stream(dev)
    ws = _workspace("prompt", _lib.lib().aria_prompt_weights_workspace_bytes(B, T, heads, kvh, first_query), dev, stream)
    call("aria_prompt_weights", q.data_ptr(), qs[0], qs[1], qs[2], k.data_ptr(), ks[0], ks[1], ks[2],
         _DTYPES[q.dtype], B, T, heads, kvh, dh, lp, scale if scale is not None else 1.0 / math.sqrt(dh),
         first_query, out.data_ptr(), out.stride(0), out.stride(1), ws[0], ws[1], stream)
    return out


def evict(kv: PagedKV, weights: torch.Tensor, slot_pos: torch.Tensor, next_pos: torch.Tensor, keep: int, *,
          recent: int = 0, sinks: int = 0, weights_out: torch.Tensor | None = None,
          slot_pos_out: torch.Tensor | None = None, lens_out: torch.Tensor | None = None) -> torch.Tensor:
    """Cut every row of more than `keep` slots down to `keep`: the positions >= next_pos[m]
    - recent and < sinks stay, then the largest weights (ties: the lowest slot).  The
    survivors past `keep` move into the freed slots, in order; weights f32 and slot_pos
    int32 [M][kv_heads][cap] move with them, in place or into the given outputs, and freed
    slots end with weight 0 and position -1.  Returns lens_out (int32 [M], another tensor
    than kv.lens) = min(lens, keep); copy it to kv.lens once every layer that shares kv.lens
    has been evicted from."""
    if lens_out is None:
        lens_out = torch.empty_like(kv.lens)
    dev = kv.index
    stream = _stream(dev)
    ws = _held("evict", dev, stream)
    if fastcall().evict(kv._ref, kv.M, kv.kv_heads, dev, kv._lens_ptr, keep, recent, sinks, ws[0], ws[1], stream, weights,
                        slot_pos, next_pos, weights_out, slot_pos_out, lens_out):
        return lens_out
    if _current_device() != kv.index:
        with torch.cuda.device(kv.index):
            return evict(kv, weights, slot_pos, next_pos, keep, recent=recent, sinks=sinks, weights_out=weights_out,
                         slot_pos_out=slot_pos_out, lens_out=lens_out)
    _int32(keep=keep, recent=recent, sinks=sinks)
    shape = weights.shape
    if weights.dim() != 3 or shape[:2] != (kv.M, kv.kv_heads):
        raise ValueError("weights must be [M][kv_heads][cap]")
    wi = _want(weights, "weights", torch.float32, shape, dev)
    pi = _want(slot_pos, "slot_pos", torch.int32, shape, dev)
    wo = wi if weights_out is None else _want(weights_out, "weights_out", torch.float32, shape, dev)
    po = pi if slot_pos_out is None else _want(slot_pos_out, "slot_pos_out", torch.int32, shape, dev)
    npp = _want(next_pos, "next_pos", torch.int32, (kv.M,), dev)
    lp = _want(lens_out, "lens_out", torch.int32, (kv.M,), dev)
    if lp == kv.lens.data_ptr() and kv.M > 0:
        raise ValueError("lens_out must not be kv.lens")
    ws = _workspace("evict", kv._evict_bytes(keep), dev, stream)
    call("aria_cache_evict", kv._ref, kv.M, wi, wo, pi, po, shape[2], npp, keep, recent, sinks, lp, ws[0], ws[1], stream)
    return lens_out
