"""What is measured of the operators that serve tokens from a paged, bounded KV cache.

Four operators: attention of one new token over a paged cache (`attention_paged`), the attention weight that
every prompt position has received (`prompt_weights`), eviction from the cache by that accumulated weight
(`evict`) and the adjustment of logits before the next token is chosen (`adjust`).  `run` computes a case in
elementary torch operations in 32 bits, or, where `own` is true, through this package's entry points; `exact`
is each operator's definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ cases
def listed() -> list[dict]:
    return [
        # one user, 256 cached positions of the 14 x 64 decoder: the latency of a call
        dict(name="attend_single", op="attend", M=1, Hkv=14, G=1, dh=64, page=16, top=256, ragged=False, dtype="f16",
             append=True, weights=False, head_major=False),
        # a small batch of chats of any length (some just begun, one empty), with the weights that eviction needs
        dict(name="attend_ragged_weights", op="attend", M=16, Hkv=14, G=1, dh=64, page=16, top=2048, ragged=True,
             dtype="f16", append=True, weights=True, head_major=False),
        # few long documents with shared key/value heads of 128 (32 query heads), pages stored head by head
        dict(name="attend_long_shared", op="attend", M=3, Hkv=8, G=4, dh=128, page=64, top=32749, ragged=False,
             dtype="bf16", append=False, weights=False, head_major=True),
        # a full server: 64 sequences up to 8191 positions
        dict(name="attend_full", op="attend", M=64, Hkv=14, G=1, dh=64, page=32, top=8191, ragged=True, dtype="f16",
             append=True, weights=False, head_major=False),
        # the prompt of one user
        dict(name="prompt_short", op="prompt", B=1, T=509, Hkv=14, G=1, dh=64, dtype="f16", first=0, packed=True),
        # a batch of prompts at the decoder's full length
        dict(name="prompt_batch", op="prompt", B=4, T=2048, Hkv=14, G=1, dh=64, dtype="f16", first=0, packed=True),
        # long prompts with shared heads of 128, counted from the prompt's second quarter on
        dict(name="prompt_long_shared", op="prompt", B=2, T=8190, Hkv=8, G=4, dh=128, dtype="bf16", first=2047,
             packed=False),
        # a full cache makes room for one token at every step
        dict(name="evict_one", op="evict", M=4, Hkv=14, dh=64, page=16, top=2049, ragged=False, keep=2048, recent=256,
             sinks=4, dtype="f16", head_major=False),
        # after the prompts of 64 sequences: half of each cache goes
        dict(name="evict_half", op="evict", M=64, Hkv=14, dh=64, page=32, top=8191, ragged=True, keep=4096, recent=511,
             sinks=4, dtype="f16", head_major=False),
        # one user's next token: penalties over a short history, no grammar
        dict(name="logits_single", op="logits", M=1, V=31500, hist=300, dtype="f32", biases=3, grammar=False),
        # a batch of the decoder's f32 logits with grammar masks
        dict(name="logits_batch", op="logits", M=64, V=31500, hist=2048, dtype="f32", biases=17, grammar=True),
        # a large batch over a large, odd vocabulary, half-precision logits
        dict(name="logits_large", op="logits", M=256, V=131071, hist=4096, dtype="f16", biases=64, grammar=True),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(max(v, lo), hi)


def _size(rng, lo: int, hi: int) -> int:
    """Spread over the logarithm of the range; half of them odd."""
    v = _log_int(rng, lo, hi)
    if rng.random() < 0.5:
        v |= 1
    v = min(v, hi)
    return v if v != 3072 else 3073


def draw(rng) -> dict:
    op = rng.choice(["attend", "attend", "prompt", "evict", "logits"])
    if op == "attend":
        dh = rng.choice([32, 64, 64, 128, 128, 256])
        Hkv, G = _log_int(rng, 1, 16), rng.choice([1, 1, 2, 3, 4, 7, 8, 12, 16])
        top, M = _size(rng, 1, 65536), _size(rng, 1, 192)
        while M > 1 and M * top * Hkv * dh > 64 * 4096 * 14 * 64:
            M = max(1, M // 2)
        while M * top * Hkv * dh * max(1, G / 4) > 64 * 4096 * 14 * 64:
            top = max(1, top // 2) | 1
        return dict(op=op, M=M, Hkv=Hkv, G=G, dh=dh, page=rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 128]), top=top,
                    ragged=rng.random() < 0.6, dtype=rng.choice(["f16", "f16", "bf16"]), append=rng.random() < 0.6,
                    weights=rng.random() < 0.4, head_major=rng.random() < 0.4)
    if op == "prompt":
        dh, T = rng.choice([64, 64, 128]), _size(rng, 2, 8192)
        Hkv, G = _log_int(rng, 1, 16), rng.choice([1, 1, 2, 3, 4, 8])
        B = _size(rng, 1, 16)
        while B > 1 and B * Hkv * G * T * T > 64 * 8190 ** 2 // 2:
            B = max(1, B // 2)
        first = rng.choice([0, 0, T // 2, max(0, T - 64), rng.randrange(T)])
        return dict(op=op, B=B, T=T, Hkv=Hkv, G=G, dh=dh, dtype=rng.choice(["f16", "f16", "bf16"]), first=first,
                    packed=rng.random() < 0.5)
    if op == "evict":
        dh, Hkv = rng.choice([32, 64, 64, 128, 256]), _log_int(rng, 1, 16)
        top, M = _size(rng, 2, 65536), _size(rng, 1, 128)
        while M > 1 and M * top * Hkv * dh > 64 * 4096 * 14 * 64:
            M = max(1, M // 2)
        keep = max(1, min(top, int(top * rng.choice([0.1, 0.25, 0.5, 0.75, 0.95, 1.0]))))
        recent = rng.randrange(keep + 1) // 2
        sinks = min(4, keep - recent)
        return dict(op=op, M=M, Hkv=Hkv, dh=dh, page=rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 128]), top=top,
                    ragged=rng.random() < 0.5, keep=keep, recent=recent, sinks=sinks,
                    dtype=rng.choice(["f16", "f16", "bf16"]), head_major=rng.random() < 0.4)
    V, M = _size(rng, 257, 262144), _size(rng, 1, 512)
    while M > 1 and M * V > 256 * 131071:
        M = max(1, M // 2)
    return dict(op="logits", M=M, V=V, hist=_size(rng, 1, 16384), dtype=rng.choice(["f32", "f32", "f16", "bf16"]),
                biases=rng.choice([0, 1, 16, 100]), grammar=rng.random() < 0.6)


# ------------------------------------------------------------------ inputs
def _gen(seed: int, salt: int) -> torch.Generator:
    g = torch.Generator(device=DEVICE)
    g.manual_seed((seed * 1000003 + salt) & 0x7FFFFFFF)
    return g


def _randn(shape, dtype, g, gain: float = 1.0) -> torch.Tensor:
    if dtype == torch.float32:
        return torch.randn(shape, generator=g, device=DEVICE) * gain
    x = torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)
    return x if gain == 1.0 else x * gain


def _lens(case, g) -> list[int]:
    """Slots in use per sequence: all `top`, or spread over 0 .. top with one empty and one full.  The lengths
    are the case's; which sequence has which is the seed's."""
    M, top = case["M"], case["top"]
    if not case["ragged"]:
        return [top] * M
    rng = random.Random(M * 65537 + top)
    n = [rng.randint(0, top) for _ in range(M)]
    n[0] = top
    if M > 2:
        n[M // 2] = 0
    return [n[i] for i in torch.randperm(M, generator=g, device=DEVICE).tolist()]


def _pages(case, n: list[int], dtype, g, room: int):
    """K and V pages, and a table that scatters every sequence's pages over the pool (-1 past the last one)."""
    H, dh, ps = case["Hkv"], case["dh"], case["page"]
    width = max(1, -(-(case["top"] + room) // ps))
    need = [-(-(x + room) // ps) for x in n]
    total = sum(need) + 3
    perm = torch.randperm(total, generator=g, device=DEVICE).to(torch.int32).cpu()
    table = torch.full((len(n), width), -1, dtype=torch.int32)
    at = 0
    for m, c in enumerate(need):
        table[m, :c] = perm[at:at + c]
        at += c
    shape = (total, H, ps, dh) if case["head_major"] else (total, ps, H, dh)
    k, v = _randn(shape, dtype, g), _randn(shape, dtype, g)
    if case["head_major"]:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return k, v, table.to(DEVICE), width * ps


def prepare(case: dict, seed: int) -> dict:
    op = case["op"]
    g = _gen(seed, 17)
    st = {"case": case}
    if op == "attend":
        M, H, dh, dt = case["M"], case["Hkv"], case["dh"], _DT[case["dtype"]]
        Hq = H * case["G"]
        # lens counts the slots in use before the call; with append the call adds one
        n = [max(0, x - 1) if case["append"] else x for x in _lens(case, g)]
        st["k"], st["v"], st["table"], cap = _pages(case, n, dt, g, 1 if case["append"] else 0)
        st["lens_list"] = n
        st["lens"] = torch.tensor(n, dtype=torch.int32, device=DEVICE)
        # q, k and v of the new token lie side by side, as the QKV projection leaves them
        row = _randn((M, (Hq + 2 * H) * dh), dt, g)
        row[:, :Hq * dh] *= 2.0
        st["q"] = row[:, :Hq * dh].view(M, Hq, dh)
        st["k_new"] = row[:, Hq * dh:(Hq + H) * dh].view(M, H, dh) if case["append"] else None
        st["v_new"] = row[:, (Hq + H) * dh:].view(M, H, dh) if case["append"] else None
        st["out"] = torch.zeros(M, Hq, dh, dtype=dt, device=DEVICE)
        if case["weights"]:
            st["w"] = torch.rand(M, H, cap, generator=g, device=DEVICE)
            st["w_out"] = torch.zeros_like(st["w"])
            st["slot_pos"] = torch.arange(cap, dtype=torch.int32, device=DEVICE).expand(M, H, cap).contiguous()
            st["positions"] = st["lens"] + 5
    elif op == "prompt":
        B, T, H, dh, dt = case["B"], case["T"], case["Hkv"], case["dh"], _DT[case["dtype"]]
        Hq = H * case["G"]
        if case["packed"]:
            row = _randn((B, T, (Hq + 2 * H) * dh), dt, g)
            row[..., :Hq * dh] *= 2.0
            st["q"] = row[..., :Hq * dh].unflatten(2, (Hq, dh))
            st["k"] = row[..., Hq * dh:(Hq + H) * dh].unflatten(2, (H, dh))
        else:
            st["q"] = _randn((B, T, Hq, dh), dt, g, 2.0)
            st["k"] = _randn((B, T, H, dh), dt, g)
        # the log-sum-exp rows that the prompt's attention returned
        lse = torch.empty(B, Hq, T, device=DEVICE)
        future = torch.ones(T, T, dtype=torch.bool, device=DEVICE).triu(1)
        for b in range(B):
            for h in range(Hq):
                s = st["q"][b, :, h].float() @ st["k"][b, :, h // case["G"]].float().T / math.sqrt(dh)
                lse[b, h] = torch.logsumexp(s.masked_fill_(future, -math.inf), 1)
        st["lse"] = lse
        st["w_out"] = torch.zeros(B, H, T, device=DEVICE)
    elif op == "evict":
        M, H, dt = case["M"], case["Hkv"], _DT[case["dtype"]]
        n = _lens(case, g)
        st["k"], st["v"], st["table"], cap = _pages(case, n, dt, g, 0)
        st["lens"] = torch.tensor(n, dtype=torch.int32, device=DEVICE)
        st["lens_list"] = n
        # a few positions receive most of the weight
        st["w"] = torch.exp(2.0 * torch.randn(M, H, cap, generator=g, device=DEVICE))
        # slots hold positions in any order once a cache has been evicted from
        pos = torch.arange(cap, dtype=torch.int32, device=DEVICE).expand(M, H, cap).contiguous()
        swap = torch.randint(0, max(n), (2,), generator=g, device=DEVICE)
        pos[:, :, swap] = pos[:, :, swap.flip(0)]
        st["slot_pos"] = pos
        st["next_pos"] = st["lens"].clone()
        st["w_out"], st["pos_out"] = torch.zeros_like(st["w"]), torch.full_like(pos, -1)
        st["lens_out"] = torch.zeros_like(st["lens"])
    else:
        M, V = case["M"], case["V"]
        dt = _DT[case["dtype"]]
        st["logits"] = (torch.randn(M, V, generator=g, device=DEVICE) * 3.0).to(dt)
        st["out"] = torch.zeros(M, V, dtype=dt, device=DEVICE)
        hl = torch.randint(0, case["hist"] + 1, (M,), generator=g, device=DEVICE, dtype=torch.int32)
        hl[0] = case["hist"]
        # frequent tokens repeat: the square of a uniform number favours low indices
        u = torch.rand(M, case["hist"], generator=g, device=DEVICE)
        st["history"] = (u * u * (V - 1)).to(torch.int32)
        st["history_lens"] = hl
        st["prompt_lens"] = (hl.float() * torch.rand(M, generator=g, device=DEVICE)).to(torch.int32)
        st["repetition"] = 1.0 + 0.3 * torch.rand(M, generator=g, device=DEVICE)
        st["frequency"] = 0.5 * torch.rand(M, generator=g, device=DEVICE)
        st["presence"] = 0.5 * torch.rand(M, generator=g, device=DEVICE)
        nb = case["biases"]
        st["bias_tokens"] = st["bias_values"] = None
        if nb:
            st["bias_tokens"] = torch.randint(-1, V, (M, nb), generator=g, device=DEVICE, dtype=torch.int32)
            st["bias_values"] = torch.randn(M, nb, generator=g, device=DEVICE) * 2.0
            # a token that is biased once only: later entries of the same token are switched off
            t, order = st["bias_tokens"].sort(dim=1, stable=True)
            dup = torch.zeros_like(t, dtype=torch.bool)
            dup[:, 1:] = t[:, 1:] == t[:, :-1]
            st["bias_tokens"] = torch.where(dup, -1, t).gather(1, order.argsort(dim=1)).contiguous()
        st["allowed"] = None
        if case["grammar"]:
            st["allowed"] = torch.randint(-2**31, 2**31, (M, (V + 31) // 32), generator=g, device=DEVICE,
                                          dtype=torch.int64).to(torch.int32)
    if own and "table" in st:
        _cache(st)
    return st


# ------------------------------------------------------------------ one pass
def run(state: dict):
    op = state["case"]["op"]
    if own:
        return {"attend": _own_attend, "prompt": _own_prompt, "evict": _own_evict, "logits": _own_logits}[op](state)
    return {"attend": _plain_attend, "prompt": _plain_prompt, "evict": _plain_evict, "logits": _plain_logits}[op](state)


def _cache(st):
    """The handle a program keeps for a layer's cache."""
    if "kv" not in st:
        from aria_b200.paged import PagedKV
        st["kv"] = PagedKV(st["k"], st["v"], st["table"], st["lens"])
    return st["kv"]


def _own_attend(st):
    from aria_b200.paged import attention_paged
    kw = {}
    if st["case"]["weights"]:
        kw = dict(weights=st["w"], weights_out=st["w_out"], slot_pos=st["slot_pos"] if st["case"]["append"] else None,
                  positions=st["positions"] if st["case"]["append"] else None)
    out, lse = attention_paged(st["q"], _cache(st), k_new=st["k_new"], v_new=st["v_new"], out=st["out"],
                               want_lse=True, **kw)
    return _attend_outputs(st, out, lse)


def _attend_outputs(st, out, lse):
    r = {"out": out, "lse": lse}
    if st["case"]["append"]:
        r["k_pages"], r["v_pages"] = st["k"], st["v"]
    if st["case"]["weights"]:
        r["weights"] = st["w_out"]
        if st["case"]["append"]:
            r["slot_pos"] = st["slot_pos"]
    return r


def _plain_attend(st):
    c = st["case"]
    M, H, G, dh, ps = c["M"], c["Hkv"], c["G"], c["dh"], c["page"]
    lse = torch.full((M, H * G), -math.inf, device=DEVICE)
    out = st["out"]
    for m in range(M):
        n = st["lens_list"][m]
        if c["append"]:
            page, slot = st["table"][m, n // ps].long().view(1), torch.full((1,), n % ps, device=DEVICE)
            st["k"][page, slot] = st["k_new"][m:m + 1]
            st["v"][page, slot] = st["v_new"][m:m + 1]
            if c["weights"]:
                st["slot_pos"][m, :, n] = st["positions"][m]
            n += 1
        if n == 0:
            out[m] = 0
            continue
        pg = st["table"][m, :-(-n // ps)].long()
        k = st["k"][pg].flatten(0, 1)[:n].float()  # [n][H][dh]
        v = st["v"][pg].flatten(0, 1)[:n].float()
        q = st["q"][m].float().view(H, G, dh)
        s = torch.matmul(q, k.permute(1, 2, 0)) * (1.0 / math.sqrt(dh))  # [H][G][n]
        mx = s.amax(2, keepdim=True)
        p = torch.exp(s - mx)
        z = p.sum(2, keepdim=True)
        p = p / z
        out[m] = torch.matmul(p, v.transpose(0, 1)).view(H * G, dh).to(out.dtype)
        lse[m] = (mx + torch.log(z)).view(-1)
        if c["weights"]:
            add = p.sum(1)
            st["w_out"][m, :, :n] = add
            old = n - 1 if c["append"] else n
            st["w_out"][m, :, :old] += st["w"][m, :, :old]
    return _attend_outputs(st, out, lse)


def _own_prompt(st):
    from aria_b200.paged import prompt_weights
    return prompt_weights(st["q"], st["k"], st["lse"], out=st["w_out"], first_query=st["case"]["first"])


def _plain_prompt(st):
    c = st["case"]
    B, T, H, G, dh, first = c["B"], c["T"], c["Hkv"], c["G"], c["dh"], c["first"]
    w = st["w_out"]
    t = torch.arange(first, T, device=DEVICE).view(-1, 1)
    hidden = torch.arange(T, device=DEVICE).view(1, -1) > t
    for b in range(B):
        for hk in range(H):
            kt = st["k"][b, :, hk].float().T
            acc = torch.zeros(T, device=DEVICE)
            for h in range(hk * G, (hk + 1) * G):
                s = st["q"][b, first:, h].float() @ kt
                p = torch.exp(s * (1.0 / math.sqrt(dh)) - st["lse"][b, h, first:].view(-1, 1))
                acc += p.masked_fill_(hidden, 0.0).sum(0)
            w[b, hk] = acc
    return w


def _own_evict(st):
    from aria_b200.paged import evict
    c = st["case"]
    evict(_cache(st), st["w"], st["slot_pos"], st["next_pos"], c["keep"], recent=c["recent"], sinks=c["sinks"],
          weights_out=st["w_out"], slot_pos_out=st["pos_out"], lens_out=st["lens_out"])
    return _evict_outputs(st)


def _evict_outputs(st):
    return {"k_pages": st["k"], "v_pages": st["v"], "weights": st["w_out"], "slot_pos": st["pos_out"],
            "lens": st["lens_out"]}


def _plain_evict(st):
    c = st["case"]
    H, ps, keep = c["Hkv"], c["page"], c["keep"]
    heads = torch.arange(H, device=DEVICE)
    st["lens_out"].copy_(st["lens"].clamp(max=keep))
    for m, n in enumerate(st["lens_list"]):
        w, pos = st["w"][m, :, :n], st["slot_pos"][m, :, :n]
        st["w_out"][m, :, :n] = w
        st["pos_out"][m, :, :n] = pos
        if n <= keep:
            continue
        safe = (pos >= st["next_pos"][m] - c["recent"]) | (pos < c["sinks"])
        rank = torch.where(safe, torch.full_like(w, math.inf), w).sort(dim=1, descending=True, stable=True)[1]
        kept = torch.zeros(H, n, dtype=torch.bool, device=DEVICE)
        kept.scatter_(1, rank[:, :keep], True)
        h_to, to = torch.nonzero(~kept[:, :keep], as_tuple=True)     # holes, head by head, lowest slot first
        h_from, frm = torch.nonzero(kept[:, keep:], as_tuple=True)   # survivors that have to move
        frm = frm + keep
        st["w_out"][m, h_to, to] = w[h_from, frm]
        st["pos_out"][m, h_to, to] = pos[h_from, frm]
        st["w_out"][m, :, keep:n] = 0.0
        st["pos_out"][m, :, keep:n] = -1
        tab = st["table"][m].long()
        for pages in (st["k"], st["v"]):
            pages[tab[to // ps], to % ps, heads[h_to]] = pages[tab[frm // ps], frm % ps, heads[h_from]]
    return _evict_outputs(st)


def _own_logits(st):
    from aria_b200.logits import adjust
    out, token = adjust(st["logits"], out=st["out"], history=st["history"], history_lens=st["history_lens"],
                        prompt_lens=st["prompt_lens"], repetition=st["repetition"], frequency=st["frequency"],
                        presence=st["presence"], bias_tokens=st["bias_tokens"], bias_values=st["bias_values"],
                        allowed=st["allowed"], want_token=True)
    return {"logits": out, "token": token}


def _plain_logits(st):
    M, V = st["logits"].shape
    x = st["logits"].float()
    at = torch.arange(st["history"].shape[1], device=DEVICE).view(1, -1)
    used = at < st["history_lens"].view(-1, 1)
    said = used & (at >= st["prompt_lens"].view(-1, 1))
    tok = st["history"].long()
    seen = torch.zeros(M, V, device=DEVICE).scatter_add_(1, tok, used.float()) > 0
    count = torch.zeros(M, V, device=DEVICE).scatter_add_(1, tok, said.float())
    r = st["repetition"].view(-1, 1)
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"].view(-1, 1) * count
    x = x - torch.where(count > 0, st["presence"].view(-1, 1).expand(M, V), torch.zeros_like(x))
    if st["bias_tokens"] is not None:
        bt = st["bias_tokens"].long()
        on = bt >= 0
        b = torch.zeros(M, V, device=DEVICE).scatter_add_(1, bt.clamp(min=0), st["bias_values"] * on)
        x = x + b
    if st["allowed"] is not None:
        v = torch.arange(V, device=DEVICE)
        bit = (st["allowed"][:, v // 32] >> (v % 32).to(torch.int32)) & 1
        x = torch.where(bit == 1, x, torch.full_like(x, -math.inf))
    best = x.amax(1, keepdim=True)
    token = torch.where(x == best, torch.arange(V, device=DEVICE), V).amin(1)
    token = torch.where(best.view(-1) > -math.inf, token, -1).to(torch.int32)
    st["out"].copy_(x)
    return {"logits": st["out"], "token": token}


# ------------------------------------------------------------------ what a pass cannot do without
def _mean_len(case) -> float:
    return case["top"] * (0.5 if case["ragged"] and case["M"] > 1 else 1.0)


def work(case: dict) -> dict:
    op = case["op"]
    if op == "attend":
        Hq, e = case["Hkv"] * case["G"], 2
        n = _mean_len(case) * case["M"]
        b = 2 * n * case["Hkv"] * case["dh"] * e + 2 * case["M"] * Hq * case["dh"] * e + 4 * case["M"] * Hq
        b += 4 * n / case["page"]
        if case["append"]:
            b += 4 * case["M"] * case["Hkv"] * case["dh"] * e
        if case["weights"]:
            b += 8 * n * case["Hkv"]
        return {"bytes": b, "flops": 4 * n * Hq * case["dh"]}
    if op == "prompt":
        B, T, Hq = case["B"], case["T"], case["Hkv"] * case["G"]
        rows = T - case["first"]
        pairs = B * Hq * (rows * (rows + 1) / 2 + rows * case["first"])
        b = B * rows * Hq * (case["dh"] * 2 + 4) + B * T * case["Hkv"] * (case["dh"] * 2 + 4)
        return {"bytes": b, "flops": 2 * case["dh"] * pairs}
    if op == "evict":
        # a slot survives with probability keep / n, so keep (1 - keep / n) holes are filled
        top, keep, rows = case["top"], case["keep"], case["M"] * case["Hkv"]
        if case["ragged"] and case["M"] > 1:
            # lengths uniform on 0 .. top: the mean of keep (1 - keep / n) over n in keep .. top
            moved = keep * ((top - keep) - keep * math.log(top / keep)) / top if top > keep else 0.0
        else:
            moved = keep * max(0.0, 1 - keep / top)
        n = _mean_len(case)
        return {"bytes": rows * (n * 16 + moved * 2 * 2 * case["dh"] * 2), "flops": rows * n}
    M, V = case["M"], case["V"]
    e = 4 if case["dtype"] == "f32" else 2
    b = M * V * 2 * e + M * case["hist"] * 0.5 * 4 + M * case["biases"] * 8
    if case["grammar"]:
        b += M * V / 8
    return {"bytes": b, "flops": 4.0 * M * V}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    return {"attend": _exact_attend, "prompt": _exact_prompt, "evict": _exact_evict, "logits": _exact_logits}[
        case["op"]](case, st)


def _exact_attend(case, st):
    """Head by head: out = sum_j exp(s_j) v_j / sum_j exp(s_j) with s = q.k / sqrt(dh)."""
    M, H, G, dh, ps = case["M"], case["Hkv"], case["G"], case["dh"], case["page"]
    out = torch.zeros(M, H * G, dh, dtype=torch.float64, device=DEVICE)
    lse = torch.full((M, H * G), -math.inf, dtype=torch.float64, device=DEVICE)
    w = None
    if case["weights"]:
        w = torch.zeros_like(st["w"], dtype=torch.float64)
    for m in range(M):
        n0 = st["lens_list"][m]
        j = torch.arange(n0, device=DEVICE)
        page, off = st["table"][m].long()[j // ps], j % ps
        for hk in range(H):
            keys, vals = st["k"][page, off, hk].double(), st["v"][page, off, hk].double()
            if case["append"]:
                keys = torch.cat([keys, st["k_new"][m, hk].double().view(1, -1)])
                vals = torch.cat([vals, st["v_new"][m, hk].double().view(1, -1)])
            if keys.shape[0] == 0:
                continue
            hs = slice(hk * G, (hk + 1) * G)
            s = st["q"][m, hs].double() @ keys.T / math.sqrt(dh)
            lse[m, hs] = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[m, hs].view(-1, 1))
            out[m, hs] = p @ vals
            if w is not None:
                w[m, hk, :keys.shape[0]] = p.sum(0)
                w[m, hk, :n0] += st["w"][m, hk, :n0].double()
    r = {"out": out, "lse": lse}
    if case["append"]:
        m = torch.arange(M, device=DEVICE)
        at = st["lens"].long()
        page = st["table"].long()[m, at // ps]
        st["k"][page, at % ps] = st["k_new"]
        st["v"][page, at % ps] = st["v_new"]
        r["k_pages"], r["v_pages"] = st["k"], st["v"]
    if case["weights"]:
        r["weights"] = w
        if case["append"]:
            m = torch.arange(M, device=DEVICE)
            st["slot_pos"][m, :, st["lens"].long()] = st["positions"].view(-1, 1).expand(M, H)
            r["slot_pos"] = st["slot_pos"]
    return r


def _exact_prompt(case, st):
    """w[b][hk][s] = sum over the group's heads and t >= max(s, first) of exp(q_t.k_s / sqrt(dh) - lse_t)."""
    B, T, H, G, dh, first = case["B"], case["T"], case["Hkv"], case["G"], case["dh"], case["first"]
    w = torch.zeros(B, H, T, dtype=torch.float64, device=DEVICE)
    step = 1024
    for b in range(B):
        for h in range(H * G):
            keys = st["k"][b, :, h // G].double()
            for t0 in range(first, T, step):
                t1 = min(T, t0 + step)
                p = torch.exp(st["q"][b, t0:t1, h].double() @ keys[:t1].T / math.sqrt(dh)
                              - st["lse"][b, h, t0:t1].double().view(-1, 1))
                w[b, h // G, :t1] += torch.tril(p, diagonal=t0).sum(0)
    return w


def _exact_evict(case, st):
    """Row by row on the host's order of (weight, slot), moved values taken as they are."""
    M, H, ps, keep = case["M"], case["Hkv"], case["page"], case["keep"]
    if sum(st["lens_list"]) * H > 1_500_000:
        return None
    w, pos = st["w"].cpu().double(), st["slot_pos"].cpu()
    w_out, pos_out = torch.zeros_like(w), torch.full_like(pos, -1)
    nxt = st["next_pos"].tolist()
    for m in range(M):
        n = st["lens_list"][m]
        tab = st["table"][m].long()
        for h in range(H):
            ww, pp = w[m, h, :n].numpy(), pos[m, h, :n].numpy()
            w_out[m, h, :n], pos_out[m, h, :n] = w[m, h, :n], pos[m, h, :n]
            if n <= keep:
                continue
            safe = (pp >= nxt[m] - case["recent"]) | (pp < case["sinks"])
            order = sorted(range(n), key=lambda i: (not safe[i], 0.0 if safe[i] else -ww[i], i))
            kept = set(order[:keep])
            to = [i for i in range(keep) if i not in kept]
            frm = sorted(i for i in kept if i >= keep)
            w_out[m, h, keep:n], pos_out[m, h, keep:n] = 0.0, -1
            if not to:
                continue
            a, b = torch.tensor(to), torch.tensor(frm)
            w_out[m, h, a], pos_out[m, h, a] = w[m, h, b], pos[m, h, b]
            a, b = a.to(DEVICE), b.to(DEVICE)
            for pages in (st["k"], st["v"]):
                pages[tab[a // ps], a % ps, h] = pages[tab[b // ps], b % ps, h]
    return {"k_pages": st["k"], "v_pages": st["v"], "weights": w_out.to(DEVICE), "slot_pos": pos_out.to(DEVICE),
            "lens": torch.tensor([min(n, keep) for n in st["lens_list"]], dtype=torch.int32, device=DEVICE)}


def _exact_logits(case, st):
    """Token by token of each row's history; the chosen token is a choice among rounded values: no value here."""
    x = st["logits"].double()
    V = case["V"]
    for m in range(case["M"]):
        n, n0 = int(st["history_lens"][m]), int(st["prompt_lens"][m])
        r, f, a = (float(st[k][m]) for k in ("repetition", "frequency", "presence"))
        tokens = st["history"][m, :n].long()
        once = torch.unique(tokens)
        l = x[m, once]
        x[m, once] = torch.where(l > 0, l / r, l * r)
        said, times = torch.unique(tokens[n0:], return_counts=True)
        x[m, said] -= f * times.double() + a
        if st["bias_tokens"] is not None:
            bt, bv = st["bias_tokens"][m].long(), st["bias_values"][m].double()
            x[m, bt[bt >= 0]] += bv[bt >= 0]
        if st["allowed"] is not None:
            bits = (st["allowed"][m].long().view(-1, 1) >> torch.arange(32, device=DEVICE)) & 1
            x[m, bits.view(-1)[:V] == 0] = -math.inf
    return {"logits": x, "token": None}
