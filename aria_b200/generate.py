"""Generation with a bounded cache: the decoder of aria_b200/decoder.py over a paged
KV cache that keeps the `budget` slots of each head with the largest accumulated
attention weight (and the newest and first positions), its logits adjusted and the next
token chosen on the GPU.

    dec = BoundedDecoder(DecoderWeights(EfkolosConfig()), M=2, budget=256)
    tokens = dec.generate(prompts, 100, repetition=1.2)

Per prompt and layer: the prompt's attention fills the cache and returns its log-sum-exp
rows, `prompt_weights` adds up what every position received, `evict` cuts the cache to the
budget.  Per token and layer: `attention_paged` stores the new rows, attends and adds to
the weights; per token: `logits.adjust`; and once a row has outgrown the budget by `slack`
slots, `evict` again.  No call waits for the GPU.

    python -m aria_b200.generate --prompt 400 --tokens 200 --budget 128
"""
from __future__ import annotations

import argparse

import torch

from .decoder import Decoder, DecoderWeights, sinusoidal_positions
from .logits import adjust
from .paged import PagedKV, attention_paged, evict, prompt_weights

__all__ = ["BoundedDecoder"]


class BoundedDecoder(Decoder):
    """A Decoder whose caches (weights.max_seq slots per sequence, in pages) never hold
    more than budget + slack slots of a sequence after its prompt.  recent, sinks: the
    newest and first positions that are always kept.  Sequences grow past max_seq: their
    position table, a formula, is extended as they do."""

    def __init__(self, weights: DecoderWeights, M: int = 1, *, budget: int = 256, recent: int = 32, sinks: int = 4,
                 slack: int = 16, page_size: int = 16, device="cuda"):
        if page_size <= 0 or not 0 < budget <= budget + slack < weights.max_seq or recent + sinks > budget:
            raise ValueError("needs a page_size, recent + sinks <= budget and budget + slack < max_seq = "
                             f"{weights.max_seq}")
        cap = -(-weights.max_seq // page_size) * page_size  # whole pages
        super().__init__(weights, M, device, cache_rows=cap)
        cfg = self.cfg
        self.budget, self.recent, self.sinks, self.slack = budget, recent, sinks, slack
        self.lens = torch.zeros(M, dtype=torch.int32, device=device)
        self._lens_next = torch.zeros_like(self.lens)
        self.kv = [PagedKV.contiguous(k, v, cfg.num_heads, self.lens, page_size)
                   for k, v in zip(self.k_cache, self.v_cache)]
        shape = (M, cfg.num_heads, cap)
        self.weights = [torch.zeros(shape, dtype=torch.float32, device=device) for _ in self.kv]
        self.slot_pos = [torch.zeros(shape, dtype=torch.int32, device=device) for _ in self.kv]
        self._prompt_pos = torch.arange(cap, dtype=torch.int32, device=device).expand(shape)
        self.used = 0      # slots in use, the same for every sequence
        self.position = 0  # of the next token, the same for every sequence

    def _attend(self, i: int) -> None:
        M, H, dh = self.M, self.cfg.num_heads, self.cfg.head_dim
        x = self.qkv.view(M, 3, H, dh)
        attention_paged(x[:, 0], self.kv[i], k_new=x[:, 1], v_new=x[:, 2], out=self.att.view(M, H, dh),
                        weights=self.weights[i], slot_pos=self.slot_pos[i], positions=self.positions)

    def _reach(self, positions: int) -> None:
        """Rows of the position table for this many positions."""
        rows = self.pos_embed.shape[0]
        if positions > rows:
            table = sinusoidal_positions(max(positions, 2 * rows), self.cfg.d_model, self.pos_embed.device)
            table[:rows] = self.pos_embed
            self.pos_embed = table

    def _evict(self) -> None:
        """Every layer's rows down to the budget (they share one length)."""
        if self.used <= self.budget:
            return
        for i, kv in enumerate(self.kv):
            evict(kv, self.weights[i], self.slot_pos[i], self.positions, self.budget, recent=self.recent,
                  sinks=self.sinks, lens_out=self._lens_next)
        self.lens.copy_(self._lens_next)
        self.used = self.budget

    def run_prefill(self, T: int, fill_cache: bool = True, after_attention=None) -> torch.Tensor:
        """Decoder.run_prefill; with fill_cache the caches then hold at most `budget` slots and
        self.positions the position of the next token."""
        if not fill_cache:
            return super().run_prefill(T, False, after_attention)
        M, H, dh = self.M, self.cfg.num_heads, self.cfg.head_dim

        def count(i, qkv, lse):
            x = qkv.view(M, T, 3, H, dh)
            prompt_weights(x[:, :, 0], x[:, :, 1], lse, out=self.weights[i])
            self.slot_pos[i].copy_(self._prompt_pos)
            if after_attention is not None:
                after_attention(i, qkv, lse)

        logits = super().run_prefill(T, True, count)
        self.positions.fill_(T)
        self.lens.fill_(T)
        self.used = self.position = T
        self._evict()
        return logits

    def run(self) -> torch.Tensor:
        """One step for self.tokens at self.positions, after which both the lengths and the
        positions stand at the next token; returns the f32 logits [M][vocab].  (Decoder.run
        leaves positions to the caller; here the caches' lengths move with them.)  Not for
        graphs: when to evict is decided on the host."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a BoundedDecoder's step cannot be captured: evictions are decided on the host")
        self._reach(self.position + 1)
        logits = super().run()
        self.positions.add_(1)
        self.lens.add_(1)
        self.used += 1
        self.position += 1
        if self.used >= self.budget + self.slack:
            self._evict()
        return logits

    def advance(self) -> torch.Tensor:
        """run() under the name that says what it does."""
        return self.run()

    def step(self, tokens, positions=None) -> torch.Tensor:
        """The next token of every sequence.  Tokens are stored in the order of the calls, so
        positions, where given, have to be the next ones: self.position for every sequence."""
        if positions is not None:
            at = torch.as_tensor(positions).reshape(-1).tolist()
            if at != [self.position] * self.M:
                raise ValueError(f"the next position of every sequence is {self.position}, got {at}")
        self.tokens.copy_(torch.as_tensor(tokens, dtype=torch.int32))
        return self.run()

    @property
    def launches(self) -> int:
        """Kernels of one run, without the evictions that come every `slack` steps."""
        return super().launches + self.cfg.num_layers

    def prefill_launches(self, fill_cache: bool = True) -> int:
        """Kernels of one run_prefill, without the eviction at its end."""
        return super().prefill_launches(fill_cache) + (self.cfg.num_layers if fill_cache else 0)

    def generate(self, prompts, steps: int, *, repetition: float = 1.0, frequency: float = 0.0, presence: float = 0.0,
                 bias_tokens: torch.Tensor | None = None, bias_values: torch.Tensor | None = None,
                 allowed: torch.Tensor | None = None) -> torch.Tensor:
        """Greedy tokens [M][steps] (int32, on the device) after prompts [M][T]; the
        penalties count the prompt (repetition) and what was generated (all three), biases
        and the mask are those of logits.adjust."""
        prompts = torch.as_tensor(prompts, dtype=torch.int32)
        M, T = self.M, prompts.shape[1]
        dev = self.h.device
        self._reach(T + steps)
        history = torch.zeros(M, T + steps, dtype=torch.int32, device=dev)
        logits = self.prefill(prompts).view(M, T, -1)[:, -1].float().contiguous()
        history[:, :T] = prompts.to(dev)
        n, n_prompt = (torch.full((M,), T, dtype=torch.int32, device=dev) for _ in range(2))
        params = {k: torch.full((M,), v, dtype=torch.float32, device=dev)
                  for k, v in (("repetition", repetition), ("frequency", frequency), ("presence", presence))}
        for s in range(steps):
            adjust(logits, out=logits, history=history, history_lens=n, prompt_lens=n_prompt, bias_tokens=bias_tokens,
                   bias_values=bias_values, allowed=allowed, token=self.tokens, **params)
            history[:, T + s] = self.tokens
            n.add_(1)
            if s + 1 < steps:
                logits = self.advance()
        return history[:, T:]


def main() -> None:
    from .efkolos import EfkolosConfig
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--sequences", type=int, default=2)
    ap.add_argument("--prompt", type=int, default=400)
    ap.add_argument("--tokens", type=int, default=200)
    ap.add_argument("--budget", type=int, default=128)
    ap.add_argument("--layers", type=int, default=20)
    a = ap.parse_args()
    cfg = EfkolosConfig(num_layers=a.layers)
    dec = BoundedDecoder(DecoderWeights(cfg, max_seq=max(a.prompt, a.budget) + 64), a.sequences, budget=a.budget)
    g = torch.Generator().manual_seed(0)
    prompts = torch.randint(0, cfg.vocab_size, (a.sequences, a.prompt), generator=g)
    dec.generate(prompts, 4, repetition=1.2)  # (first launches)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    tokens = dec.generate(prompts, a.tokens, repetition=1.2, frequency=0.1)
    end.record()
    end.synchronize()
    ms = start.elapsed_time(end)
    print(tokens[:, :16].tolist())
    print(f"{a.sequences} sequences x ({a.prompt} + {a.tokens}) tokens, at most {a.budget + dec.slack} cached: "
          f"{ms:.1f} ms")


if __name__ == "__main__":
    main()
