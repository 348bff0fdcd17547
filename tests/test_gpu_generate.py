"""Generation over the bounded, paged cache (aria_b200/generate.py)."""
import numpy as np
import pytest
import torch

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


@pytest.fixture(scope="module")
def weights():
    from aria_b200.decoder import DecoderWeights
    from aria_b200.efkolos import EfkolosConfig
    return DecoderWeights(EfkolosConfig(num_layers=3, d_model=256, num_heads=4, ffn_dim=512, vocab_size=1000),
                          max_seq=128)


def _prompts(M, T):
    return torch.randint(0, 1000, (M, T), generator=torch.Generator().manual_seed(T))


def test_without_eviction_it_is_the_decoder(weights):
    """A budget that is never reached: the logits of every step are the contiguous-cache
    decoder's, up to the rounding of the f16 attention outputs (|logits| < 4; each layer's
    output differs by at most 2^-10 relative, three layers and the head: 2e-2)."""
    from aria_b200.decoder import Decoder
    from aria_b200.generate import BoundedDecoder
    M, T = 3, 20
    p = _prompts(M, T)
    a, b = Decoder(weights, M), BoundedDecoder(weights, M, budget=100, slack=8)
    la, lb = a.prefill(p), b.prefill(p)
    assert torch.equal(la, lb)
    tok = la.view(M, T, -1)[:, -1].argmax(1).to(torch.int32)
    for s in range(12):
        xa = a.step(tok, [T + s] * M).clone()
        b.tokens.copy_(tok)
        xb = b.advance()
        assert (xa - xb).abs().max().item() <= 2e-2
        tok = xa.argmax(1).to(torch.int32)
    for i in range(3):  # every query's weights add up to 1
        n = T + 12
        assert torch.allclose(b.weights[i][:, :, :n].sum(2), torch.full((M, 4), float(n), device="cuda"), rtol=2e-3)
        assert torch.equal(b.slot_pos[i][:, :, :n], torch.arange(n, dtype=torch.int32, device="cuda").expand(M, 4, n))


def test_bounded_generation(weights):
    """Through several evictions: never more than budget + slack slots, the newest and first
    positions among them, each position once; the same tokens again; tokens a mask forbids
    never appear; a repetition penalty changes the outcome."""
    from aria_b200.generate import BoundedDecoder
    from aria_b200.logits import allowed_mask
    M, T, steps = 2, 90, 70
    dec = BoundedDecoder(weights, M, budget=32, recent=8, sinks=2, slack=8)
    p = _prompts(M, T)
    ok = torch.ones(1, 1000, dtype=torch.bool, device="cuda")
    ok[:, 500:] = False
    mask = allowed_mask(ok)
    first = dec.generate(p, steps, allowed=mask).clone()
    assert first.shape == (M, steps) and int(first.max()) < 500 and int(first.min()) >= 0
    n = dec.used
    assert 32 <= n < 40 and dec.lens.tolist() == [n] * M and dec.positions.tolist() == [T + steps - 1] * M
    last = T + steps - 2
    for i in range(3):
        pos = dec.slot_pos[i][:, :, :n].cpu().numpy()
        for m in range(M):
            for h in range(4):
                got = set(pos[m, h].tolist())
                assert len(got) == n and max(got) == last and {0, 1} <= got
                assert set(range(last - (n - 32) - 7, last + 1)) <= got  # newest 8 at the last eviction, and since
        assert bool(torch.isfinite(dec.weights[i][:, :, :n]).all()) and bool((dec.weights[i][:, :, :n] > 0).all())
    assert torch.equal(dec.generate(p, steps, allowed=mask), first)
    other = dec.generate(p, steps, repetition=5.0, frequency=2.0, presence=1.0)
    assert len(np.unique(other[0].cpu().numpy())) > len(np.unique(first[0].cpu().numpy()))


def test_bounded_decoder_refuses():
    from aria_b200.decoder import DecoderWeights
    from aria_b200.efkolos import EfkolosConfig
    from aria_b200.generate import BoundedDecoder
    w = DecoderWeights(EfkolosConfig(num_layers=1, d_model=128, num_heads=2, ffn_dim=256, vocab_size=64), max_seq=64)
    with pytest.raises(ValueError):
        BoundedDecoder(w, 1, budget=64)
    with pytest.raises(ValueError):
        BoundedDecoder(w, 1, budget=8, recent=7, sinks=2)
