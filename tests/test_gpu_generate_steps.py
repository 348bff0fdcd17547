"""BoundedDecoder through the methods that it shares with Decoder."""
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


@pytest.mark.parametrize("way", ["step", "step at positions", "run", "advance"])
def test_every_way_to_step_is_the_decoders(weights, way):
    """After the same prompt, without eviction: the logits of Decoder.step, up to the rounding of the
    f16 attention outputs (2e-2, as derived in test_gpu_generate.py), and every slot in its place."""
    from aria_b200.decoder import Decoder
    from aria_b200.generate import BoundedDecoder
    M, T, n = 3, 20, 9
    p = _prompts(M, T)
    a, b = Decoder(weights, M), BoundedDecoder(weights, M, budget=100, slack=8)
    la = a.prefill(p)
    b._prefill_buffers(T)["tok"].copy_(p.to(torch.int32).reshape(-1))
    assert torch.equal(b.run_prefill(T), la)  # (what prefill calls, and the caller may)
    tok = la.view(M, T, -1)[:, -1].argmax(1).to(torch.int32)
    for s in range(n):
        xa = a.step(tok, [T + s] * M).clone()
        if way == "step":
            xb = b.step(tok)
        elif way == "step at positions":
            xb = b.step(tok, [T + s] * M)
        else:
            b.tokens.copy_(tok)
            xb = getattr(b, way)()
        assert (xa - xb).abs().max().item() <= 2e-2, s
        tok = xa.argmax(1).to(torch.int32)
    assert b.used == b.position == T + n and b.lens.tolist() == b.positions.tolist() == [T + n] * M
    for i in range(3):
        assert torch.equal(b.slot_pos[i][:, :, :T + n],
                           torch.arange(T + n, dtype=torch.int32, device="cuda").expand(M, 4, T + n))
        # the caches hold the same rows, up to what the layers below differ by
        assert (a.k_cache[i][:, :T + n].float() - b.k_cache[i][:, :T + n].float()).abs().max().item() <= 2e-2


def test_steps_without_a_prompt(weights):
    from aria_b200.decoder import Decoder
    from aria_b200.generate import BoundedDecoder
    a, b = Decoder(weights, 2), BoundedDecoder(weights, 2, budget=64, slack=8)
    for s in range(5):
        tok = [17 * s + 3, 5 * s]
        assert (a.step(tok, [s, s]) - b.step(tok)).abs().max().item() <= 2e-2


def test_positions_out_of_order_are_refused(weights):
    from aria_b200.generate import BoundedDecoder
    b = BoundedDecoder(weights, 2, budget=100, slack=8)
    b.prefill(_prompts(2, 10))
    before = b.k_cache[0].clone()
    for bad in ([9, 9], [11, 11], [10, 9], [10]):
        with pytest.raises(ValueError):
            b.step([1, 2], bad)
    assert torch.equal(b.k_cache[0], before) and b.used == 10
    b.step([1, 2], torch.tensor([10, 10]))


def test_launches_are_counted(weights):
    """The kernels of a step and of a prompt: the paged attention is two where the decoder's is one,
    the prompt weights are one more."""
    from aria_b200.decoder import Decoder
    from aria_b200.generate import BoundedDecoder
    a, b = Decoder(weights, 2), BoundedDecoder(weights, 2, budget=100, slack=8)
    assert b.launches == a.launches + 3 and b.prefill_launches() == a.prefill_launches() + 3
    assert b.prefill_launches(False) == a.prefill_launches(False)


def test_a_capture_is_refused(weights):
    from aria_b200.generate import BoundedDecoder
    b = BoundedDecoder(weights, 1, budget=100, slack=8)
    b.prefill(_prompts(1, 10))
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            b.run()
    torch.cuda.synchronize()
    assert b.used == b.position == 10
    b.step([3])


def test_positions_past_the_cache_have_their_own_embedding(weights):
    """Bounded caches of 128 slots, sequences of 230 positions: the logits are those of weights whose
    position table was made for 512, bit for bit (nothing else depends on max_seq)."""
    from aria_b200.decoder import DecoderWeights
    from aria_b200.generate import BoundedDecoder
    M, T, steps = 2, 90, 140
    wide = DecoderWeights(weights.cfg, max_seq=512)
    kw = dict(budget=48, recent=8, sinks=2, slack=8)
    a, b = BoundedDecoder(weights, M, **kw), BoundedDecoder(wide, M, **kw)
    p = _prompts(M, T)
    assert torch.equal(a.prefill(p), b.prefill(p))
    for s in range(steps):
        tok = torch.full((M,), (37 * s) % 1000, dtype=torch.int32, device="cuda")
        for d in (a, b):
            d.tokens.copy_(tok)
        assert torch.equal(a.advance(), b.advance()), T + s
    assert a.positions.tolist() == [T + steps] * M
    assert torch.equal(BoundedDecoder(weights, M, **kw).generate(p, steps),
                       BoundedDecoder(wide, M, **kw).generate(p, steps))


def test_lengths_that_are_no_multiple_of_a_page():
    """max_seq 101 in pages of 16 and of 7: the same tokens as in pages of 1 (whose slots are the same)."""
    from aria_b200.decoder import DecoderWeights
    from aria_b200.efkolos import EfkolosConfig
    from aria_b200.generate import BoundedDecoder
    w = DecoderWeights(EfkolosConfig(num_layers=1, d_model=128, num_heads=2, ffn_dim=256, vocab_size=200), max_seq=101)
    p = torch.randint(0, 200, (2, 101), generator=torch.Generator().manual_seed(1))
    tokens = [BoundedDecoder(w, 2, budget=80, slack=20, page_size=ps).generate(p, 40) for ps in (1, 16, 7)]
    assert torch.equal(tokens[0], tokens[1]) and torch.equal(tokens[0], tokens[2])


@pytest.mark.parametrize("prompt", [40, 41, 401])
def test_the_command(monkeypatch, capsys, prompt):
    """python -m aria_b200.generate for prompts of any length."""
    import sys

    from aria_b200 import generate
    monkeypatch.setattr(sys, "argv", ["generate", "--prompt", str(prompt), "--tokens", "9", "--budget", "48", "--layers",
                                      "1"])
    generate.main()
    assert f"2 sequences x ({prompt} + 9) tokens" in capsys.readouterr().out
