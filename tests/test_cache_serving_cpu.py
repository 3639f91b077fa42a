"""The decoder's serving paths with the operators' kernels compiled for the CPU: their checks, and decoding within a bounded
cache against a plain loop."""

import pytest
import torch

from tests.simt.cache_ops import on_the_cpu

VOCAB = 23


def _model(**kw):
    from bittorch_b200.utils.decoder import DecoderConfig, TernaryDecoder

    torch.manual_seed(0)
    cfg = dict(vocab_size=VOCAB, dim=32, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=48, max_seq_len=40)
    cfg.update(kw)
    model = TernaryDecoder(DecoderConfig(backend="python", **cfg)).eval()
    with torch.no_grad():
        model.head.weight.mul_(4)                                           # clear choices: a rounding decides no token
    return model


def _prompt(b, t, seed=1):
    return torch.randint(0, VOCAB, (b, t), generator=torch.Generator().manual_seed(seed))


def test_decode_tokens_in_grad_mode_and_outside_the_cache(monkeypatch):
    """No graph is built, and nothing is written for a step whose slots or positions do not exist."""
    from bittorch_b200.utils.decoder import CacheStep

    model, prompt, tokens = _model(), _prompt(2, 6), _prompt(2, 3, 2)
    with on_the_cpu(monkeypatch):
        cache = model.new_cache(2)
        with torch.no_grad():
            want = model(torch.cat([prompt, tokens], 1))[:, 6:]
            model(prompt, cache, 0)
        step = lambda at, first: CacheStep(torch.tensor(at), torch.tensor(first)[:, None] + torch.arange(3))
        before = [x.clone() for layer in cache for x in layer]
        for at, first in (([6, 38], [6, 6]), ([6, -1], [6, 6]), ([6, 6], [6, 38]), ([6, 6], [-1, 6]), ([40, 40], [6, 6])):
            with pytest.raises(ValueError, match="do not fit|negative"):
                model.decode_tokens(tokens, cache, step(at, first))
        assert all(torch.equal(x, old) for x, old in zip((x for layer in cache for x in layer), before))
        with torch.enable_grad():
            got = model.decode_tokens(tokens, cache, step([6, 6], [6, 6]))
        assert not got.requires_grad and torch.allclose(got, want, rtol=1e-4, atol=1e-4 * float(want.abs().max()))
        model.decode_tokens(tokens, cache, step([37, 9], [37, 9]))          # up to the last slot


@pytest.mark.parametrize("vocab,beams,new,most", [(70, 33, 2, 32), (70, 64, 5, 32), (70, 65, 1, 64), (5, 6, 1, 5), (5, 6, 3, 5), (70, 0, 3, 32)])
def test_beam_search_refuses_its_beams_before_it_starts(monkeypatch, vocab, beams, new, most):
    model = _model(vocab_size=vocab, n_layers=1)
    monkeypatch.setattr(model, "forward", lambda *a, **k: pytest.fail("the prompt was run"))
    with pytest.raises(ValueError, match=f"1 to {most} beams"):
        model.generate_beam(_prompt(1, 3) % vocab, beams, new)


def test_beam_search_takes_the_beams_that_it_can(monkeypatch):
    model = _model(vocab_size=70, n_layers=1)
    with on_the_cpu(monkeypatch):
        for beams, new in ((64, 1), (32, 2)):
            sequences, scores = model.generate_beam(_prompt(1, 3), beams, new)
            assert sequences.shape == (1, beams, 3 + new) and bool((scores[:, :-1] >= scores[:, 1:]).all())


@pytest.mark.parametrize("change", [dict(window=0), dict(window=-3), dict(slack=0), dict(budget=0), dict(sinks=-1), dict(recent=-1), dict(recent=11), dict(sinks=13)])
def test_a_bounded_cache_refuses_its_sizes_before_it_starts(monkeypatch, change):
    model = _model()
    for name in ("forward", "new_cache"):
        monkeypatch.setattr(model, name, lambda *a, **k: pytest.fail("the prompt was run"))
    with pytest.raises(ValueError, match="window|budget"):
        model.generate_evicting(_prompt(1, 6), 4, **{**dict(budget=12, sinks=2, window=6, slack=3), **change})
