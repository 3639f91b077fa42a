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


def plain_evicting(model, prompt, new_tokens, budget, sinks, recent, window, slack):
    """generate_evicting token by token in float64: every layer, sequence and key/value head keeps a list of (rotated key, value,
    collected weight).  -> (tokens, how often it evicted, smallest relative gap between the lightest slot kept and the
    heaviest dropped, smallest gap between the two largest logits): the gaps say how far float32 may be off."""
    import copy
    import math

    from bittorch_b200.utils.decoder import apply_rope_positions
    from tests import cache_reference as ref

    model = copy.deepcopy(model).cpu().double()
    cfg = model.cfg
    hkv, group = cfg.n_kv_heads, cfg.n_heads // cfg.n_kv_heads
    out, evictions, gap, margin = [], 0, math.inf, math.inf
    with torch.no_grad():
        for b in range(prompt.shape[0]):
            seq = prompt[b].tolist()
            state = [[[] for _ in range(hkv)] for _ in model.blocks]

            def feed(token, at):
                x = model.tok(torch.tensor([[token]]))
                for block, heads in zip(model.blocks, state):
                    q, k, v = block.attn._qkv(block.norm1(x))
                    q, k = (apply_rope_positions(y, model.rope_cos, model.rope_sin, torch.tensor([[at]])) for y in (q, k))
                    row = []
                    for h, slots in enumerate(heads):
                        slots.append([k[0, h, 0], v[0, h, 0], 0.0])
                        keys, values = torch.stack([s[0] for s in slots]), torch.stack([s[1] for s in slots])
                        for j in range(group):
                            p = torch.softmax(keys @ q[0, h * group + j, 0] / math.sqrt(cfg.head_dim), 0)
                            row.append(p @ values)
                            if at >= len(prompt[b]) - window:
                                for s, w in zip(slots, p.tolist()):
                                    s[2] += w
                    x = x + block.attn.proj(torch.cat(row)[None, None])
                    x = x + block.mlp(block.norm2(x))
                logits = model.head(model.norm(x))[0, 0]
                top = logits.topk(2).values
                return int(logits.argmax()), float(top[0] - top[1])

            def evict():
                nonlocal evictions, gap
                for heads in state:
                    for h, slots in enumerate(heads):
                        mass = torch.tensor([s[2] for s in slots], dtype=torch.float64)
                        keep = ref.keep_slots(mass, len(slots), budget, sinks, recent)
                        if len(keep) < len(slots):
                            evictions += 1
                            middle = range(sinks, len(slots) - recent)
                            kept, dropped = [mass[i] for i in middle if i in keep], [mass[i] for i in middle if i not in keep]
                            if kept:
                                gap = min(gap, float(min(kept) / max(dropped)) - 1)
                        heads[h] = [slots[i] for i in keep]

            for at, token in enumerate(seq):
                nxt, clear = feed(token, at)
            evict()
            filled = min(len(seq), budget)
            for i in range(1, new_tokens + 1):
                seq.append(nxt)
                margin = min(margin, clear)
                if i == new_tokens:
                    break
                if filled == budget + slack:
                    evict()
                    filled = budget
                nxt, clear = feed(nxt, len(seq) - 1)
                filled += 1
            out.append(seq)
    return torch.tensor(out), evictions, gap, margin


@pytest.mark.parametrize("budget,sinks,recent,window,slack,prompt", [(10, 2, 3, 6, 3, 17), (14, 3, 11, 1, 2, 9)])
def test_a_bounded_cache_against_the_plain_loop(monkeypatch, budget, sinks, recent, window, slack, prompt):
    """Lengths, positions, weights and slots through several evictions in place.  Keys, values and weights in float32 are off by
    about 1e-6 of themselves; the gaps show that no choice of a token or a slot is closer than that."""
    model = _model()
    tokens = _prompt(2, prompt, 5)
    want, evictions, gap, margin = plain_evicting(model, tokens, 14, budget, sinks, recent, window, slack)
    assert evictions >= 8 and gap > 1e-4 and margin > 1e-4
    with on_the_cpu(monkeypatch):
        got = model.generate_evicting(tokens, 14, budget=budget, sinks=sinks, recent=recent, window=window, slack=slack)
    assert torch.equal(got, want)


@pytest.mark.parametrize("tokens,parents", [
    (lambda cur: cur, torch.tensor([-2])), (lambda cur: torch.cat([cur, cur], 1), torch.tensor([[-1, 0], [-2, -1]])),
    (lambda cur: (cur + 1) % VOCAB, torch.tensor([-1])), (lambda cur: cur[:, :0], torch.zeros(0, dtype=torch.long)),
])
def test_a_draft_must_begin_with_the_current_token(monkeypatch, tokens, parents):
    """A root that is unused keeps nothing (the loop would not end), another token would be taken for the model's choice."""
    model, calls = _model(n_layers=1), []

    def draft(sequence, current):
        calls.append(1)
        assert len(calls) < 30, "no progress"
        return tokens(current), parents

    with on_the_cpu(monkeypatch):
        with pytest.raises(ValueError, match="begin with the current token"):
            model.generate_speculative(_prompt(2, 4), 6, draft)


def test_a_finished_sequence_may_have_any_tree(monkeypatch):
    """What is drafted for a sequence that has its tokens changes nothing."""
    model = _model(n_layers=1)
    prompt = _prompt(2, 4)
    want = model.generate_greedy(prompt, 9)

    def draft(sequence, current):
        """Right chains of three for the first sequence, which ends early; then an unused root there."""
        n = (sequence >= 0).sum(1)
        chain = torch.stack([want[0, (n[0] + i).clamp(max=12)] for i in range(3)])
        tokens = torch.stack([chain, current[1].expand(3)])
        tokens[0, 0] = current[0, 0] if n[0] < 13 else 0
        return tokens, torch.tensor([[-1, 0, 1] if n[0] < 13 else [-2, -2, -2], [-1, -2, -2]])

    with on_the_cpu(monkeypatch):
        assert torch.equal(model.generate_speculative(prompt, 9, draft), want)
