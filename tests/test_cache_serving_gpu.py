"""The decoder's serving paths on the operators over the key/value cache (GPU): drafted trees, beams, bounded caches, the
fused single-token step; and the operators together, as a decoding loop uses them, against their plain forms."""

import pytest
import torch

from tests import cache_reference as ref
from tests.conftest import needs_real_gpu

pytestmark = [pytest.mark.gpu, needs_real_gpu]

VOCAB = 65


def _model(dtype=torch.float32, packed=False, **kw):
    from bittorch_b200.utils.decoder import DecoderConfig, TernaryDecoder

    torch.manual_seed(0)
    cfg = dict(vocab_size=VOCAB, dim=256, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=320, max_seq_len=96)
    cfg.update(kw)
    model = TernaryDecoder(DecoderConfig(backend="cuda" if packed else "python", **cfg)).cuda().eval().to(dtype)
    with torch.no_grad():
        model.head.weight.mul_(4)                                           # clear choices: a rounding decides no token
    return model.to_inference() if packed else model


def _prompt(b, t, seed=1):
    return torch.randint(0, VOCAB, (b, t), generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("dtype,packed,tol", [(torch.float32, False, 1e-4), (torch.float32, True, 4e-2), (torch.bfloat16, False, 4e-2),
                                              (torch.bfloat16, True, 4e-2)])
def test_fused_attention_step_follows_the_plain_step(dtype, tol, packed):
    """Same weights, attention of the fixed-shape step as framework operations and as the operator: the float32 arithmetic
    differs by its order (relative 1e-6 per layer), bf16 by one rounding of the scores, the weights and the output.
    The packed form rounds every layer's input to 8 bits, and a difference of any size can move an element that lies on
    the border between two codes: by 1/127 of the row's largest, that is 1.5e-3 of the norm of a normal row of 256
    (16 largest / 3).  A float32 difference of 1e-6 does so to an element with probability 127 * 2e-6, to one of the 2500
    inputs of a pass with probability one half; sixteen such moves in one pass (which nothing but a fault would bring about)
    make 16 * 1.5e-3 = 2.4e-2 before the layers behind them.  So 4e-2 there."""
    from bittorch_b200.utils.decoder import GreedyDecodeGraph

    plain, fused = _model(dtype, packed), _model(dtype, packed, fused_attention=True)
    prompt = _prompt(3, 9)
    with torch.no_grad():
        ca, cb = plain.new_cache(3), fused.new_cache(3)
        plain(prompt, ca, 0), fused(prompt, cb, 0)
        for i in range(4):
            tok, pos = _prompt(3, 1, 10 + i), torch.tensor([9 + i]).cuda()
            a, b = plain.decode_step(tok, ca, pos).float(), fused.decode_step(tok, cb, pos).float()
            assert float((a - b).norm() / a.norm()) < tol
        first = fused(prompt, fused.new_cache(3), 0)[:, -1].argmax(-1, keepdim=True)
        cache = fused.new_cache(3)
        fused(prompt, cache, 0)
        eager = [(k.clone(), v.clone()) for k, v in cache]
        want, tok = [], first
        for i in range(12):
            want.append(tok)
            tok = fused.decode_step(tok, eager, torch.tensor([9 + i]).cuda())[:, -1].argmax(-1, keepdim=True)
    loop = GreedyDecodeGraph(fused, 3, cache=cache)
    loop.start(first, 9)
    loop.run(12)
    torch.cuda.synchronize()
    assert torch.equal(loop.history[:, 9:21], torch.cat(want, dim=1))


def test_a_drafted_tree_gets_the_logits_of_its_paths():
    """Every node's logits are those of the sequence that ends with its path, at ragged lengths."""
    from bittorch_b200 import ops

    model = _model()
    parents = torch.tensor([[-1, 0, 0, 1, 1, 2, 5], [-1, 0, 1, 2, 2, -2, -2]]).cuda()
    tree = ops.tree_mask(parents)
    lens = [11, 4]
    prompt, tokens = _prompt(2, 11), _prompt(2, 7, seed=3)
    with torch.no_grad():
        cache = model.new_cache(2)
        model(prompt, cache, 0)                                             # sequence 1 uses its first 4 slots only
        logits = model.decode_tree(tokens, cache, torch.tensor(lens).cuda(), tree)
        for b in range(2):
            for i in range(7):
                if parents[b, i] == -2:
                    continue
                path = tree[b, i].nonzero()[:, 0]
                want = model(torch.cat([prompt[b, :lens[b]], tokens[b, path]])[None])[0, -1]
                assert torch.allclose(logits[b, i], want, rtol=1e-4, atol=1e-4 * float(want.abs().max()))
    with pytest.raises(ValueError, match="do not fit"):
        model.decode_tree(tokens, cache, torch.tensor([90, 3]).cuda(), tree)


def test_speculative_decoding_gives_the_greedy_tokens():
    """Whatever is drafted: the right continuation beside wrong ones, nothing but wrong ones, the root alone."""
    model = _model()
    prompt, new = _prompt(3, 5), 40
    want = model.generate_greedy(prompt, new)
    g = torch.Generator().manual_seed(7)
    calls = []

    def oracle_draft(seq, current):
        """A chain of up to 4 right tokens with a wrong sibling at each step, of random length."""
        calls.append(1)
        b, n = seq.shape
        depth = int(torch.randint(0, 5, (1,), generator=g))
        tokens = torch.zeros(b, 1 + 2 * depth, dtype=torch.long, device="cuda")
        tokens[:, 0] = current[:, 0]
        parents = [-1]
        at = 0
        filled = (seq >= 0).sum(dim=1)
        for d in range(depth):
            right = want.gather(1, (filled + 1 + d).clamp(max=want.shape[1] - 1)[:, None])[:, 0]
            tokens[:, 1 + 2 * d] = (right + 1) % VOCAB
            tokens[:, 2 + 2 * d] = right
            parents += [at, at]
            at = 2 + 2 * d
        return tokens, torch.tensor(parents, device="cuda")

    got = model.generate_speculative(prompt, new, oracle_draft)
    assert torch.equal(got, want)
    assert len(calls) < new                                                 # several tokens a pass
    got = model.generate_speculative(prompt, 6, lambda seq, cur: (torch.cat([cur, (cur + 1) % VOCAB], 1), torch.tensor([-1, 0], device="cuda")))
    assert torch.equal(got, want[:, :11])
    full = model.generate_speculative(prompt, 91, lambda seq, cur: (cur.repeat(1, 3), torch.tensor([-1, 0, 1], device="cuda")))
    assert torch.equal(full, model.generate_greedy(prompt, 91))             # up to the last slot of the cache


def test_packed_models_serve_too():
    """The packed form on every serving path: its tokens are the choices of the same model fed with the whole sequence,
    up to what an 8-bit code on a border moves (4e-2 of the logits' scale, see above)."""
    model = _model(torch.bfloat16, packed=True)
    prompt = _prompt(2, 6)
    spec = model.generate_speculative(prompt, 20, lambda seq, cur: (torch.cat([cur, cur, (cur + 1) % VOCAB], 1), torch.tensor([-1, 0, 0], device="cuda")))
    evicting = model.generate_evicting(prompt, 20, budget=90, slack=2)
    with torch.no_grad():
        for tokens in (spec, evicting):
            assert tokens.shape == (2, 26) and torch.equal(tokens[:, :6], prompt)
            logits = model(tokens)[:, 5:-1].float()
            chosen = logits.gather(-1, tokens[:, 6:, None])[..., 0]
            assert float((logits.amax(-1) - chosen).max()) < 0.1 * float(logits.abs().max())
    sequences, scores = model.generate_beam(prompt, 3, 8)
    assert sequences.shape == (2, 3, 14) and bool((scores[:, :-1] >= scores[:, 1:]).all()) and bool(scores.isfinite().all())


@pytest.mark.parametrize("end_token", [None, 7])
def test_beam_search_is_the_plain_search(end_token):
    """generate_beam against a search that recomputes whole sequences and sorts every candidate in float64."""
    model = _model()
    prompt, beams, new = _prompt(2, 4), 4, 10
    got, scores = model.generate_beam(prompt, beams, new, end_token)
    with torch.no_grad():
        for b in range(2):
            live = [(0.0, prompt[b].tolist(), False)]
            for _ in range(new):
                cand = []
                for w, (s, seq, done) in enumerate(live):
                    if done:
                        cand.append((s, -(w * VOCAB + end_token), seq + [end_token], True))
                        continue
                    lp = torch.log_softmax(model(torch.tensor([seq]).cuda())[0, -1].double(), -1).tolist()
                    cand += [(s + lp[v], -(w * VOCAB + v), seq + [v], v == end_token) for v in range(VOCAB)]
                cand.sort(key=lambda c: (c[0], c[1]), reverse=True)
                live = [(c[0], c[2], c[3]) for c in cand[:beams]]
            assert got[b].tolist() == [seq for _, seq, _ in live]
            assert torch.allclose(scores[b].double().cpu(), torch.tensor([s for s, _, _ in live], dtype=torch.float64), atol=1e-3)


def test_a_bounded_cache_that_holds_everything_changes_nothing():
    model = _model()
    prompt = _prompt(2, 20)
    want = model.generate_greedy(prompt, 30)
    assert torch.equal(model.generate_evicting(prompt, 30, budget=96, slack=8), want)
    short = model.generate_evicting(prompt, 30, budget=12, sinks=2, recent=5, window=6, slack=3)
    assert short.shape == want.shape and torch.equal(short[:, :20], prompt) and bool(((short >= 0) & (short < VOCAB)).all())
    assert torch.equal(short[:, 20], want[:, 20])                           # the first token sees the whole prompt


def test_the_operators_together_against_their_plain_forms():
    """A decoding loop of beams over a bounded cache on the operators alone: attend (adding the weights up), select,
    reorder, evict, four rounds, every state against the plain forms in 64 bits fed with the same inputs."""
    from bittorch_b200 import ops

    g = torch.Generator().manual_seed(11)
    b, w, h, hkv, d, s, budget = 2, 3, 8, 2, 64, 24, 16
    n = 18
    k, v = (torch.randn(b * w, hkv, s, d, generator=g).bfloat16().cuda() for _ in range(2))
    mass = torch.zeros(b * w, hkv, s, device="cuda")
    lengths = torch.full((b * w,), n, dtype=torch.int64, device="cuda")
    scores = torch.randn(b, w, generator=g).cuda()
    proj = (torch.randn(h * d, 50, generator=g) / 8).cuda()
    for step in range(12):
        q = (torch.randn(b * w, h, 1, d, generator=g) * 2).bfloat16().cuda()
        new = torch.randn(2, b * w, hkv, d, generator=g).bfloat16().cuda()
        k[:, :, n], v[:, :, n] = new[0], new[1]
        want, want_mass, largest = ref.attention(q, k, v, lengths, None, None, mass)
        out = ops.tree_attention(q, k, v, lengths, mass=mass)
        half = 2.0 ** -9
        assert bool(((out.double().cpu() - want).abs() <= (half + 8e-6 * (1 + largest)) * float(v.abs().max()) + half * want.abs() + 1e-6).all())
        assert torch.allclose(mass.double().cpu(), want_mass, rtol=1e-6, atol=8e-6 * (1 + largest) * 4)
        lengths += 1
        n += 1
        logits = (out.float().transpose(1, 2).reshape(b, w, h * d) @ proj)
        wanted = ref.select(logits, scores, w)
        scores, tokens, parents = ops.beam_select(logits, scores)
        assert torch.equal(tokens.cpu(), wanted[1]) and torch.equal(parents.cpu(), wanted[2])
        before = [k.clone(), v.clone()]
        ops.reorder_cache([k, v], parents, lengths[::w].contiguous())
        source = (parents + torch.arange(b, device="cuda")[:, None] * w).reshape(-1)
        for x, old in zip((k, v), before):
            assert torch.equal(x[:, :, :n], old[source][:, :, :n])
        mass = mass[source].contiguous()
        if n == s:
            before = [k.clone(), v.clone(), mass.clone()]
            keep, counts = ops.evict_cache(k, v, mass, lengths, budget, 2, 6)
            for i in range(b * w):
                for j in range(hkv):
                    slots = ref.keep_slots(before[2][i, j].cpu(), n, budget, 2, 6)
                    assert keep[i, j].tolist() == slots
                    for x, old in zip((k, v, mass), before):
                        assert torch.equal(x[i, j, :budget], old[i, j, slots])
            lengths, n = counts, budget
