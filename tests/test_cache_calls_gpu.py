"""Calls of the operators over a key/value cache that their documentation allows and that lie off the usual path (GPU)."""

import pytest
import torch

from tests import cache_reference as ref
from tests.conftest import needs_real_gpu
from tests.test_cache_operators_gpu import _close, _ops
from tests.test_cache_serving_cpu import _model, _prompt, plain_evicting

pytestmark = [pytest.mark.gpu, needs_real_gpu]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_last_dimensions_of_one_element_with_any_stride(dtype):
    ops = _ops()
    g = torch.Generator().manual_seed(0)
    q = torch.randn(2, 5, 4, 3, generator=g).to(dtype).cuda()[..., ::3].transpose(1, 2)
    k, v = (torch.randn(2, 2, 9, 1, generator=g).to(dtype).cuda() for _ in range(2))
    lengths = torch.tensor([4, 2]).cuda()
    want, _, largest = ref.attention(q, k, v, lengths)
    _close(ops.tree_attention(q, k, v, lengths), want, float(v.abs().max()), dtype, largest)
    keep = torch.randint(0, 20, (4, 8, 5), generator=g).cuda()[:, :, ::5]
    k, v = (torch.randn(4, 8, 20, 4, generator=g).to(dtype).cuda() for _ in range(2))
    want = [x.gather(2, keep[..., None].expand(4, 8, 1, 4)) for x in (k, v)]
    out = [torch.zeros(4, 8, 1, 4, dtype=dtype, device="cuda") for _ in range(2)]
    ops.compact_cache(k, v, keep, torch.ones(4, dtype=torch.int64, device="cuda"), out=out)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    logits, scores = torch.randn(3, 4, 2, generator=g).to(dtype).cuda()[..., ::2], torch.randn(3, 4, generator=g).cuda()
    got, want = ops.beam_select(logits, scores), ref.select(logits, scores, 4)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2]) and torch.equal(got[0].double().cpu(), want[0])


@pytest.mark.parametrize("budget,sinks,recent,window,slack,prompt", [(10, 2, 3, 6, 3, 17), (6, 0, 0, 17, 1, 17), (14, 3, 11, 1, 2, 9), (24, 4, 10, 32, 8, 60)])
def test_a_bounded_cache_against_the_plain_loop(budget, sinks, recent, window, slack, prompt):
    """As on the CPU: lengths, positions, weights and slots through several evictions in place."""
    model = _model(max_seq_len=120)
    tokens = _prompt(2, prompt, 5)
    want, evictions, gap, margin = plain_evicting(model, tokens, 40, budget, sinks, recent, window, slack)
    assert evictions >= 8 and gap > 1e-4 and margin > 1e-4                  # float32 is off by about 1e-6
    got = model.cuda().generate_evicting(tokens.cuda(), 40, budget=budget, sinks=sinks, recent=recent, window=window, slack=slack)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("packed", [False, True])
def test_a_captured_step_of_several_tokens(packed):
    """decode_tokens in a graph: the checks that read lengths back are left out there, and a replay goes by what the tensors hold."""
    from bittorch_b200.utils.decoder import CacheStep
    from tests.test_cache_serving_gpu import _model as model_of, _prompt as prompt_of

    model = model_of(torch.bfloat16 if packed else torch.float32, packed)
    prompt = prompt_of(2, 20)
    cache = model.new_cache(2)
    with torch.no_grad():
        model(prompt, cache, 0)
    tokens, lengths = prompt_of(2, 5, 3), torch.tensor([20, 11]).cuda()
    step = CacheStep(lengths, lengths[:, None] + torch.arange(5, device="cuda"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            model.decode_tokens(tokens, cache, step)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = model.decode_tokens(tokens, cache, step)
    for at, seed in (([3, 17], 5), ([20, 0], 6)):
        tokens.copy_(prompt_of(2, 5, seed))
        lengths.copy_(torch.tensor(at))
        step.positions.copy_(lengths[:, None] + torch.arange(5, device="cuda"))
        mine = [tuple(x.clone() for x in layer) for layer in cache]
        want = model.decode_tokens(tokens, mine, step)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert all(torch.equal(x, y) for a, b in zip(cache, mine) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_operands_in_one_buffer(dtype):
    """Queries and output, keys and values, layers and rows side by side in one buffer: taken, and right; where they meet, refused."""
    ops = _ops()
    g = torch.Generator().manual_seed(8)
    both = torch.randn(2, 6, 3, 128, generator=g).to(dtype).cuda()
    q, out = both[..., :64], both[..., 64:]
    slots = torch.randn(2, 90, 2, 3, 64, generator=g).to(dtype).cuda()      # batch, slot, keys or values, head, column
    k, v = slots[:, :, 0].transpose(1, 2), slots[:, :, 1].transpose(1, 2)
    lengths = torch.tensor([70, 5]).cuda()
    want, _, largest = ref.attention(q, k, v, lengths)
    ops.tree_attention(q, k, v, lengths, out=out)
    _close(out, want, float(v.abs().max()), dtype, largest)
    keep, counts = torch.tensor([[[1, 4, 6]]]).cuda().expand(2, 3, 3), torch.tensor([3, 2]).cuda()
    want = [x.gather(2, keep[..., None].expand(2, 3, 3, 64)) for x in (k, v)]
    ops.compact_cache(k, v, keep, counts)
    for x, w in zip((k, v), want):
        assert torch.equal(x[0, :, :3], w[0]) and torch.equal(x[1, :, :2], w[1, :, :2])
    with pytest.raises(RuntimeError, match="same memory"):
        ops.compact_cache(slots[:, :80, 0].transpose(1, 2), slots[:, 10:, 0].transpose(1, 2), keep, counts)
    layers = torch.randn(4, 3, 2, 2, 50, 64, generator=g).to(dtype).cuda()  # row, layer, keys or values, head, slot, column
    views, parents = [layers[:, i, j] for i in range(3) for j in range(2)], torch.tensor([[1, 0], [0, 0]]).cuda()
    before, source = [x.clone() for x in views], [1, 0, 2, 2]
    ops.reorder_cache(views, parents, torch.tensor([50, 33]).cuda())
    for x, old in zip(views, before):
        for row in range(4):
            n = (50, 33)[row // 2]
            assert torch.equal(x[row, :, :n], old[source[row], :, :n]) and torch.equal(x[row, :, n:], old[row, :, n:])
    with pytest.raises(RuntimeError, match="share memory"):
        ops.reorder_cache([layers[:, 0, 0], layers[:, 0].reshape(4, -1)[:, 64:64 + 6400].view(4, 2, 50, 64)], parents, torch.tensor([50, 33]).cuda())
