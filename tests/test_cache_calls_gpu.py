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
