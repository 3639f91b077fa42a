"""How far the log-sums of beam_select may be off (csrc/beam_select.cuh derives 54 * 2^-24), on the kernels compiled for the CPU
and on a GPU."""

import pytest
import torch

from tests import cache_reference as ref
from tests.conftest import needs_real_gpu

BOUND = 54 * 2.0 ** -24


def _rows(v, dtype, g):
    """Peaked, flat and random rows, and rows whose mass lies about 7 powers of two below the largest logit."""
    rows = [torch.full((v,), -30.0).index_fill(0, torch.randperm(v, generator=g)[:n], 0.3) + 1e-3 * torch.randn(v, generator=g) for n in (1, 2, 3, 5)]
    rows += [torch.zeros(v), torch.randn(v, generator=g) * 0.01, torch.randn(v, generator=g) * 3, torch.rand(v, generator=g) * 20 - 10]
    low = torch.full((v,), -7.7 * 0.6931) + 1e-2 * torch.randn(v, generator=g)
    low[torch.randperm(v, generator=g)[:max(1, v // 1024)]] = 0.0
    return torch.stack(rows + [low]).to(dtype)


def _errors(select, v, dtype, g):
    """Of the log-sums, one row to a sequence: the scores are chosen so that the best candidate's sum is near 0, where float32 has
    room enough."""
    logits = _rows(v, dtype, g)[:, None]
    x = logits.double()
    logsum = torch.logsumexp(x, -1)
    scores = (logsum - x.amax(-1)).float()
    got, tokens, _ = select(logits, scores)
    want = scores.double() + x.amax(-1) - logsum
    assert torch.equal(tokens[:, 0], logits[:, 0].float().argmax(-1))
    return (got.double() - want).abs().max()


def _ordered(select, dtype, g):
    """Two beams of peaked rows: the second's best is ahead by little more than twice the bound."""
    for _ in range(4):
        logits = _rows(3001, dtype, g)[[1, 3]][None]
        x = logits.double()
        best = x.amax(-1) - torch.logsumexp(x, -1)
        scores = torch.zeros(1, 2)
        scores[0, 0] = best[0, 1] - best[0, 0]                              # equal but for a rounding of at most 2^-24
        scores[0, 0] -= 2.3 * BOUND
        got = select(logits, scores)
        want = ref.select(logits, scores, 1)
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2]) and int(got[2]) == 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_log_sums_on_the_cpu(dtype):
    from tests.simt import cache_harness as H

    g = torch.Generator().manual_seed(0)
    select = lambda x, s: H.beam_select(x, s, 1)
    assert float(_errors(select, 9000, dtype, g)) <= BOUND
    _ordered(select, dtype, g)


@pytest.mark.gpu
@needs_real_gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_log_sums_on_the_gpu(dtype):
    from bittorch_b200 import ops

    g = torch.Generator().manual_seed(1)
    select = lambda x, s: [y.cpu() for y in ops.beam_select(x.cuda(), s.cuda(), 1)]
    for v in (1000, 8192, 50257):
        error = float(_errors(select, v, dtype, g))
        print(v, dtype, error)
        assert error <= BOUND
    _ordered(select, dtype, g)
