"""The host side of the operators over a key/value cache (plans, strides, pointers, checks), with the kernels compiled for
the CPU behind ``bittorch_b200.ops``."""

import pytest
import torch

from tests import cache_reference as ref
from tests.simt.cache_ops import on_the_cpu


def test_last_dimensions_of_one_element_with_any_stride(monkeypatch):
    """Where the last dimension has one element its stride says nothing: pointer and strides must be of one tensor."""
    g = torch.Generator().manual_seed(0)
    with on_the_cpu(monkeypatch) as (ops, _):
        # q [B, H, T, 1] as a slice whose last stride is 3
        q = torch.randn(2, 5, 4, 3, generator=g)[..., ::3].transpose(1, 2)
        k, v = (torch.randn(2, 2, 9, 1, generator=g) for _ in range(2))
        lengths = torch.tensor([4, 2])
        want, _, largest = ref.attention(q, k, v, lengths)
        got = ops.tree_attention(q, k, v, lengths)
        # a score is a product, rounded with its factor three times (3 2^-24 of itself); with the exponential (2^-23) and sums of
        # at most 9 terms a weight is off by (3 largest + 11) 2^-24 of itself, a quotient of two sums by twice that
        assert float((got.double() - want).abs().max()) <= 2 * (3 * largest + 12) * 2.0 ** -24 * float(v.abs().max())

        # one kept slot, a column of a longer list
        keep = torch.randint(0, 20, (4, 8, 5), generator=g)[:, :, ::5]
        k, v = (torch.randn(4, 8, 20, 4, generator=g) for _ in range(2))
        want = [x.gather(2, keep[..., None].expand(4, 8, 1, 4)) for x in (k, v)]
        out = [torch.zeros(4, 8, 1, 4) for _ in range(2)]
        ops.compact_cache(k, v, keep, torch.ones(4, dtype=torch.int64), out=out)
        assert all(torch.equal(a, b) for a, b in zip(out, want))

        # a vocabulary of one token
        logits = torch.randn(3, 4, 2, generator=g)[..., ::2]
        scores = torch.randn(3, 4, generator=g)
        got = ops.beam_select(logits, scores)
        want = ref.select(logits, scores, 4)
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2]) and torch.equal(got[0].double(), want[0])


@pytest.mark.parametrize("shape", [(2, 3, 4, 1), (2, 3, 4, 6)])
def test_plans_take_the_strides_of_the_tensor_that_is_read(monkeypatch, shape):
    """Every operand that a call may copy first: pointer and strides agree, whichever tensor is read."""
    b, h, t, d = shape
    with on_the_cpu(monkeypatch) as (ops, calls):
        q = torch.randn(b, h, t, 2 * d)[..., ::2]
        ops.tree_attention(q, torch.randn(b, h, 9, d), torch.randn(b, h, 9, d), torch.zeros(b, dtype=torch.int64))
        args = calls.pop()[1]
        own = args[0] == q.data_ptr()
        assert own == (d == 1) and list(args[10][:3]) == list((q if own else q.contiguous()).stride()[:3])
        keep = torch.zeros(b, h, 2 * d, dtype=torch.int64)[..., ::2]
        ops.compact_cache(torch.randn(b, h, 9, 4), torch.randn(b, h, 9, 4), keep, torch.ones(b, dtype=torch.int64))
        args = calls.pop()[1]
        own = args[11] == keep.data_ptr()
        assert own == (d == 1) and list(args[12:14]) == list((keep if own else keep.contiguous()).stride()[:2])
        logits = torch.randn(b, h, 2 * d)[..., ::2]
        ops.beam_select(logits, torch.zeros(b, h), 1)
        args = calls.pop()[1]
        own = args[0] == logits.data_ptr()
        assert own == (d == 1) and list(args[5:7]) == list((logits if own else logits.contiguous()).stride()[:2])
