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


def test_shared_memory_is_found_exactly():
    """Every pair of random views of one buffer against the elements that they hold."""
    import numpy as np
    from bittorch_b200 import _cache

    rng = np.random.default_rng(0)
    found = {True: 0, False: 0}
    for _ in range(3000):
        pair = []
        for _ in range(2):
            base = torch.zeros(int(rng.integers(1, 5)), int(rng.integers(1, 5)), int(rng.integers(2, 9)), int(rng.integers(1, 7)))
            view = base.permute(*rng.permutation(4).tolist())
            view = view[tuple(slice(int(rng.integers(0, n)), None, int(rng.integers(1, 3))) for n in view.shape)]
            pair.append((view.shape, view.stride(), [torch.float32, torch.bfloat16][int(rng.integers(2))], view.storage_offset()))
        if rng.random() < 0.5:
            pair[1] = (*pair[0][:2], pair[1][2], pair[1][3])
        at = [x[3] * x[2].itemsize + int(rng.integers(0, 40)) * 2 for x in pair]
        held = [set((p + x[2].itemsize * np.add.outer(sum(np.ix_(*[np.arange(n) * st for n, st in zip(x[0], x[1])])), np.zeros(1, int)).reshape(-1, 1)
                     + np.arange(x[2].itemsize)).reshape(-1).tolist()) for p, x in zip(at, pair)]
        want = bool(held[0] & held[1])
        a, b = (tuple(x[:3]) for x in pair)
        assert _cache._meet(a, b, at[1] - at[0]) == want == _cache._meet(b, a, at[0] - at[1])
        found[want] += 1
    assert min(found.values()) > 100


def test_a_compaction_refuses_partly_shared_memory(monkeypatch):
    """An output that begins some slots into the cache, keys and values that overlap; views of one buffer that hold no common
    element are taken."""
    g = torch.Generator().manual_seed(1)
    with on_the_cpu(monkeypatch) as (ops, _):
        buf = torch.randn(2, 3, 20, 8, generator=g)
        k, v = buf[:, :, :10], torch.randn(2, 3, 10, 8, generator=g)
        keep, counts = torch.tensor([[[1, 4, 6]]]).expand(2, 3, 3), torch.tensor([3, 2])
        mass, lengths = torch.rand(2, 3, 10, generator=g), torch.tensor([10, 9])
        for first in (0, 1, 9):                                             # they meet in slots first .. 9
            with pytest.raises(RuntimeError, match="other memory"):
                ops.compact_cache(k, v, keep, counts, out=(buf[:, :, first:first + 5], torch.empty(2, 3, 5, 8)))
            with pytest.raises(RuntimeError, match="other memory"):
                ops.evict_cache(k, v, mass, lengths, 5, out=(torch.empty(2, 3, 5, 8), buf[:, :, first:first + 5], torch.empty(2, 3, 5)))
        big = torch.randn(2, 3, 9, 8, generator=g)
        with pytest.raises(RuntimeError, match="other memory"):
            ops.compact_cache(k, v, keep, counts, out=(big[:, :, :5], big[:, :, 4:]))
        with pytest.raises(RuntimeError, match="same memory"):
            ops.compact_cache(buf[:, :, :10], buf[:, :, 9:19], keep, counts)
        with pytest.raises(RuntimeError, match="same memory"):
            ops.evict_cache(buf[:, :, :10], buf[:, :, 9:19], mass, lengths, 5)
        with pytest.raises(RuntimeError, match="other memory"):
            ops.evict_cache(k, v, mass, lengths, 5, out=(torch.empty(2, 3, 5, 8), torch.empty(2, 3, 5, 8), mass[:, :, 3:8]))
        # the two halves of one buffer, as output and as keys and values; heads and slots in turn
        want = [k.gather(2, keep[..., None].expand(2, 3, 3, 8)), v.gather(2, keep[..., None].expand(2, 3, 3, 8))]
        out = (buf[:, :, 10:15], torch.zeros(2, 3, 5, 8))
        ops.compact_cache(k, v, keep, counts, out=out)
        for x, w in zip(out, want):
            assert torch.equal(x[0, :, :3], w[0]) and torch.equal(x[1, :, :2], w[1, :, :2])
        pair = torch.randn(2, 10, 2, 3, 8, generator=g)
        k, v = pair[:, :, 0].transpose(1, 2), pair[:, :, 1].transpose(1, 2)
        want = [k.gather(2, keep[..., None].expand(2, 3, 3, 8)), v.gather(2, keep[..., None].expand(2, 3, 3, 8))]
        ops.compact_cache(k, v, keep, counts)
        for x, w in zip((k, v), want):
            assert torch.equal(x[0, :, :3], w[0]) and torch.equal(x[1, :, :2], w[1, :, :2])


def test_attention_refuses_shared_memory_and_nothing_else(monkeypatch):
    """An output beside the queries in one buffer is memory of its own; one that meets an operand is not, nor is such a mass."""
    g = torch.Generator().manual_seed(2)
    with on_the_cpu(monkeypatch) as (ops, _):
        both = torch.randn(2, 3, 4, 16, generator=g)                        # queries and output in one buffer, row by row
        q, out = both[..., :8], both[..., 8:]
        slots = torch.randn(2, 2, 3, 9, 8, generator=g)
        k, v = slots[0], slots[1]
        lengths = torch.tensor([5, 2])
        want, _, largest = ref.attention(q, k, v, lengths)
        assert ops.tree_attention(q, k, v, lengths, out=out) is out
        # as in the CPU tests of the kernels: 4e-6 (1 + largest) for scores and sums, one rounding
        assert torch.allclose(out.double(), want, rtol=2.0 ** -24, atol=4e-6 * (1 + largest))
        whole = torch.randn(2, 3, 6, 8, generator=g)
        with pytest.raises(RuntimeError, match="other memory"):
            ops.tree_attention(whole[:, :, :4], k, v, lengths, out=whole[:, :, 2:])
        with pytest.raises(RuntimeError, match="other memory"):
            ops.tree_attention(q, k, v, lengths, out=k[:, :, :4])
        with pytest.raises(RuntimeError, match="other memory"):
            ops.tree_attention(q, k, v, lengths, mass=v.reshape(-1)[:54].view(2, 3, 9))
        with pytest.raises(RuntimeError, match="other memory"):
            ops.tree_attention(q, k, v, lengths, mass=both.view(-1)[8:8 + 54].view(2, 3, 9), out=out)
        mass = torch.zeros(2, 3, 10)
        ops.tree_attention(q, k, v, lengths, mass=mass[:, :, 1:])
        assert torch.allclose(mass.sum(-1), torch.full((2, 3), 4.0), rtol=1e-5) and bool((mass[:, :, 0] == 0).all())


def test_reordering_refuses_views_that_meet(monkeypatch):
    """Views of one buffer that interleave are taken, strided ones that have elements in common are not."""
    g = torch.Generator().manual_seed(3)
    parents, lengths = torch.tensor([[1, 0, 2], [0, 0, 1]]), torch.tensor([5, 7])
    source = (parents + torch.arange(2)[:, None] * 3).reshape(-1)
    with on_the_cpu(monkeypatch) as (ops, _):
        layers = torch.randn(6, 4, 2, 2, 7, 8, generator=g)                 # row, layer, keys or values, head, slot, column
        views = [layers[:, i, j] for i in range(4) for j in range(2)]
        before = [x.clone() for x in views]
        ops.reorder_cache(views, parents, lengths)
        for x, old in zip(views, before):
            for row in range(6):
                n = int(lengths[row // 3])
                assert torch.equal(x[row, :, :n], old[source[row], :, :n]) and torch.equal(x[row, :, n:], old[row, :, n:])
        buf = torch.randn(6, 2, 12, 8, generator=g)
        for first in (0, 1, 5):                                             # they meet in slots first .. 6
            with pytest.raises(RuntimeError, match="share memory"):
                ops.reorder_cache([buf[:, :, first:first + 7], torch.randn(6, 2, 7, 8), buf[:, :, :7]], parents, lengths)
        wide = torch.randn(6, 2, 7, 12, generator=g)
        with pytest.raises(RuntimeError, match="share memory"):
            ops.reorder_cache([wide[..., :8], wide[..., 4:]], parents, lengths)
        ops.reorder_cache([wide[..., :6], wide[..., 6:]], parents, lengths)


def test_tangents_are_refused():
    """Forward-mode differentiation does not show in requires_grad: a dual tensor's tangent must not be lost in silence."""
    import torch.autograd.forward_ad as fwd
    from bittorch_b200 import ops

    k, v, mass, n = torch.zeros(2, 3, 10, 8), torch.zeros(2, 3, 10, 8), torch.zeros(2, 3, 10), torch.zeros(2, dtype=torch.int64)
    q, keep = torch.zeros(2, 3, 1, 8), torch.zeros(2, 3, 4, dtype=torch.int64)
    x, s, parents = torch.zeros(2, 3, 50), torch.zeros(2, 3), torch.zeros(1, 2, dtype=torch.int64)
    calls = [(lambda *a: ops.tree_attention(*a, n), (q, k, v)), (lambda a, b: ops.tree_attention(q, a, v, n, mass=b), (k, mass)),
             (lambda a, b: ops.compact_cache(a, b, keep, n), (k, v)), (lambda *a: ops.evict_cache(*a, n, 4, 1, 1), (k, v, mass)),
             (ops.beam_select, (x, s)), (lambda a, b: ops.reorder_cache([a, b], parents, n[:1]), (k, v))]
    for call, args in calls:
        for i in range(len(args)):
            for quiet in (False, True):
                with fwd.dual_level(), torch.set_grad_enabled(not quiet):
                    dual = [fwd.make_dual(a, torch.ones_like(a)) if j == i else a for j, a in enumerate(args)]
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        call(*dual)
                    with pytest.raises(RuntimeError, match="CUDA"):        # no tangent: as outside a dual level
                        call(*args)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda a: ops.tree_attention(a, k, v, n), (q,), (torch.ones_like(q),))


def test_what_a_call_writes_counts_as_changed(monkeypatch):
    """Version counters of the tensors that are written, of those alone; a graph that has saved one refuses to go back."""
    g = torch.Generator().manual_seed(4)
    with on_the_cpu(monkeypatch) as (ops, _):
        k, v, q = torch.randn(2, 3, 10, 8, generator=g), torch.randn(2, 3, 10, 8, generator=g), torch.randn(2, 3, 1, 8, generator=g)
        mass, n, keep = torch.rand(2, 3, 10, generator=g), torch.tensor([9, 8]), torch.arange(4).expand(2, 3, 4)
        out, small = torch.empty_like(q), (torch.zeros(2, 3, 5, 8), torch.zeros(2, 3, 5, 8), torch.zeros(2, 3, 5))
        calls = [(lambda: ops.tree_attention(q, k, v, n), ()), (lambda: ops.tree_attention(q, k, v, n, mass=mass, out=out), (mass, out)),
                 (lambda: ops.evict_cache(k, v, mass, n, 5, out=small), small), (lambda: ops.evict_cache(k, v, mass, n, 5), (k, v, mass)),
                 (lambda: ops.compact_cache(k, v, keep, n, out=small[:2]), small[:2]), (lambda: ops.compact_cache(k, v, keep, n), (k, v)),
                 (lambda: ops.compact_cache(k, v, keep, n, mass=mass), (k, v, mass)),
                 (lambda: ops.reorder_cache([k, v], torch.tensor([[1, 0]]), n[:1]), (k, v)), (lambda: ops.evict_select(mass, n, 5, 1, 1), ()),
                 (lambda: ops.beam_select(q[:, :, 0], mass[:, :, 0]), ())]
        every = (q, k, v, mass, n, out, *small)
        for call, written in calls:
            before = [t._version for t in every]
            call()
            for t, old in zip(every, before):
                assert (t._version > old) == any(t is w for w in written)
        w = torch.ones(8, requires_grad=True)
        loss = (k * w).sum()                                                # saves k
        with torch.no_grad():
            ops.compact_cache(k, v, keep, n)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        with torch.inference_mode():                                        # tensors without a counter
            a, b = k.clone(), v.clone()
            ops.compact_cache(a, b, keep, n)


def test_numbers_of_any_kind(monkeypatch):
    """Scales and end tokens as numpy numbers or tensors of one element are taken by their value; nothing is kept of them."""
    import numpy as np
    from bittorch_b200 import _cache

    g = torch.Generator().manual_seed(6)
    with on_the_cpu(monkeypatch) as (ops, _):
        q, k, v = torch.randn(2, 2, 1, 8, generator=g), torch.randn(2, 2, 9, 8, generator=g), torch.randn(2, 2, 9, 8, generator=g)
        n, half = torch.tensor([5, 7]), torch.tensor(0.5)
        want = ops.tree_attention(q, k, v, n, scale=0.5)
        for scale in (half, torch.tensor([0.5]), np.float32(0.5), np.float64(0.5)):
            assert torch.equal(ops.tree_attention(q, k, v, n, scale=scale), want)
        assert _cache._attention_plan.cache_info().currsize == 1
        half.fill_(float("inf"))
        with pytest.raises(RuntimeError, match="scale must be finite"):
            ops.tree_attention(q, k, v, n, scale=half)
        x, s, done = torch.randn(2, 3, 20, generator=g), torch.randn(2, 3, generator=g), torch.tensor([[True, False, True], [False, True, False]])
        want = ops.beam_select(x, s, 4, done, 7)
        for end in (torch.tensor(7), np.int64(7), np.uint8(7)):
            assert all(torch.equal(a, b) for a, b in zip(ops.beam_select(x, s, np.int32(4), done, end), want))
        assert _cache._beam_plan.cache_info().currsize == 1
