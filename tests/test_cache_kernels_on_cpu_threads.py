"""The kernels over a key/value cache, their shipped sources executed on the CPU with one OS thread per CUDA thread
(tests/simt/), against the plain forms in 64 bits of tests/cache_reference.py.  Not covered here: the tensor-core kernels
of the attention."""

import pytest
import torch

from tests import cache_reference as ref
from tests.simt import cache_harness as H


def _cache(g, b, hkv, s, d, used, dtype, layout="bhsd"):
    """Keys and values with NaN in every slot that is not in use."""
    pair = []
    for _ in range(2):
        if layout == "bshd":
            x = torch.randn(b, s, hkv, d, generator=g).to(dtype).transpose(1, 2)
        else:
            x = torch.randn(b, hkv, s, d, generator=g).to(dtype)
        for i, n in enumerate(used):
            x[i, :, n:] = float("nan")
        pair.append(x)
    return pair


def _tolerance(dtype, largest):
    """float32 arithmetic on the inputs as they are: scores are off by at most (D + 2) 2^-24 of their absolute sum (below
    largest * 8 here), which moves a weight by that relative amount; sums of at most 300 terms; one rounding of the
    output.  4e-6 * (1 + largest) covers the first two for D <= 128."""
    return 4e-6 * (1 + largest), torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("b,h,hkv,t,s,d,lens,dtype,trees,sms", [
    (1, 1, 1, 1, 1, 1, [0], torch.float32, None, 1),
    (2, 4, 2, 1, 70, 20, [0, 69], torch.float32, None, 1),
    (2, 6, 2, 7, 100, 16, [33, 93], torch.float32, "one", 1),
    (3, 2, 1, 5, 140, 66, [135, 64, 1], torch.bfloat16, "each", 3),
    (1, 8, 1, 3, 200, 64, [197], torch.float16, None, 4),
    (2, 1, 1, 18, 90, 7, [72, 3], torch.float32, "blank", 2),
    (1, 2, 2, 4, 40, 130, [38], torch.float32, None, 1),                     # two of the four new slots do not exist
])
def test_attention_kernel(b, h, hkv, t, s, d, lens, dtype, trees, sms):
    H.set_sm_count(sms)
    g = torch.Generator().manual_seed(b * 100 + s)
    k, v = _cache(g, b, hkv, s, d, [n + t for n in lens], dtype, "bshd" if s % 3 == 1 else "bhsd")
    q = torch.randn(b, t, h, d, generator=g).to(dtype).transpose(1, 2)
    tree = None
    if trees == "one":
        tree = torch.rand(t, t, generator=g) < 0.5
    elif trees in ("each", "blank"):
        tree = torch.rand(b, t, t, generator=g) < 0.4
        if trees == "blank":
            tree[1, 4:] = False
            lens = [lens[0], 0]
            k[1, :, t:], v[1, :, t:] = float("nan"), float("nan")
            v[0, :, lens[0] + 2] = float("inf")                            # seen by some of the tokens only
    lengths = torch.tensor(lens, dtype=torch.int32 if s % 2 else torch.int64)
    mass = torch.rand(b, hkv, s, generator=g) if t < 8 else None
    want, want_mass, largest = ref.attention(q, k, v, lengths, tree, None, mass)
    got = H.tree_attention(q, k, v, lengths, tree, None, mass)
    atol, rtol = _tolerance(dtype, largest)
    finite = want.isfinite()
    assert torch.equal(got.double()[~finite].isnan(), want[~finite].isnan()) and bool((~got[~finite].isfinite()).all())
    assert torch.allclose(got.double()[finite], want[finite], rtol=rtol + atol, atol=atol)
    if mass is not None:
        assert torch.allclose(mass.double(), want_mass, rtol=1e-6, atol=atol)


@pytest.mark.parametrize("n,budget,sinks,recent,kind", [
    (50, 20, 4, 5, "random"), (64, 64, 0, 0, "random"), (40, 50, 4, 4, "random"), (1500, 300, 3, 100, "random"),
    (1100, 33, 2, 11, "ties"), (200, 10, 4, 6, "random"), (90, 30, 0, 0, "special"), (77, 1, 0, 0, "ties"), (77, 1, 0, 1, "random"),
])
def test_evict_select_kernel(n, budget, sinks, recent, kind):
    g = torch.Generator().manual_seed(n)
    s = n + 7
    mass = torch.rand(2, 2, s, generator=g) ** 4
    if kind == "ties":
        mass = (mass * 3).floor()
    if kind == "special":
        for i, x in enumerate((float("nan"), float("inf"), -1.0, -0.0, 0.0, float("-inf"), float("nan"), -0.0, 1e-42)):
            mass[:, :, 5 * i + 2] = x
        mass[:, :, 45:] = 0.0
    lengths = torch.tensor([n, n // 2])
    keep, counts = H.evict_select(mass, lengths, budget, sinks, recent)
    for b, m in enumerate(lengths.tolist()):
        for h in range(2):
            want = ref.keep_slots(mass[b, h], m, budget, sinks, recent)
            assert keep[b, h, :len(want)].tolist() == want and bool((keep[b, h, len(want):] == -1).all())
            assert int(counts[b]) == len(want)


@pytest.mark.parametrize("d,dtype,in_place,heads", [(8, torch.float32, True, 2), (9, torch.bfloat16, True, 1), (40, torch.float16, False, 2),
                                                    (3, torch.float32, False, 1), (64, torch.bfloat16, True, 2)])
def test_compact_kernel(d, dtype, in_place, heads):
    g = torch.Generator().manual_seed(d)
    b, hkv, s, n = 2, 2, 1300, 1100
    H.set_sm_count(2)
    k, v = (torch.randn(b, hkv, s, d, generator=g).to(dtype) for _ in range(2))
    mass = torch.rand(b, hkv, s, generator=g)
    first = torch.tensor([3, 0])
    counts = torch.tensor([n - 50, 17])
    keep = torch.stack([torch.stack([torch.randperm(s - 3, generator=g)[:n].sort().values + 3 for _ in range(heads)]) for _ in range(b)])
    if not in_place:
        keep[0, 0, 5], keep[1, 0, 2] = -1, s                               # skipped
    s_out = s if in_place else n
    out = [k.clone(), v.clone(), mass.clone()] if in_place else [torch.full((b, hkv, s_out, d), 7.0, dtype=dtype) for _ in range(2)] + [
        torch.full((b, hkv, s_out), 7.0)]
    want = [x.clone() for x in out]
    for i in range(b):
        for h in range(hkv):
            row = keep[i, h % heads].tolist()
            for j in range(int(counts[i])):
                if 0 <= row[j] < s and int(first[i]) + j < s_out:
                    for w, x in zip(want, (k, v, mass)):
                        w[i, h, int(first[i]) + j] = x[i, h, row[j]]
            want[2][i, h, int(first[i]) + int(counts[i]):] = 0.0
    if in_place:
        H.compact_cache(*out[:2], keep, counts, first, out[2])
    else:
        H.compact_cache(k, v, keep, counts, first, mass, out)
    for w, x in zip(want, out):
        assert torch.equal(w, x)


@pytest.mark.parametrize("b,w,v,n,dtype,kind", [
    (1, 1, 1, 1, torch.float32, "plain"), (2, 3, 65, 6, torch.float32, "plain"), (1, 2, 9001, 5, torch.bfloat16, "plain"),
    (1, 3, 4100, 7, torch.float32, "finished"), (2, 2, 33, 8, torch.float16, "ties"), (1, 4, 20, 30, torch.float32, "dead"),
    (1, 2, 8200, 64, torch.float16, "ties"), (1, 40, 50, 64, torch.float32, "plain"),
])
def test_beam_select_kernels(b, w, v, n, dtype, kind):
    g = torch.Generator().manual_seed(v)
    logits = (torch.randn(b, w, v + 3, generator=g) * 3).to(dtype)[:, :, 1:v + 1]
    scores = torch.randn(b, w, generator=g)
    finished = end = None
    if kind == "ties":                                                      # equal rows: every rank is decided by the place
        logits = logits.round()
        logits[:, 1:] = logits[:, :1]
        scores[:] = -1.0
    elif kind == "finished":
        finished, end = torch.tensor([[True, False, True]]), 2
    elif kind == "dead":
        scores[0, 0] = float("-inf")
        logits[0, 1] = float("-inf")
        logits[0, 2, 3:] = float("nan")
        finished, end = torch.tensor([[False, False, False, True]]), 19
    want, tokens, parents = ref.select(logits, scores, n, finished, end)
    got = H.beam_select(logits, scores, n, finished, end)
    assert torch.equal(got[1], tokens) and torch.equal(got[2], parents)
    assert torch.allclose(got[0].double(), want, rtol=2.0 ** -23, atol=1e-6)


@pytest.mark.parametrize("w,d,dtype,lens,start,layout", [(4, 8, torch.float32, [9, 5], 0, "bhsd"), (2, 3, torch.bfloat16, [7, 0], 2, "bhsd"),
                                                       (13, 16, torch.float16, [11, 11], 0, "bshd"), (20, 5, torch.float32, [3, 4], 1, "bshd")])
def test_reorder_kernel(w, d, dtype, lens, start, layout):
    g = torch.Generator().manual_seed(w)
    b, hkv, s, tensors = 2, 2, 11, 3
    caches = []
    for _ in range(tensors):
        x = torch.randn(b * w, s, hkv, d, generator=g).to(dtype).transpose(1, 2)
        caches.append(x if layout == "bshd" else x.contiguous())
    parents = torch.randint(0, w, (b, w), generator=g)
    parents[1, 0], parents[0, w - 1] = w, -1                                # outside: stays
    want = [c.clone() for c in caches]
    for x, c in zip(want, caches):
        for i in range(b):
            for j in range(w):
                src = int(parents[i, j])
                if 0 <= src < w:
                    x[i * w + j, :, start:lens[i]] = c[i * w + src, :, start:lens[i]]
    H.reorder_cache(caches, parents, torch.tensor(lens), start)
    for x, c in zip(want, caches):
        assert torch.equal(x, c)
