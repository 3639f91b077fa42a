"""The operators over a key/value cache on the GPU, through bittorch_b200.ops, against the plain forms in 64 bits."""

import pytest
import torch

from tests import cache_reference as ref
from tests.conftest import needs_real_gpu

pytestmark = [pytest.mark.gpu, needs_real_gpu]

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _ops():
    from bittorch_b200 import ops

    return ops


def _cache(g, b, hkv, s, d, used, dtype, layout="bhsd"):
    """Keys and values with NaN in every slot that is not in use."""
    pair = []
    for _ in range(2):
        if layout == "bshd":
            x = torch.randn(b, s, hkv, d, generator=g).to(dtype).transpose(1, 2)
        elif layout == "odd":                                              # rows that no vector load can take
            x = torch.randn(b, hkv, s, d + 1, generator=g).to(dtype)[..., 1:]
        else:
            x = torch.randn(b, hkv, s, d, generator=g).to(dtype)
        for i, n in enumerate(used):
            x[i, :, n:] = float("nan")
        pair.append(x.cuda() if layout == "bhsd" else x.cuda().as_strided(x.size(), x.stride()) if layout == "bshd" else _odd(x))
    return pair


def _odd(x):
    y = torch.empty(*x.shape[:3], x.shape[3] + 1, dtype=x.dtype, device="cuda")[..., 1:]
    return y.copy_(x)


def _close(got, want, v_largest, dtype, largest):
    """Scores are float32 sums of D exact (16-bit types) or once rounded products: off by at most D 2^-24 sum|q k| scale,
    below 2e-6 * (1 + largest) * 4 for the sizes here, and a weight by as much, relatively.  With a 16-bit type a weight is
    rounded to it once more (eps / 2 of itself) for the product with the values, so an output is off by eps / 2 of
    sum p |v| <= eps / 2 * max|v|, and by eps / 2 of itself at the end."""
    half = torch.finfo(dtype).eps / 2
    score = 8e-6 * (1 + largest)
    atol = (score + (0 if dtype == torch.float32 else half)) * v_largest + 1e-6
    off = (got.double().cpu() - want).abs()
    assert bool((off <= atol + half * want.abs()).all()), (float(off.max()), atol)


def _attention_case(b, h, hkv, t, s, d, lens, dtype, trees=None, layout="bhsd", with_mass=False, seed=0, scale=None, stretch=1.0):
    ops = _ops()
    g = torch.Generator().manual_seed(seed + b * 1000 + s + d + t)
    k, v = _cache(g, b, hkv, s, d, [min(n + t, s) for n in lens], dtype, layout)
    q = (torch.randn(b, t, h, d, generator=g) * stretch).to(dtype).transpose(1, 2).cuda()
    tree = None
    if trees == "one":
        tree = (torch.rand(t, t, generator=g) < 0.5).cuda()
    elif trees == "each":
        tree = (torch.rand(b, t, t, generator=g) < 0.4).cuda()
        tree[b - 1, t // 2:] = False
    lengths = torch.tensor(lens, dtype=torch.int32 if s % 2 else torch.int64).cuda()
    mass = torch.rand(b, hkv, s, generator=g).cuda() if with_mass else None
    want, want_mass, largest = ref.attention(q, k, v, lengths, tree, scale, mass)
    got = ops.tree_attention(q, k, v, lengths, tree, scale, mass)
    assert got.shape == q.shape and got.dtype == dtype
    _close(got, want, float(v[v.isfinite()].abs().max()), dtype, largest)
    if with_mass:
        assert torch.allclose(mass.double().cpu(), want_mass, rtol=1e-6, atol=8e-6 * (1 + largest) * (h // hkv) * t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,h,hkv,t,s,d,lens", [
    (1, 1, 1, 1, 1, 1, [0]), (1, 20, 20, 1, 600, 128, [517]), (3, 8, 1, 1, 333, 64, [0, 332, 64]), (2, 16, 2, 1, 1100, 128, [1099, 63]),
    (2, 40, 8, 1, 257, 96, [256, 128]), (1, 4, 4, 1, 70, 256, [65]), (2, 3, 1, 1, 129, 80, [128, 127]), (1, 32, 1, 1, 200, 128, [199]),
])
def test_single_token(b, h, hkv, t, s, d, lens, dtype):
    _attention_case(b, h, hkv, t, s, d, lens, dtype)
    _attention_case(b, h, hkv, t, s, d, lens, dtype, with_mass=True, seed=1, stretch=3.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,h,hkv,t,s,d,lens,trees", [
    (2, 4, 4, 7, 128, 64, [33, 121], "one"), (2, 8, 2, 5, 300, 128, [0, 290], None), (3, 4, 1, 61, 320, 128, [0, 255, 200], "each"),
    (1, 8, 1, 33, 600, 64, [513], "each"), (2, 2, 2, 64, 64, 128, [0, 0], "one"), (1, 6, 2, 130, 450, 128, [300], None),
    (1, 2, 1, 9, 77, 32, [70], None), (2, 5, 1, 17, 200, 96, [64, 127], "each"), (1, 4, 2, 65, 333, 64, [200], "one"),
])
def test_trees(b, h, hkv, t, s, d, lens, trees, dtype):
    _attention_case(b, h, hkv, t, s, d, lens, dtype, trees)
    _attention_case(b, h, hkv, t, s, d, lens, dtype, trees, with_mass=t < 20, seed=2, stretch=3.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,h,hkv,t,s,d,lens,trees", [
    (2, 9, 3, 16, 700, 128, [0, 650], "each"),               # three heads of one tile each: two together, one alone
    (2, 8, 2, 75, 400, 64, [320, 129], "one"),               # three tiles a head: two share its keys, the third goes with the next head's
    (1, 4, 1, 32, 5200, 128, [5100], "one"),                 # fewer blocks than CTAs
    (9, 4, 2, 20, 1500, 64, [1400, 0, 127, 128, 129, 1, 600, 1280, 256], "each"),
    (1, 2, 1, 250, 700, 128, [333], "one"), (1, 3, 1, 300, 520, 64, [100], None), (2, 2, 2, 17, 17, 128, [0, 5], None),
])
def test_many_rows(b, h, hkv, t, s, d, lens, trees, dtype):
    """Rows in tiles of 128, pairs of tiles of one head or two, pieces of a sequence on several CTAs."""
    from bittorch_b200 import _C

    _attention_case(b, h, hkv, t, s, d, lens, dtype, trees, stretch=2.0)
    assert _C.device_status() == 0


@pytest.mark.parametrize("t", [1, 24])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7, 40.0])
def test_scales(t, scale):
    """Any finite scale: uniform weights, the smallest products first, weights that are all but one-hot (where a score moves
    the running maximum by far more than a float's exponent can take)."""
    for dtype in (torch.float32, torch.bfloat16):
        _attention_case(2, 4, 2, t, 300, 64, [260, 70], dtype, "one", scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,d", [(1, 128), (9, 64), (40, 128), (1, 20)])
def test_other_layouts(t, d, dtype):
    for layout in ("bshd", "odd"):
        _attention_case(2, 4, 2, t, 210, d, [100, 210 - t], dtype, "one", layout, with_mass=t == 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,d,g", [(1, 128, 4), (6, 64, 2), (48, 128, 4)])
def test_nothing_reaches_a_token_that_does_not_see_it(t, d, g, dtype):
    """Infinities and NaN in slots behind the new tokens, and in new tokens that other tokens see: a token's result
    depends on what it sees alone, bit for bit."""
    ops = _ops()
    gen = torch.Generator().manual_seed(t)
    b, hkv, s, n = 2, 2, 200, 130
    k, v = (torch.randn(b, hkv, s, d, generator=gen).to(dtype).cuda() for _ in range(2))
    q = torch.randn(b, hkv * g, t, d, generator=gen).to(dtype).cuda()
    lengths = torch.tensor([n, 0]).cuda()
    tree = torch.eye(t, dtype=torch.bool, device="cuda")
    tree[t - 1, 0] = True
    clean = ops.tree_attention(q, k, v, lengths, tree)
    for bad in (float("nan"), float("inf"), -float("inf")):
        k2, v2 = k.clone(), v.clone()
        for i, m in enumerate((n, 0)):
            k2[i, :, m + t:], v2[i, :, m + t:] = bad, bad
            if t > 1:
                k2[i, :, m], v2[i, :, m] = bad, bad                        # the first new token: seen by itself and the last
        got = ops.tree_attention(q, k2, v2, lengths, tree)
        unharmed = slice(1, t - 1) if t > 1 else slice(0, 1)
        assert torch.equal(got[:, :, unharmed], clean[:, :, unharmed])
        if t > 1:
            assert bool((~got[:, :, 0].isfinite()).all()) or bad == -float("inf")
    blank = torch.zeros(t, t, dtype=torch.bool, device="cuda")
    got = ops.tree_attention(q, k, v, lengths, blank)
    assert bool((got[1] == 0).all()) and bool(got[0].isfinite().all())     # sequence 1 sees nothing at all
    mass = torch.zeros(b, hkv, s, device="cuda")
    ops.tree_attention(q, k, v, lengths, blank, mass=mass)
    assert bool((mass[1] == 0).all()) and torch.allclose(mass[0].sum(-1), torch.full((hkv,), float(g * t), device="cuda"), rtol=1e-4)
    assert bool((mass[0, :, n:] == 0).all())


def test_values_given_for_the_output_and_expanded_caches():
    """An output of the caller's with its own strides; a cache that all sequences share (stride 0), read only."""
    ops = _ops()
    g = torch.Generator().manual_seed(5)
    for t, d in ((1, 128), (33, 128), (3, 40)):
        k, v = (torch.randn(1, 2, 200, d, generator=g).bfloat16().cuda().expand(3, 2, 200, d) for _ in range(2))
        q = torch.randn(3, 4, t, d, generator=g).bfloat16().cuda()
        lengths = torch.tensor([150, 0, 199 - t]).cuda()
        want = ops.tree_attention(q, k.contiguous(), v.contiguous(), lengths)
        buf = torch.full((3, 4, t, 2 * d), 7.0, dtype=torch.bfloat16, device="cuda")
        got = ops.tree_attention(q, k, v, lengths, out=buf[..., :d])
        assert torch.allclose(got.float(), want.float(), rtol=2e-2, atol=2e-2) and bool((buf[..., d:] == 7).all())
        with pytest.raises(RuntimeError, match="other memory"):
            ops.tree_attention(q, k, v, lengths, out=q)


def test_long_cache_offsets_pass_32_bits():
    """2^31 elements lie between the first and the last slot that are read."""
    ops = _ops()
    if torch.cuda.mem_get_info()[0] < 30e9:
        pytest.skip("needs 20 GB of free device memory")
    b, hkv, s, d = 2, 2, 1 << 22, 256
    k = torch.empty(b, hkv, s, d, dtype=torch.bfloat16, device="cuda")     # 4 * 2^30 elements, never filled
    v = torch.empty_like(k)
    assert k.numel() > 1 << 31
    g = torch.Generator().manual_seed(0)
    n, t = 40, 3
    lengths = torch.tensor([n, n]).cuda()
    small = [torch.randn(b, hkv, n + t, d, generator=g).bfloat16().cuda() for _ in range(2)]
    k[:, :, :n + t], v[:, :, :n + t] = small[0], small[1]
    q = torch.randn(b, 4, t, d, generator=g).bfloat16().cuda()
    want = ops.tree_attention(q, small[0], small[1], lengths)
    got = ops.tree_attention(q, k, v, lengths)
    assert torch.allclose(got.float(), want.float(), atol=2e-2, rtol=2e-2)
    keep = torch.tensor([[[1, 5, n + t - 1]], [[0, 7, s - 1]]]).cuda()
    k[:, :, s - 1], v[:, :, s - 1] = 3.0, 4.0
    ops.compact_cache(k, v, keep, torch.tensor([3, 3]).cuda())
    assert torch.equal(k[0, :, 2], small[0][0, :, n + t - 1]) and bool((k[1, :, 2] == 3).all()) and bool((v[1, :, 2] == 4).all())
    k[:, 1, s - 2:] = torch.tensor([1.0, 2.0], device="cuda").view(2, 1, 1).bfloat16()
    ops.reorder_cache([k], torch.tensor([[1, 0]]).cuda(), torch.tensor([s]).cuda(), start=s - 2)
    assert bool((k[0, 1, s - 2:] == 2).all()) and bool((k[1, 1, s - 2:] == 1).all())


def test_two_streams_and_a_replayed_graph_agree_with_plain_calls():
    ops = _ops()
    g = torch.Generator().manual_seed(3)
    b, h, hkv, s, d = 3, 8, 2, 900, 128
    k, v = (torch.randn(b, hkv, s, d, generator=g).bfloat16().cuda() for _ in range(2))
    qs = [torch.randn(b, h, t, d, generator=g).bfloat16().cuda() for t in (1, 24)]
    lengths = torch.tensor([5, 800, 333]).cuda()
    logits = torch.randn(b, 4, 20000, generator=g).cuda()
    scores = torch.randn(b, 4, generator=g).cuda()

    def work():
        return [ops.tree_attention(q, k, v, lengths) for q in qs] + list(ops.beam_select(logits, scores))

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = work()
    torch.cuda.synchronize()
    for x in got:
        assert all(torch.equal(a, c) for a, c in zip(x, want))
    graphs = []
    for st in streams:                                                      # two graphs, replayed at the same time
        st.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = work()
        graphs.append((graph, out))
    lengths.copy_(torch.tensor([0, 876, 12]))                               # a captured call goes by the device's lengths
    want = work()
    torch.cuda.synchronize()
    for _ in range(3):
        for st, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, c) for a, c in zip(out, want))


@pytest.mark.parametrize("n,budget,sinks,recent,kind,s", [
    (50, 20, 4, 5, "random", 57), (1500, 300, 3, 100, "random", 1507), (40000, 2048, 4, 512, "random", 40001), (1100, 33, 2, 11, "ties", 1100),
    (90, 30, 0, 0, "special", 97), (77, 1, 0, 0, "ties", 80), (77, 1, 0, 1, "random", 77), (5000, 4999, 4, 9, "ties", 6000), (300, 300, 0, 0, "ties", 301),
])
def test_evict(n, budget, sinks, recent, kind, s):
    ops = _ops()
    g = torch.Generator().manual_seed(n)
    b, hkv, d = 2, 3, 16
    mass = torch.rand(b, hkv, s, generator=g) ** 4
    if kind == "ties":
        mass = (mass * 3).floor()
    if kind == "special":
        for i, x in enumerate((float("nan"), float("inf"), -1.0, -0.0, 0.0, float("-inf"), float("nan"), -0.0, 1e-42)):
            mass[:, :, 5 * i + 2] = x
        mass[:, :, 45:] = 0.0
    k, v = (torch.randn(b, hkv, s, d, generator=g).half() for _ in range(2))
    lens = [n, n // 2]
    want = [[ref.keep_slots(mass[i, j], m, budget, sinks, recent) for j in range(hkv)] for i, m in enumerate(lens)]
    dev = [x.cuda() for x in (k, v, mass)]
    lengths = torch.tensor(lens, dtype=torch.int32).cuda()
    out = [torch.full((b, hkv, budget + 3, d), 7.0).half().cuda(), torch.full((b, hkv, budget + 3, d), 7.0).half().cuda(),
           torch.full((b, hkv, budget + 3), 7.0).cuda()]
    keep, counts = ops.evict_cache(*dev, lengths, budget, sinks, recent, out=out)
    keep2, counts2 = ops.evict_cache(*dev, lengths, budget, sinks, recent)     # and in place
    assert torch.equal(keep, keep2) and torch.equal(counts, counts2)
    for i in range(b):
        assert int(counts[i]) == len(want[i][0])
        for j in range(hkv):
            slots = want[i][j]
            m = len(slots)
            assert keep[i, j, :m].tolist() == slots and bool((keep[i, j, m:] == -1).all())
            for full, cut, same in zip((k, v), out, dev):
                assert torch.equal(cut[i, j, :m].cpu(), full[i, j, slots]) and bool((cut[i, j, m:] == 7).all())
                assert torch.equal(same[i, j, :m].cpu(), full[i, j, slots]) and torch.equal(same[i, j, m:].cpu(), full[i, j, m:])
            for cut in (out[2], dev[2]):
                assert torch.equal(cut[i, j, :m].cpu().nan_to_num(9), mass[i, j, slots].nan_to_num(9)) and bool((cut[i, j, m:] == 0).all())


@pytest.mark.parametrize("dtype,d", [(torch.float32, 33), (torch.float16, 17), (torch.bfloat16, 128), (torch.bfloat16, 20)])
def test_accepted_path_moves_to_the_front(dtype, d):
    """What a verified tree leaves: some of the new slots move to first + j, one list for all heads, strided caches."""
    ops = _ops()
    g = torch.Generator().manual_seed(d)
    b, hkv, s = 3, 4, 90
    k, v = (torch.randn(b, s, hkv, d, generator=g).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    first = torch.tensor([10, 0, 80]).cuda()
    keep = torch.tensor([[[11, 13, 14, 16]], [[0, 1, 5, 89]], [[82, 85, 200, -7]]]).cuda()
    counts = torch.tensor([3, 4, 9]).cuda()                                 # more than there are: clamped
    want = [k.clone(), v.clone()]
    for w, x in zip(want, (k, v)):
        for i in range(b):
            for j in range(min(4, int(counts[i]))):
                src = int(keep[i, 0, j])
                if 0 <= src < s:
                    w[i, :, int(first[i]) + j] = x[i, :, src]
    ops.compact_cache(k, v, keep, counts, first)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


@pytest.mark.parametrize("b,w,v,n,dtype,kind", [
    (1, 1, 1, 1, torch.float32, "plain"), (2, 3, 65, 6, torch.float32, "plain"), (4, 8, 32000, 16, torch.bfloat16, "plain"),
    (3, 5, 50001, 7, torch.float16, "finished"), (2, 2, 33, 8, torch.float16, "ties"), (1, 4, 20, 30, torch.float32, "dead"),
    (2, 3, 9001, 64, torch.bfloat16, "ties"), (1, 64, 20003, 64, torch.float32, "plain"), (2, 64, 70001, 64, torch.bfloat16, "equal"),
    (2, 4, 300, 5, torch.bfloat16, "finished"),
])
def test_beam_select(b, w, v, n, dtype, kind):
    ops = _ops()
    g = torch.Generator().manual_seed(v + w)
    logits = (torch.randn(b, w, v + 3, generator=g) * 3).to(dtype)[:, :, 1:v + 1]
    scores = torch.randn(b, w, generator=g)
    finished = end = None
    if kind in ("ties", "equal"):                                           # equal rows: every rank is decided by the place
        logits = torch.zeros_like(logits) if kind == "equal" else logits.round()
        logits[:, 1:] = logits[:, :1].clone()
        scores[:] = -1.0
    elif kind == "finished":
        finished, end = torch.rand(b, w, generator=g) < 0.5, 2
        finished[b - 1] = True
    elif kind == "dead":
        scores[0, 0] = float("-inf")
        logits[0, 1] = float("-inf")
        logits[0, 2, 3:] = float("nan")
        finished, end = torch.tensor([[False, False, False, True]]), 19
    want, tokens, parents = ref.select(logits, scores, n, finished, end)
    dev = torch.empty(b, w, v + 3, dtype=dtype, device="cuda")[:, :, 1:v + 1]
    got = ops.beam_select(dev.copy_(logits), scores.cuda(), n, None if finished is None else finished.cuda(), end)
    assert torch.equal(got[1].cpu(), tokens) and torch.equal(got[2].cpu(), parents)
    # the log-sum: float32 exponentials off by 2^-22 each at most, summed; the score's own rounding
    fine = want.isfinite()
    assert torch.equal(got[0].cpu()[~fine].double(), want[~fine])
    assert torch.allclose(got[0].double().cpu()[fine], want[fine], rtol=2.0 ** -24, atol=3e-7)


@pytest.mark.parametrize("w,d,dtype,lens,start,layout,tensors", [
    (4, 64, torch.float32, [97], 0, "bhsd", 8), (2, 3, torch.bfloat16, [7, 0], 2, "bhsd", 1), (13, 16, torch.float16, [61, 100], 0, "bshd", 3),
    (32, 128, torch.bfloat16, [70], 11, "bshd", 5), (8, 128, torch.bfloat16, [100, 40], 0, "bhsd", 70), (3, 20, torch.float16, [100], 100, "bhsd", 2),
    (1, 8, torch.float32, [9], 0, "bhsd", 2),
])
def test_reorder(w, d, dtype, lens, start, layout, tensors):
    ops = _ops()
    g = torch.Generator().manual_seed(w)
    b, hkv, s = len(lens), 2, 100
    caches = []
    for _ in range(tensors):
        x = torch.randn(b * w, s, hkv, d, generator=g).to(dtype).cuda().transpose(1, 2)
        caches.append(x if layout == "bshd" else x.contiguous())
    parents = torch.randint(0, w, (b, w), generator=g)
    parents[0, w - 1] = w                                                   # outside: stays
    want = [c.clone() for c in caches]
    for x, c in zip(want, caches):
        for i in range(b):
            for j in range(w):
                src = int(parents[i, j])
                if 0 <= src < w:
                    x[i * w + j, :, start:lens[i]] = c[i * w + src, :, start:lens[i]]
    ops.reorder_cache(caches, parents.cuda(), torch.tensor(lens).cuda(), start)
    for x, c in zip(want, caches):
        assert torch.equal(x, c)
