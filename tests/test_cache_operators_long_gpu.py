"""tree_attention on the GPU with many rows over long caches: the sizes at which the tensor-memory kernel takes over
(batch x key/value heads x tiles of 16 rows x slots x head size above 1.3e7; more than 64 tiles or 128 rows)."""

import pytest
import torch

from tests.conftest import needs_real_gpu
from tests.test_cache_operators_gpu import _attention_case, _ops

pytestmark = [pytest.mark.gpu, needs_real_gpu]

HALF = [torch.bfloat16, torch.float16]


def _large(b, h, hkv, t, s, d):
    rows = h // hkv * t
    tiles = b * hkv * -(-rows // 16)
    assert d in (64, 128) and tiles * s * d > 1.3e7 and (rows > 128 or tiles > 64)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("b,h,hkv,t,s,d,lens,trees", [
    (8, 9, 3, 16, 1501, 128, [0, 1490, 127, 128, 129, 1, 700, 255], "each"),    # three heads of one tile each: two together, one alone
    (2, 8, 2, 75, 2800, 64, [320, 2700], "one"),                                # three tiles a head: two share its keys, the third goes with the next head's
    (12, 4, 1, 32, 1100, 128, [1068, 0, 96, 97, 95, 1000, 512, 511, 513, 1, 31, 33], "one"),
    (11, 4, 2, 20, 3100, 64, [3000, 0, 127, 128, 129, 1, 600, 1280, 256, 108, 3080], "each"),
    (1, 2, 1, 250, 3300, 128, [333], "one"), (1, 3, 1, 300, 3600, 64, [100], None), (1, 8, 1, 33, 12001, 64, [11900], "each"),
    (17, 2, 2, 17, 1600, 128, [0, 5, 1583, 111, 112, 110, 1, 2, 3, 900, 901, 902, 64, 65, 66, 67, 1500], None),
    (2, 6, 2, 130, 1100, 128, [970, 64], "each"), (2, 20, 20, 17, 2700, 128, [2683, 2000], "one"),
])
def test_many_rows_over_long_caches(b, h, hkv, t, s, d, lens, trees, dtype):
    """Rows in tiles of 128, pairs of tiles of one head or two, pieces of a sequence on several CTAs, caches that are full."""
    from bittorch_b200 import _C

    _large(b, h, hkv, t, s, d)
    _attention_case(b, h, hkv, t, s, d, lens, dtype, trees, stretch=2.0)
    assert _C.device_status() == 0


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7, 40.0])
def test_scales_over_long_caches(scale):
    """As test_scales (a scale below zero is the few-rows kernel's)."""
    _large(2, 8, 2, 48, 2304, 128)
    for dtype in HALF:
        _attention_case(2, 8, 2, 48, 2304, 128, [260, 70], dtype, "one", scale=scale)


@pytest.mark.parametrize("layout", ["bshd", "odd"])
@pytest.mark.parametrize("dtype", HALF)
def test_other_layouts_over_long_caches(layout, dtype):
    """Caches with the heads inside the slots; rows that TMA cannot take (the generic kernel's)."""
    _large(2, 8, 2, 48, 2304, 128)
    _attention_case(2, 8, 2, 48, 2304, 128, [100, 2250], dtype, "one", layout)


@pytest.mark.parametrize("dtype", HALF)
def test_nothing_reaches_a_token_that_does_not_see_it_over_long_caches(dtype):
    """Infinities and NaN in slots behind the new tokens, and in new tokens that other tokens see; rows that see nothing."""
    ops = _ops()
    gen = torch.Generator().manual_seed(1)
    b, hkv, g, t, s, d, n = 2, 2, 4, 48, 2304, 128, 130
    _large(b, hkv * g, hkv, t, s, d)
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
            k2[i, :, m], v2[i, :, m] = bad, bad
        got = ops.tree_attention(q, k2, v2, lengths, tree)
        assert torch.equal(got[:, :, 1:t - 1], clean[:, :, 1:t - 1])
        assert bool((~got[:, :, 0].isfinite()).all()) or bad == -float("inf")
    got = ops.tree_attention(q, k, v, lengths, torch.zeros(t, t, dtype=torch.bool, device="cuda"))
    assert bool((got[1] == 0).all()) and bool(got[0].isfinite().all())


def test_expanded_caches_and_a_given_output():
    ops = _ops()
    g = torch.Generator().manual_seed(5)
    _large(4, 8, 2, 48, 2304, 64)
    k, v = (torch.randn(1, 2, 2304, 64, generator=g).bfloat16().cuda().expand(4, 2, 2304, 64) for _ in range(2))
    q = torch.randn(4, 8, 48, 64, generator=g).bfloat16().cuda()
    lengths = torch.tensor([1500, 0, 2256, 77]).cuda()
    want = ops.tree_attention(q, k.contiguous(), v.contiguous(), lengths)
    buf = torch.full((4, 8, 48, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got = ops.tree_attention(q, k, v, lengths, out=buf[..., :64])
    # each result is within eps / 2 of the weights' rounding (of sum p |v| <= 5) and eps / 2 of its own of the exact value
    assert float((got.float() - want.float()).abs().max()) <= 2 * (5 + 5) * 2 ** -8 and bool((buf[..., 64:] == 7).all())


def test_two_streams_and_a_replayed_graph_over_long_caches():
    """Calls at the same time have their own workspaces, and a graph goes by the device's lengths."""
    ops = _ops()
    g = torch.Generator().manual_seed(3)
    _large(2, 8, 2, 48, 2304, 128)
    k, v = (torch.randn(2, 2, 2304, 128, generator=g).bfloat16().cuda() for _ in range(2))
    qs = [torch.randn(2, 8, t, 128, generator=g).bfloat16().cuda() for t in (48, 61)]
    lengths = torch.tensor([2240, 333]).cuda()

    def work():
        return [ops.tree_attention(q, k, v, lengths) for q in qs]

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
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = work()
        graphs.append((graph, out))
    lengths.copy_(torch.tensor([0, 1700]))
    want = work()
    torch.cuda.synchronize()
    for _ in range(3):
        for st, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, c) for a, c in zip(out, want))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("d", [8, 16, 40, 72, 88, 104, 120, 136, 192, 248, 256])
def test_head_sizes(d, dtype):
    """Head sizes between and beyond the ones that a kernel is built for: rows padded with zeros."""
    _attention_case(2, 8, 2, 1, 310, d, [300, 64], dtype)
    _attention_case(2, 4, 2, 9, 310, d, [301, 1], dtype, "each", stretch=2.0)
    _attention_case(1, 6, 1, 4, 150, d, [140], dtype, "one", "bshd", with_mass=True)
