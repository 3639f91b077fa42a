"""tree_attention on the GPU, tensor-memory kernel: new tokens that end up in several blocks of 128 slots, with the second
tile of a head delayed where the first is not (its running maximum moves there, and its output is rescaled)."""

import pytest
import torch

from tests import cache_reference as ref
from tests.conftest import needs_real_gpu
from tests.test_cache_operators_gpu import _cache, _close, _ops
from tests.test_cache_operators_long_gpu import HALF, _large

pytestmark = [pytest.mark.gpu, needs_real_gpu]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("b,h,hkv,t,s,d,lens", [
    (2, 8, 2, 61, 2304, 128, [100, 1900]),                                  # two blocks with new tokens
    (2, 4, 2, 130, 3100, 64, [127, 2000]),                                  # two or three
    (1, 2, 1, 250, 3300, 128, [333]),                                       # three, tiles of both heads
    (12, 8, 2, 61, 700, 64, [67 + 128 * (i % 4) for i in range(12)]),       # pieces of one to five blocks, one after the other
    (3, 8, 4, 80, 900, 128, [0, 60, 128]),                                  # sequences that are new tokens alone, or nearly
])
def test_new_tokens_in_neighbouring_blocks(b, h, hkv, t, s, d, lens, dtype):
    from bittorch_b200 import _C

    ops = _ops()
    _large(b, h, hkv, t, s, d)
    g = torch.Generator().manual_seed(t + s)
    k, v = _cache(g, b, hkv, s, d, [n + t for n in lens], dtype)
    q = torch.randn(b, h, t, d, generator=g).to(dtype)
    group, u = h // hkv, torch.randn(d, generator=g)
    rows = torch.arange(group * t).reshape(group, t) % 256 >= 128           # those of every second tile
    q.view(b, hkv, group, t, d)[:, :, rows] = (3 * u).to(dtype)
    for i, n in enumerate(lens):
        last = (n + t - 1) // 128 * 128                                     # the last block's new tokens: scores 9 sqrt(d) above the others
        k[i, :, max(last, n):n + t] = (3 * u).to(dtype).cuda()
    tree = torch.rand(t, t, generator=g) < 0.5
    tree[:, t - 1] = True
    q, tree, lengths = q.cuda(), tree.cuda(), torch.tensor(lens).cuda()
    want, _, largest = ref.attention(q, k, v, lengths, tree)
    got = ops.tree_attention(q, k, v, lengths, tree)
    _close(got, want, float(v[v.isfinite()].abs().max()), dtype, largest)
    for _ in range(50):
        assert torch.equal(ops.tree_attention(q, k, v, lengths, tree), got)
    assert _C.device_status() == 0


@pytest.mark.parametrize("tiles", [0, 1, 5, 12])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_a_call_whose_wait_runs_out_leaves_nan_and_a_status(dtype, d, tiles):
    """The give-up path: the role that brings the tiles leaves after some of them, as it does when its wait runs out, and all
    others follow (every wait of theirs has a limit).  What was finished before is right, the rest is NaN, nothing is left
    unwritten, and the next call is as ever."""
    from bittorch_b200 import _C

    ops = _ops()
    b, h, hkv, t, s = 24, 32, 8, 61, 2304                                   # about 19 places of the line for each CTA
    _large(b, h, hkv, t, s, d)
    g = torch.Generator().manual_seed(tiles)
    k, v = (torch.randn(b, hkv, s, d, generator=g).to(dtype).cuda() for _ in range(2))
    q = torch.randn(b, h, t, d, generator=g).to(dtype).cuda()
    tree = (torch.rand(t, t, generator=g) < 0.5).cuda()
    lengths = torch.tensor([100, 2200, 0, 1300, 64, 2243] * 4).cuda()
    clean = ops.tree_attention(q, k, v, lengths, tree)
    assert _C.device_status() == 0
    out = torch.full((b, h, t, d), 7.0, dtype=dtype, device="cuda")
    _C.set_tuning(_C.TUNE_ATTENTION_GIVE_UP, tiles)
    try:
        ops.tree_attention(q, k, v, lengths, tree, out=out)
        torch.cuda.synchronize()
    finally:
        _C.set_tuning(_C.TUNE_ATTENTION_GIVE_UP, -1)
    assert _C.device_status() == 4
    lost = out.isnan().any(-1)
    assert bool(lost.any()) and bool(out.isnan().all(-1)[lost].all())
    assert bool(lost.all()) or tiles > 0
    assert torch.equal(out[~lost], clean[~lost])
    assert torch.equal(ops.tree_attention(q, k, v, lengths, tree), clean) and _C.device_status() == 0


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("b,h,hkv,t,s,d,lens,trees", [
    (1, 2, 1, 65, 12001, 128, [0], None), (1, 2, 1, 65, 12001, 128, [500], "one"), (1, 2, 1, 65, 12001, 128, [1100], "each"),
    (1, 8, 1, 33, 12001, 64, [5], "one"), (2, 8, 1, 33, 7001, 64, [0, 300], "each"), (3, 4, 1, 40, 12001, 128, [1, 0, 255], None),
    (5, 4, 1, 33, 7001, 64, [3, 0, 5, 1, 2], "one"),
])
def test_fewer_places_than_ctas(b, h, hkv, t, s, d, lens, trees, dtype):
    """Little work in a large cache: the line of blocks (with the places that the end of a pair counts as) is shorter than the
    number of CTAs, so that some have none, and a pair is in as many pieces as it has blocks."""
    from bittorch_b200 import _C
    from tests.test_cache_operators_gpu import _attention_case

    _large(b, h, hkv, t, s, d)
    pairs = -(-hkv * -(-(h // hkv * t) // 128) // 2)
    assert sum(-(-(n + t) // 128) + 8 for n in lens) * pairs < torch.cuda.get_device_properties(0).multi_processor_count
    _attention_case(b, h, hkv, t, s, d, lens, dtype, trees, stretch=2.0)
    assert _C.device_status() == 0


def _squares(q, k, v, lengths, tree):
    """-> out, sum p^2 v^2, sum p |v| and the largest |score|, float64 [B, H, T, D]."""
    b, h, t, d = q.shape
    group, s = h // k.shape[1], k.shape[2]
    q, k, v = q.double(), k.double().repeat_interleave(group, 1), v.double().repeat_interleave(group, 1)
    slot, token = torch.arange(s, device=q.device), torch.arange(t, device=q.device)
    n = lengths[:, None, None]
    own = (slot - n).clamp(0, t - 1).expand(b, t, s)
    sees = (slot < n) | ((slot < n + t) & tree.expand(b, t, t).gather(2, own))
    x = (q @ k.nan_to_num().transpose(2, 3)) * d ** -0.5
    largest = float(x.abs()[sees[:, None].expand_as(x)].max())
    p = torch.softmax(x.masked_fill(~sees[:, None], float("-inf")), -1)
    v = v.nan_to_num()
    return p @ v, (p * p) @ (v * v), p @ v.abs(), largest


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("b,h,hkv,t,s,d,lens", [
    (2, 20, 20, 1, 600, 128, [517, 598]), (2, 16, 2, 5, 800, 64, [700, 555]), (4, 8, 2, 7, 700, 96, [600, 611, 650, 500]), (2, 16, 4, 4, 640, 80, [600, 620]),
    (2, 8, 2, 61, 2304, 128, [1900, 700]), (2, 8, 2, 130, 3100, 64, [2900, 1000]),
])
def test_the_error_as_a_whole(b, h, hkv, t, s, d, lens, dtype):
    """The root mean square of the errors.  With u = eps / 2 a weight's rounding is off by u of itself at most and, over
    many slots, independently, so that an output is off by u sqrt(sum p^2 v^2) in the mean (0.4 of it in fact); its own
    rounding by u of itself; scores in float32 move every weight by 8e-6 (1 + largest) of itself at most.  One slot of 600 that
    was lost or counted twice would be far outside."""
    ops = _ops()
    g = torch.Generator().manual_seed(s + d)
    k, v = _cache(g, b, hkv, s, d, [n + t for n in lens], dtype)
    q = torch.randn(b, h, t, d, generator=g).to(dtype).cuda()
    tree = (torch.rand(b, t, t, generator=g) < 0.5).cuda() | torch.eye(t, dtype=torch.bool, device="cuda")
    lengths = torch.tensor(lens).cuda()
    want, squares, sums, largest = _squares(q, k, v, lengths, tree)
    got = ops.tree_attention(q, k, v, lengths, tree).double()
    u = torch.finfo(dtype).eps / 2
    bound = float((u * u * (squares + want * want)).mean().sqrt()) + 8e-6 * (1 + largest) * float((sums * sums).mean().sqrt())
    error = float((got - want).square().mean().sqrt())
    assert error <= bound, (error, bound)
    v[:, :, min(lens) // 2] = 0                                             # the bound tells one committed slot more or less
    without = ops.tree_attention(q, k, v, lengths, tree).double()
    assert float((without - want).square().mean().sqrt()) > 2 * bound
