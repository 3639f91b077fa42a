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
