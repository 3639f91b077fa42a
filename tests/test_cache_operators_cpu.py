"""What needs no GPU of the operators over a key/value cache: the boundary, the refusals, the tree masks."""

import ctypes
import os
import re

import pytest
import torch

from bittorch_b200 import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_header_the_library_and_the_binding_agree():
    from bittorch_b200 import _build, _cache

    text = open(os.path.join(ROOT, "include", "bittorch_b200_cache.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    declared = dict(re.findall(r"\b(bt_[a-z0-9_]+)\s*\(([^)]*)\)", text))
    assert sorted(declared) == sorted(_cache.EXPORTED)
    lib = ctypes.CDLL(_build.build())
    for name, args in declared.items():
        assert hasattr(lib, name)
        assert len(args.split(",")) == len(_cache._SIGNATURES[name][0]), name


def test_the_library_refuses_bad_sizes_and_pointers():
    from bittorch_b200 import _cache

    p = ctypes.c_void_p
    lib = _cache._C._lib
    err = lambda: lib.bt_last_error().decode()
    st = (ctypes.c_int64 * 12)(*[4] * 12)
    args = lambda **kw: [kw.get("q", p(16)), p(16), p(16), kw.get("dtype", 0), 1, kw.get("h", 2), 1, 1, kw.get("s", 8), kw.get("d", 4), st, p(16), 1, 1,
                         None, 0, kw.get("scale", 1.0), None, 0, 0, p(16), p(16), kw.get("bytes", 1 << 20), None]
    assert lib.bt_tree_attention(*args(q=None)) == 1 and "NULL" in err()
    assert lib.bt_tree_attention(*args(dtype=7)) == 1 and "dtype" in err()
    assert lib.bt_tree_attention(*args(h=0)) == 1 and "empty" in err()
    assert lib.bt_tree_attention(*args(d=257)) == 3 and "head size" in err()
    assert lib.bt_tree_attention(*args(s=1 << 31)) == 3
    assert lib.bt_tree_attention(*args(scale=float("nan"))) == 1 and "scale" in err()
    assert lib.bt_tree_attention(*args(s=4096, bytes=0)) == 1 and "workspace" in err()
    assert lib.bt_tree_attention_workspace(1, 2, 1, 1, 4096, 300, 0, 0) == 0
    assert lib.bt_evict_select(p(16), 8, 8, 1, 1, 8, p(16), 1, 1, 4, 3, 2, p(16), p(16), None) == 1 and "budget" in err()
    assert lib.bt_evict_select(None, 8, 8, 1, 1, 8, p(16), 1, 1, 4, 0, 0, p(16), p(16), None) == 1 and "NULL" in err()
    assert lib.bt_compact_cache(p(16), p(32), p(16), p(64), 0, 1, 1, 8, 8, 4, st, p(16), 1, 1, 4, p(16), None, None, None, None, None) == 1
    assert "in place" in err()
    assert lib.bt_compact_cache(p(16), p(32), p(48), p(64), 0, 1, 1, 8, 8, 4, st, p(16), 1, 1, 4, p(16), None, p(16), None, None, None) == 1
    assert "together" in err()
    assert lib.bt_beam_select(p(16), 0, 1, 65, 9, 9, 9, p(16), None, 0, 4, p(16), p(16), p(16), p(16), 1 << 20, None) == 3 and "beams" in err()
    assert lib.bt_beam_select(p(16), 0, 1, 2, 3, 9, 9, p(16), None, 0, 7, p(16), p(16), p(16), p(16), 1 << 20, None) == 1
    assert lib.bt_beam_select(p(16), 0, 1, 2, 9, 9, 9, p(16), p(16), 9, 4, p(16), p(16), p(16), p(16), 1 << 20, None) == 1 and "end token" in err()
    assert lib.bt_reorder_cache((p * 1)(16), 1, 0, 1, 33, 1, 8, 4, st, p(16), p(16), 1, 1, 0, None) == 3 and "beams" in err()
    assert lib.bt_reorder_cache((p * 1)(None), 1, 0, 1, 3, 1, 8, 4, st, p(16), p(16), 1, 1, 0, None) == 1 and "NULL" in err()


def _attention_args(**kw):
    b, h, hkv, t, s, d = (kw.get(k, x) for k, x in (("b", 2), ("h", 4), ("hkv", 2), ("t", 3), ("s", 10), ("d", 8)))
    args = dict(q=torch.zeros(b, h, t, d), k_cache=torch.zeros(b, hkv, s, d), v_cache=torch.zeros(b, hkv, s, d), lengths=torch.zeros(b, dtype=torch.int64))
    return args


@pytest.mark.parametrize("change,message", [
    (lambda a: a.update(q=a["q"][0]), "q must be 4D"),
    (lambda a: a.update(q=a["q"].half()), "cache's type"),
    (lambda a: a.update(q=a["q"].double(), k_cache=a["k_cache"].double(), v_cache=a["v_cache"].double()), "float32, float16 or bfloat16"),
    (lambda a: a.update(v_cache=a["v_cache"][:, :, :5]), "one shape"),
    (lambda a: a.update(q=a["q"][:, :3]), "multiple"),
    (lambda a: a.update(q=torch.zeros(2, 4, 11, 8)), "do not fit"),
    (lambda a: a.update(q=torch.zeros(2, 4, 0, 8)), "empty"),
    (lambda a: a.update(q=torch.zeros(3, 4, 3, 8)), "differ"),
    (lambda a: a.update(k_cache=torch.zeros(2, 2, 8, 10).transpose(2, 3)), "contiguous"),
    (lambda a: a.update(lengths=torch.zeros(3, dtype=torch.int64)), "lengths must be"),
    (lambda a: a.update(lengths=torch.zeros(2)), "int64 or int32"),
    (lambda a: a.update(tree=torch.ones(3, 3)), "tree must be bool"),
    (lambda a: a.update(tree=torch.ones(3, 4, dtype=torch.bool)), "tree must be bool"),
    (lambda a: a.update(scale=float("inf")), "scale"),
    (lambda a: a.update(mass=torch.zeros(2, 2, 9)), "mass must be"),
    (lambda a: a.update(mass=torch.zeros(1, 1, 10).expand(2, 2, 10)), "share no memory"),
    (lambda a: a.update(out=torch.zeros(2, 4, 3, 9)), "out must be"),
    (lambda a: a["q"].requires_grad_(), "no backward"),
    (lambda a: None, "All tensors must be CUDA"),
])
def test_tree_attention_refuses(change, message):
    args = _attention_args()
    change(args)
    with pytest.raises(RuntimeError, match=message):
        ops.tree_attention(**args)
    if message == "no backward":
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            ops.tree_attention(**args)


def test_the_other_operators_refuse():
    k, mass, n = torch.zeros(2, 3, 10, 8), torch.zeros(2, 3, 10), torch.zeros(2, dtype=torch.int64)
    keep = torch.zeros(2, 3, 4, dtype=torch.int64)

    def refuses(message, fn, *args, **kw):
        with pytest.raises(RuntimeError, match=message):
            fn(*args, **kw)

    refuses("mass must be", ops.evict_select, mass.half(), n, 4, 1, 1)
    refuses("budget", ops.evict_select, mass, n, 0, 0, 0)
    refuses("budget", ops.evict_select, mass, n, 4, 3, 2)
    refuses("CUDA", ops.evict_select, mass, n, 4, 1, 1)
    refuses("mass must be", ops.evict_cache, k, k.clone(), mass[:, :, :9], n, 4)
    refuses("at least 4 slots", ops.evict_cache, k, k.clone(), mass, n, 4, 1, 1, out=(k[:, :, :3].clone(), k[:, :, :3].clone(), mass[:, :, :3].clone()))
    refuses("one shape", ops.compact_cache, k, k[:, :2], keep, n)
    refuses("keep must be", ops.compact_cache, k, k.clone(), keep.int(), n)
    refuses("keep must be", ops.compact_cache, k, k.clone(), keep[:, :2], n)
    refuses("counts must be", ops.compact_cache, k, k.clone(), keep, n.int())
    refuses("first must be", ops.compact_cache, k, k.clone(), keep, n, first=n[:1])
    refuses("third", ops.compact_cache, k, k.clone(), keep, n, mass=mass, out=(k.clone(), k.clone()))
    refuses("other memory", ops.compact_cache, k, k.clone(), keep, n, out=(k, k.clone()))
    refuses("share no memory", ops.compact_cache, k[:, :1].expand(2, 3, 10, 8), k.clone(), keep, n)
    refuses("same memory", ops.compact_cache, k, k, keep, n)
    refuses("same memory", ops.evict_cache, k, k, mass, n, 4, 1, 1)
    refuses("other memory", ops.evict_cache, k, k.clone(), mass, n, 4, 1, 1, out=(k, k.clone(), mass.clone()))
    refuses("CUDA", ops.compact_cache, k, k.clone(), keep, n)
    x, s = torch.zeros(2, 3, 50), torch.zeros(2, 3)
    refuses("logits must be", ops.beam_select, x[0], s)
    refuses("logits must be", ops.beam_select, x.double(), s)
    refuses("scores must be", ops.beam_select, x, s[:, :2])
    refuses("select must be", ops.beam_select, x, s, 65)
    refuses("select must be", ops.beam_select, x[:, :, :2], s, 7)
    refuses("beams are supported", ops.beam_select, torch.zeros(1, 65, 9), torch.zeros(1, 65))
    refuses("come together", ops.beam_select, x, s, 3, s > 0)
    refuses("outside the vocabulary", ops.beam_select, x, s, 3, s > 0, 50)
    refuses("finished must be", ops.beam_select, x, s, 3, s, 5)
    refuses("CUDA", ops.beam_select, x, s, 3)
    parents = torch.zeros(1, 2, dtype=torch.int64)
    refuses("no cache", ops.reorder_cache, [], parents, n[:1])
    refuses("parents must be", ops.reorder_cache, [k], parents.int(), n[:1])
    refuses("beams are supported", ops.reorder_cache, [k], torch.zeros(1, 33, dtype=torch.int64), n[:1])
    refuses("cache tensors must be", ops.reorder_cache, [k], torch.zeros(1, 3, dtype=torch.int64), n[:1])
    refuses("one shape", ops.reorder_cache, [k, k[:, :, :5]], parents, n[:1])
    refuses("negative", ops.reorder_cache, [k], parents, n[:1], start=-1)
    refuses("share no memory", ops.reorder_cache, [k[:, :1].expand(2, 3, 10, 8)], parents, n[:1])
    refuses("CUDA", ops.reorder_cache, [k, k], parents, n[:1])


def test_tree_mask_is_the_ancestors():
    parents = torch.tensor([[-1, 0, 0, 1, 3, -1, 5], [-1, -1, 1, 2, -2, -2, 2]])
    mask = ops.tree_mask(parents)
    assert mask.dtype == torch.bool and mask.shape == (2, 7, 7)
    for b in range(2):
        for i in range(7):
            want, at = set(), i if parents[b, i] != -2 else -1
            while at >= 0:
                want.add(at)
                at = int(parents[b, at])
            assert set(mask[b, i].nonzero()[:, 0].tolist()) == want
        assert torch.equal(ops.tree_mask(parents[b]), mask[b])
    for bad in ([0], [-1, 1], [-3], [-2, 0]):
        with pytest.raises(RuntimeError, match="parent"):
            ops.tree_mask(torch.tensor(bad))
    with pytest.raises(RuntimeError, match="int32 or int64"):
        ops.tree_mask(torch.zeros(3))
