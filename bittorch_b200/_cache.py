"""ctypes binding of the operators over a key/value cache (include/bittorch_b200_cache.h), and their argument checks.

The entry points live in the same library as ``_C``'s; they are bound here, on first use, so that a caller of the
linear layers alone needs none of them.  Shapes and types are checked before devices, with messages as
``RuntimeError``; nothing here computes on the CPU.
"""

from __future__ import annotations

import ctypes
import functools
import math
import operator
from typing import Optional, Sequence, Tuple

import torch
import torch.autograd.forward_ad as _forward_ad
from torch import Tensor

from . import _C

_p, _i64, _int, _f32, _size = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_size_t

BEAM_MAX_SELECT = 64
BEAM_MAX_BEAMS = 64
REORDER_MAX_BEAMS = 32
ATTENTION_MAX_HEAD_DIM = 256

_SIGNATURES = {
    "bt_tree_attention_workspace": ([_i64] * 6 + [_int, _int], _size),
    "bt_tree_attention": ([_p, _p, _p, _int] + [_i64] * 6 + [_p, _p, _int, _i64, _p, _i64, _f32, _p, _i64, _i64, _p, _p, _size, _p], _int),
    "bt_evict_select": ([_p, _i64, _i64, _i64, _i64, _i64, _p, _int, _i64, _i64, _i64, _i64, _p, _p, _p], _int),
    "bt_compact_cache": ([_p, _p, _p, _p, _int] + [_i64] * 5 + [_p, _p, _i64, _i64, _i64, _p, _p, _p, _p, _p, _p], _int),
    "bt_beam_select_workspace": ([_i64, _i64, _i64, _int, _i64], _size),
    "bt_beam_select": ([_p, _int] + [_i64] * 5 + [_p, _p, _i64, _i64, _p, _p, _p, _p, _size, _p], _int),
    "bt_reorder_cache": ([_p, _i64, _int] + [_i64] * 5 + [_p, _p, _p, _int, _i64, _i64, _p], _int),
}
EXPORTED = tuple(_SIGNATURES)


def _bind():
    fns = {}
    for name, (argtypes, restype) in _SIGNATURES.items():
        try:
            fn = getattr(_C._lib, name)
        except AttributeError as exc:
            raise ImportError(f"bittorch_b200: {_C.LIB_PATH} is stale (no symbol {name}); rebuild it with "
                              "`python -m bittorch_b200._build`") from exc
        fn.argtypes, fn.restype = argtypes, restype
        fns[name] = fn
    return fns


_fn = _bind()
_tree_attention, _tree_attention_workspace = _fn["bt_tree_attention"], _fn["bt_tree_attention_workspace"]
_evict_select, _compact_cache = _fn["bt_evict_select"], _fn["bt_compact_cache"]
_beam_select, _beam_select_workspace = _fn["bt_beam_select"], _fn["bt_beam_select_workspace"]
_reorder_cache = _fn["bt_reorder_cache"]

_DT = _C._DT
# What a call writes in place counts as changed: autograd refuses to go back through a graph that has saved it
_written = torch.autograd.graph.increment_version
_SIX, _TWELVE, _FOUR = _i64 * 6, _i64 * 12, _i64 * 4


def _fail(text: str):
    raise RuntimeError(text)


def _require(ok: bool, text: str) -> None:
    if not ok:
        raise RuntimeError(text)


def _no_gradient(what: str, *tensors: Optional[Tensor]) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                _fail(f"{what} has no backward pass: call it under torch.no_grad()")
    if _forward_ad._current_level >= 0 and any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        _fail(f"{what} has no forward-mode derivative: its output would lose the tangent")


def _on_one_device(what: str, *tensors: Optional[Tensor]) -> torch.device:
    dev = tensors[0].device
    for t in tensors:
        if t is not None:
            if not t.is_cuda:
                _fail("All tensors must be CUDA")
            if t.device != dev:
                _fail(f"{what}: all tensors must be on one device")
    return dev


def _plain_memory(t: Tensor) -> bool:
    """No two elements of ``t`` share memory (what is written in place must not)."""
    if t.is_contiguous():
        return True
    span = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        if stride < span:
            return False
        span = stride * size
    return True


def _span(shape, stride, dtype: torch.dtype) -> int:
    """Bytes from the first element of a tensor to behind its last."""
    return (1 + sum((n - 1) * st for n, st in zip(shape, stride))) * dtype.itemsize


@functools.lru_cache(maxsize=1024)
def _meet(a_sig, b_sig, distance: int) -> bool:
    """Whether tensors of these shapes, strides and types have a byte in common, the second ``distance`` bytes behind the
    first.  A byte of the first less one of the second is a sum of steps, each taken a bounded number of times; from the
    longest step down, what is left must be within reach of the shorter ones, which for the nested strides of a tensor
    leaves one or two numbers to try.  Layouts that take more than 4096 trials count as meeting."""
    steps = {}
    for (shape, stride, dtype), sign in ((a_sig, 1), (b_sig, -1)):
        for n, st in (*zip(shape, (st * dtype.itemsize for st in stride)), (dtype.itemsize, 1)):
            if n > 1 and st > 0:
                low, high = steps.get(st, (0, 0))
                steps[st] = (low - (n - 1), high) if sign < 0 else (low, high + n - 1)
    order = sorted(steps, reverse=True)
    reach = [0]                                            # of the steps from a place on, each counted from its lowest number
    for st in reversed(order):
        reach.insert(0, reach[0] + st * (steps[st][1] - steps[st][0]))
    trials = 0

    def solve(i: int, left: int) -> bool:
        nonlocal trials
        trials += 1
        if trials > 4096 or left == 0:
            return True
        if i == len(order) or left > reach[i]:
            return False
        st = order[i]
        most = min(left // st, steps[st][1] - steps[st][0])
        least = max(0, -((reach[i + 1] - left) // st))
        return any(solve(i + 1, left - n * st) for n in range(most, least - 1, -1))

    target = distance - sum(st * low for st, (low, _) in steps.items())
    return target >= 0 and solve(0, target)


def _behind_one_another(addresses, spans) -> bool:
    """Whether tensors lie one behind the other: the usual case, in which none shares memory with another."""
    end = 0
    for at, span in sorted(zip(addresses, spans)):
        if at < end:
            return False
        end = at + span
    return True


def _apart(sigs, addresses, spans, written: int) -> bool:
    """Whether the first ``written`` of the tensors share no memory with one another or with the rest, which may share theirs."""
    if _behind_one_another(addresses, spans):
        return True
    for i in range(written):
        for j in range(i + 1, len(sigs)):
            distance = addresses[j] - addresses[i]
            if -spans[j] < distance < spans[i] and _meet(sigs[i], sigs[j], distance):
                return False
    return True


def _rows(t: Tensor) -> Tensor:
    """``t`` with the elements of its last dimension side by side: itself, or a copy.  Plans and calls both go by it, so that
    strides and pointer are of one tensor (a single element lies beside itself whatever its stride says)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _call(index: int, fn, *args) -> None:
    """Enqueue on the current stream of device ``index``."""
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _C._check(rc)


def _lengths(lengths: Tensor, batch: int) -> Tuple[int, int]:
    """(is int64, stride): one length for the batch, or one per sequence."""
    if lengths.dim() != 1 or lengths.shape[0] not in (1, batch):
        _fail(f"lengths must be [{batch}] or [1], got {list(lengths.shape)}")
    if lengths.dtype is not torch.int64 and lengths.dtype is not torch.int32:
        _fail(f"lengths must be int64 or int32, got {lengths.dtype}")
    return (1 if lengths.dtype is torch.int64 else 0), (0 if lengths.shape[0] == 1 else lengths.stride(0))


def _cache_pair(what: str, k: Tensor, v: Tensor) -> None:
    if k.dim() != 4 or k.shape != v.shape:
        _fail(f"{what}: keys and values must be 4D [B, Hkv, S, D] of one shape")
    if k.dtype != v.dtype or k.dtype not in _DT:
        _fail(f"{what}: keys and values must both be float32, float16 or bfloat16, got {k.dtype} and {v.dtype}")
    if k.numel() == 0:
        _fail(f"{what}: the cache is empty")
    if (k.stride(3) != 1 or v.stride(3) != 1) and k.shape[3] != 1:
        _fail(f"{what}: the head dimension of a cache must be contiguous")


def _same_device(what: str, first: Tensor, *rest: Optional[Tensor]) -> int:
    """The CUDA device index that all tensors are on."""
    index = first.get_device()                         # -1: not on a device
    for t in rest:
        if t is not None and t.get_device() != index:
            _on_one_device(what, first, *rest)
    if index < 0 or not first.is_cuda:
        _fail("All tensors must be CUDA")
    return index


def _sig(t: Optional[Tensor]):
    """What the checks of a call go by: a call whose tensors have been seen with these is not checked again."""
    return None if t is None else (t.shape, t.stride(), t.dtype)


@functools.lru_cache(maxsize=1024)
def _attention_plan(q_sig, k_sig, v_sig, len_sig, tree_sig, scale, mass_sig, out_sig, index):
    """Checks the arguments of tree_attention; -> (what the C call takes of shapes and strides, workspace bytes)."""
    q, k, v, lengths, tree, mass, out = (None if x is None else torch.empty_strided(x[0], x[1], dtype=x[2], device="meta")
                                         for x in (q_sig, k_sig, v_sig, len_sig, tree_sig, mass_sig, out_sig))
    if q.dim() != 4:
        _fail("q must be 4D [B, H, T, D]")
    b, h, t, d = q.shape
    _cache_pair("tree_attention", k, v)
    if q.dtype != k.dtype:
        _fail(f"q must have the cache's type {k.dtype}, got {q.dtype}")
    if k.shape[0] != b or k.shape[3] != d:
        _fail(f"q {list(q.shape)} and the cache {list(k.shape)} differ in batch or head size")
    hkv, s = k.shape[1], k.shape[2]
    if q.numel() == 0:
        _fail("q is empty")
    if h % hkv:
        _fail(f"{h} query heads are not a multiple of {hkv} key/value heads")
    if d > ATTENTION_MAX_HEAD_DIM:
        _fail(f"head sizes up to {ATTENTION_MAX_HEAD_DIM} are supported, got {d}")
    if t > s:
        _fail(f"{t} new tokens do not fit a cache of {s} slots")
    len64, len_stride = _lengths(lengths, b)
    tree_sb = 0
    if tree is not None:
        if tree.dtype is not torch.bool or tuple(tree.shape) not in ((t, t), (b, t, t)):
            _fail(f"tree must be bool [{t}, {t}] or [{b}, {t}, {t}], got {tree.dtype} {list(tree.shape)}")
        tree_sb = t * t if tree.dim() == 3 else 0
    if not math.isfinite(scale):
        _fail("scale must be finite")
    if mass is not None:
        if mass.dtype is not torch.float32 or mass.shape != k.shape[:3]:
            _fail(f"mass must be float32 {list(k.shape[:3])}, got {mass.dtype} {list(mass.shape)}")
        if (mass.stride(2) != 1 and s != 1) or not _plain_memory(mass):
            _fail("mass must have contiguous slots that share no memory")
    if out is not None:
        if out.shape != q.shape or out.dtype != q.dtype:
            _fail(f"out must be {q.dtype} {list(q.shape)}, got {out.dtype} {list(out.shape)}")
        if (out.stride(3) != 1 and d != 1) or not _plain_memory(out):
            _fail("out must have a contiguous head dimension and share no memory with itself")
    if index < 0:
        return None
    out_strides = (t * h * d, d, h * d, 1) if out is None else out.stride()      # [B, T, H * D]: as the next projection reads it
    strides = _TWELVE(*_rows(q).stride()[:3], *k.stride()[:3], *v.stride()[:3], *out_strides[:3])
    code = _DT[q.dtype]
    sizes = (b, h, hkv, t, s, d)
    with torch.cuda.device(index):                     # the workspace depends on the device's SM count
        need = _tree_attention_workspace(*sizes, code, mass is not None)
    sigs = [sig for sig in (out_sig, mass_sig, q_sig, k_sig, v_sig) if sig is not None]
    memory = (sigs, [_span(*sig) for sig in sigs])
    return ((code, *sizes, strides), (len64, len_stride), tree_sb, ((0, 0) if mass is None else mass.stride()[:2]), need, out_strides, memory,
            _rows(q) is not q)


def tree_attention(q: Tensor, k: Tensor, v: Tensor, lengths: Tensor, tree: Optional[Tensor], scale: Optional[float],
                   mass: Optional[Tensor], out: Optional[Tensor]) -> Tensor:
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    plan = _attention_plan(_sig(q), _sig(k), _sig(v), _sig(lengths), _sig(tree), scale, _sig(mass), _sig(out), q.get_device())
    if torch.is_grad_enabled() or _forward_ad._current_level >= 0:
        _no_gradient("tree_attention", q, k, v, mass, out)
    index = _same_device("tree_attention", q, k, v, lengths, tree, mass, out)
    head, lens, tree_sb, mass_strides, need, out_strides, (sigs, spans), copy_q = plan
    written = None
    if out is not None or mass is not None:
        written = [t for t in (out, mass) if t is not None]
        if not _apart(sigs, [t.data_ptr() for t in (*written, q, k, v)], spans, len(written)):
            _fail("out and mass must be other memory than the queries and the cache, and than each other")
    if copy_q:
        q = q.contiguous()
    if tree is not None and not tree.is_contiguous():
        tree = tree.contiguous()
    dev = q.device
    if out is None:
        out = torch.empty_strided(q.shape, out_strides, dtype=q.dtype, device=dev)
    work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(index, _tree_attention, q.data_ptr(), k.data_ptr(), v.data_ptr(), *head, lengths.data_ptr(), *lens,
          None if tree is None else tree.data_ptr(), tree_sb, scale, None if mass is None else mass.data_ptr(), *mass_strides,
          out.data_ptr(), None if work is None else work.data_ptr(), need)
    if written is not None:
        _written(written)
    return out


@functools.lru_cache(maxsize=1024)
def _evict_plan(mass_sig, len_sig, budget, sinks, recent):
    mass, lengths = (torch.empty_strided(x[0], x[1], dtype=x[2], device="meta") for x in (mass_sig, len_sig))
    if mass.dim() != 3 or mass.dtype is not torch.float32 or mass.numel() == 0:
        _fail(f"mass must be float32 [B, Hkv, S], got {mass.dtype} {list(mass.shape)}")
    if mass.stride(2) != 1 and mass.shape[2] != 1:
        _fail("mass must have contiguous slots")
    b, hkv, s = mass.shape
    if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
        _fail(f"a budget of {budget} slots must be positive and hold {sinks} sinks and {recent} recent slots")
    return (b, hkv, s), mass.stride()[:2], _lengths(lengths, b)


def evict_select(mass: Tensor, lengths: Tensor, budget: int, sinks: int, recent: int) -> Tuple[Tensor, Tensor]:
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    sizes, strides, lens = _evict_plan(_sig(mass), _sig(lengths), budget, sinks, recent)
    index = _same_device("evict_select", mass, lengths)
    b, hkv, _ = sizes
    keep = torch.empty((b, hkv, budget), dtype=torch.int64, device=mass.device)
    counts = torch.empty((b,), dtype=torch.int64, device=mass.device)
    _call(index, _evict_select, mass.data_ptr(), *strides, *sizes, lengths.data_ptr(), *lens, budget, sinks, recent, keep.data_ptr(),
          counts.data_ptr())
    return keep, counts


@functools.lru_cache(maxsize=1024)
def _compact_plan(k_sig, v_sig, keep_sig, counts_sig, first_sig, mass_sig, out_sigs):
    make = lambda x: None if x is None else torch.empty_strided(x[0], x[1], dtype=x[2], device="meta")
    k, v, keep, counts, first, mass = (make(x) for x in (k_sig, v_sig, keep_sig, counts_sig, first_sig, mass_sig))
    _cache_pair("compact_cache", k, v)
    b, hkv, s, d = k.shape
    if out_sigs is None:
        k_out, v_out, mass_out = k, v, mass
    else:
        if len(out_sigs) != (2 if mass is None else 3):
            _fail("out must be (keys, values), with the mass third where one is given")
        k_out, v_out, mass_out = make(out_sigs[0]), make(out_sigs[1]), (make(out_sigs[2]) if mass is not None else None)
        _cache_pair("compact_cache", k_out, v_out)
        if k_out.dtype != k.dtype or k_out.shape[:2] != k.shape[:2] or k_out.shape[3] != d:
            _fail(f"out must be {k.dtype} [{b}, {hkv}, slots, {d}], got {k_out.dtype} {list(k_out.shape)}")
    s_out = k_out.shape[2]
    if keep.dim() != 3 or keep.dtype is not torch.int64 or keep.shape[0] != b or keep.shape[1] not in (1, hkv) or keep.shape[2] == 0:
        _fail(f"keep must be int64 [{b}, {hkv} or 1, n], got {keep.dtype} {list(keep.shape)}")
    for name, t in (("counts", counts), ("first", first)):
        if t is not None and (t.dtype is not torch.int64 or tuple(t.shape) != (b,)):
            _fail(f"{name} must be int64 [{b}], got {t.dtype} {list(t.shape)}")
    if mass is not None:
        for m, slots in ((mass, s), (mass_out, s_out)):
            if m.dtype is not torch.float32 or tuple(m.shape) != (b, hkv, slots) or (m.stride(2) != 1 and slots != 1):
                _fail(f"mass must be float32 [{b}, {hkv}, {slots}] with contiguous slots, got {m.dtype} {list(m.shape)}")
    if not (_plain_memory(k_out) and _plain_memory(v_out) and (mass_out is None or _plain_memory(mass_out))):
        _fail("compact_cache: what is written must share no memory with itself")
    n = keep.shape[2]
    keep_strides = _rows(keep).stride()
    strides = _TWELVE(*k.stride()[:3], *v.stride()[:3], *k_out.stride()[:3], *v_out.stride()[:3])
    mass_strides = None if mass is None else _FOUR(*mass.stride()[:2], *mass_out.stride()[:2])
    sigs = [*(out_sigs or ()), *(sig for sig in (k_sig, v_sig, mass_sig) if sig is not None)]
    memory = (sigs, [_span(*sig) for sig in sigs], 2 if mass is None else 3)          # as _apart takes it
    return ((_DT[k.dtype], b, hkv, s, s_out, d, strides), (keep_strides[0], keep_strides[1] if keep.shape[1] == hkv else 0, n), mass_strides,
            memory, _rows(keep) is not keep)


def compact_cache(k: Tensor, v: Tensor, keep: Tensor, counts: Tensor, first: Optional[Tensor], mass: Optional[Tensor],
                  out: Optional[Sequence[Tensor]]) -> None:
    head, tail, mass_strides, (sigs, spans, written), copy_keep = _compact_plan(_sig(k), _sig(v), _sig(keep), _sig(counts), _sig(first), _sig(mass),
                                                                                None if out is None else tuple([_sig(x) for x in out]))
    k_out, v_out, mass_out = (k, v, mass) if out is None else (out[0], out[1], out[2] if mass is not None else None)
    if torch.is_grad_enabled() or _forward_ad._current_level >= 0:
        _no_gradient("compact_cache", k, v, k_out, v_out, mass, mass_out)
    at = [t.data_ptr() for t in ((k, v) if mass is None else (k, v, mass))]
    to = at if out is None else [t.data_ptr() for t in out]
    if not _apart(sigs, at if out is None else to + at, spans, written):
        _fail("keys and values (and mass) that share the same memory cannot be compacted in place" if out is None else
              "out must be other memory than the cache and share none within itself (leave it out to compact in place)")
    index = _same_device("compact_cache", k, v, k_out, v_out, keep, counts, first, mass, mass_out)
    if copy_keep:
        keep = keep.contiguous()
    counts = counts.contiguous()
    first = None if first is None else first.contiguous()
    _call(index, _compact_cache, *at[:2], *to[:2], *head, keep.data_ptr(), *tail, counts.data_ptr(), None if first is None else first.data_ptr(),
          None if mass is None else at[2], None if mass is None else to[2], mass_strides)
    _written((k_out, v_out) if mass is None else (k_out, v_out, mass_out))


@functools.lru_cache(maxsize=1024)
def _evict_cache_plan(k_sig, v_sig, mass_sig, len_sig, budget, sinks, recent, out_sigs):
    if len(k_sig[0]) != 4 or mass_sig[0] != k_sig[0][:3]:
        _fail(f"mass must be float32 {list(k_sig[0][:3])}, got {mass_sig[2]} {list(mass_sig[0])}")
    if out_sigs is not None and (len(out_sigs) != 3 or len(out_sigs[0][0]) != 4 or out_sigs[0][0][2] < budget):
        _fail(f"out must be (keys, values, mass) of at least {budget} slots")
    b, hkv = mass_sig[0][:2]
    select = _evict_plan(mass_sig, len_sig, budget, sinks, recent)
    keep = (torch.Size((b, hkv, budget)), (hkv * budget, budget, 1), torch.int64)
    return select, _compact_plan(k_sig, v_sig, keep, (torch.Size((b,)), (1,), torch.int64), None, mass_sig, out_sigs)


def evict_cache(k: Tensor, v: Tensor, mass: Tensor, lengths: Tensor, budget: int, sinks: int, recent: int,
                out: Optional[Sequence[Tensor]]) -> Tuple[Tensor, Tensor]:
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    (sizes, strides, lens), (head, tail, mass_strides, (sigs, spans, written), _) = _evict_cache_plan(
        _sig(k), _sig(v), _sig(mass), _sig(lengths), budget, sinks, recent, None if out is None else tuple([_sig(x) for x in out]))
    k_out, v_out, mass_out = (k, v, mass) if out is None else out
    if torch.is_grad_enabled() or _forward_ad._current_level >= 0:
        _no_gradient("evict_cache", k, v, k_out, v_out, mass, mass_out)
    at = [k.data_ptr(), v.data_ptr(), mass.data_ptr()]
    to = at if out is None else [k_out.data_ptr(), v_out.data_ptr(), mass_out.data_ptr()]
    if not _apart(sigs, at if out is None else to + at, spans, written):
        _fail("keys, values and mass that share the same memory cannot be evicted from in place" if out is None else
              "out must be other memory than the cache and share none within itself (leave it out to evict in place)")
    if out is None:
        index = _same_device("evict_cache", k, v, mass, lengths)
    else:
        index = _same_device("evict_cache", k, v, mass, lengths, k_out, v_out, mass_out)
    b, hkv, _ = sizes
    keep = torch.empty((b, hkv, budget), dtype=torch.int64, device=k.device)
    counts = torch.empty((b,), dtype=torch.int64, device=k.device)
    keep_at, counts_at = keep.data_ptr(), counts.data_ptr()
    _call(index, _evict_select, at[2], *strides, *sizes, lengths.data_ptr(), *lens, budget, sinks, recent, keep_at, counts_at)
    _call(index, _compact_cache, at[0], at[1], to[0], to[1], *head, keep_at, *tail, counts_at, None, at[2], to[2], mass_strides)
    _written((k_out, v_out, mass_out))
    return keep, counts


@functools.lru_cache(maxsize=1024)
def _beam_plan(logits_sig, scores_sig, select, finished_sig, end_token):
    logits, scores, finished = (None if x is None else torch.empty_strided(x[0], x[1], dtype=x[2], device="meta")
                                for x in (logits_sig, scores_sig, finished_sig))
    if logits.dim() != 3 or logits.dtype not in _DT:
        _fail(f"logits must be float32, float16 or bfloat16 [B, beams, vocabulary], got {logits.dtype} {list(logits.shape)}")
    b, w, vocab = logits.shape
    if logits.numel() == 0:
        _fail("logits are empty")
    n = w if select is None else select
    if scores.dtype is not torch.float32 or scores.shape != (b, w):
        _fail(f"scores must be float32 [{b}, {w}], got {scores.dtype} {list(scores.shape)}")
    if not 1 <= w <= BEAM_MAX_BEAMS:
        _fail(f"up to {BEAM_MAX_BEAMS} beams are supported, got {w}")
    if not 1 <= n <= min(BEAM_MAX_SELECT, w * vocab):
        _fail(f"select must be 1 to {min(BEAM_MAX_SELECT, w * vocab)}, got {n}")
    if (finished is None) != (end_token is None):
        _fail("finished and end_token come together")
    if finished is not None:
        if finished.dtype is not torch.bool or finished.shape != (b, w):
            _fail(f"finished must be bool [{b}, {w}], got {finished.dtype} {list(finished.shape)}")
        if not 0 <= end_token < vocab:
            _fail(f"end_token {end_token} is outside the vocabulary of {vocab}")
    code = _DT[logits.dtype]
    return (code, b, w, vocab, *_rows(logits).stride()[:2]), n, _beam_select_workspace(b, w, vocab, code, n), _rows(logits) is not logits


def beam_select(logits: Tensor, scores: Tensor, select: Optional[int], finished: Optional[Tensor],
                end_token: Optional[int]) -> Tuple[Tensor, Tensor, Tensor]:
    select = None if select is None else int(select)
    end_token = None if end_token is None else operator.index(end_token)
    head, n, need, copy_logits = _beam_plan(_sig(logits), _sig(scores), select, _sig(finished), end_token)
    if torch.is_grad_enabled() or _forward_ad._current_level >= 0:
        _no_gradient("beam_select", logits, scores)
    index = _same_device("beam_select", logits, scores, finished)
    if copy_logits:
        logits = logits.contiguous()
    if not scores.is_contiguous():
        scores = scores.contiguous()
    if finished is not None and not finished.is_contiguous():
        finished = finished.contiguous()
    dev, b = logits.device, head[1]
    out = torch.empty((b, n), dtype=torch.float32, device=dev)
    tokens = torch.empty((b, n), dtype=torch.int64, device=dev)
    parents = torch.empty((b, n), dtype=torch.int64, device=dev)
    work = torch.empty(need, dtype=torch.uint8, device=dev)
    _call(index, _beam_select, logits.data_ptr(), *head, scores.data_ptr(), None if finished is None else finished.data_ptr(),
          0 if end_token is None else end_token, n, out.data_ptr(), tokens.data_ptr(), parents.data_ptr(), work.data_ptr(), need)
    return out, tokens, parents


@functools.lru_cache(maxsize=1024)
def _reorder_plan(sigs, parents_sig, len_sig, start):
    parents, lengths = (torch.empty_strided(x[0], x[1], dtype=x[2], device="meta") for x in (parents_sig, len_sig))
    if len(sigs) == 0:
        _fail("reorder_cache: no cache tensors")
    if parents.dim() != 2 or parents.dtype is not torch.int64 or parents.numel() == 0:
        _fail(f"parents must be int64 [B, beams], got {parents.dtype} {list(parents.shape)}")
    b, w = parents.shape
    if w > REORDER_MAX_BEAMS:
        _fail(f"up to {REORDER_MAX_BEAMS} beams are supported, got {w}")
    shape, _, dtype = sigs[0]
    if len(shape) != 4 or shape[0] != b * w or 0 in shape or dtype not in _DT:
        _fail(f"cache tensors must be float32, float16 or bfloat16 [{b * w}, Hkv, S, D], got {dtype} {list(shape)}")
    _require(start >= 0, "start must not be negative")
    strides = []
    for size, stride, kind in sigs:
        if size != shape or kind != dtype:
            _fail("reorder_cache: all cache tensors must have one shape and type")
        if (stride[3] != 1 and shape[3] != 1) or not _plain_memory(torch.empty_strided(size, stride, dtype=kind, device="meta")):
            _fail("reorder_cache: cache tensors must have a contiguous head dimension and share no memory with themselves")
        strides += stride[:3]
    count = len(sigs)
    spans = [_span(*sig) for sig in sigs]
    return ((count, _DT[dtype], b, w, *shape[1:], (_i64 * (3 * count))(*strides)), _lengths(lengths, b),
            spans, _p * count, functools.lru_cache(maxsize=16)(lambda offsets: _apart(sigs, offsets, spans, count)))


def reorder_cache(caches: Sequence[Tensor], parents: Tensor, lengths: Tensor, start: int) -> None:
    start = int(start)
    head, lens, spans, pointer_array, views_apart = _reorder_plan(tuple([_sig(c) for c in caches]), _sig(parents), _sig(lengths), start)
    if torch.is_grad_enabled() or _forward_ad._current_level >= 0:
        _no_gradient("reorder_cache", *caches)
    index = _same_device("reorder_cache", parents, lengths, *caches)
    pointers = [c.data_ptr() for c in caches]
    if len(pointers) > 1:
        # views of one buffer are looked at element by element, once for their distances
        if not _behind_one_another(pointers, spans) and not views_apart(tuple([p - pointers[0] for p in pointers])):
            _fail("reorder_cache: a cache tensor is listed twice, or two share memory")
    if not parents.is_contiguous():
        parents = parents.contiguous()
    _call(index, _reorder_cache, pointer_array(*pointers), *head, parents.data_ptr(), lengths.data_ptr(), *lens, start)
    _written(caches)
