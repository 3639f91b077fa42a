"""libbt_simt_cache.so: the kernels over a key/value cache compiled for the CPU, called with torch CPU tensors.
TEST INFRASTRUCTURE ONLY.  Same entry points and argument order as include/bittorch_b200_cache.h."""

from __future__ import annotations

import ctypes
import os
import subprocess

import torch

from tests.simt.harness import CSRC, HERE, ROOT, cuda_include_dir

LIB = os.path.join(HERE, "libbt_simt_cache.so")
DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_lib = None


def build() -> str:
    """g++, about 10 s.  `-fsanitize=address` finds reads outside the caller's buffers (see tests/simt/harness.py)."""
    sources = [os.path.join(HERE, f) for f in ("cache_lib.cpp", "simt_host.h")]
    sources += [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cuh")]
    sources += [os.path.join(ROOT, "include", f) for f in os.listdir(os.path.join(ROOT, "include"))]
    if not os.path.exists(LIB) or any(os.path.getmtime(s) > os.path.getmtime(LIB) for s in sources):
        subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-ffp-contract=off", "-fno-fast-math", "-fPIC", "-shared", "-pthread",
                               "-Wno-attributes", *os.environ.get("SIMT_CXXFLAGS", "").split(), "-I" + cuda_include_dir(), "-o", LIB,
                               os.path.join(HERE, "cache_lib.cpp")])
    return LIB


def lib():
    global _lib
    if _lib is None:
        from bittorch_b200 import _cache

        _lib = ctypes.CDLL(build())
        _lib.bt_last_error.restype = ctypes.c_char_p
        _lib.simt_take_errors.argtypes = [ctypes.c_char_p, ctypes.c_size_t]
        for name, (argtypes, restype) in _cache._SIGNATURES.items():
            fn = getattr(_lib, name)
            fn.argtypes, fn.restype = argtypes, restype
    return _lib


def check(rc: int) -> None:
    buf = ctypes.create_string_buffer(512)
    broken = lib().simt_take_errors(buf, 512)
    if rc != 0:
        raise RuntimeError(lib().bt_last_error().decode() or f"status {rc}")
    if broken:
        raise RuntimeError(f"emulated hardware rule broken: {buf.value.decode()}")


def set_sm_count(n: int) -> None:
    lib().simt_set_sm_count(n)


def ptr(t):
    return None if t is None else t.data_ptr()


def _i64s(*values):
    return (ctypes.c_int64 * len(values))(*values)


def _len(lengths):
    return int(lengths.dtype == torch.int64), (0 if lengths.numel() == 1 else lengths.stride(0))


def aligned_bytes(n):
    raw = torch.empty(n + 16, dtype=torch.uint8)
    off = (-raw.data_ptr()) % 16
    return raw[off:off + n]


def tree_attention(q, k, v, lengths, tree=None, scale=None, mass=None):
    b, h, t, d = q.shape
    hkv, s = k.shape[1], k.shape[2]
    out = torch.empty(b, t, h, d, dtype=q.dtype).transpose(1, 2)
    code = DT[q.dtype]
    need = lib().bt_tree_attention_workspace(b, h, hkv, t, s, d, code, int(mass is not None))
    work = aligned_bytes(need)
    i64, stride = _len(lengths)
    check(lib().bt_tree_attention(ptr(q), ptr(k), ptr(v), code, b, h, hkv, t, s, d,
                                  _i64s(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3]), ptr(lengths), i64, stride,
                                  ptr(tree), 0 if tree is None or tree.dim() == 2 else t * t, d ** -0.5 if scale is None else scale,
                                  ptr(mass), *((0, 0) if mass is None else mass.stride()[:2]), ptr(out), ptr(work) if need else None, need, None))
    return out


def evict_select(mass, lengths, budget, sinks, recent):
    b, hkv, s = mass.shape
    keep, counts = torch.empty(b, hkv, budget, dtype=torch.int64), torch.empty(b, dtype=torch.int64)
    i64, stride = _len(lengths)
    check(lib().bt_evict_select(ptr(mass), mass.stride(0), mass.stride(1), b, hkv, s, ptr(lengths), i64, stride, budget, sinks, recent,
                                ptr(keep), ptr(counts), None))
    return keep, counts


def compact_cache(k, v, keep, counts, first=None, mass=None, out=None):
    b, hkv, s, d = k.shape
    ko, vo, mo = (k, v, mass) if out is None else (out[0], out[1], out[2] if mass is not None else None)
    check(lib().bt_compact_cache(ptr(k), ptr(v), ptr(ko), ptr(vo), DT[k.dtype], b, hkv, s, ko.shape[2], d,
                                 _i64s(*k.stride()[:3], *v.stride()[:3], *ko.stride()[:3], *vo.stride()[:3]), ptr(keep), keep.stride(0),
                                 keep.stride(1) if keep.shape[1] == hkv else 0, keep.shape[2], ptr(counts), ptr(first), ptr(mass), ptr(mo),
                                 None if mass is None else _i64s(*mass.stride()[:2], *mo.stride()[:2]), None))


def beam_select(logits, scores, n, finished=None, end_token=None):
    b, w, v = logits.shape
    need = lib().bt_beam_select_workspace(b, w, v, DT[logits.dtype], n)
    work = aligned_bytes(need)
    out, tokens, parents = torch.empty(b, n), torch.empty(b, n, dtype=torch.int64), torch.empty(b, n, dtype=torch.int64)
    check(lib().bt_beam_select(ptr(logits), DT[logits.dtype], b, w, v, logits.stride(0), logits.stride(1), ptr(scores), ptr(finished),
                               0 if end_token is None else end_token, n, ptr(out), ptr(tokens), ptr(parents), ptr(work), need, None))
    return out, tokens, parents


def reorder_cache(caches, parents, lengths, start=0):
    n = len(caches)
    rows, hkv, s, d = caches[0].shape
    b, w = parents.shape
    i64, stride = _len(lengths)
    strides = [x for c in caches for x in c.stride()[:3]]
    check(lib().bt_reorder_cache((ctypes.c_void_p * n)(*[c.data_ptr() for c in caches]), n, DT[caches[0].dtype], b, w, hkv, s, d,
                                 _i64s(*strides), ptr(parents), ptr(lengths), i64, stride, start, None))
