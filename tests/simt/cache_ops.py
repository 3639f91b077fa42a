"""``bittorch_b200.ops`` over the cache kernels that are compiled for the CPU: the whole host side of a call (checks, plans,
strides, pointers) with CPU tensors.  TEST INFRASTRUCTURE ONLY."""

from __future__ import annotations

import contextlib

import torch

from tests.simt import cache_harness as H

_PLANS = ("_attention_plan", "_evict_plan", "_compact_plan", "_evict_cache_plan", "_beam_plan", "_reorder_plan")


@contextlib.contextmanager
def on_the_cpu(monkeypatch):
    """Within it the operators take CPU tensors.  Gives the list of (entry point, arguments) of the calls that were made."""
    from bittorch_b200 import _cache, ops

    lib, calls = H.lib(), []

    def call(index, fn, *args):
        calls.append((fn.__name__, args))
        H.check(fn(*args, None))

    def clear():
        for name in _PLANS:
            getattr(_cache, name).cache_clear()

    with monkeypatch.context() as m:
        for name in _cache.EXPORTED:
            m.setattr(_cache, name[2:], getattr(lib, name))
        m.setattr(_cache, "_call", call)
        m.setattr(_cache, "_same_device", lambda *a: 0)
        m.setattr(torch.Tensor, "get_device", lambda self: 0)
        m.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
        clear()
        try:
            yield ops, calls
        finally:
            clear()
