"""The Python side of the operators around the layer, on the CPU."""
import ctypes

import pytest
import torch

from moe_b200 import _lib, ops


LIBRARY = _lib.load()


def size(fmt, t, k):
    n = ctypes.c_size_t()
    assert LIBRARY.moe_fp4_linear_workspace_size(fmt, t, k, ctypes.byref(n)) == 0
    return n.value


class Library:
    """The library, but products want `more` bytes of workspace."""

    def __init__(self, more):
        self.more = more

    def moe_fp4_linear_workspace_size(self, fmt, t, k, n):
        n._obj.value = size(fmt, t, k) + self.more
        return 0


@pytest.mark.parametrize("more", [0, 768])
@pytest.mark.parametrize("t", [1, 4, 5, 16, 129])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_the_library_tells_the_workspace_size(monkeypatch, fmt, t, more):
    """How much a product wants, and from how many tokens on, is the library's to say."""
    k, n = 96, 8
    want = size(ops._FORMATS[fmt], t, k) + more
    monkeypatch.setattr(ops, "_gpu", lambda t, name: 0)
    monkeypatch.setattr(ops, "_same", lambda t, name, index: None)
    got = []
    monkeypatch.setattr(ops, "_call", lambda name, index, *args: got.append((name, args)))
    if more:
        monkeypatch.setattr(_lib, "load", lambda: Library(more))
    cached = getattr(ops, "_linear_workspace", None)
    if cached is not None:
        cached.cache_clear()
    try:
        ops.linear_fp4(torch.zeros(t, k, dtype=torch.bfloat16), torch.zeros(n, k // 2, dtype=torch.uint8),
                       torch.zeros(ops.fp4_scales_shape(n, k, fmt), dtype=torch.uint8), fmt)
    finally:
        if cached is not None:
            cached.cache_clear()
    (name, args), = got
    assert name == "moe_fp4_linear" and args[-1] == want and (args[-2] is None) == (want == 0)
