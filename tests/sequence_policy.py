"""Shared helpers of the tests of the recurrence, token log-prob, policy and preference operators."""
import numpy as np
import pytest
import torch

from conftest import pkg

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# Half of each type's smallest step near 0 (its subnormals).
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def load_ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    p = pkg()
    p.load()
    return p.ops


def near(got, want, error, what=""):
    """got (a tensor) is want (fp64) within `error`, plus the rounding to got's type; NaN and infinities agree."""
    g = got.detach().cpu().double().numpy()
    want, error = np.asarray(want, np.float64), np.broadcast_to(np.asarray(error, np.float64), np.shape(want))
    assert g.shape == want.shape, (what, g.shape, want.shape)
    odd = ~np.isfinite(want)
    assert np.array_equal(np.isnan(g), np.isnan(want)), f"{what}: NaN in other places"
    inf = np.isinf(want)
    assert np.array_equal(g[inf], want[inf]), f"{what}: infinities differ"
    room = error + HALF_STEP[got.dtype] * (np.abs(want) + error) + TINY[got.dtype]
    off = np.abs(np.where(odd, 0.0, g - np.where(odd, 0.0, want)))
    bad = (off > room) & ~odd
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.size} off, worst {np.nanmax(np.where(bad, off / room, 0)):.3g} "
                           f"times the bound at {np.argwhere(bad)[0]}")


def bits(t):
    t = t.detach()
    return t.contiguous().view({4: torch.int32, 2: torch.int16, 8: torch.int64, 1: torch.uint8}[t.element_size()])


def same_bits(a, b):
    return torch.equal(bits(a), bits(b))


def captured(fn):
    """fn captured into a CUDA graph (after one eager call): (graph, what the captured call returned)."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out
