"""Serving calls on inputs at the edge of their definitions: zero, infinite and
NaN values, rows that see little or nothing, rows and sequences nobody owns.

Tolerances are those of test_gpu_paged.py unless a test derives its own.
"""

import ctypes
import math

import numpy as np
import pytest
import torch

from conftest import has_gpu
from test_gpu_paged import ACT, CACHE, CACHES, Setup, compare, gen, settle, tolerance, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    if not has_gpu():
        pytest.skip("no CUDA device")
    from lbr_b200 import paged as m
    return m


def place(s, b, pos):
    return int(s.table[b, pos // s.page]), pos % s.page


def owners(s):
    """(sequence, position) of every row of q."""
    return [(b, n - m + i) for b, (n, m) in enumerate(zip(s.lens, s.new)) for i in range(m)]


# ------------------------------------------------------------------ small heads in the cache
@pytest.mark.parametrize("cache", ["f32", "bf16", "i8", "f8"])
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("heads,dim,n", [(5, 16, 5), (7, 16, 7), (3, 16, 3), (19, 16, 5000), (33, 16, 5000), (5, 32, 5), (9, 48, 7)])
def test_write_of_tokens_that_fill_no_warp(paged, cache, act, heads, dim, n):
    """Tokens of a few lanes, whose block ends inside a warp; nothing else of the cache changes."""
    g, page = gen(29), 16
    n_pages = -(-n // page) + 2
    pages = [torch.full((n_pages, page, heads, dim), 3.0, device="cuda").to(CACHE[cache]) for _ in "kv"]
    scale = [torch.full((n_pages, page, heads), 5.0, device="cuda") if cache in ("i8", "f8") else None for _ in "kv"]
    k, v = (torch.randn(n, heads, dim, generator=g, device="cuda").to(ACT[act]) for _ in "kv")
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:n]
    paged.kv_write(k, v, pages[0], pages[1], slots, k_scale=scale[0], v_scale=scale[1])
    paged.check_stream()
    other = torch.ones(n_pages * page, dtype=torch.bool, device="cuda")
    other[slots] = False
    for x, p, sc in zip((k, v), pages, scale):
        got = p.flatten(0, 1).float()
        assert bool((got[other] == 3.0).all())
        x = x.float()
        if sc is None:
            assert torch.equal(got[slots], x.to(CACHE[cache]).float())
            continue
        sc = sc.flatten(0, 1)
        assert bool((sc[other] == 5.0).all())
        # half a code (i8: scale / 2; e4m3: 2^-4 of the value or 2^-10 scales), with the products' own roundings
        top = x.abs().amax(-1, keepdim=True)
        tol = top / 127 * 0.5001 if cache == "i8" else torch.maximum(x.abs() * 2.0 ** -4, top / 448 * 2.0 ** -10) * 1.0001
        assert bool(((got[slots] * sc[slots][..., None] - x).abs() <= tol + x.abs() * 2.0 ** -22).all())
