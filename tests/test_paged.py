"""Serving calls without a GPU: structure layout, refusals that need no device."""

import ctypes

import pytest
import torch

from lbr_b200 import executor

paged = pytest.importorskip("lbr_b200.paged")


def test_structs_match_the_header():
    """Sizes the C compiler gives the structures of include/b200exec.h (LP64)."""
    sizes = {paged.RtKvCache: 104, paged.RtKvWrite: 168, paged.RtKvRead: 200, paged.RtPagedAttention: 232,
             paged.RtVerifyDraft: 112}
    for struct, size in sizes.items():
        assert ctypes.sizeof(struct) == size, struct.__name__


@pytest.mark.skipif(not executor.LIB_PATH.exists(), reason="library not built")
def test_calls_need_init_and_arguments():
    lib = ctypes.CDLL(str(executor.LIB_PATH))
    for name in ("rt_kv_write", "rt_kv_read", "rt_verify_draft"):
        fn = getattr(lib, name)
        fn.argtypes, fn.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
        assert fn(None, None) != 0
    lib.rt_paged_attention_workspace.restype = ctypes.c_size_t
    assert lib.rt_paged_attention_workspace(None) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 4, 64)
    pages = torch.zeros(3, 16, 4, 64)
    c = paged.RtKvCache()
    with pytest.raises(ValueError, match="CUDA"):
        paged._cache(c, pages, pages, None, None)
    with pytest.raises(TypeError):
        paged._cache(c, pages.half(), pages.half(), None, None)
    with pytest.raises(TypeError):
        paged._rows(x.half(), "k", (2, 4, 64), x.device)
    with pytest.raises(ValueError):
        paged._rows(x, "k", (2, 5, 64), x.device)
    with pytest.raises(ValueError):
        paged._rows(x.transpose(1, 2), "k", (2, 64, 4), x.device)
    with pytest.raises(TypeError):
        paged._index(torch.zeros(4), "slots", 4, torch.int64, x.device)
    with pytest.raises(ValueError):
        paged._index(torch.zeros(8, dtype=torch.int64)[::2], "slots", 4, torch.int64, x.device)
