"""Serving calls without a GPU: structure layout, refusals that need no device."""

import ctypes

import pytest
import torch

from lbr_b200 import executor

paged = pytest.importorskip("lbr_b200.paged")


def test_structs_match_the_header():
    """Sizes the C compiler gives the structures of include/b200exec.h (LP64)."""
    sizes = {paged.RtKvCache: 104, paged.RtKvWrite: 168, paged.RtKvRead: 200, paged.RtPagedAttention: 232,
             paged.RtVerifyDraft: 120}
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


@pytest.mark.skipif(not executor.LIB_PATH.exists(), reason="library not built")
def test_refusals_before_any_device():
    x = torch.zeros(2, 4, 64)
    pages = torch.zeros(3, 16, 4, 64)
    slots = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        paged.kv_write(x, x, pages, pages, slots)
    with pytest.raises(TypeError, match="cache holds"):
        paged.kv_write(x, x, pages.half(), pages.half(), slots)
    with pytest.raises(TypeError, match="v_pages"):
        paged.kv_write(x, x, pages, pages.bfloat16(), slots)
    with pytest.raises(TypeError, match="tensor"):
        paged.kv_write(None, x, pages, pages, slots)
    with pytest.raises(TypeError, match="dtype"):
        paged.kv_read(pages, pages, slots, None, slots, 1, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.verify_draft(x, x[:, :3], slots, slots, slots)
