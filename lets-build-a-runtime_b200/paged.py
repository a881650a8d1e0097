"""Serving calls: a paged key/value cache, attention over it, drafted tokens.

The reference generates text by re-planning and re-running the whole prefix for
every token (run_gpt2.py:92-113).  These calls are what a decoder keeps beside
its planned graph instead: :func:`kv_write` stores the keys and values of new
tokens in the pages of a cache (quantised for 8-bit caches), :func:`paged_attention`
attends over them, :func:`kv_read` reads them back and :func:`verify_draft`
settles which drafted tokens stand.

They take CUDA tensors of the device the library runs on, enqueue on torch's
current stream and do not wait, so they can be captured into a CUDA graph.
Arguments are checked before anything is enqueued: a wrong type, shape or device
raises ``TypeError`` / ``ValueError``, a refusal of the library
``CudaRuntimeError`` with its status.  Slots, page numbers and lengths live on
the device; the kernels skip what is out of range and :func:`check_stream` raises
for it.
"""

from __future__ import annotations

import ctypes
import importlib.util

import torch

from .executor import LIB_PATH, CudaRuntimeError, load_library

_I64x2, _I64x3 = ctypes.c_int64 * 2, ctypes.c_int64 * 3
_vp, _i, _f, _l = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_int64


# The structures of include/b200exec.h, for callers of the C ABI.
class RtKvCache(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("stride", _I64x3),
                ("scale_stride", _I64x3), ("dtype", _i), ("n_pages", _i), ("page_size", _i), ("n_heads", _i),
                ("head_dim", _i), ("flags", _i)]


class RtKvWrite(ctypes.Structure):
    _fields_ = [("cache", RtKvCache), ("k", _vp), ("v", _vp), ("k_stride", _I64x2), ("v_stride", _I64x2),
                ("slots", _vp), ("dtype", _i), ("n_tokens", _i)]


class RtKvRead(ctypes.Structure):
    _fields_ = [("cache", RtKvCache), ("k_out", _vp), ("v_out", _vp), ("k_stride", _I64x2), ("v_stride", _I64x2),
                ("page_table", _vp), ("table_stride", _l), ("start", _vp), ("cu", _vp), ("dtype", _i),
                ("n_seqs", _i), ("table_width", _i), ("n_rows", _i)]


class RtPagedAttention(ctypes.Structure):
    _fields_ = [("cache", RtKvCache), ("q", _vp), ("out", _vp), ("lse", _vp), ("q_stride", _I64x2),
                ("out_stride", _I64x2), ("page_table", _vp), ("table_stride", _l), ("kv_lens", _vp),
                ("cu_new", _vp), ("scale", _f), ("dtype", _i), ("n_seqs", _i), ("table_width", _i),
                ("n_q_heads", _i), ("total_new", _i), ("max_new", _i), ("max_kv", _i), ("causal", _i),
                ("window", _i)]


class RtVerifyDraft(ctypes.Structure):
    _fields_ = [("target", _vp), ("draft", _vp), ("target_stride", _I64x2), ("draft_stride", _I64x2),
                ("draft_tokens", _vp), ("draft_lens", _vp), ("accept_u", _vp), ("sample_u", _vp), ("tokens", _vp),
                ("accepted", _vp), ("dtype", _i), ("n_seqs", _i), ("n_drafts", _i), ("vocab", _i), ("flags", _i)]


_dtypes = {torch.float32: 0, torch.bfloat16: 1}
_module = None


def _calls():
    """b200paged, the native side of these calls (raises if it has not been built: no fallback)."""
    global _module
    if _module is None:
        load_library()      # the module links to it
        paths = list(LIB_PATH.parent.glob("b200paged*.so"))
        if not paths:
            raise RuntimeError(f"b200paged not found in {LIB_PATH.parent} -- run build() first")
        spec = importlib.util.spec_from_file_location("b200paged", paths[0])
        m = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(m)
        m.set_status_error(CudaRuntimeError)
        _module = m
    return _module


def kv_write(k, v, k_pages, v_pages, slots, *, k_scale=None, v_scale=None) -> None:
    """Store the keys and values ``[tokens, heads, head_dim]`` of new tokens in a cache.

    ``k_pages`` / ``v_pages``: ``[pages, page_size, heads, head_dim]`` (any strides, the same for both,
    with contiguous features on 16-byte boundaries); ``slots``: int64 ``[tokens]``, ``page * page_size + position in
    the page``, negative to skip a token.  int8 and float8_e4m3fn caches take ``k_scale`` /
    ``v_scale``, float32 ``[pages, page_size, heads]``, and are written with one scale per token and
    head: ``scale = max|x| * (1/M)``, ``code = round(x * ((1/max|x|) * M))``, M = 127 or 448.
    """
    (_module or _calls()).kv_write(k, v, k_pages, v_pages, slots, k_scale, v_scale)


def kv_read(k_pages, v_pages, page_table, start, cu, total, *, k_scale=None, v_scale=None, dtype=torch.float32,
            out=None):
    """Read cached positions back as dense ``(k, v)``, each ``[total, heads, head_dim]``.

    Row ``cu[b] + i`` is position ``start[b] + i`` of sequence b (``start`` None: from 0); ``cu``:
    int32 ``[sequences + 1]``, ``total`` = its last value as the host knows it.  ``out``: a pair of
    tensors to write instead of new ones of ``dtype`` (float32 / bfloat16).  Rows past the last sequence's are zeros.
    """
    if dtype not in _dtypes:
        raise TypeError(f"dtype must be float32 or bfloat16, got {dtype}")
    ko, vo = (None, None) if out is None else out
    return (_module or _calls()).kv_read(k_pages, v_pages, page_table, start, cu, total, k_scale, v_scale,
                                         _dtypes[dtype], ko, vo)


def paged_attention(q, k_pages, v_pages, page_table, kv_lens, cu_new, *, k_scale=None, v_scale=None, scale=None,
                    causal=True, window=0, max_new=None, max_kv=None, out=None, lse=None):
    """Attention of new tokens ``q [tokens, query heads, head_dim]`` over their sequences' cached positions.

    Sequence b brings tokens ``cu_new[b] .. cu_new[b+1]-1`` of ``q`` and has ``kv_lens[b]`` cached
    positions, its new tokens' own included (write them first); ``page_table``: int32 ``[sequences,
    pages]``.  New token i of n stands at ``kv_lens[b] - n + i`` and sees what is at or before it
    (``causal``) and less than ``window`` positions back (0: no window).  Query head h reads cache head
    ``h // (query heads / cache heads)``.  A token that sees nothing gives zeros, and so does a row of ``q``
    that no sequence owns (before ``cu_new[0]``, from ``cu_new[-1]`` on).

    ``scale``: default 1/sqrt(head_dim).  ``max_new`` / ``max_kv``: the host's bounds on new and cached
    tokens of a sequence (default: the tokens of q, the width of the table); they only choose how the
    work is split.  ``lse``: float32 ``[tokens, query heads]`` to receive log-sum-exp.  Returns ``out``.
    """
    return (_module or _calls()).paged_attention(q, k_pages, v_pages, page_table, kv_lens, cu_new, k_scale, v_scale,
                                                 scale, causal, window, max_new, max_kv, out, lse)


def verify_draft(target, draft, draft_tokens, accept_u, sample_u, *, draft_lens=None):
    """Accept drafted tokens against the target's probabilities and sample the token that follows.

    ``target [sequences, drafts + 1, vocab]`` and ``draft [sequences, drafts, vocab]`` are probabilities
    (float32 or bfloat16; ``draft`` None: the drafts were certain, as from a lookup), ``draft_tokens``
    int32 ``[sequences, drafts]``, ``accept_u`` / ``sample_u`` uniform numbers in [0, 1), float32
    ``[sequences, drafts]`` / ``[sequences]``; ``draft_lens`` int32 where sequences have fewer drafts.
    Draft i stands while ``accept_u * draft(x) < target(x)``; the token after the last one that stands is
    sampled from ``max(target - draft, 0)``, or from the target after all of them.

    Returns ``(tokens, accepted)``: int32 ``[sequences, drafts + 1]`` with the accepted drafts, the sampled
    token and -1 from there on, and int32 ``[sequences]``.
    """
    return (_module or _calls()).verify_draft(target, draft, draft_tokens, accept_u, sample_u, draft_lens)


def check_stream(device=0) -> None:
    """Wait for torch's current stream on `device` and raise for what serving calls reported (of all streams)."""
    (_module or _calls()).check_stream(device if isinstance(device, int) else device.index)
