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

import torch

from .executor import CudaRuntimeError, check, load_library

_I64x2, _I64x3 = ctypes.c_int64 * 2, ctypes.c_int64 * 3
_vp, _i, _f, _l = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_int64


class RtKvCache(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("stride", _I64x3),
                ("scale_stride", _I64x3), ("dtype", _i), ("n_pages", _i), ("page_size", _i), ("n_heads", _i),
                ("head_dim", _i)]


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
                ("accepted", _vp), ("dtype", _i), ("n_seqs", _i), ("n_drafts", _i), ("vocab", _i)]


ACT_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
CACHE_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float8_e4m3fn: 2, torch.int8: 3}

_lib = None
_device = -1


def _library(device: torch.device):
    """The library, initialised on `device` (the first CUDA tensor's, once per process)."""
    global _lib, _device
    if _lib is None or _device != device.index:
        lib = load_library()
        for name, struct in (("rt_kv_write", RtKvWrite), ("rt_kv_read", RtKvRead),
                             ("rt_verify_draft", RtVerifyDraft)):
            fn = getattr(lib, name)
            fn.argtypes, fn.restype = [ctypes.POINTER(struct), _vp], _i
        lib.rt_paged_attention_workspace.argtypes = [ctypes.POINTER(RtPagedAttention)]
        lib.rt_paged_attention_workspace.restype = ctypes.c_size_t
        lib.rt_paged_attention.argtypes = [ctypes.POINTER(RtPagedAttention), _vp, ctypes.c_size_t, _vp]
        lib.rt_paged_attention.restype = _i
        lib.rt_check_stream.argtypes, lib.rt_check_stream.restype = [_vp], _i
        check(lib, lib.rt_init(device.index), "rt_init")
        _lib, _device = lib, device.index
    return _lib


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _index(t, name: str, n: int, dtype, device) -> int:
    """Address of a contiguous index / number vector of `n` elements."""
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    _need(t.device == device, f"{name} is on {t.device}, expected {device}")
    _need(t.numel() == n and t.is_contiguous(), f"{name} must be contiguous with {n} elements, got {tuple(t.shape)}")
    return t.data_ptr()


def _cache(c: RtKvCache, k_pages, v_pages, k_scale, v_scale) -> None:
    code = CACHE_DTYPES.get(k_pages.dtype)
    if code is None or v_pages.dtype is not k_pages.dtype:
        raise TypeError(f"a cache holds float32, bfloat16, float8_e4m3fn or int8, got {k_pages.dtype} / {v_pages.dtype}")
    _need(k_pages.is_cuda and k_pages.device == v_pages.device, "cache pages must be CUDA tensors of one device")
    _need(k_pages.dim() == 4 and k_pages.shape == v_pages.shape,
          f"cache pages must be [pages, page_size, heads, head_dim], got {tuple(k_pages.shape)} / {tuple(v_pages.shape)}")
    st = k_pages.stride()
    _need(st[3] == 1 and v_pages.stride() == st, "k_pages and v_pages need the same strides and contiguous features")
    c.k, c.v, c.dtype = k_pages.data_ptr(), v_pages.data_ptr(), code
    c.n_pages, c.page_size, c.n_heads, c.head_dim = k_pages.shape
    c.stride[0], c.stride[1], c.stride[2] = st[0], st[1], st[2]
    if code >= 2:
        _need(k_scale is not None and v_scale is not None, "an 8-bit cache needs k_scale and v_scale")
        if k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32:
            raise TypeError("scales must be float32")
        _need(k_scale.shape == k_pages.shape[:3] and v_scale.shape == k_pages.shape[:3]
              and k_scale.stride() == v_scale.stride() and k_scale.device == v_scale.device == k_pages.device,
              "scales must be [pages, page_size, heads] beside their pages, with the same strides")
        c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        st = k_scale.stride()
        c.scale_stride[0], c.scale_stride[1], c.scale_stride[2] = st
    else:
        _need(k_scale is None and v_scale is None, "only an 8-bit cache has scales")


def _rows(t, name: str, shape: tuple, device, dtype=None) -> int:
    """dtype code of a dense [rows, heads, features] operand with contiguous features."""
    code = ACT_DTYPES.get(t.dtype)
    if code is None or (dtype is not None and t.dtype is not dtype):
        raise TypeError(f"{name} must be {dtype or 'float32 or bfloat16'}, got {t.dtype}")
    _need(t.device == device, f"{name} is on {t.device}, expected {device}")
    _need(t.shape == shape, f"{name} must be {shape}, got {tuple(t.shape)}")
    _need(t.stride(-1) == 1 or shape[-1] == 1, f"{name} needs contiguous features")
    return code


def _table(x, page_table, n: int, device) -> None:
    if page_table.dtype is not torch.int32:
        raise TypeError(f"page_table must be int32, got {page_table.dtype}")
    _need(page_table.device == device and page_table.dim() == 2 and page_table.shape[0] == n,
          f"page_table must be [{n}, pages] on {device}, got {tuple(page_table.shape)} on {page_table.device}")
    _need(page_table.shape[1] <= 1 or page_table.stride(1) == 1, "page_table needs contiguous rows")
    x.page_table, x.table_stride, x.table_width = page_table.data_ptr(), page_table.stride(0), page_table.shape[1]


def kv_write(k, v, k_pages, v_pages, slots, *, k_scale=None, v_scale=None) -> None:
    """Store the keys and values ``[tokens, heads, head_dim]`` of new tokens in a cache.

    ``k_pages`` / ``v_pages``: ``[pages, page_size, heads, head_dim]`` (any strides with contiguous
    features on 16-byte boundaries); ``slots``: int64 ``[tokens]``, ``page * page_size + position in
    the page``, negative to skip a token.  int8 and float8_e4m3fn caches take ``k_scale`` /
    ``v_scale``, float32 ``[pages, page_size, heads]``, and are written with one scale per token and
    head: ``scale = max|x| * (1/M)``, ``code = round(x * ((1/max|x|) * M))``, M = 127 or 448.
    """
    lib = _library(k_pages.device)
    w = RtKvWrite()
    _cache(w.cache, k_pages, v_pages, k_scale, v_scale)
    dev = k_pages.device
    shape = (k.shape[0], w.cache.n_heads, w.cache.head_dim)
    w.dtype = _rows(k, "k", shape, dev)
    _rows(v, "v", shape, dev, k.dtype)
    w.k, w.v, w.n_tokens = k.data_ptr(), v.data_ptr(), shape[0]
    w.k_stride[0], w.k_stride[1] = k.stride(0), k.stride(1)
    w.v_stride[0], w.v_stride[1] = v.stride(0), v.stride(1)
    w.slots = _index(slots, "slots", shape[0], torch.int64, dev)
    check(lib, lib.rt_kv_write(w, _stream(dev)), "kv_write")


def kv_read(k_pages, v_pages, page_table, start, cu, total, *, k_scale=None, v_scale=None, dtype=torch.float32,
            out=None):
    """Read cached positions back as dense ``(k, v)``, each ``[total, heads, head_dim]``.

    Row ``cu[b] + i`` is position ``start[b] + i`` of sequence b (``start`` None: from 0); ``cu``:
    int32 ``[sequences + 1]``, ``total`` = its last value as the host knows it.  ``out``: a pair of
    tensors to write instead of new ones of ``dtype`` (float32 / bfloat16).
    """
    lib = _library(k_pages.device)
    r = RtKvRead()
    _cache(r.cache, k_pages, v_pages, k_scale, v_scale)
    dev = k_pages.device
    shape = (total, r.cache.n_heads, r.cache.head_dim)
    if out is None:
        if dtype not in ACT_DTYPES:
            raise TypeError(f"dtype must be float32 or bfloat16, got {dtype}")
        k, v = torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev)
    else:
        k, v = out
    r.dtype = _rows(k, "k out", shape, dev)
    _rows(v, "v out", shape, dev, k.dtype)
    r.k_out, r.v_out, r.n_rows, r.n_seqs = k.data_ptr(), v.data_ptr(), total, cu.numel() - 1
    r.k_stride[0], r.k_stride[1] = k.stride(0), k.stride(1)
    r.v_stride[0], r.v_stride[1] = v.stride(0), v.stride(1)
    _table(r, page_table, r.n_seqs, dev)
    r.start = None if start is None else _index(start, "start", r.n_seqs, torch.int32, dev)
    r.cu = _index(cu, "cu", r.n_seqs + 1, torch.int32, dev)
    check(lib, lib.rt_kv_read(r, _stream(dev)), "kv_read")
    return k, v


def paged_attention(q, k_pages, v_pages, page_table, kv_lens, cu_new, *, k_scale=None, v_scale=None, scale=None,
                    causal=True, window=0, max_new=None, max_kv=None, out=None, lse=None):
    """Attention of new tokens ``q [tokens, query heads, head_dim]`` over their sequences' cached positions.

    Sequence b brings tokens ``cu_new[b] .. cu_new[b+1]-1`` of ``q`` and has ``kv_lens[b]`` cached
    positions, its new tokens' own included (write them first); ``page_table``: int32 ``[sequences,
    pages]``.  New token i of n stands at ``kv_lens[b] - n + i`` and sees what is at or before it
    (``causal``) and less than ``window`` positions back (0: no window).  Query head h reads cache head
    ``h // (query heads / cache heads)``.  A token that sees nothing gives zeros.

    ``scale``: default 1/sqrt(head_dim).  ``max_new`` / ``max_kv``: the host's bounds on new and cached
    tokens of a sequence (default: the tokens of q, the width of the table); they only choose how the
    work is split.  ``lse``: float32 ``[tokens, query heads]`` to receive log-sum-exp.  Returns ``out``.
    """
    lib = _library(k_pages.device)
    p = RtPagedAttention()
    _cache(p.cache, k_pages, v_pages, k_scale, v_scale)
    dev = k_pages.device
    _need(q.dim() == 3, f"q must be [tokens, heads, head_dim], got {tuple(q.shape)}")
    shape = (q.shape[0], q.shape[1], p.cache.head_dim)
    p.dtype = _rows(q, "q", shape, dev)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=dev)
    else:
        _rows(out, "out", shape, dev, q.dtype)
    p.q, p.out, p.total_new, p.n_q_heads = q.data_ptr(), out.data_ptr(), shape[0], shape[1]
    p.q_stride[0], p.q_stride[1] = q.stride(0), q.stride(1)
    p.out_stride[0], p.out_stride[1] = out.stride(0), out.stride(1)
    p.lse = None if lse is None else _index(lse, "lse", shape[0] * shape[1], torch.float32, dev)
    p.n_seqs = kv_lens.numel()
    _table(p, page_table, p.n_seqs, dev)
    p.kv_lens = _index(kv_lens, "kv_lens", p.n_seqs, torch.int32, dev)
    p.cu_new = _index(cu_new, "cu_new", p.n_seqs + 1, torch.int32, dev)
    p.scale = p.cache.head_dim ** -0.5 if scale is None else scale
    p.causal, p.window = int(causal), window
    p.max_new = shape[0] if max_new is None else max_new
    p.max_kv = p.table_width * p.cache.page_size if max_kv is None else max_kv
    n = lib.rt_paged_attention_workspace(p)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    check(lib, lib.rt_paged_attention(p, ws.data_ptr() if n else None, n, _stream(dev)), "paged_attention")
    return out


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
    lib = _library(target.device)
    v, dev = RtVerifyDraft(), target.device
    _need(target.is_cuda and target.dim() == 3 and target.shape[1] >= 1,
          f"target must be a CUDA tensor [sequences, drafts + 1, vocab], got {tuple(target.shape)}")
    B, n, V = target.shape
    n -= 1
    v.dtype = _rows(target, "target", (B, n + 1, V), dev)
    v.target, v.n_seqs, v.n_drafts, v.vocab = target.data_ptr(), B, n, V
    v.target_stride[0], v.target_stride[1] = target.stride(0), target.stride(1)
    if draft is not None:
        _rows(draft, "draft", (B, n, V), dev, target.dtype)
        v.draft = draft.data_ptr()
        v.draft_stride[0], v.draft_stride[1] = draft.stride(0), draft.stride(1)
    v.draft_tokens = _index(draft_tokens, "draft_tokens", B * n, torch.int32, dev)
    v.accept_u = _index(accept_u, "accept_u", B * n, torch.float32, dev)
    v.sample_u = _index(sample_u, "sample_u", B, torch.float32, dev)
    v.draft_lens = None if draft_lens is None else _index(draft_lens, "draft_lens", B, torch.int32, dev)
    tokens = torch.empty((B, n + 1), dtype=torch.int32, device=dev)
    accepted = torch.empty(B, dtype=torch.int32, device=dev)
    v.tokens, v.accepted = tokens.data_ptr(), accepted.data_ptr()
    check(lib, lib.rt_verify_draft(v, _stream(dev)), "verify_draft")
    return tokens, accepted


def check_stream(device=0) -> None:
    """Wait for torch's current stream on `device` and raise for what its kernels reported."""
    dev = torch.device("cuda", device) if isinstance(device, int) else device
    lib = _library(dev)
    check(lib, lib.rt_check_stream(_stream(dev)), "check_stream")
