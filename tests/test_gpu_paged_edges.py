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


# ------------------------------------------------------------------ value rows of zeros
@pytest.mark.parametrize("cache,act", CACHES)
@pytest.mark.parametrize("dim,lens,new", [(64, [200, 90], [200, 60]), (128, [700], [100]), (64, [300], [1]), (64, [700] * 4, [100] * 4)])
def test_value_rows_of_zeros(paged, cache, act, dim, lens, new):
    """The first token's values or the first 300, scattered ones, and all of one head."""
    hkv = 2 if len(lens) < 4 else 16                    # (several tiles in a row in a block)
    s = Setup(cache, act, 2 * hkv, hkv, dim, 16, lens, new, seed=20)
    for b, n in enumerate(lens):
        for pos in [*range(1 if b % 2 == 0 else min(300, n)), *range(5, n, 7)]:
            s.pages["v"][place(s, b, pos)] = 0
            if s.scale["v"] is not None:
                s.scale["v"][place(s, b, pos)] = 0      # as kv_write stores a row of zeros
    for b, n in enumerate(lens):
        for pos in range(n):
            pg, off = place(s, b, pos)
            s.pages["v"][pg, off, 1] = 0
            if s.scale["v"] is not None:
                s.scale["v"][pg, off, 1] = 0
    lse = torch.empty(s.q.shape[:2], device="cuda")
    out = s.attend(paged, lse=lse)
    compare(s, out, act)
    assert bool((out[:, 2:4] == 0).all())               # query heads of the head without values
    _, want = s.expected()
    assert float((lse.double() - want).abs().max()) < (1e-4 if act == "f32" else 2e-2)


# ------------------------------------------------------------------ NaN scores
@pytest.mark.parametrize("cache,act", CACHES)
@pytest.mark.parametrize("lens,new,bounds", [
    ([33], [1], {}),                                    # one block, a warp has the newest position to itself
    ([33], [1], {"max_kv": 33, "max_new": 1}),
    ([5000], [1], {"max_new": 1}),                      # cut over many blocks
    ([400] * 70, [1] * 70, {"max_new": 1, "max_kv": 600}),   # a warp has a head to itself
    ([2000, 300], [5, 60], {"max_new": 60}),            # tiles
])
def test_nan_queries_and_keys_give_nan(paged, cache, act, lens, new, bounds):
    """softmax of a NaN score is NaN, and so is its log-sum-exp, however the work is split."""
    def run(change):
        s = Setup(cache, act, 4, 2, 64, 16, lens, new, seed=21)
        ref, want = s.expected()
        hit = change(s)                                 # [rows, query heads] that must be NaN
        lse = torch.empty(s.q.shape[:2], device="cuda")
        out = s.attend(paged, lse=lse, **bounds)
        assert bool(out[hit].isnan().all()) and bool(lse[hit].isnan().all())
        assert bool(out[~hit].isfinite().all()) and bool(lse[~hit].isfinite().all())
        assert float((out.double() - ref)[~hit].abs().max()) <= tolerance(s, act)

    def query(s):
        hit = torch.zeros(s.q.shape[:2], dtype=torch.bool, device="cuda")
        hit[::3, 1] = hit[0, 2] = True
        s.q[hit] = math.nan
        return hit

    def newest_key(s):                                  # of cache head 1: query heads 2 and 3
        for b, n in enumerate(s.lens):
            pg, off = place(s, b, n - 1)
            if s.scale["k"] is None:
                s.pages["k"][pg, off, 1] = math.nan
            else:
                s.scale["k"][pg, off, 1] = math.nan
        hit = torch.zeros(s.q.shape[:2], dtype=torch.bool, device="cuda")
        for r, (b, pos) in enumerate(owners(s)):
            hit[r, 2:] = pos == s.lens[b] - 1
        return hit
    run(query)
    run(newest_key)


# ------------------------------------------------------------------ values that are not finite
@pytest.mark.parametrize("cache,act", [("f32", "f32"), ("bf16", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("dim,new,window,back", [(d, n, w, b) for d, n, w in [(64, 300, 0), (128, 300, 0), (64, 300, 100), (128, 300, 100),
                                                                              (64, 6, 0), (64, 6, 4)]
                                                 for b in (1, 5, 40, 120, 239, 255, 299) if b <= n])
def test_only_rows_that_see_a_value_get_it(paged, cache, act, dim, new, window, back):
    """An infinite value `back` positions from the end: rows that see it are not finite, the rest are as without it."""
    s = Setup(cache, act, 4, 2, dim, 16, [500], [new], seed=22)
    ref, _ = s.expected(window=window)
    pos = 500 - back
    pg, off = place(s, 0, pos)
    s.pages["v"][pg, off, 0, 3] = math.inf
    out = s.attend(paged, window=window)
    at = torch.arange(500 - new, 500, device="cuda")
    hit = torch.zeros(s.q.shape[:2], dtype=torch.bool, device="cuda")
    hit[:, :2] = ((at >= pos) & (at < pos + window if window else at >= 0))[:, None]
    assert bool((~out.isfinite()).any(-1).eq(hit).all())
    assert float((out.double() - ref)[~hit].abs().max()) <= tolerance(Setup(cache, act, 4, 2, dim, 16, [500], [new], seed=22), act)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("new,lens", [(6, 230), (6, 3000), (70, 230), (300, 500)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_codes_that_are_nan(paged, act, new, lens, which):
    """Codes 0x7f / 0xff of an e4m3 cache at positions that only later rows see."""
    s = Setup("f8", act, 4, 2, 64, 16, [lens], [new], seed=23)
    ref, _ = s.expected()
    pos = lens - 4
    pg, off = place(s, 0, pos)
    s.pages[which].view(torch.uint8)[pg, off, 0, 3] = 0x7f
    s.pages[which].view(torch.uint8)[pg, off, 0, 60] = 0xff
    out = s.attend(paged)
    at = torch.arange(lens - new, lens, device="cuda")
    hit = torch.zeros(s.q.shape[:2], dtype=torch.bool, device="cuda")
    hit[:, :2] = (at >= pos)[:, None]
    assert bool((~out.isfinite()).any(-1).eq(hit).all())
    assert float((out.double() - ref)[~hit].abs().max()) <= tolerance(Setup("f8", act, 4, 2, 64, 16, [lens], [new], seed=23), act)


# ------------------------------------------------------------------ scores far below zero
@pytest.mark.parametrize("cache,act", CACHES)
@pytest.mark.parametrize("dim", [64, 128])
def test_low_scores_under_a_window(paged, cache, act, dim):
    """All scores near -150, rows of a tile that see nothing of its first keys.

    A score is off by 2^-19 of |q||k| scale (bf16 activations: 2^-10, a q of one fp16 part), which
    changes weights by as much and an output by at most twice that of the largest value.  There are
    enough heads and sequences for several tiles in a row in a block."""
    s = Setup(cache, act, 16, 16, dim, 16, [700, 300, 650, 512], [300] * 4, seed=24)
    a = math.sqrt(150 / math.sqrt(dim))
    s.q.copy_((a + 0.1 * s.q.float()).to(s.q.dtype))
    k = -a + 0.1 * torch.randn(s.pages["k"].shape, generator=gen(25), device="cuda")
    if s.scale["k"] is not None:
        m = 448.0 if cache == "f8" else 127.0
        s.scale["k"] = k.abs().amax(-1) / m
        k = k / s.scale["k"][..., None]
        k = k.round() if cache == "i8" else k
    s.pages["k"] = k.to(CACHE[cache])
    vmax = float(values(s.pages["v"], s.scale["v"]).nan_to_num(0, 0, 0).abs().max())
    tol = 2 * 165 * 2.0 ** -19 * vmax if act == "f32" else (2 * 165 * 2.0 ** -10 + 2.0 ** -7) * vmax
    for window in (200, 100):
        out = s.attend(paged, window=window)
        ref, _ = s.expected(window=window)
        assert bool(out.isfinite().all())
        assert float((out.double() - ref).abs().max()) <= tol


# ------------------------------------------------------------------ rows and sequences nobody owns
@pytest.mark.parametrize("cache,act", [("f32", "f32"), ("bf16", "bf16"), ("i8", "f32")])
@pytest.mark.parametrize("seqs,new", [(3, 1), (40, 1), (3, 50), (40, 20)])
def test_rows_without_a_sequence_are_zero(paged, cache, act, seqs, new):
    """Padding before the first and after the last sequence's tokens."""
    lens = [50 + 3 * i for i in range(seqs)]
    s = Setup(cache, act, 4, 2, 64, 16, lens, [new] * seqs, seed=26)
    ref, _ = s.expected()
    n = len(s.q)
    q = torch.randn(n + 12, 4, 64, device="cuda").to(ACT[act])
    q[5:5 + n] = s.q
    out = torch.full_like(q, 7.0)
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    paged.paged_attention(q, s.pages["k"], s.pages["v"], s.table, s.lens_t, s.cu + 5, **s.kw(), out=out, lse=lse)
    paged.check_stream()
    assert float((out[5:5 + n].double() - ref).abs().max()) <= tolerance(s, act)
    pad = torch.ones(n + 12, dtype=torch.bool, device="cuda")
    pad[5:5 + n] = False
    assert bool((out[pad] == 0).all()) and bool((lse[pad] == -math.inf).all())
    assert bool(lse[~pad].isfinite().all())


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("seqs", [3, 40])
def test_rows_of_a_refused_sequence_are_zero(paged, new, seqs):
    """Offsets past the end of q: the sequence is left out and reported, its rows are zeros."""
    from lbr_b200.executor import CudaRuntimeError
    s = Setup("f32", "f32", 4, 2, 64, 16, [60] * seqs, [new] * seqs, seed=27)
    ref, _ = s.expected()
    cu = s.cu.clone()
    cu[-1] += 100
    out = torch.full_like(s.q, 7.0)
    lse = torch.full(s.q.shape[:2], 7.0, device="cuda")
    paged.check_stream()
    paged.paged_attention(s.q, s.pages["k"], s.pages["v"], s.table, s.lens_t, cu, out=out, lse=lse)
    with pytest.raises(CudaRuntimeError, match="out of range"):
        paged.check_stream()
    assert bool((out[-new:] == 0).all()) and bool((lse[-new:] == -math.inf).all())
    assert float((out[:-new].double() - ref[:-new]).abs().max()) <= tolerance(s, "f32")


def test_attention_without_sequences(paged):
    pages = torch.randn(3, 16, 2, 64, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    table, cu = torch.zeros(0, 4, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    for n in (1, 9, 100):
        out, lse = torch.full((n, 4, 64), 7.0, device="cuda"), torch.full((n, 4), 7.0, device="cuda")
        paged.paged_attention(torch.randn(n, 4, 64, device="cuda"), pages, pages, table, none, cu, out=out, lse=lse)
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    paged.check_stream()


def test_read_without_sequences(paged):
    pages = torch.randn(3, 16, 2, 64, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    table, cu = torch.zeros(0, 4, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    for start in (None, none):
        k, v = torch.full((9, 2, 64), 7.0, device="cuda"), torch.full((9, 2, 64), 7.0, device="cuda")
        paged.kv_read(pages, pages, table, start, cu, 9, out=(k, v))
        assert bool((k == 0).all()) and bool((v == 0).all())
    paged.check_stream()


# ------------------------------------------------------------------ windows as large as integers go
@pytest.mark.parametrize("new", [7, 60])
@pytest.mark.parametrize("causal", [True, False])
def test_largest_window(paged, new, causal):
    """More new tokens than positions, so that some stand before the first: a window that hides nothing."""
    s = Setup("f32", "f32", 4, 2, 64, 16, [3, 40], [new, new], seed=28)
    compare(s, s.attend(paged, window=2 ** 31 - 1, causal=causal), "f32", causal=causal)


# ------------------------------------------------------------------ drafted tokens
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("V", [9, 1000, 40000])
def test_certain_draft_that_takes_all_the_mass(paged, act, V):
    """A refused certain draft on a row whose only mass is its token: sampled from the target's row."""
    target = torch.zeros(3, 3, V, device="cuda")
    x = torch.tensor([[0, 1], [V - 1, 2], [V // 2, 3]], dtype=torch.int32, device="cuda")
    for b in range(3):
        target[b, 0, int(x[b, 0])] = 0.5
        target[b, 1] = 1.0 / V
    target = target.to(ACT[act])
    au, su = torch.full((3, 2), 0.9, device="cuda"), torch.tensor([0.0, 0.5, 0.999], device="cuda")
    got, acc = paged.verify_draft(target, None, x, au, su)
    want, wacc = settle(target.float().cpu().numpy(), None, x.cpu().numpy(), au.cpu().numpy(), su.cpu().numpy())
    np.testing.assert_array_equal(acc.cpu().numpy(), wacc)
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    assert got[:, 0].tolist() == x[:, 0].tolist()
    paged.check_stream()


@pytest.mark.parametrize("B", [1, 2, 19, 37, 74])
def test_verify_while_other_work_holds_the_gpu(paged, B):
    """A sequence's blocks exchange their sums wherever and whenever they get to run: the same answer next to
    products on another stream that take SMs at other times."""
    V = 20011
    target = torch.softmax(2 * torch.randn(B, 3, V, generator=gen(33), device="cuda"), -1)
    draft = torch.softmax(2 * torch.randn(B, 2, V, generator=gen(34), device="cuda"), -1)
    x = torch.randint(0, V, (B, 2), generator=gen(35), device="cuda").to(torch.int32)
    au, su = torch.rand(B, 2, generator=gen(36), device="cuda"), torch.rand(B, generator=gen(37), device="cuda")
    want, wacc = settle(*(t.cpu().numpy() for t in (target, draft, x, au, su)))
    side, a = torch.cuda.Stream(), torch.randn(1000, 1000, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    results = []
    for _ in range(20):
        with torch.cuda.stream(side):
            a = torch.tanh(a @ a)
        results.append(paged.verify_draft(target, draft, x, au, su))
    torch.cuda.current_stream().wait_stream(side)
    paged.check_stream()
    for got, acc in results:
        np.testing.assert_array_equal(acc.cpu().numpy(), wacc)
        np.testing.assert_array_equal(got.cpu().numpy(), want)


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


# ------------------------------------------------------------------ what one caller's mistake does to others
def test_a_bad_slot_does_not_fail_planned_work(paged):
    from lbr_b200.copnode import COpNode
    from lbr_b200.executor import CudaRuntimeError, load_library
    lib = load_library()
    x = torch.zeros(1, 4, 64, device="cuda")
    pages = torch.zeros(2, 16, 4, 64, device="cuda")
    paged.kv_write(x, x, pages, pages.clone(), torch.zeros(1, dtype=torch.int64, device="cuda"))
    paged.check_stream()
    paged.kv_write(x, x, pages, pages.clone(), torch.tensor([10 ** 6], device="cuda"))
    torch.cuda.synchronize()
    arr = (COpNode * 1)()                               # one GELU of 256 elements
    arr[0].op, arr[0].n_inputs, arr[0].n_dims, arr[0].elem_size = 104, 1, 1, 4
    arr[0].inputs[0], arr[0].output = lib.rt_alloc(1024), lib.rt_alloc(1024)
    arr[0].out_shape[0] = 256
    assert lib.rt_execute(arr, 1, 0) == 0
    assert lib.rt_synchronize() == 0
    with pytest.raises(CudaRuntimeError, match="slot"):
        paged.check_stream()
    paged.check_stream()


# ------------------------------------------------------------------ shapes
def test_refusals_by_shape(paged):
    """Operands of the right number of elements in another order or shape."""
    s = Setup("f32", "f32", 4, 2, 64, 16, [40, 50], [3, 3], seed=30)
    kp, vp, q = s.pages["k"], s.pages["v"], s.q

    def attend(**kw):
        a = {"kv_lens": s.lens_t, "cu_new": s.cu, **kw}
        return paged.paged_attention(q, kp, vp, s.table, a.pop("kv_lens"), a.pop("cu_new"), **a)
    attend()
    with pytest.raises(ValueError, match="lse"):
        attend(lse=torch.empty(4, 6, device="cuda"))
    with pytest.raises(ValueError, match="lse"):
        attend(lse=torch.empty(24, device="cuda"))
    with pytest.raises(ValueError, match="kv_lens"):
        attend(kv_lens=s.lens_t[:, None])
    with pytest.raises(ValueError, match="cu_new"):
        attend(cu_new=s.cu[None])
    i32 = {"dtype": torch.int32, "device": "cuda"}
    with pytest.raises(ValueError, match="slots"):
        paged.kv_write(s.k, s.v, kp, vp, torch.zeros(2, 3, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="start"):
        paged.kv_read(kp, vp, s.table, torch.zeros(2, 1, **i32), s.cu, 6)
    with pytest.raises(ValueError, match="cu"):
        paged.kv_read(kp, vp, s.table, None, s.cu[:, None], 6)
    p, x, u = torch.rand(2, 4, 50, device="cuda"), torch.zeros(2, 3, **i32), torch.rand(2, 3, device="cuda")
    paged.verify_draft(p, p[:, :3], x, u, u[:, 0].contiguous())
    with pytest.raises(ValueError, match="draft_tokens"):
        paged.verify_draft(p, p[:, :3], x.view(3, 2), u, u[:, 0].contiguous())
    with pytest.raises(ValueError, match="accept_u"):
        paged.verify_draft(p, p[:, :3], x, u.view(3, 2), u[:, 0].contiguous())
    with pytest.raises(ValueError, match="sample_u"):
        paged.verify_draft(p, p[:, :3], x, u, u[:, :1].contiguous())
    with pytest.raises(ValueError, match="draft_lens"):
        paged.verify_draft(p, p[:, :3], x, u, u[:, 0].contiguous(), draft_lens=torch.zeros(2, 1, **i32))
    paged.check_stream()


def test_read_refuses_rows_that_overlap(paged):
    from lbr_b200.executor import CudaRuntimeError
    s = Setup("f32", "f32", 2, 2, 64, 16, [40], [3], seed=31)
    one = torch.zeros(1, 2, 64, device="cuda")
    with pytest.raises(CudaRuntimeError, match="overlap"):
        paged.kv_read(s.pages["k"], s.pages["v"], s.table, None, s.cu, 3, out=(one.expand(3, 2, 64), one.expand(3, 2, 64)))
    heads = torch.zeros(3, 1, 64, device="cuda")
    with pytest.raises(CudaRuntimeError, match="overlap"):
        paged.kv_read(s.pages["k"], s.pages["v"], s.table, None, s.cu, 3, out=(torch.zeros(3, 2, 64, device="cuda"), heads.expand(3, 2, 64)))


def test_causal_must_have_a_truth_value(paged):
    s = Setup("f32", "f32", 2, 2, 64, 16, [40], [3], seed=32)
    with pytest.raises(TypeError, match="causal"):
        s.attend(paged, causal=np.ones(2))


# ------------------------------------------------------------------ the library's life
def in_a_process(code):
    import pathlib
    import subprocess
    import sys
    root = pathlib.Path(__file__).resolve().parents[1]
    head = ("import torch, sys\n"
            f"sys.path.insert(0, {str(root)!r})\n"
            "import __graft_entry__\n"
            "__graft_entry__.load_package()\n"
            "from lbr_b200 import paged\n"
            "from lbr_b200.executor import CudaRuntimeError, load_library\n"
            "lib = load_library()\n"
            "x, p = torch.ones(2, 4, 64, device='cuda'), torch.zeros(3, 16, 4, 64, device='cuda')\n"
            "write = lambda *at: paged.kv_write(x, x, p, p.clone(), torch.tensor(at, device='cuda'))\n")
    r = subprocess.run([sys.executable, "-c", head + code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_destroy_waits_for_serving_calls(paged):
    """Calls still under way on the caller's stream, with something to report, when the library ends."""
    in_a_process("write(1, 2)\n"
                 "a = torch.randn(4000, 4000, device='cuda')\n"
                 "side = torch.cuda.Stream()\n"
                 "torch.cuda.synchronize()\n"
                 "with torch.cuda.stream(side):\n"
                 "    at = torch.tensor([10 ** 6, 10 ** 7], device='cuda')\n"
                 "    for _ in range(20): a = torch.tanh(a @ a)\n"
                 "    paged.kv_write(x, x, p, p, at)\n"
                 "assert lib.rt_destroy() == 0\n"
                 "assert side.query()\n"
                 "assert lib.rt_init(0) == 0\n"
                 "torch.cuda.synchronize()\n")


def test_calls_after_destroy_start_the_library_again(paged):
    in_a_process("write(1, 2)\n"
                 "paged.check_stream()\n"
                 "assert lib.rt_destroy() == 0\n"
                 "write(3, 4)\n"
                 "paged.check_stream()\n"
                 "write(3, 10 ** 6)\n"
                 "try:\n"
                 "    paged.check_stream()\n"
                 "except CudaRuntimeError as e:\n"
                 "    assert 'slot' in str(e)\n"
                 "else:\n"
                 "    raise SystemExit('nothing reported')\n")


# ------------------------------------------------------------------ how good bf16 outputs are
@pytest.mark.parametrize("cache", ["f32", "bf16", "i8", "f8"])
@pytest.mark.parametrize("hq,hkv,dim,lens,new", [
    (4, 2, 128, [3001, 700], [1, 1]),                   # few rows, over many blocks
    (8, 2, 64, [9000], [5]),                            # a drafted run
    (4, 2, 128, [2500], [300]),                         # tiles, two row tiles an item
    (2, 2, 64, [4000, 130], [60, 100]),                 # tiles, alternate key tiles
])
def test_bf16_outputs_are_as_good_as_their_weights(paged, cache, hq, hkv, dim, lens, new):
    """Weights w_j in bf16 are off by e_j, |e_j| <= 2^-8 of them and of either sign, evenly spread: an output
    by sum w_j e_j v_j, whose standard deviation is at most 2^-8 / sqrt(3) sqrt(sum w_j^2 v_j^2); six of them,
    the output's own rounding (2^-8 of it), and 2^-18 of the largest value for scores and sums.  That is little
    enough to notice a key tile that is left out, which a bound by the largest value is not."""
    s = Setup(cache, "bf16", hq, hkv, dim, 16, lens, new, seed=40)
    out = s.attend(paged, max_new=max(new), max_kv=max(lens)).double()
    group, r0 = hq // hkv, 0
    for b, (n, m) in enumerate(zip(lens, new)):
        pos = torch.arange(n, device="cuda")
        pg, off = s.table[b].long()[pos // 16], pos % 16
        k, v = (values(s.pages[x], s.scale[x])[pg, off].repeat_interleave(group, 1) for x in "kv")
        z = torch.einsum("qhd,khd->hqk", s.q[r0:r0 + m].double(), k) * dim ** -0.5
        z = z.masked_fill(pos > torch.arange(n - m, n, device="cuda")[:, None], -math.inf)
        w = torch.softmax(z, -1)
        want = torch.einsum("hqk,khd->qhd", w, v)
        spread = torch.einsum("hqk,khd->qhd", w * w, v * v).sqrt()
        tol = 2.0 ** -8 * (want.abs() + 6 / 3 ** 0.5 * spread) + 2.0 ** -18 * v.abs().max()
        got = out[r0:r0 + m]
        assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())
        if n > 256:
            z[..., 128:256] = -math.inf                 # a tile lost
            lost = torch.einsum("hqk,khd->qhd", torch.softmax(z, -1), v)
            assert not bool(((got - lost).abs() <= tol).all(0).all(0).any())
        r0 += m


# ------------------------------------------------------------------ graphs
@pytest.mark.parametrize("cache,act,hq,lens,new", [("i8", "f32", 8, [3000, 90], [1, 1]), ("bf16", "bf16", 8, [700, 300], [200, 40]),
                                                   ("f8", "bf16", 16, [2000] * 40, [3] * 40)])
def test_calls_of_two_launches_in_a_graph(paged, cache, act, hq, lens, new):
    """Write, attention that is cut over blocks and joined, and verification by clusters, captured once and
    replayed on other contents."""
    s = Setup(cache, act, hq, 4, 64, 16, lens, new, seed=41)
    slots = torch.cat([s.table[b].long()[p // 16] * 16 + p % 16
                       for b, (n, m) in enumerate(zip(lens, new)) for p in [torch.arange(n - m, n, device="cuda")]])
    V = 30011
    target = torch.softmax(2 * torch.randn(3, 3, V, generator=gen(42), device="cuda"), -1)
    draft = torch.softmax(2 * torch.randn(3, 2, V, generator=gen(43), device="cuda"), -1)
    x = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    au, su = torch.rand(3, 2, device="cuda"), torch.rand(3, device="cuda")
    out = torch.empty_like(s.q)

    def calls():
        paged.kv_write(s.k, s.v, s.pages["k"], s.pages["v"], slots, **s.kw())
        s.attend(paged, max_new=max(new), max_kv=max(lens), out=out)
        return paged.verify_draft(target, draft, x, au, su)
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, accepted = calls()
    for i in range(3):
        for t in (s.q, s.k, s.v):
            t.copy_(torch.randn(t.shape, generator=gen(50 + i), device="cuda"))
        x.copy_(torch.randint(0, V, x.shape, generator=gen(60 + i), device="cuda"))
        au.uniform_(0, 1, generator=gen(70 + i))
        out.fill_(7.0)
        graph.replay()
        paged.check_stream()
        compare(s, out, act)
        want, wacc = settle(*(t.cpu().numpy() for t in (target, draft, x, au, su)))
        np.testing.assert_array_equal(accepted.cpu().numpy(), wacc)
        np.testing.assert_array_equal(tokens.cpu().numpy(), want)


@pytest.mark.parametrize("cache,act", CACHES)
@pytest.mark.parametrize("new,lens", [(1, 40), (5, 3000), (60, 300), (300, 500)])
def test_values_do_not_enter_the_log_sum_exp(paged, cache, act, new, lens):
    """A value that is not finite makes outputs NaN; the softmax's sum knows nothing of it."""
    s = Setup(cache, act, 4, 2, 64, 16, [lens], [new], seed=44)
    _, want = s.expected()
    for pos in (lens - 1, lens - new // 2 - 1, 3):
        pg, off = place(s, 0, pos)
        if s.scale["v"] is None:
            s.pages["v"][pg, off, 0, 5] = math.nan
        else:
            s.scale["v"][pg, off, 0] = math.nan
    lse = torch.empty(s.q.shape[:2], device="cuda")
    out = s.attend(paged, lse=lse)
    assert bool(out[:, :2].isnan().any(-1).all()) and bool(out[:, 2:].isfinite().all())
    assert float((lse.double() - want).abs().max()) < (1e-4 if act == "f32" else 2e-2)


@pytest.mark.parametrize("cache,act", CACHES)
@pytest.mark.parametrize("heads,seqs,new", [(2, 1, 1), (2, 1, 80), (16, 4, 80), (8, 3, 200)])
@pytest.mark.parametrize("powers", [(None, 40), (None, 60), (-60, 60), (60, None), (-40, None, 40, 0)])
def test_values_of_far_apart_sizes(paged, cache, act, heads, seqs, new, powers):
    """Values of every 128 positions times a power of two of their own, or zero: what weighs little in the output
    still weighs in full in the sum and the log-sum-exp."""
    s = Setup(cache, act, heads, heads, 64, 16, [700 + 30 * b for b in range(seqs)], [new] * seqs, seed=45)
    for b, n in enumerate(s.lens):
        for i in range(0, n, 16):
            f, pg = powers[i // 128 % len(powers)], int(s.table[b, i // 16])
            f = 0.0 if f is None else 2.0 ** f
            if s.scale["v"] is None:
                s.pages["v"][pg] = torch.where(s.pages["v"][pg].isnan(), s.pages["v"][pg], s.pages["v"][pg] * f)
            else:
                s.scale["v"][pg] *= f
    lse = torch.empty(s.q.shape[:2], device="cuda")
    out = s.attend(paged, lse=lse)
    ref, want = s.expected()
    compare(s, out, act)
    assert float((lse.double() - want).abs().max()) < (1e-4 if act == "f32" else 2e-2)


@pytest.mark.parametrize("cache,act", CACHES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sink", [0, 70, 130, 200])
def test_a_position_that_outweighs_all_others(paged, cache, act, dim, sink):
    """One key with a score some 200 above the rest, and larger values far behind it: every weight but one
    underflows, and the output is that position's values."""
    s = Setup(cache, act, 32, 16, dim, 16, [1500, 900, 1200, 1400, 1100], [100, 100, 64, 80, 90], seed=46)
    for b, n in enumerate(s.lens):
        at = place(s, b, sink)
        if s.scale["k"] is None:
            s.pages["k"][at] = 8.0
        else:
            s.pages["k"][at] = torch.full((dim,), 100.0, device="cuda").to(CACHE[cache])
            s.scale["k"][at] = 0.08
        for i in range(384 // 16, -(-n // 16)):         # whole pages
            pg = int(s.table[b, i])
            if s.scale["v"] is None:
                s.pages["v"][pg] *= 16
            else:
                s.scale["v"][pg] *= 16
    s.q.copy_((200 * dim ** 0.5 / (8 * dim) + 0.1 * s.q.float()).to(s.q.dtype))
    out = s.attend(paged)
    ref, _ = s.expected()
    assert bool(out.isfinite().all())
    # the one weight is 1 up to fp32 rounding: the values' own form (22 bits), then the output's rounding
    assert float((out.double() - ref).abs().max()) <= (2.0 ** -19 if act == "f32" else 2.0 ** -8) * float(ref.abs().max())
