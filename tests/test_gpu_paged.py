"""Paged key/value cache, attention over it and draft verification on the GPU.

Every operator is compared with its definition in 64 bits.  Tolerances:

* storing and reading back: float caches hold the value in their type exactly, 8 bits
  half a code (i8: scale/2; e4m3: 2^-4 of the value or 2^-10 scales) plus the
  rounding of the read's type;
* attention, fp32: products and sums carry at least 21 significant bits, so an
  output is within 2^-19 of the largest value it averages (|out| <= max |v|), a
  score within 2^-19 of |q| |k| scale, which scales the weights by as much:
  (2^-19 (1 + 2 max |q||k| scale)) max|v|, below 1e-4 at these sizes;
* attention, bf16 output: the output's own rounding, 2^-8 of its value, and
  weights rounded to bf16 (2^-8, relative, averaged): 2^-7 max|v|;
* draft verification: whole numbers, equal.
"""

import math

import numpy as np
import pytest
import torch

from conftest import has_gpu

pytestmark = pytest.mark.gpu

CACHE = {"f32": torch.float32, "bf16": torch.bfloat16, "f8": torch.float8_e4m3fn, "i8": torch.int8}
ACT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def paged():
    if not has_gpu():
        pytest.skip("no CUDA device")
    from lbr_b200 import paged as m
    return m


def gen(seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def values(pages, scale):
    """What a cache stands for, in 64 bits."""
    x = pages.double()
    return x if scale is None else x * scale.double()[..., None]


class Setup:
    """A cache of random contents with shuffled pages and poisoned unused slots."""

    def __init__(self, cache, act, hq, hkv, dim, page, lens, new, seed=0, poison=True, layout="slots", spread=1.0):
        g, dev = gen(seed), "cuda"
        self.lens, self.new, self.page, self.dim = lens, new, page, dim
        per = [-(-max(n, 0) // page) for n in lens]
        n_pages = sum(per) + 2
        order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
        width = max(per + [1])
        self.table = torch.zeros(len(lens), width, dtype=torch.int32, device=dev)
        used, at = torch.zeros(n_pages, page, dtype=torch.bool, device=dev), 0
        for b, n in enumerate(per):
            ids = order[at:at + n]
            self.table[b, :n] = ids
            for i in range(n):
                used[ids[i].long(), :min(page, lens[b] - i * page)] = True
            at += n
        shape = (n_pages, page, hkv, dim)
        self.scale = {"k": None, "v": None}
        self.pages = {}
        for x in "kv":
            y = torch.randn(shape, generator=g, device=dev) * spread
            if cache in ("f8", "i8"):
                m = 448.0 if cache == "f8" else 127.0
                s = y.abs().amax(-1) / m
                code = y / s[..., None]
                self.pages[x] = (code.round() if cache == "i8" else code).to(CACHE[cache])
                self.scale[x] = s
                if poison:
                    self.scale[x] = torch.where(used[..., None], s, torch.full_like(s, math.nan))
            else:
                if poison:
                    y = torch.where(used[..., None, None], y, torch.full_like(y, math.nan))
                self.pages[x] = y.to(CACHE[cache])
        if layout == "heads":      # [pages, heads, page, dim] in memory
            for x in "kv":
                self.pages[x] = self.pages[x].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
                if self.scale[x] is not None:
                    self.scale[x] = self.scale[x].permute(0, 2, 1).contiguous().permute(0, 2, 1)
        self.lens_t = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.cu = torch.tensor(np.cumsum([0] + new), dtype=torch.int32, device=dev)
        qkv = torch.randn(sum(new), hq + 2 * hkv, dim, generator=g, device=dev).to(ACT[act])
        self.q, self.k, self.v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]

    def kw(self):
        return {"k_scale": self.scale["k"], "v_scale": self.scale["v"]}

    def attend(self, paged, **kw):
        return paged.paged_attention(self.q, self.pages["k"], self.pages["v"], self.table, self.lens_t, self.cu,
                                     **self.kw(), **kw)

    def expected(self, causal=True, window=0, scale=None):
        scale = self.dim ** -0.5 if scale is None else scale
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        lse = torch.full(self.q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        group = self.q.shape[1] // self.pages["k"].shape[2]
        cu = self.cu.tolist()
        for b, (n, m) in enumerate(zip(self.lens, self.new)):
            if n == 0 or m == 0:
                continue
            pos = torch.arange(n, device="cuda")
            pg, off = self.table[b].long()[pos // self.page], pos % self.page
            k, v = (values(self.pages[x], self.scale[x])[pg, off].repeat_interleave(group, 1) for x in "kv")
            at = torch.arange(n - m, n, device="cuda")[:, None]
            seen = pos <= at if causal else torch.ones_like(pos <= at)
            if window:
                seen = seen & (pos > at - window)
            z = torch.einsum("qhd,khd->hqk", self.q[cu[b]:cu[b + 1]].double(), k) * scale
            z = z.masked_fill(~seen, -math.inf)
            some = seen.any(-1)
            p = torch.softmax(torch.where(some[:, None], z, torch.zeros_like(z)), -1)
            # a position no row sees must not enter, whatever it holds
            o = torch.stack([torch.einsum("hk,khd->hd", p[:, i][:, seen[i]], v[seen[i]]) for i in range(m)]) \
                if m <= 64 else torch.einsum("hqk,khd->qhd", p, v)
            out[cu[b]:cu[b + 1]] = torch.where(some[:, None, None], o, torch.zeros_like(o))
            lse[cu[b]:cu[b + 1]] = torch.where(some, torch.logsumexp(z, -1), torch.full_like(z[..., 0], -math.inf)).T
        return out, lse


def tolerance(s, act):
    vmax = max(float(values(s.pages["v"], s.scale["v"]).nan_to_num(0, 0, 0).abs().max()), 1e-30)
    if act == "bf16":
        return 2.0 ** -7 * vmax
    return min(1e-4, 2.0 ** -19 * (1 + 2 * float(s.q.double().norm(dim=-1).max()) * s.dim ** 0.5 * vmax * s.dim ** -0.5)) * max(vmax, 1.0)


def compare(s, out, act, **kw):
    ref, _ = s.expected(**kw)
    assert torch.isfinite(out).all()
    err = float((out.double() - ref).abs().max()) if ref.numel() else 0.0
    assert err <= tolerance(s, act), f"max abs error {err:.3e}, allowed {tolerance(s, act):.3e}"


CACHES = [("f32", "f32"), ("bf16", "f32"), ("i8", "f32"), ("f8", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("i8", "bf16"), ("f8", "bf16")]


@pytest.mark.parametrize("cache,act", CACHES)
@pytest.mark.parametrize("hq,hkv,dim,page,lens,new", [
    (4, 4, 64, 16, [1], [1]),                                   # the first token of all
    (12, 12, 64, 16, [200], [1]),
    (16, 8, 128, 16, [1, 127, 128, 129, 700, 3001], [1] * 6),   # tile edges
    (8, 1, 128, 64, [513, 40], [1, 1]),                         # eight heads share one
    (16, 1, 64, 32, [300, 5], [1, 1]),                          # sixteen
    (32, 1, 128, 32, [260], [1]),                               # more rows than a small tile
    (4, 2, 16, 16, [33, 50], [1, 3]),                           # small head dim
    (4, 2, 96, 24, [100, 257], [2, 1]),                         # head dim off a power of two, odd pages
    (6, 2, 80, 1, [70], [5]),                                   # pages of one slot, three heads to one
    (5, 5, 32, 7, [29, 300], [4, 1]),                           # odd everything
])
def test_attention_few_rows(paged, cache, act, hq, hkv, dim, page, lens, new):
    s = Setup(cache, act, hq, hkv, dim, page, lens, new)
    compare(s, s.attend(paged), act)


@pytest.mark.parametrize("cache,act", CACHES)
@pytest.mark.parametrize("hq,hkv,dim,page,lens,new", [
    (4, 2, 128, 16, [5, 600], [5, 5]),                          # a whole short prompt; a drafted run
    (8, 8, 64, 64, [300], [300]),                               # a prompt from nothing
    (4, 2, 128, 24, [1000, 130, 77], [129, 1, 77]),             # a mixed step, odd pages
    (16, 4, 128, 128, [520], [260]),
    (2, 1, 64, 48, [900], [513]),
    (3, 1, 112, 16, [150], [60]),                               # head dim the tensor tiles do not take
])
def test_attention_chunks(paged, cache, act, hq, hkv, dim, page, lens, new):
    s = Setup(cache, act, hq, hkv, dim, page, lens, new, seed=1)
    compare(s, s.attend(paged), act)


@pytest.mark.parametrize("cache,act", [("f32", "f32"), ("bf16", "bf16"), ("i8", "f32"), ("f8", "bf16")])
def test_attention_empty_sequences_and_rows(paged, cache, act):
    """Lengths of zero, sequences without new tokens, more new tokens than positions: rows that
    see nothing are zero and their lse is -inf."""
    for new in ([0, 3, 2, 1, 0], [0, 40, 30, 1, 0]):
        s = Setup(cache, act, 8, 4, 64, 16, [0, 0, 1, 20, 300], new)
        lse = torch.empty(sum(new), 8, device="cuda")
        out = s.attend(paged, lse=lse)
        ref, rl = s.expected()
        compare(s, out, act)
        assert torch.equal(torch.isinf(lse), torch.isinf(rl))
        fin = torch.isfinite(rl)
        assert float((lse.double() - rl)[fin].abs().max()) < (1e-4 if act == "f32" else 2e-2)


@pytest.mark.parametrize("cache,act", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("i8", "f32"), ("f8", "bf16")])
@pytest.mark.parametrize("window", [1, 5, 128, 1000])
def test_attention_window(paged, cache, act, window):
    s = Setup(cache, act, 8, 4, 128, 16, [1, 130, 700, 900], [1, 2, 1, 150], seed=2)
    compare(s, s.attend(paged, window=window), act, window=window)


@pytest.mark.parametrize("cache,act", [("f32", "f32"), ("bf16", "bf16"), ("i8", "f32")])
def test_attention_not_causal_and_scaled(paged, cache, act):
    s = Setup(cache, act, 4, 4, 64, 32, [200, 31], [70, 4], seed=3)
    compare(s, s.attend(paged, causal=False, scale=0.05), act, causal=False, scale=0.05)


@pytest.mark.parametrize("cache", ["f32", "bf16"])
@pytest.mark.parametrize("new", [6, 70])
def test_masked_values_do_not_enter(paged, cache, new):
    """A later token's keys and values may hold anything: earlier tokens do not see them, later do."""
    s = Setup(cache, "f32" if cache == "f32" else "bf16", 4, 2, 64, 16, [230], [new], seed=4)
    bad = 225                                              # a position only the last tokens see
    pg, off = int(s.table[0, bad // 16]), bad % 16
    s.pages["v"][pg, off, 0, 3] = math.inf
    s.pages["v"][pg, off, 1, 5] = math.nan
    s.pages["k"][pg, off] = math.nan
    out = s.attend(paged).double()
    first = new - (230 - bad)                              # tokens before this one do not see it
    clean = Setup(cache, "f32" if cache == "f32" else "bf16", 4, 2, 64, 16, [230], [new], seed=4)
    ref, _ = clean.expected()
    assert torch.isfinite(out[:first]).all()
    assert float((out[:first] - ref[:first]).abs().max()) <= tolerance(clean, "f32" if cache == "f32" else "bf16")
    assert not torch.isfinite(out[first:]).all()


@pytest.mark.parametrize("cache,act", [("f32", "f32"), ("bf16", "bf16"), ("i8", "f32"), ("f8", "bf16")])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_layouts_and_strides(paged, cache, act, new):
    """Heads-first pages, out and q as views of wider tensors, a table with spare columns."""
    s = Setup(cache, act, 8, 2, 64, 16, [130, 400], [new, new], seed=5, layout="heads")
    wide = torch.full((2 * new, 10, 72), 7.0, dtype=ACT[act], device="cuda")
    out = wide[:, 1:9, 4:68]
    table = torch.full((2, s.table.shape[1] + 3), -1, dtype=torch.int32, device="cuda")
    table[:, :s.table.shape[1]] = s.table
    s.table = table[:, :s.table.shape[1]]
    got = s.attend(paged, out=out)
    assert got is out
    compare(s, out, act)
    keep = torch.ones_like(wide, dtype=torch.bool)
    keep[:, 1:9, 4:68] = False
    assert bool((wide[keep] == 7.0).all())


@pytest.mark.parametrize("cache,act", [("f32", "f32"), ("bf16", "bf16"), ("i8", "f32"), ("f8", "f32")])
@pytest.mark.parametrize("lens,new,bounds", [([40, 9000], [1, 1], {}), ([40, 9000], [1, 1], {"max_kv": 9000, "max_new": 1}),
                                             ([2500, 600], [200, 3], {"max_kv": 64, "max_new": 1}),
                                             ([2500, 600], [3, 3], {"max_kv": 2500, "max_new": 2500})])
def test_bounds_do_not_change_results(paged, cache, act, lens, new, bounds):
    """max_new / max_kv steer the split only; and a call gives the same bits every time."""
    s = Setup(cache, act, 8, 4, 128, 32, lens, new, seed=6)
    out = s.attend(paged, **bounds)
    compare(s, out, act)
    for _ in range(3):
        assert torch.equal(out, s.attend(paged, **bounds))


@pytest.mark.parametrize("cache", ["i8", "f8"])
def test_scales_far_apart(paged, cache):
    """Value scales that differ by 2^20 between tokens."""
    for new in (1, 80):
        s = Setup(cache, "f32", 4, 2, 64, 16, [500], [new], seed=7)
        f = torch.exp2(torch.randint(-10, 10, s.scale["v"].shape, device="cuda", generator=gen(1)).float())
        s.scale["v"] = s.scale["v"] * f
        compare(s, s.attend(paged), "f32")


@pytest.mark.parametrize("cache,act", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("i8", "f32")])
@pytest.mark.parametrize("new", [1, 64])
def test_large_scores(paged, cache, act, new):
    """Scores of hundreds: the running maximum has to move, weights underflow."""
    s = Setup(cache, act, 4, 2, 128, 16, [700], [new], seed=8, spread=6.0)
    ref, _ = s.expected()
    out = s.attend(paged).double()
    assert torch.isfinite(out).all()
    # a score is off by 2^-19 |q||k| scale ~ 2^-19 * 12 * 72 / 11 (fp32), which moves a weight by as much
    tol = 1e-3 if act == "f32" else 2.0 ** -6 * 36
    assert float((out - ref).abs().max()) < tol


def test_bad_pages_and_lengths_are_reported(paged):
    from lbr_b200.executor import CudaRuntimeError
    s = Setup("f32", "f32", 4, 4, 64, 16, [100], [1])
    paged.check_stream()
    table = s.table.clone()
    table[0, 2] = 10 ** 6
    for t, lens in ((table, s.lens_t), (s.table, s.lens_t + 1000)):
        out = paged.paged_attention(s.q, s.pages["k"], s.pages["v"], t, lens, s.cu)
        with pytest.raises(CudaRuntimeError, match="out of range"):
            paged.check_stream()
        assert out.shape == s.q.shape
    with pytest.raises(CudaRuntimeError):
        paged.kv_write(s.k, s.v, s.pages["k"], s.pages["v"], torch.tensor([10 ** 9], device="cuda"))
        paged.check_stream()
    paged.check_stream()


# ------------------------------------------------------------------ write and read
@pytest.mark.parametrize("cache", ["f32", "bf16", "i8", "f8"])
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("heads,dim,page,n,offset", [(12, 64, 16, 1, 0), (8, 128, 64, 333, 0), (1, 16, 3, 50, 0),
                                                     (5, 96, 24, 77, 1), (2, 112, 128, 300, 2)])
def test_write_and_read_back(paged, cache, act, heads, dim, page, n, offset):
    g = gen(9)
    n_pages = -(-n // page) + 2
    pages = [torch.zeros(n_pages, page, heads, dim, device="cuda").to(CACHE[cache]) for _ in range(2)]
    scale = [torch.zeros(n_pages, page, heads, device="cuda") for _ in range(2)] if cache in ("i8", "f8") else [None, None]
    # rows of a wider projection, shifted off 16 bytes by `offset` elements
    wide = torch.randn(n, 2 * heads, dim + 8, generator=g, device="cuda").to(ACT[act])
    k, v = wide[:, :heads, offset:offset + dim], wide[:, heads:, offset:offset + dim]
    order = torch.randperm(n_pages, generator=g, device="cuda")
    pos = torch.arange(n, device="cuda")
    slots = order[pos // page] * page + pos % page
    if n > 3:
        slots[2] = -1                                   # a padding token
    paged.kv_write(k, v, pages[0], pages[1], slots, k_scale=scale[0], v_scale=scale[1])
    table = order[None, :-2].to(torch.int32) if n_pages > 2 else order[None].to(torch.int32)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    for out in ("f32", "bf16"):
        got = paged.kv_read(pages[0], pages[1], table, None, cu, n, k_scale=scale[0], v_scale=scale[1], dtype=ACT[out])
        for x, y in zip((k, v), got):
            assert y.dtype is ACT[out]
            if cache in ("f32", "bf16"):                # nothing but the types' own rounding
                x = x.to(CACHE[cache]).to(ACT[out])
            x, y = x.double(), y.double()
            if n > 3:
                assert bool((y[2] == 0).all())
                x, y = torch.cat([x[:2], x[3:]]), torch.cat([y[:2], y[3:]])
            top = x.abs().amax(-1, keepdim=True)
            tol = {"f32": 0 * x, "bf16": 0 * x, "i8": top / 127 * 0.5001,
                   "f8": torch.maximum(x.abs() * 2.0 ** -4, top / 448 * 2.0 ** -10) * 1.0001}[cache]
            if cache in ("i8", "f8"):
                tol = tol + ((x.abs() + tol) * 2.0 ** -8 if out == "bf16" else x.abs() * 2.0 ** -22)
            assert bool(((x - y).abs() <= tol).all())
    paged.check_stream()


@pytest.mark.parametrize("cache", ["i8", "f8"])
def test_quantised_codes_follow_the_definition(paged, cache):
    """Codes and scales bit for bit, with zero, tiny, huge and non-finite heads."""
    heads, dim, n, m = 4, 64, 40, np.float32(127 if cache == "i8" else 448)
    x = torch.randn(n, heads, dim, generator=gen(10), device="cuda")
    x[0] = 0
    x[1] *= 1e-35
    x[2] *= 1e30
    x[3, 0, 5], x[3, 1, 6], x[3, 2, 7] = math.inf, -math.inf, math.nan
    pages = [torch.ones(3, 16, heads, dim, device="cuda").to(CACHE[cache]) for _ in range(2)]
    scale = [torch.ones(3, 16, heads, device="cuda") for _ in range(2)]
    paged.kv_write(x, x, pages[0], pages[1], torch.arange(n, device="cuda"), k_scale=scale[0], v_scale=scale[1])
    h = x.cpu().numpy()
    with np.errstate(all="ignore"):
        top = np.abs(h).max(-1)
        live = (top >= np.float32(2.0 ** -100)) & np.isfinite(top)
        want = np.where(live, top * (np.float32(1) / m), np.float32(0)).astype(np.float32)
        inv = np.where(live, (np.float32(1) / top) * m, 0).astype(np.float32)
        code = np.where(live[..., None], h * inv[..., None], 0).astype(np.float32)
        want = np.where(np.isfinite(top), want, np.float32("nan"))
    code = torch.from_numpy(np.rint(code) if cache == "i8" else np.clip(code, -448, 448)).to(CACHE[cache])
    for i in range(2):
        assert torch.equal(pages[i].flatten(0, 1)[:n].cpu().view(torch.int8), code.view(torch.int8))
        np.testing.assert_array_equal(scale[i].flatten(0, 1)[:n].cpu().numpy(), want)
        assert bool((scale[i].flatten(0, 1)[n:] == 1).all())


def test_read_ranges(paged):
    """Ranges that start inside pages, empty ranges, rows past the last range."""
    g = gen(11)
    pages = [torch.randn(9, 8, 2, 32, generator=g, device="cuda") for _ in range(2)]
    table = torch.tensor([[3, 1, 4, 0], [8, 2, 0, 0], [5, 0, 0, 0]], dtype=torch.int32, device="cuda")
    start, count = [5, 0, 7], [20, 0, 1]
    cu = torch.tensor(np.cumsum([0] + count), dtype=torch.int32, device="cuda")
    k, v = paged.kv_read(pages[0], pages[1], table, torch.tensor(start, dtype=torch.int32, device="cuda"), cu, 24)
    for x, p in ((k, pages[0]), (v, pages[1])):
        rows = [p[int(table[b, j // 8]), j % 8] for b in range(3) for j in range(start[b], start[b] + count[b])]
        assert torch.equal(x[:21], torch.stack(rows))
        assert bool((x[21:] == 0).all())
    paged.check_stream()


# ------------------------------------------------------------------ drafted tokens
def settle(target, draft, tokens, au, su, lens=None):
    """The definition with Python integers."""
    B, N1, V = target.shape
    N = N1 - 1
    out, acc = -np.ones((B, N1), np.int64), np.zeros(B, np.int64)
    f = np.float32
    for b in range(B):
        n = N if lens is None else int(lens[b])
        a = 0
        while a < n:
            x = int(tokens[b, a])
            if not 0 <= x < V:
                break
            q = f(1) if draft is None else f(draft[b, a, x])
            if not f(au[b, a]) * q < f(target[b, a, x]):
                break
            a += 1
        acc[b] = a
        out[b, :a] = tokens[b, :a]
        row = target[b, a].astype(f)
        w = row
        if a < n:
            q = np.zeros(V, f)
            if draft is not None:
                q = draft[b, a].astype(f)
            elif 0 <= int(tokens[b, a]) < V:
                q[int(tokens[b, a])] = 1
            with np.errstate(invalid="ignore"):
                w = row - q
        for ws in (w, row):
            ws = np.where(ws > 0, np.minimum(ws, f(1)), f(0))
            m = [int(z) for z in np.floor(ws.astype(np.float64) * 2.0 ** 40)]
            total = sum(m)
            if total:
                break
        if total:
            t = (int(np.floor(min(max(float(su[b]), 0.0) * 2.0 ** 24, 2.0 ** 24 - 1))) * total) >> 24
            c = np.cumsum(np.array(m, dtype=object))
            out[b, a] = int(np.argmax(c > t))
    return out, acc


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("B,N,V", [(1, 1, 7), (3, 4, 1000), (20, 7, 4099), (2, 3, 50001), (5, 0, 333), (1, 4, 300001)])
def test_verify_draft(paged, act, B, N, V):
    g = gen(12)
    target = torch.softmax(2 * torch.randn(B, N + 1, V, generator=g, device="cuda"), -1).to(ACT[act])
    draft = torch.softmax(target[:, :N].float().log() + 0.5 * torch.randn(B, N, V, generator=g, device="cuda"), -1).to(ACT[act])
    tokens = torch.multinomial(draft.float().reshape(-1, V), 1, generator=g).view(B, N).to(torch.int32) if N else \
        torch.zeros(B, 0, dtype=torch.int32, device="cuda")
    au, su = torch.rand(B, N, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")
    lens = torch.randint(0, N + 1, (B,), generator=g, device="cuda").to(torch.int32)
    for d in (draft, None):
        for n in (None, lens):
            got, acc = paged.verify_draft(target, d, tokens, au, su, draft_lens=n)
            want, wacc = settle(target.float().cpu().numpy(), None if d is None else d.float().cpu().numpy(),
                                tokens.cpu().numpy(), au.cpu().numpy(), su.cpu().numpy(), None if n is None else n.tolist())
            np.testing.assert_array_equal(acc.cpu().numpy(), wacc)
            np.testing.assert_array_equal(got.cpu().numpy(), want)
    paged.check_stream()


def test_verify_extremes(paged):
    """Uniform numbers at the ends, a draft equal to its target, rows without mass, NaN, one-hot rows."""
    V = 100
    target = torch.full((6, 2, V), 1.0 / V, device="cuda")
    draft = target[:, :1].clone()
    target[1, 0] = 0
    target[1, 0, 17] = 1
    target[2, 0] = 0                                    # nothing to sample from
    target[3, 0, :50] = math.nan
    target[4, 1] = 0
    target[4, 1, 99] = 1e-13                            # below the fixed-point unit: no mass
    tokens = torch.tensor([[3], [17], [5], [60], [2], [200]], dtype=torch.int32, device="cuda")
    au = torch.tensor([[0.9999999], [0.5], [0.5], [1.0], [0.0], [0.0]], device="cuda")
    for u in (0.0, 0.5, 1.0 - 2.0 ** -24, 1.0):
        su = torch.full((6,), u, device="cuda")
        got, acc = paged.verify_draft(target, draft, tokens, au, su)
        want, wacc = settle(target.cpu().numpy(), draft.cpu().numpy(), tokens.cpu().numpy(), au.cpu().numpy(), su.cpu().numpy())
        np.testing.assert_array_equal(acc.cpu().numpy(), wacc)
        np.testing.assert_array_equal(got.cpu().numpy(), want)
    from lbr_b200.executor import CudaRuntimeError
    with pytest.raises(CudaRuntimeError, match="out of range"):
        paged.check_stream()                            # token 200 of 100


def test_verify_keeps_the_target_distribution(paged):
    """Over many uniform numbers the first emitted token follows the target, whatever the draft."""
    V, B = 8, 200000
    g = gen(13)
    p = torch.softmax(torch.randn(V, generator=g, device="cuda"), 0)
    q = torch.softmax(torch.randn(V, generator=g, device="cuda"), 0)
    target, draft = p.expand(B // 10, 2, V), q.expand(B // 10, 1, V)
    count = torch.zeros(V, device="cuda")
    for _ in range(10):
        tokens = torch.multinomial(q, B // 10, replacement=True, generator=g)[:, None].to(torch.int32)
        got, _ = paged.verify_draft(target, draft, tokens, torch.rand(B // 10, 1, generator=g, device="cuda"),
                                    torch.rand(B // 10, generator=g, device="cuda"))
        count += torch.bincount(got[:, 0].long(), minlength=V)
    # a count's standard deviation is sqrt(B p (1 - p)): five of them
    assert bool(((count / B - p).abs() < 5 * (p * (1 - p) / B).sqrt()).all())


# ------------------------------------------------------------------ streams, graphs, refusals
def test_stream_and_graph(paged):
    """Calls follow torch's current stream, and can be captured and replayed on new contents."""
    s = Setup("i8", "f32", 8, 4, 64, 16, [400, 90], [1, 1], seed=14)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = s.attend(paged, max_kv=400, max_new=1)
    side.synchronize()
    compare(s, a, "f32")
    out = torch.empty_like(a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.attend(paged, max_kv=400, max_new=1, out=out)
    s.q.copy_(torch.randn(s.q.shape, device="cuda"))
    s.lens_t.copy_(torch.tensor([250, 1], dtype=torch.int32))
    s.lens = [250, 1]
    graph.replay()
    torch.cuda.synchronize()
    compare(s, out, "f32")
    paged.check_stream()


def test_refusals(paged):
    from lbr_b200.executor import CudaRuntimeError
    s = Setup("i8", "f32", 8, 4, 64, 16, [100], [1])
    kp, vp, q, t, n, cu, kw = s.pages["k"], s.pages["v"], s.q, s.table, s.lens_t, s.cu, s.kw()
    with pytest.raises(ValueError, match="8-bit"):
        paged.paged_attention(q, kp, vp, t, n, cu)
    with pytest.raises(TypeError):
        paged.paged_attention(q.half(), kp, vp, t, n, cu, **kw)
    with pytest.raises(ValueError):
        paged.paged_attention(q[:, :, :32], kp, vp, t, n, cu, **kw)
    with pytest.raises(TypeError):
        paged.paged_attention(q, kp, vp, t.long(), n, cu, **kw)
    with pytest.raises(ValueError):
        paged.paged_attention(q, kp, vp, t, n.cpu(), cu, **kw)
    with pytest.raises(CudaRuntimeError):
        paged.paged_attention(q[:, :7], kp, vp, t, n, cu, **kw)          # 7 query heads over 4
    with pytest.raises(CudaRuntimeError):
        paged.paged_attention(q, kp, vp, t, n, cu, window=-1, **kw)
    with pytest.raises(CudaRuntimeError):
        paged.paged_attention(q, kp, vp, t, n, cu, scale=0.0, **kw)
    wide = torch.zeros(4, 16, 4, 68, device="cuda")[..., 2:66]           # rows off 16 bytes
    with pytest.raises(CudaRuntimeError, match="16"):
        paged.paged_attention(q, wide, wide, t, n, cu)
    big = torch.zeros(2, 16, 4, 144, device="cuda")
    with pytest.raises(CudaRuntimeError, match="head_dim"):
        paged.kv_write(torch.zeros(1, 4, 144, device="cuda"), torch.zeros(1, 4, 144, device="cuda"), big, big,
                       torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(TypeError):
        paged.kv_write(s.k, s.v.bfloat16(), kp, vp, torch.zeros(1, dtype=torch.int64, device="cuda"), **kw)
    with pytest.raises(TypeError):
        paged.kv_write(s.k, s.v, kp, vp, torch.zeros(1, dtype=torch.int32, device="cuda"), **kw)
    with pytest.raises(ValueError):
        paged.kv_read(kp, vp, t, None, cu, 1, out=(q, q), **kw)
    p = torch.zeros(2, 3, 50, device="cuda")
    x, u = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, device="cuda")
    with pytest.raises(ValueError):
        paged.verify_draft(p, p, x, u, u[:, 0].contiguous())
    with pytest.raises(TypeError):
        paged.verify_draft(p, p[:, :2].bfloat16(), x, u, u[:, 0].contiguous())
    # a host pointer through the C ABI
    import ctypes
    from lbr_b200.executor import load_library
    lib = load_library()
    lib.rt_kv_write.argtypes, lib.rt_kv_write.restype = [ctypes.POINTER(paged.RtKvWrite), ctypes.c_void_p], ctypes.c_int
    a = paged.RtKvWrite()
    c = a.cache
    c.k, c.v, c.k_scale, c.v_scale = kp.data_ptr(), vp.data_ptr(), kw["k_scale"].data_ptr(), kw["v_scale"].data_ptr()
    c.stride[:], c.scale_stride[:] = kp.stride()[:3], kw["k_scale"].stride()
    c.dtype, (c.n_pages, c.page_size, c.n_heads, c.head_dim) = 3, kp.shape
    slots = torch.full((1,), 5, dtype=torch.int64, device="cuda")
    k = torch.zeros(1, 4, 64, device="cuda")
    a.k = a.v = k.data_ptr()
    a.k_stride[:] = a.v_stride[:] = (256, 64)
    a.slots, a.n_tokens = slots.data_ptr(), 1
    assert lib.rt_kv_write(a, None) == 0
    host = torch.zeros(1, 4, 64)
    a.k = host.data_ptr()
    assert lib.rt_kv_write(a, None) == 5            # RT_ERR_HOST_POINTER
    a.k = None
    assert lib.rt_kv_write(a, None) == 4            # RT_ERR_NULL_POINTER
    a.k, a.dtype = k.data_ptr(), 2
    assert lib.rt_kv_write(a, None) == 7            # RT_ERR_UNSUPPORTED
    paged.check_stream()


@pytest.mark.parametrize("cache,act", CACHES)
@pytest.mark.parametrize("hq,hkv,dim,new", [(8, 2, 128, 5), (4, 4, 64, 33), (8, 2, 128, 9), (16, 8, 64, 16), (2, 2, 128, 31)])
def test_attention_around_the_kernels_row_limits(paged, cache, act, hq, hkv, dim, new):
    """16 to 36 rows a cache head, where calls change kernels."""
    s = Setup(cache, act, hq, hkv, dim, 24, [new, 700, 2 * new + 1, 64], [new, new, new - 1, 1], seed=new)
    compare(s, s.attend(paged), act)


@pytest.mark.parametrize("cache,act", [("f32", "f32"), ("bf16", "bf16"), ("i8", "f32")])
@pytest.mark.parametrize("seqs,new", [(32, 1), (33, 1), (129, 3), (600, 1), (600, 2), (40, 50)])
def test_attention_of_many_sequences(paged, cache, act, seqs, new):
    lens = [(37 * i) % 150 for i in range(seqs)]
    s = Setup(cache, act, 4, 2, 64, 8, lens, [min(new, n) for n in lens], seed=seqs)
    compare(s, s.attend(paged), act)


@pytest.mark.parametrize("new", [1, 40])
def test_offsets_beyond_32_bits(paged, new):
    """The same sequences on pages at both ends of a cache of more than 2^32 bytes and elements a side."""
    page, heads, dim, n_pages = 64, 8, 128, 70000
    assert n_pages * page * heads * dim > 2 ** 32
    big = {x: torch.empty(n_pages, page, heads, dim, dtype=torch.int8, device="cuda") for x in "kv"}
    scale = {x: torch.empty(n_pages, page, heads, device="cuda") for x in "kv"}
    s = Setup("i8", "f32", 16, heads, dim, page, [300, 1000], [new, new])
    used = s.pages["k"].shape[0]
    move = torch.arange(used, device="cuda")
    move[1::2] = n_pages - move[1::2]
    for x in "kv":
        big[x][move], scale[x][move] = s.pages[x], s.scale[x]
    table = move[s.table.long()].to(torch.int32)
    near = s.attend(paged)
    far = paged.paged_attention(s.q, big["k"], big["v"], table, s.lens_t, s.cu, k_scale=scale["k"], v_scale=scale["v"])
    assert torch.equal(near, far)
    slots = torch.tensor([n_pages * page - 1, 3 * page + 1], device="cuda")
    k, v = (torch.randn(2, heads, dim, device="cuda") for _ in "kv")
    paged.kv_write(k, v, big["k"], big["v"], slots, k_scale=scale["k"], v_scale=scale["v"])
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    last = torch.tensor([[n_pages - 1]], dtype=torch.int32, device="cuda")
    start = torch.tensor([page - 1], dtype=torch.int32, device="cuda")
    got = paged.kv_read(big["k"], big["v"], last, start, cu, 1, k_scale=scale["k"], v_scale=scale["v"])
    for x, y in zip((k, v), got):
        # half a code of scale, and the products' roundings
        assert ((x[0] - y[0]).abs() <= x[0].abs().amax(-1, keepdim=True) / 127 * (0.5 + 2.0 ** -14)).all()
    paged.check_stream()


def settle_row(row, u):
    """The token for each u from one row's weights, whole numbers up to 2^63."""
    m = np.floor(np.clip(row.astype(np.float64), 0, 1) * 2.0 ** 40).astype(np.int64)
    c = np.cumsum(m)
    return [int(np.searchsorted(c, (int(np.floor(float(x) * 2.0 ** 24)) * int(c[-1])) >> 24, side="right")) for x in u]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("B,V,off", [(160, 1200001, 3), (80, 40000, 5), (1, 4194304, 1), (40, 16384, 7), (3, 6, 2), (160, 21, 1)])
def test_verify_long_rows_at_any_alignment(paged, act, B, V, off):
    g = gen(14)
    logits = torch.randn(V + 8, generator=g, device="cuda")
    row = torch.softmax(3 * logits, 0).to(ACT[act])[off:off + V]
    u = torch.rand(B, generator=g, device="cuda")
    none = torch.zeros(B, 0, device="cuda")
    got, acc = paged.verify_draft(row.expand(B, 1, V), None, none.to(torch.int32), none, u)
    assert (acc == 0).all() and got[:, 0].tolist() == settle_row(row.float().cpu().numpy(), u.cpu().numpy())
    # a refused draft whose distribution is the target's own, at another alignment: nothing is left of the
    # difference, and the target's row is read in a second pass
    other = torch.empty(V + 16, dtype=ACT[act], device="cuda")[off + 5:off + 5 + V].copy_(row)
    x = torch.zeros(B, 1, dtype=torch.int32, device="cuda")
    got, acc = paged.verify_draft(row.expand(B, 2, V), other.expand(B, 1, V), x, torch.ones(B, 1, device="cuda"), u)
    assert (acc == 0).all() and got[:, 0].tolist() == settle_row(row.float().cpu().numpy(), u.cpu().numpy())
    paged.check_stream()


@pytest.mark.parametrize("heads,dim,page,lens,start", [(1, 16, 5, [1, 0, 70, 3], None), (3, 16, 7, [40] * 50, 3),
                                                       (40, 128, 16, [5, 33], 2), (5, 80, 1, [129, 1, 2], 1)])
@pytest.mark.parametrize("cache,act", [("f32", "bf16"), ("bf16", "f32"), ("i8", "f32"), ("f8", "bf16")])
def test_read_shapes(paged, cache, act, heads, dim, page, lens, start):
    s = Setup(cache, act, heads, heads, dim, page, [n + (start or 0) for n in lens], lens)
    at = None if start is None else torch.full((len(lens),), start, dtype=torch.int32, device="cuda")
    got = paged.kv_read(s.pages["k"], s.pages["v"], s.table, at, s.cu, sum(lens), dtype=ACT[act], **s.kw())
    for x, y in zip("kv", got):
        pages = s.pages[x].float() if s.scale[x] is None else s.pages[x].float() * s.scale[x][..., None]
        want = torch.cat([pages[s.table[b].long()].flatten(0, 1)[start or 0:][:n] for b, n in enumerate(lens)])
        assert torch.equal(y, want.to(ACT[act]))
    paged.check_stream()
