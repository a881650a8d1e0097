"""The serving operators over a paged key/value cache, as workloads.

Four operators that a decoder needs around its planned graph once it generates text:

* ``kv_write``         -- store the keys and values of new tokens in the pages of a cache, quantised
                          to 8 bits per token and head where the cache holds 8 bits;
* ``kv_read``          -- read ranges of positions back out of the pages as dense rows;
* ``paged_attention``  -- attention of a chunk of new tokens (one token, a drafted run, a piece of a
                          prompt) over all cached positions of its sequence;
* ``verify_draft``     -- accept or reject drafted tokens against the target's probabilities and
                          sample the token that follows, from given random numbers.

``run`` computes them in plain torch operations, or with ``own`` through the package's entry points.
"""
import math
import random

import torch

own = False

ACT = {"f32": torch.float32, "bf16": torch.bfloat16}
CACHE = {"f32": torch.float32, "bf16": torch.bfloat16, "f8": torch.float8_e4m3fn, "i8": torch.int8}
BYTES = {"f32": 4, "bf16": 2, "f8": 1, "i8": 1}
QMAX = {"f8": 448.0, "i8": 127.0}   # largest code of the 8-bit formats
TINY = 2.0 ** -100                  # a token whose largest magnitude is below this is stored as zeros
ONE = 1 << 40                       # fixed-point unit of the sampling weights


# ------------------------------------------------------------------ the cases
def _cache_case(name, op, act, cache, heads, dim, page, seqs, longest, new):
    return {"name": name, "op": op, "act": act, "cache": cache, "heads": heads, "dim": dim, "page": page,
            "seqs": seqs, "longest": longest, "new": new}


def _attn_case(name, act, cache, q_heads, heads, dim, page, seqs, longest, new, ragged=False, window=0):
    return {"name": name, "op": "attention", "act": act, "cache": cache, "q_heads": q_heads, "heads": heads,
            "dim": dim, "page": page, "seqs": seqs, "longest": longest, "new": new, "ragged": ragged,
            "window": window}


def _verify_case(name, probs, seqs, drafts, vocab, greedy_draft=False):
    return {"name": name, "op": "verify", "probs": probs, "seqs": seqs, "drafts": drafts, "vocab": vocab,
            "greedy_draft": greedy_draft}


def listed():
    return [
        # a decode step of a small batch appends one token per sequence: pure latency
        _cache_case("append_token_i8", "write", "f32", "i8", 12, 64, 16, 8, 500, 1),
        # four prompts' keys and values enter an 8-bit floating-point cache at once
        _cache_case("append_prompts_f8", "write", "bf16", "f8", 8, 128, 64, 4, 6000, 4096),
        # a short shared prefix is taken out of the cache
        _cache_case("read_prefix_i8", "read", "bf16", "i8", 12, 64, 16, 1, 100, 100),
        # a batch of long sequences is read back, for another device or another engine
        _cache_case("read_batch_f8", "read", "f32", "f8", 8, 128, 24, 12, 8192, 8192),
        # one user, one token, a short context, full precision: the smallest call
        _attn_case("decode_one_f32", "f32", "f32", 12, 12, 64, 16, 1, 200, 1),
        # a batch decodes one token each, contexts of every length, 8-bit integers
        _attn_case("decode_batch_i8", "f32", "i8", 16, 8, 128, 16, 64, 8192, 1),
        # two very long documents: few rows, a long axis
        _attn_case("decode_long_bf16", "bf16", "bf16", 16, 8, 128, 128, 2, 131072, 1),
        # four drafted tokens and the one before them, checked in one pass of the target
        _attn_case("drafted_run_f8", "bf16", "f8", 32, 8, 128, 32, 32, 4096, 5),
        # a piece of a long prompt over what came before it
        _attn_case("prompt_chunk_bf16", "bf16", "bf16", 16, 8, 128, 64, 1, 16384, 4096),
        # a mixed step: prompts' pieces and single tokens together, odd pages, fp32 activations
        _attn_case("mixed_step_i8", "f32", "i8", 12, 12, 64, 24, 9, 8000, 1400, True),
        # one sequence's drafted tokens
        _verify_case("verify_one", "f32", 1, 4, 32000),
        # a batch's drafted tokens over a large vocabulary of odd size
        _verify_case("verify_batch", "f32", 128, 7, 131071),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "attention", "attention", "attention", "verify"])
    if kind == "verify":
        seqs, vocab = _log(rng, 1, 128), _log(rng, 1000, 131071)
        return _nameless(_verify_case("", rng.choice(["f32", "bf16"]), seqs, rng.randint(1, 7), vocab,
                                      rng.random() < 0.3))
    act, cache = rng.choice(["f32", "bf16"]), rng.choice(["f32", "bf16", "f8", "i8"])
    dim, page = rng.choice([64, 128]), rng.choice([16, 24, 32, 64, 128])
    heads, group = rng.choice([4, 8, 12]), rng.choice([1, 2, 4])
    if kind in ("write", "read"):
        cache = rng.choice(["f8", "i8"])
        new = _log(rng, 1, 4096)
        return _nameless(_cache_case("", kind, act, cache, heads, dim, page, _log(rng, 1, 12), new + _log(rng, 1, 4000), new))
    form = rng.choice(["token", "run", "chunk"])
    window = rng.choice([0, 0, 0, 1000])
    if form == "token":     # single tokens: at most a quarter of a million cached positions in all
        longest = _log(rng, 16, 131072)
        seqs = _log(rng, 1, max(1, min(256, 262144 // longest)))
        return _nameless(_attn_case("", act, cache, heads * group, heads, dim, page, seqs, longest, 1, False, window))
    if form == "run":
        longest = _log(rng, 64, 8192)
        seqs = _log(rng, 1, max(1, min(64, 131072 // longest)))
        return _nameless(_attn_case("", act, cache, heads * group, heads, dim, page, seqs, longest,
                                    rng.randint(2, 9), False, window))
    new = _log(rng, 100, 2048)
    longest = new + _log(rng, 1, 6000)
    return _nameless(_attn_case("", act, cache, heads, max(1, heads // group), dim, page, rng.randint(1, 3), longest,
                                new, rng.random() < 0.5, window))


def _nameless(case):
    return {k: v for k, v in case.items() if k != "name"}


def _lengths(case):
    """(cached positions, new tokens) of each sequence; the cached positions include the new tokens."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["longest"], case["new"]))
    lens, new = [], []
    for b in range(case["seqs"]):
        n = case["new"]
        if case.get("ragged") and b:   # mixed steps: some sequences bring one token, others part of a chunk
            n = 1 if b % 3 == 0 else rng.randint(1, n)
        elif case["op"] in ("write", "read") and b:
            n = rng.randint((n + 1) // 2, n)
        lens.append(case["longest"] if b == 0 else rng.randint(n, case["longest"]))
        new.append(n)
    return lens, new


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    if case["op"] == "verify":
        return _prepare_verify(case, g, dev)
    lens, new = _lengths(case)
    page, heads, dim, act = case["page"], case["heads"], case["dim"], ACT[case["act"]]
    pages = [-(-n // page) for n in lens]
    n_pages = sum(pages) + 3                      # a few pages belong to nobody
    perm = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    first = [0]
    for n in pages:
        first.append(first[-1] + n)
    host_row = torch.zeros(len(lens), max(pages), dtype=torch.int64)
    for b, n in enumerate(pages):                 # rows past a sequence's last page keep page 0
        host_row[b, :n] = torch.arange(first[b], first[b] + n)
    table = perm[host_row.to(dev)].contiguous()
    s = {"case": case, "table": table, "max_kv": max(lens), "max_new": max(new), "total": sum(new),
         "lens": torch.tensor(lens, dtype=torch.int32, device=dev),
         "cu": torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)}
    shape = (n_pages, page, heads, dim)
    for x in ("k", "v"):
        s[x + "_pages"], s[x + "_scale"] = _pool(shape, case["cache"], g, dev)
    q_heads = case.get("q_heads", 0)
    # the projections' output: queries, keys and values of a token side by side, as a model has them
    qkv = torch.randn(s["total"], q_heads + 2 * heads, dim, generator=g, device=dev).to(act)
    s["q"], s["k"], s["v"] = qkv[:, :q_heads], qkv[:, q_heads:q_heads + heads], qkv[:, q_heads + heads:]
    if case["op"] == "attention":
        return s
    # the new tokens are the last positions of their sequences
    start = s["lens"] - (s["cu"][1:] - s["cu"][:-1])
    owner = torch.repeat_interleave(torch.arange(len(new), device=dev), torch.tensor(new, device=dev))
    pos = start[owner].long() + torch.arange(s["total"], device=dev) - s["cu"][owner].long()
    s["start"] = start
    s["slots"] = table[owner, pos // page].long() * page + pos % page
    return s


def _pool(shape, cache, g, dev):
    """A cache that has been written: unit-variance values, quantised per token and head for 8 bits."""
    if cache in ("f32", "bf16"):
        return torch.randn(shape, generator=g, device=dev).to(CACHE[cache]), None
    codes = torch.empty(shape, dtype=CACHE[cache], device=dev)
    scale = torch.empty(shape[:3], dtype=torch.float32, device=dev)
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for i in range(0, shape[0], step):
        n = min(step, shape[0] - i)
        codes[i:i + n], scale[i:i + n] = _quantise(torch.randn((n,) + shape[1:], generator=g, device=dev), cache)
    return codes, scale


def _prepare_verify(case, g, dev):
    B, N, V = case["seqs"], case["drafts"], case["vocab"]
    dt = ACT[case["probs"]]

    def rows(n, base=None):
        out = torch.empty(B, n, V, dtype=dt, device=dev)
        for b in range(B):   # peaked, as a trained model's are; the draft's are near the target's
            z = torch.randn(n, V, generator=g, device=dev)
            z = 4.0 * z if base is None else base[b, :n].float().clamp_min(1e-30).log() + 0.7 * z
            out[b] = torch.softmax(z, -1).to(dt)
        return out

    target = rows(N + 1)
    draft = rows(N, target)
    pick = torch.multinomial(draft.view(B * N, V).float().clamp_min(0), 1, generator=g).view(B, N)
    return {"case": case, "target": target, "draft": None if case["greedy_draft"] else draft,
            "tokens": pick.to(torch.int32), "accept_u": torch.rand(B, N, generator=g, device=dev),
            "sample_u": torch.rand(B, generator=g, device=dev)}


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    with torch.no_grad():
        if op == "verify":
            return _plain_verify(state)
        if op == "attention":
            return {"out": _plain_attention(state)}
        if op == "write":
            _plain_write(state)
        return _plain_read(state)


def _own(s, op):
    from __graft_entry__ import load_package
    load_package()
    from lbr_b200 import paged
    if op == "verify":
        tokens, accepted = paged.verify_draft(s["target"], s["draft"], s["tokens"], s["accept_u"], s["sample_u"])
        return {"tokens": tokens, "accepted": accepted}
    if op == "attention":
        return {"out": paged.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cu"],
                                             k_scale=s["k_scale"], v_scale=s["v_scale"],
                                             window=s["case"]["window"], max_new=s["max_new"], max_kv=s["max_kv"])}
    if op == "write":
        paged.kv_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"],
                       k_scale=s["k_scale"], v_scale=s["v_scale"])
    k, v = paged.kv_read(s["k_pages"], s["v_pages"], s["table"], s["start"], s["cu"], s["total"],
                         k_scale=s["k_scale"], v_scale=s["v_scale"], dtype=s["k"].dtype)
    return {"k": k, "v": v}


def _quantise(x, cache):
    """Codes and one scale per token and head: scale = largest magnitude / largest code."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    some = top >= TINY
    inv = torch.where(some, QMAX[cache] / top, torch.zeros_like(top))
    code = x * inv
    code = code.round() if cache == "i8" else code.clamp(-448.0, 448.0)
    scale = torch.where(some, top / QMAX[cache], torch.zeros_like(top))
    return code.to(CACHE[cache]), scale.squeeze(-1)


def _plain_write(s):
    cache = s["case"]["cache"]
    for x in ("k", "v"):
        codes, scale = _quantise(s[x], cache)
        s[x + "_pages"].view(torch.int8).flatten(0, 1)[s["slots"]] = codes.view(torch.int8)
        s[x + "_scale"].flatten(0, 1)[s["slots"]] = scale


def _plain_read(s):
    page = s["case"]["page"]
    rows = torch.arange(s["total"], device=s["cu"].device)
    owner = torch.searchsorted(s["cu"][1:].long(), rows, right=True)
    pos = s["start"][owner].long() + rows - s["cu"][owner].long()
    slot = s["table"][owner, pos // page].long() * page + pos % page
    out = {}
    for x in ("k", "v"):
        codes = s[x + "_pages"].view(torch.int8).flatten(0, 1)[slot].view(CACHE[s["case"]["cache"]]).float()
        out[x] = (codes * s[x + "_scale"].flatten(0, 1)[slot][..., None]).to(s["k"].dtype)
    return out


def _plain_attention(s):
    c = s["case"]
    dev, page, heads, dim = s["cu"].device, c["page"], c["heads"], c["dim"]
    lens, cu, L, Q = s["lens"].long(), s["cu"].long(), s["max_kv"], s["max_new"]
    B, group = lens.numel(), c["q_heads"] // heads
    pos = torch.arange(L, device=dev)
    where = s["table"][:, pos // page].long() * page + pos % page                       # [B, L]
    there = (pos < lens[:, None])[:, :, None, None]

    def dense(x):
        y = s[x + "_pages"].flatten(0, 1)
        y = (y.view(torch.int8)[where].view(y.dtype) if y.element_size() == 1 else y[where]).float()
        if s[x + "_scale"] is not None:
            y = y * s[x + "_scale"].flatten(0, 1)[where][..., None]
        return torch.where(there, y, torch.zeros((), device=dev)).permute(0, 2, 1, 3)   # [B, heads, L, dim]

    new = cu[1:] - cu[:-1]
    i = torch.arange(Q, device=dev)
    row = (cu[:-1, None] + i).clamp_max(s["total"] - 1)                                  # [B, Q]
    q = s["q"][row].float().view(B, Q, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(B, heads, group * Q, dim)
    score = torch.matmul(q, dense("k").transpose(-1, -2)).view(B, heads, group, Q, L) / math.sqrt(dim)
    at = (lens - new)[:, None] + i                                                       # a query's own position
    seen = pos <= at[..., None]
    if c["window"]:
        seen = seen & (pos > at[..., None] - c["window"])
    seen = seen[:, None, None]
    score = score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, heads, group * Q, L), dense("v")).view(B, heads, group, Q, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out)).permute(0, 3, 1, 2, 4).reshape(B, Q, -1)
    # back to the packed rows
    rows = torch.arange(s["total"], device=dev)
    owner = torch.searchsorted(cu[1:], rows, right=True)
    return out[owner, rows - cu[owner]].view(s["total"], c["q_heads"], dim).to(s["q"].dtype)


def _plain_verify(s):
    p, u, x = s["target"], s["accept_u"], s["tokens"].long()
    B, N = x.shape
    V = p.shape[-1]
    px = p[:, :N].gather(-1, x[..., None]).squeeze(-1).float()
    qx = torch.ones_like(px) if s["draft"] is None else s["draft"].gather(-1, x[..., None]).squeeze(-1).float()
    n = (u * qx < px).long().cumprod(-1).sum(-1)                                         # accepted before the first refusal
    b = torch.arange(B, device=x.device)
    row = p[b, n].float()
    at = n.clamp_max(N - 1)
    if s["draft"] is None:
        q = torch.zeros_like(row).scatter_(-1, x[b, at][:, None], 1.0)
    else:
        q = s["draft"][b, at].float()
    w = torch.where((n < N)[:, None], (row - q).clamp_min(0.0), row)
    total, cum = _mass(w)
    _, cum_row = _mass(row)                                                              # nothing left: the target's own
    cum = torch.where(total[:, None] > 0, cum, cum_row)
    total = cum[:, -1]
    m = (s["sample_u"] * float(1 << 24)).long().clamp(0, (1 << 24) - 1)
    t = m * (total >> 24) + ((m * (total & ((1 << 24) - 1))) >> 24)                      # floor(u * total)
    token = (cum <= t[:, None]).sum(-1)
    token = torch.where(total > 0, token, torch.full_like(token, -1))
    i = torch.arange(N + 1, device=x.device)
    padded = torch.cat([x, torch.zeros_like(x[:, :1])], -1)
    tokens = torch.where(i < n[:, None], padded, torch.where(i == n[:, None], token[:, None], torch.full_like(padded, -1)))
    return {"tokens": tokens.to(torch.int32), "accepted": n.to(torch.int32)}


def _mass(w):
    """Sampling weights in fixed point, so that their sums do not depend on an order."""
    cum = (w.clamp_max(1.0) * float(ONE)).long().cumsum(-1)
    return cum[:, -1], cum


# ------------------------------------------------------------------ floors
def work(case):
    if case["op"] == "verify":
        B, N, V, e = case["seqs"], case["drafts"], case["vocab"], BYTES[case["probs"]]
        rows = 1 if case["greedy_draft"] else 2      # the row where a sequence stops; a gathered value per draft
        return {"bytes": B * (rows * V * e + N * (2 * e + 8) + 4 + 4 * (N + 2)), "flops": B * V * 3}
    lens, new = _lengths(case)
    heads, dim, a, c = case["heads"], case["dim"], BYTES[case["act"]], BYTES[case["cache"]]
    row = 2 * heads * (dim * c + (4 if c == 1 else 0))        # one cached position: keys, values and their scales
    if case["op"] == "write":
        return {"bytes": sum(new) * (2 * heads * dim * a * 2 + 2 * row + 8), "flops": sum(new) * heads * dim * 8}
    if case["op"] == "read":
        return {"bytes": sum(new) * (row + 2 * heads * dim * a), "flops": sum(new) * heads * dim * 2}
    w = case["window"]
    touched = pairs = 0
    for n, m in zip(lens, new):
        touched += min(n, w + m - 1) if w else n
        for i in range(n - m + 1, n + 1):
            pairs += min(i, w) if w else i
    return {"bytes": touched * row + 2 * sum(new) * case["q_heads"] * dim * a + 4 * sum(-(-n // case["page"]) for n in lens),
            "flops": 4 * dim * case["q_heads"] * pairs}


# ------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "verify":
        return None     # whole numbers
    page, lens, new = case["page"], *_lengths(case)
    cu, table = s["cu"].tolist(), s["table"].long()
    if case["op"] == "attention":
        out = torch.zeros(s["total"], case["q_heads"], case["dim"], dtype=torch.float64, device=table.device)
        group = case["q_heads"] // case["heads"]
        for b, (n, m) in enumerate(zip(lens, new)):
            pos = torch.arange(n, device=table.device)
            pg, off = table[b, pos // page], pos % page
            at = torch.arange(n - m, n, device=table.device)[:, None]
            seen = pos <= at
            if case["window"]:
                seen &= pos > at - case["window"]
            for h in range(case["heads"]):
                k, v = (_value(s, x, pg, off, h) for x in ("k", "v"))
                for j in range(h * group, (h + 1) * group):
                    z = s["q"][cu[b]:cu[b + 1], j].double() @ k.T / math.sqrt(case["dim"])
                    out[cu[b]:cu[b + 1], j] = torch.softmax(z.masked_fill(~seen, -math.inf), -1) @ v
        return {"out": out}
    out = {}
    for x in ("k", "v"):
        if case["op"] == "write":     # each value to the nearest code of its token and head
            y = s[x].double()
            step = y.abs().amax(-1, keepdim=True) / QMAX[case["cache"]]
            z = y / step
            if case["cache"] == "i8":
                z = z.round()
            else:                     # 3 bits below the leading one, none below 2^-9
                e = torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6)))
                z = torch.round(z / 2.0 ** (e - 3)) * 2.0 ** (e - 3)
            out[x] = z * step
            continue
        got = []
        for b, (n, m) in enumerate(zip(lens, new)):
            pos = torch.arange(n - m, n, device=table.device)
            got.append(_value(s, x, table[b, pos // page], pos % page, slice(None)))
        out[x] = torch.cat(got)
    return out


def _value(s, x, pg, off, h):
    """What the cache stands for at (page, offset, head), in 64 bits."""
    codes = s[x + "_pages"]
    y = (codes.view(torch.int8)[pg, off][:, h].view(codes.dtype) if codes.element_size() == 1 else codes[pg, off][:, h]).double()
    return y if s[x + "_scale"] is None else y * s[x + "_scale"][pg, off][:, h].double()[..., None]
