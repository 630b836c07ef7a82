"""The operators that serve a grouped-head stack over an 8-bit paged cache, as measurable cases.

One decoder layer's way through a call, one operator a case:

  tables    page tables, slots and positions of a call's rows from the sequences' lengths (`kv_tables`)
  rope      per-head norm and rotary embedding of the rows' q and k (`qk_norm_rope`)
  append    K and V rows into 8-bit pages with one scale per page, head and K or V (`kv8_append`)
  prompt    causal attention over whole prompts packed one behind the other (`packed_attend`)
  attend8   one query row a sequence against the 8-bit pages (`kv8_attend`)

Pages hold 16 tokens: kv[page][kv head][K | V][16][d] in E4M3, scales[page][kv head][K | V] in f32, powers of two.
A page's scale is the smallest 2^e, e >= -100, whose 448 * 2^e holds the largest finite magnitude that was put into the page.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

PAGE = 16
E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -100
EPS, THETA = 1e-6, 1e6

# (query heads, kv heads, head dimension): the talker's stack, the Higgs body's, narrow heads in large groups, one kv head, no groups
HEADS = [(16, 8, 128), (32, 8, 128), (20, 4, 64), (14, 2, 64), (5, 1, 128), (16, 1, 128), (4, 4, 128), (4, 4, 64)]


# ---- cases ---------------------------------------------------------------------------------------------------------

def _heads(hq, hk, d):
    return {"hq": hq, "hk": hk, "d": d}


def listed():
    return [
        # a decode step of the headline batch: every sequence grows by a token
        {"name": "tables-step-64", "kind": "tables", "n": 64, "ctx_min": 128, "ctx_max": 1000, "fresh": 0, "prompt_min": 0, "prompt_max": 0, "done": 0},
        # a full server with long contexts: most sequences step, some end, new ones bring their prompts
        {"name": "tables-mixed-1000", "kind": "tables", "n": 1000, "ctx_min": 16, "ctx_max": 8000, "fresh": 60, "prompt_min": 32, "prompt_max": 512, "done": 50},
        # the rows of a decode step, and of a full start call (8192 prompt tokens)
        {"name": "rope-step-64", "kind": "rope", "rows": 64, "far": 4096, **_heads(16, 8, 128)},
        {"name": "rope-start-8192", "kind": "rope", "rows": 8192, "far": 32768, **_heads(32, 8, 128)},
        # an odd number of sessions, a token each, somewhere in their last page
        {"name": "append-step-61", "kind": "append", "n": 61, "ctx_min": 100, "ctx_max": 2000, "add_min": 1, "add_max": 1, **_heads(16, 8, 128)},
        # a burst of prompts that fills a start call
        {"name": "append-start-28", "kind": "append", "n": 28, "ctx_min": 0, "ctx_max": 0, "add_min": 32, "add_max": 512, **_heads(16, 8, 128)},
        # one new request (time to first audio), a burst of them, and one long document
        {"name": "prompt-1-77", "kind": "prompt", "n": 1, "len_min": 77, "len_max": 77, "pad": 0, **_heads(16, 8, 128)},
        {"name": "prompt-28-ragged", "kind": "prompt", "n": 28, "len_min": 32, "len_max": 512, "pad": 19, **_heads(16, 8, 128)},
        {"name": "prompt-1-8192", "kind": "prompt", "n": 1, "len_min": 8192, "len_max": 8192, "pad": 0, **_heads(32, 8, 128)},
        # one speaker, a full server, and a few very long contexts over narrow heads
        {"name": "attend8-step-1", "kind": "attend8", "n": 1, "ctx_min": 777, "ctx_max": 777, **_heads(16, 8, 128)},
        {"name": "attend8-step-128", "kind": "attend8", "n": 128, "ctx_min": 500, "ctx_max": 8000, **_heads(16, 8, 128)},
        {"name": "attend8-long-9", "kind": "attend8", "n": 9, "ctx_min": 2000, "ctx_max": 60000, **_heads(20, 4, 64)},
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables"] * 2 + ["rope"] * 2 + ["append"] * 3 + ["prompt"] * 4 + ["attend8"] * 5)
    if kind == "tables":
        n = _spread(rng, 1, 1000)
        hi = _spread(rng, 16, 8000)
        fresh = rng.randint(0, n // 8)
        lo = _spread(rng, 1, 64)
        return {"kind": kind, "n": n, "ctx_min": rng.randint(1, hi), "ctx_max": hi, "fresh": fresh, "prompt_min": lo if fresh else 0,
                "prompt_max": _spread(rng, lo, 512) if fresh else 0, "done": rng.randint(0, n // 8)}
    heads = rng.choice(HEADS)
    if kind == "rope":
        return {"kind": kind, "rows": _spread(rng, 1, 8192), "far": _spread(rng, 16, 1 << 20), **_heads(*heads)}
    if kind == "append":
        if rng.random() < 0.5:  # a decode step
            hi = _spread(rng, 1, 4000)
            return {"kind": kind, "n": _spread(rng, 1, 256), "ctx_min": rng.randint(0, hi), "ctx_max": hi, "add_min": 1, "add_max": 1, **_heads(*heads)}
        hi = _spread(rng, 2, 2048)  # prompts, or pieces of them behind what is there
        ctx = rng.choice([0, 0, rng.randint(1, 1000)])
        return {"kind": kind, "n": _spread(rng, 1, max(1, 7600 // hi)), "ctx_min": ctx, "ctx_max": ctx, "add_min": rng.randint(1, hi), "add_max": hi, **_heads(*heads)}
    if kind == "prompt":
        if rng.random() < 0.4:  # one prompt
            n = _spread(rng, 1, 8192)
            return {"kind": kind, "n": 1, "len_min": n, "len_max": n, "pad": rng.randint(0, 20), **_heads(*heads)}
        hi = _spread(rng, 4, 1024)
        return {"kind": kind, "n": _spread(rng, 2, max(2, min(64, 8192 // hi))), "len_min": rng.randint(0, hi), "len_max": hi, "pad": rng.randint(0, 20), **_heads(*heads)}
    hi = _spread(rng, 1, 60000)
    most = max(1, min(256, 128 * 8000 * 8 * 128 // (hi * heads[1] * heads[2]), 128 * 8000 * 2 // hi))
    return {"kind": kind, "n": _spread(rng, 1, most), "ctx_min": rng.randint(0, hi), "ctx_max": hi, **_heads(*heads)}


def _even(n, lo, hi):
    """n lengths evenly over [lo, hi]."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _requests(case):
    """(tokens in the cache, tokens to come) of a tables case's sequences; -1 to come: the sequence has ended."""
    ended = _even(case["done"], case["ctx_min"], case["ctx_max"])
    begun = _even(case["fresh"], case["prompt_min"], case["prompt_max"])
    rest = _even(case["n"] - len(ended) - len(begun), case["ctx_min"], case["ctx_max"])
    return [(c, -1) for c in ended] + [(0, p) for p in begun] + [(c, 1) for c in rest]


def _pages(tokens):
    return -(-tokens // PAGE)


def work(case):
    kind = case["kind"]
    if kind == "tables":
        seqs = _requests(case)
        kept = sum(_pages(c) for c, a in seqs if a >= 0)
        total = sum(_pages(c + a) for c, a in seqs if a >= 0)
        rows = sum(max(0, a) for _, a in seqs)
        # lengths in and out, additions and both prefix arrays; kept pages read, all pages written; new ones read and put into the table; a row's three words
        return {"bytes": 4 * (5 * len(seqs) + kept + total + 2 * (total - kept) + 3 * rows), "flops": 0}
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if kind == "rope":
        elems = case["rows"] * (hq + hk) * d
        return {"bytes": 4 * elems + 4 * case["rows"] + 4 * d, "flops": 7 * elems}
    if kind == "append":
        adds, ctx = _even(case["n"], case["add_min"], case["add_max"]), _even(case["n"], case["ctx_min"], case["ctx_max"])
        rows = sum(adds)
        touched = sum(_pages(c + a) - c // PAGE for c, a in zip(ctx, adds) if a)
        return {"bytes": 3 * 2 * rows * hk * d + 4 * rows + 8 * touched * hk, "flops": 2 * 2 * rows * hk * d}
    if kind == "prompt":
        lens = _even(case["n"], case["len_min"], case["len_max"])
        return {"bytes": 2 * sum(lens) * (2 * hq + 2 * hk) * d, "flops": 2 * d * hq * sum(t * (t + 1) for t in lens)}
    lens = _even(case["n"], case["ctx_min"], case["ctx_max"])
    return {"bytes": sum(lens) * 2 * hk * d + sum(_pages(t) for t in lens) * (8 * hk + 4) + 2 * 2 * case["n"] * hq * d, "flops": 4 * d * hq * sum(lens)}


# ---- what a program has in hand before the call ----------------------------------------------------------------------

def _rows(gen, rows, heads, d):
    """Rows of heads as projections give them: a few channels of a head are much larger than the others."""
    x = torch.randn(rows, heads, d, generator=gen, device="cuda")
    loud = torch.rand(heads, d, generator=gen, device="cuda")
    return (x * (0.5 + 4.0 * (loud > 0.97) + 0.5 * loud)).reshape(rows, heads * d).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = random.Random(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    empty = lambda *shape: torch.full(shape, -1, dtype=torch.int32, device="cuda")  # noqa: E731
    kind = case["kind"]
    st = {"kind": kind, **{k: case[k] for k in ("hq", "hk", "d") if k in case}}
    if kind == "tables":
        seqs = _requests(case)
        rng.shuffle(seqs)
        n, width = len(seqs), _pages(max(c + max(0, a) for c, a in seqs)) + 1
        held, total = [_pages(c) for c, _ in seqs], [_pages(c + a) if a >= 0 else 0 for c, a in seqs]
        spare = sum(max(0, t - h) for t, h in zip(total, held)) + 64
        ids = torch.randperm(sum(held) + spare, generator=gen, device="cuda").to(torch.int32)
        table = empty(n, width)
        table[torch.arange(width, device="cuda")[None] < ints(held)[:, None]] = ids[:sum(held)]
        free = empty(ids.numel())
        free[:spare] = ids[sum(held):]
        rows = sum(max(0, a) for _, a in seqs)
        st |= {"lens": ints([c for c, _ in seqs]), "add": ints([a for _, a in seqs]), "table": table, "free": free, "count": ints([spare]),
               "lens_out": empty(n), "count_out": empty(1), "indptr": empty(n + 1), "pages": empty(sum(total) + 8), "row_ptr": empty(n + 1),
               "pos": empty(rows + 3), "slot": empty(rows + 3), "seq": empty(rows + 3), "status": empty(1)}
        return st
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if kind == "rope":
        rows = case["rows"]
        st |= {"qkv": _rows(gen, rows, hq + 2 * hk, d), "pos": torch.randint(0, case["far"], (rows,), generator=gen, device="cuda").to(torch.int32),
               "out": torch.zeros(rows, (hq + hk) * d, dtype=torch.bfloat16, device="cuda")}
        for name in ("q_norm", "k_norm"):
            st[name] = (1 + 0.3 * torch.randn(d, generator=gen, device="cuda")).to(torch.bfloat16)
        return st
    if kind == "prompt":
        lens = _even(case["n"], case["len_min"], case["len_max"])
        rng.shuffle(lens)
        rows = sum(lens) + case["pad"]
        qkv = _rows(gen, rows, hq + 2 * hk, d)
        st |= {"q": qkv[:, :hq * d], "k": qkv[:, hq * d:(hq + hk) * d], "v": qkv[:, (hq + hk) * d:], "most": max(lens),
               "row_ptr": ints([0] + list(np.cumsum(lens))), "out": torch.zeros(rows, hq * d, dtype=torch.bfloat16, device="cuda")}
        return st
    ctx = _even(case["n"], case["ctx_min"], case["ctx_max"])
    adds = _even(case["n"], case["add_min"], case["add_max"]) if kind == "append" else [0] * len(ctx)
    seqs = list(zip(ctx, adds))
    rng.shuffle(seqs)
    counts = [_pages(c + a) for c, a in seqs]
    total = sum(counts) + 5
    ids = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    indptr = np.concatenate([[0], np.cumsum(counts)])
    # what pages hold: E4M3 codes of normal values, under a scale for each page and head; a page that nobody wrote holds an earlier owner's
    kv = (torch.randn(total, hk, 2, PAGE, d, generator=gen, device="cuda") * 90).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.exp2(torch.randint(-8, -5, (total, hk, 2), generator=gen, device="cuda").float())
    st |= {"kv": kv, "scales": scales}
    if kind == "append":
        slots = []
        at = ids.tolist()
        for s, (c, a) in enumerate(seqs):
            slots += [at[indptr[s] + p // PAGE] * PAGE + p % PAGE for p in range(c, c + a)]
        kvrows = _rows(gen, len(slots), 2 * hk, d)
        return st | {"k": kvrows[:, :hk * d], "v": kvrows[:, hk * d:], "slot": ints(slots)}
    return st | {"q": _rows(gen, len(seqs), hq, d), "pos": ints([c - 1 for c, _ in seqs]), "indptr": ints(list(indptr)), "pages": ids[:total - 5].contiguous(),
                 "most": max(1, max(counts)), "out": torch.zeros(len(seqs), hq * d, dtype=torch.bfloat16, device="cuda")}


# ---- the operators -----------------------------------------------------------------------------------------------------

_contexts = {}  # device -> [its context, the stream that its calls run on]


def _ops():
    """The current device's context, on the stream that the program works on at the moment."""
    device = torch.cuda.current_device()
    if device not in _contexts:
        from pega_omni_b200.ops import Ops
        _contexts[device] = [Ops(device), None]
    context = _contexts[device]
    stream = torch._C._cuda_getCurrentRawStream(device)  # torch.cuda.current_stream() makes an object, which takes longer than some of the calls
    if context[1] != stream:
        context[0].stream(stream)
        context[1] = stream
    return context[0]


def run(st):
    kind = st["kind"]
    if kind == "tables":
        if own:
            _ops().kv_tables(st["lens"], st["add"], st["table"], st["free"], st["count"], st["lens_out"], st["count_out"], st["indptr"], st["pages"],
                             st["row_ptr"], st["pos"], st["slot"], st["seq"], st["status"])
            return {k: st[k] for k in ("lens_out", "count_out", "table", "free", "indptr", "pages", "row_ptr", "pos", "slot", "seq", "status")}
        return _plain_tables(st)
    hq, hk, d = st["hq"], st["hk"], st["d"]
    if kind == "rope":
        if own:
            _ops().qk_norm_rope(st["qkv"], st["q_norm"], st["k_norm"], st["pos"], hq, hk, d, EPS, THETA, st["out"])
            return st["out"]
        return _plain_rope(st)
    if kind == "append":
        if own:
            _ops().kv8_append(st["k"], st["v"], st["slot"], st["kv"], st["scales"])
        else:
            _plain_append(st)
        return {"kv": st["kv"].view(torch.float8_e4m3fn), "scales": st["scales"]}
    if kind == "prompt":
        if own:
            _ops().packed_attend(st["q"], st["k"], st["v"], st["row_ptr"], hq, hk, d, d ** -0.5, st["out"])
            return st["out"]
        return _plain_prompt(st)
    if own:
        _ops().kv8_attend(st["q"], st["kv"], st["scales"], st["pos"], st["indptr"], st["pages"], hq, d ** -0.5, st["out"])
        return st["out"]
    return _plain_attend8(st)


def _plain_tables(st):
    lens, add, table, free, count = (st[k].long() for k in ("lens", "add", "table", "free", "count"))
    n, width = table.shape
    dev = table.device
    prefix = lambda v: torch.cat([v.new_zeros(1), v.cumsum(0)])  # noqa: E731
    gone = add == -1
    held = (lens + PAGE - 1) // PAGE
    total = torch.where(gone, 0, lens + add)
    have = torch.where(gone, 0, held)
    want = (total + PAGE - 1) // PAGE
    back = prefix(torch.where(gone, held, 0))
    needed, indptr, row_ptr = prefix(want - have), prefix(want), prefix(add.clamp(min=0))
    # the stack of free pages: what was free, then what comes back, in order
    span = torch.arange(width, device=dev)[None]
    k = torch.arange(n * width, device=dev)
    owner = torch.searchsorted(back[1:], k, right=True).clamp(max=n - 1)
    returned = table[owner, (k - back[owner]).clamp(0, width - 1)]
    top = count + back[-1] - 1

    def stack(i):
        return torch.where(i < count, free[i.clamp(0, free.numel() - 1)], returned[(i - count).clamp(0, n * width - 1)])

    status = ((lens < 0) | (add < -1) | (total > width * PAGE)).any().int() + 2 * (needed[-1] > top + 1).int() + 4 * (row_ptr[-1] > st["pos"].numel()).int() \
        + 8 * (indptr[-1] > st["pages"].numel()).int() + 16 * ((count < 0) | (count > free.numel()) | (top + 1 - needed[-1] > free.numel()))[0].int()
    ok = status == 0
    new = torch.where((span >= have[:, None]) & (span < want[:, None]), stack(top - (needed[:-1, None] + span - have[:, None])), table)
    table_out = torch.where(ok, new, table)
    place = torch.arange(free.numel(), device=dev)
    free_out = torch.where(ok & (place >= count) & (place <= top - needed[-1]), stack(place), free)
    e = torch.arange(st["pages"].numel(), device=dev)
    s = torch.searchsorted(indptr[1:], e, right=True).clamp(max=n - 1)
    pages = torch.where(ok & (e < indptr[-1]), new[s, (e - indptr[s]).clamp(0, width - 1)], st["pages"].long())
    r = torch.arange(st["pos"].numel(), device=dev)
    s = torch.searchsorted(row_ptr[1:], r, right=True).clamp(max=n - 1)
    live = ok & (r < row_ptr[-1])
    pos = torch.where(live, lens[s] + r - row_ptr[s], -1)
    slot = torch.where(live, new[s, (pos // PAGE).clamp(0, width - 1)] * PAGE + pos % PAGE, -1)
    got = {"lens_out": torch.where(ok, total, lens), "count_out": torch.where(ok, top + 1 - needed[-1], count), "table": table_out, "free": free_out,
           "indptr": torch.where(ok, indptr, 0), "pages": pages, "row_ptr": torch.where(ok, row_ptr, 0), "pos": pos, "slot": slot,
           "seq": torch.where(live, s, -1), "status": status.reshape(1)}
    return {k: v.to(torch.int32) for k, v in got.items()}


def _plain_rope(st):
    hq, hk, d = st["hq"], st["hk"], st["d"]
    x = st["qkv"][:, :(hq + hk) * d].float().reshape(-1, hq + hk, d)
    gain = torch.cat([st["q_norm"].float().expand(hq, d), st["k_norm"].float().expand(hk, d)])
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gain
    angle = st["pos"].double()[:, None] * THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device=x.device) / d)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    lo, hi = x[..., :d // 2], x[..., d // 2:]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(torch.bfloat16).reshape(-1, (hq + hk) * d)


def _plain_append(st):
    hk, d = st["hk"], st["d"]
    kv, scales, slot = st["kv"].view(torch.float8_e4m3fn), st["scales"], st["slot"].long()
    x = torch.stack([st["k"].float().reshape(-1, hk, d), st["v"].float().reshape(-1, hk, d)], 2)  # [row, head, K | V, d]
    page, off = slot // PAGE, slot % PAGE
    before = torch.cat([slot.new_full((1,), -2), slot[:-1]])
    first = (off == 0) | (before + 1 != slot)  # the rows that begin a run of rows of one page
    run_of = first.long().cumsum(0) - 1
    begin = first.nonzero()[:, 0]
    at, held = page[begin], off[begin]  # a run's page, and the tokens that it holds already
    size = torch.where(x.isfinite(), x.abs(), 0).amax(-1)
    most = torch.zeros(begin.numel(), hk, 2, device=x.device).scatter_reduce(0, run_of[:, None, None].expand_as(size), size, "amax")
    part, exp = torch.frexp(most / E4M3_MAX)
    need = torch.where(most > 0, torch.ldexp(torch.ones_like(part), torch.where(part > 0.5, exp, exp - 1)), 0).clamp(min=MIN_SCALE)
    old = torch.where((held > 0)[:, None, None], scales[at], need)
    new = torch.maximum(old, need)
    block = kv.view(torch.uint8)[at].view(torch.float8_e4m3fn)
    moved = (block.float() * (old / new)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    keep = (torch.arange(PAGE, device=x.device) < held[:, None])[:, None, None, :, None] & (new > old)[..., None, None]
    kv.view(torch.uint8)[at] = torch.where(keep, moved, block.view(torch.uint8))
    kv.view(torch.uint8)[page, :, :, off] = (x / new[run_of][..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    scales[at] = new


def _plain_prompt(st):
    hq, hk, d, most = st["hq"], st["hk"], st["d"], st["most"]
    rows, out = st["q"].shape[0], st["out"]
    ptr = st["row_ptr"].long()
    if most == 0:
        return out
    t = torch.arange(most, device=out.device)
    live = t < (ptr[1:] - ptr[:-1])[:, None]  # [sequence, token]
    at = torch.where(live, ptr[:-1, None] + t, 0)
    heads = lambda x, h: (x.float()[at] * live[..., None]).reshape(-1, most, h, d).transpose(1, 2)  # noqa: E731
    q, k, v = heads(st["q"], hq).unflatten(1, (hk, hq // hk)), heads(st["k"], hk)[:, :, None], heads(st["v"], hk)[:, :, None]
    s = (q @ k.transpose(-1, -2)).mul_(d ** -0.5)
    s.masked_fill_(t > t[:, None], -math.inf)
    p = s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = (p @ v) / p.sum(-1, keepdim=True)
    o = o.flatten(1, 2).transpose(1, 2).reshape(-1, hq * d).to(torch.bfloat16)
    padded = torch.cat([out, out.new_zeros(1, hq * d)])
    padded[torch.where(live, at, rows).reshape(-1)] = o
    return padded[:rows]


def _plain_attend8(st):
    hq, hk, d = st["hq"], st["hk"], st["d"]
    n, ptr = st["q"].shape[0], st["indptr"].long()
    e = ptr[:-1, None] + torch.arange(st["most"], device=ptr.device)
    at = st["pages"].long()[e.clamp(max=max(0, st["pages"].numel() - 1))] if st["pages"].numel() else torch.zeros_like(e)
    live = torch.arange(st["most"] * PAGE, device=ptr.device) <= st["pos"][:, None]  # [row, token]
    blocks = st["kv"][at].view(torch.float8_e4m3fn).float() * st["scales"][at][..., None, None]  # [row, page, head, K | V, token, d]
    tokens = lambda i: blocks[:, :, :, i].transpose(1, 2).reshape(n, hk, -1, d)  # noqa: E731
    k, v = tokens(0), tokens(1) * live[:, None, :, None]
    s = (st["q"].float().reshape(n, hk, hq // hk, d) @ k.transpose(-1, -2)) * d ** -0.5
    s = s.masked_fill(~live[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total == 0, 1, total)
    return o.reshape(n, hq * d).to(torch.bfloat16)


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"tables": _exact_tables, "rope": _exact_rope, "append": _exact_append, "prompt": _exact_prompt, "attend8": _exact_attend8}[case["kind"]](st)


def _exact_tables(st):
    lens, add, table, free = (st[k].cpu().numpy().copy() for k in ("lens", "add", "table", "free"))
    stack = list(free[:int(st["count"])])
    for s in np.flatnonzero(add == -1):
        stack += list(table[s, :_pages(int(lens[s]))])
    indptr, row_ptr, pages, rows = [0], [0], [], []
    for s in range(len(lens)):
        total = 0 if add[s] == -1 else int(lens[s] + add[s])
        for i in range(_pages(int(lens[s])) if add[s] != -1 else 0, _pages(total)):
            table[s, i] = stack.pop()
        pages += list(table[s, :_pages(total)])
        rows += [(s, p, table[s, p // PAGE] * PAGE + p % PAGE) for p in range(int(lens[s]), total)]
        indptr.append(len(pages))
        row_ptr.append(len(rows))
        lens[s] = total
    free[:len(stack)] = np.where(np.arange(len(stack)) < int(st["count"]), free[:len(stack)], stack)
    given = st["pages"].cpu().numpy().copy()
    given[:len(pages)] = pages
    got = {"lens_out": lens, "count_out": [len(stack)], "table": table, "free": free, "indptr": indptr, "pages": given, "row_ptr": row_ptr, "status": [0]}
    for i, name in enumerate(("seq", "pos", "slot")):
        got[name] = [r[i] for r in rows] + [-1] * (st["pos"].numel() - len(rows))
    return {k: np.asarray(v, dtype=np.int32) for k, v in got.items()}


def _exact_rope(st):
    hq, hk, d = st["hq"], st["hk"], st["d"]
    x = st["qkv"].cpu().double().numpy()[:, :(hq + hk) * d].reshape(-1, hq + hk, d)
    x = x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + EPS)
    x[:, :hq] *= st["q_norm"].cpu().double().numpy()
    x[:, hq:] *= st["k_norm"].cpu().double().numpy()
    turn = np.exp(1j * st["pos"].cpu().double().numpy()[:, None] * np.power(THETA, -2.0 * np.arange(d // 2) / d))
    z = (x[..., :d // 2] + 1j * x[..., d // 2:]) * turn[:, None]
    return np.concatenate([z.real, z.imag], -1).reshape(-1, (hq + hk) * d)


def _e4m3(x):
    """The E4M3 value nearest to each x, ties to even, at most 448 in magnitude."""
    _, e = np.frexp(np.where(x == 0, 1.0, np.abs(x)))
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.clip(np.rint(x / step) * step, -E4M3_MAX, E4M3_MAX)


def _exact_append(st):
    hk, d = st["hk"], st["d"]
    kv = st["kv"].view(torch.float8_e4m3fn).cpu().double().numpy()
    scales, slot = st["scales"].cpu().double().numpy(), st["slot"].cpu().numpy()
    x = np.stack([st["k"].cpu().double().numpy().reshape(-1, hk, d), st["v"].cpu().double().numpy().reshape(-1, hk, d)], 2)
    r = 0
    while r < len(slot):
        page, off = divmod(int(slot[r]), PAGE)
        m = 1
        while r + m < len(slot) and off + m < PAGE and slot[r + m] == slot[r] + m:
            m += 1
        new = x[r:r + m].transpose(1, 2, 0, 3)  # [head, K | V, token, d]
        top = np.abs(new).max((-1, -2))
        scale = np.where(top > 0, np.exp2(np.ceil(np.log2(np.where(top > 0, top, 1.0) / E4M3_MAX))), 0)
        scale = np.maximum(scale, MIN_SCALE)
        if off:
            scale = np.maximum(scale, scales[page])
            kv[page, :, :, :off] = _e4m3(kv[page, :, :, :off] * (scales[page] / scale)[..., None, None])
        kv[page, :, :, off:off + m] = _e4m3(new / scale[..., None, None])
        scales[page] = scale
        r += m
    return {"kv": kv, "scales": scales}


def _exact_prompt(st):
    hq, hk, d = st["hq"], st["hk"], st["d"]
    ptr = st["row_ptr"].tolist()
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    for a, b in zip(ptr, ptr[1:]):
        for h in range(hq if b > a else 0):
            g = h // (hq // hk)
            q, k, v = st["q"][a:b, h * d:(h + 1) * d].double(), st["k"][a:b, g * d:(g + 1) * d].double(), st["v"][a:b, g * d:(g + 1) * d].double()
            for i in range(0, b - a, 2048):
                j = min(b - a, i + 2048)
                w = torch.softmax((q[i:j] @ k[:j].T * d ** -0.5).masked_fill(torch.ones(j - i, j, dtype=torch.bool, device="cuda").triu(i + 1), -math.inf), -1)
                out[a + i:a + j, h * d:(h + 1) * d] = w @ v[:j]
    return out


def _exact_attend8(st):
    hq, hk, d = st["hq"], st["hk"], st["d"]
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    ptr, pos = st["indptr"].tolist(), st["pos"].tolist()
    for n, t in enumerate(p + 1 for p in pos):
        if t:
            at = st["pages"][ptr[n]:ptr[n + 1]].long()
            x = st["kv"][at].view(torch.float8_e4m3fn).double() * st["scales"][at].double()[..., None, None]
            x = x.permute(1, 2, 0, 3, 4).reshape(hk, 2, -1, d)[:, :, :t]
            w = torch.softmax(st["q"][n].double().reshape(hk, -1, d) @ x[:, 0].transpose(-1, -2) * d ** -0.5, -1)
            out[n] = (w @ x[:, 1]).reshape(-1)
    return out
