"""Workloads of the paged 8-bit KV cache: appending tokens, attention over the pages, copying and compacting pages.

Each case is one call on one layer's cache.  `run` evaluates the operator's definition with elementary torch
operations (`own = False`) or calls this library (`own = True`) on the same inputs; `exact` evaluates the definition
once more in 64 bits.

The cache: `num_pages` pages of `page` tokens for every kv head, e4m3 codes with one fp32 scale for each page and
head (value = code * scale; appended pages carry powers of two).  `table[b, i]` names the page that holds tokens
`i * page ..` of sequence b, `lens[b]` counts the tokens of sequence b with the new ones, `offs[b] .. offs[b + 1]` are
the new tokens of sequence b among the rows of k, v, q and out (one each where there are no `offs`).
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODE = torch.float8_e4m3fn
MIN_EXP = -40  # smallest scale: 2 ** -40


# ---- cases ------------------------------------------------------------------------------------------------------

def _attend(name, batch, new, ctx, ragged, q_heads, kv_heads, dim, page, dtype, layout):
    return {"name": name, "op": "attend", "batch": batch, "new": new, "ctx": ctx, "ragged": ragged, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "type": dtype, "layout": layout}


def _append(name, batch, new, ctx, ragged, kv_heads, dim, page, dtype, layout):
    return {"name": name, "op": "append", "batch": batch, "new": new, "ctx": ctx, "ragged": ragged, "kv_heads": kv_heads,
            "dim": dim, "page": page, "type": dtype, "layout": layout}


def _copy(name, pages, pairs, kv_heads, dim, page, layout):
    return {"name": name, "op": "copy", "pages": pages, "pairs": pairs, "kv_heads": kv_heads, "dim": dim, "page": page,
            "layout": layout}


def _compact(name, pages, batch, used, kv_heads, dim, page, layout):
    return {"name": name, "op": "compact", "pages": pages, "batch": batch, "used": used, "kv_heads": kv_heads, "dim": dim,
            "page": page, "layout": layout}


def listed():
    return [
        # one chat session of a small model, one token: what a call costs when there is next to nothing to read
        _attend("attend_one_short", 1, 1, 777, False, 8, 2, 64, 16, "fp16", "token"),
        # a serving batch in the middle of its answers, every sequence at its own length
        _attend("attend_batch", 32, 1, 8192, True, 32, 8, 128, 64, "bf16", "head"),
        # one session with a book in its context, one token
        _attend("attend_one_long", 1, 1, 131072, False, 32, 8, 128, 128, "fp16", "head"),
        # speculative drafts of up to 5 tokens to be checked, odd lengths, head size off the powers of two
        _attend("attend_drafts", 12, 5, 2500, True, 40, 8, 96, 32, "bf16", "token"),
        # a chunk of a long prompt over what is cached of it already
        _attend("attend_chunk", 1, 512, 16896, False, 32, 8, 128, 64, "bf16", "head"),
        # prompts of several requests, nothing cached before them
        _attend("attend_prompts", 2, 4096, 4096, True, 32, 8, 128, 64, "fp16", "head"),
        # the serving batch's new tokens, one each: small pieces into 64 pages of every head
        _append("append_tokens", 64, 1, 4096, True, 8, 128, 64, "bf16", "head"),
        # prompts of several requests
        _append("append_prompts", 4, 4096, 4096, True, 8, 128, 64, "fp16", "head"),
        # a beam forks: the half-filled last pages of a few sequences are duplicated
        _copy("copy_few", 256, 5, 8, 128, 64, "head"),
        # many sequences fork or swap places
        _copy("copy_many", 2048, 700, 8, 128, 64, "head"),
        # a small cache closes its gaps
        _compact("compact_small", 300, 6, 0.5, 2, 64, 16, "token"),
        # a large cache closes its gaps after half of its sequences have ended
        _compact("compact_large", 4096, 64, 0.5, 8, 128, 64, "head"),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case; the caps keep a drawn case below the largest listed one."""
    op = rng.choice(["attend", "attend", "attend", "attend", "append", "append", "copy", "compact"])
    kv_heads, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 80, 96, 112, 128, 128, 128, 256])
    page, dtype, layout = rng.choice([8, 16, 20, 32, 64, 64, 128, 256]), rng.choice(["fp16", "bf16"]), rng.choice(["head", "token"])
    if op == "attend":
        group = rng.choice([1, 2, 4, 4, 5, 8, 12])
        kind = rng.choice(["token", "token", "draft", "prompt"])
        batch = _log(rng, 1, 64 if kind != "prompt" else 4)
        new = 1 if kind == "token" else rng.randint(2, 16) if kind == "draft" else _log(rng, 17, 2048)
        past = rng.choice([0, _log(rng, 1, 8192)]) if kind == "prompt" else _log(rng, 1, 65536)
        while True:
            c = _attend("drawn", batch, new, new + past, rng.random() < 0.7, group * kv_heads, kv_heads, dim, page, dtype, layout)
            w, scores = work(c), batch * group * kv_heads * new * (new + past)
            if w["bytes"] < 2.5e8 and w["flops"] < 1e11 and scores < 8e8:
                return c
            if batch > 1 and (batch > 8 or rng.random() < 0.5):
                batch = max(1, batch * 2 // 3)
            elif past > new:
                past = past * 2 // 3
            else:
                new = max(1, new * 2 // 3)
    if op == "append":
        batch = _log(rng, 1, 64)
        new = rng.choice([1, _log(rng, 2, max(2, 12000 // batch))])
        return _append("drawn", batch, new, new + _log(rng, 1, 2000), rng.random() < 0.7, kv_heads, dim, page, dtype, layout)
    pages = _log(rng, 16, 2000)
    if op == "copy":
        return _copy("drawn", pages, _log(rng, 1, max(1, pages // 3)), kv_heads, min(dim, 128), min(page, 64), layout)
    return _compact("drawn", pages, _log(rng, 1, min(64, pages // 4)), rng.uniform(0.1, 0.9), kv_heads, min(dim, 128), min(page, 64), layout)


# ---- inputs -----------------------------------------------------------------------------------------------------

def _lengths(c):
    """(new tokens, tokens in all) of each sequence: a matter of the case, so that every seed's tensors have the same
    sizes; the seed decides which sequence comes where."""
    rng, pairs = random.Random("%(batch)d %(new)d %(ctx)d" % c), []
    for _ in range(c["batch"]):
        n = rng.randint(max(1, c["new"] // 4), c["new"]) if c["ragged"] else c["new"]
        past = c["ctx"] - c["new"]
        past = rng.randint(past // 8, past) if c["ragged"] else past
        pairs.append((n, n + past))
    return pairs


def _held(c):
    """Tokens of each sequence of a cache that is to be compacted."""
    rng, left, total = random.Random("%(pages)d %(batch)d" % c), max(1, int(c["pages"] * c["used"])), []
    for b in range(c["batch"]):
        n = left // (c["batch"] - b)
        n = min(left, rng.randint((n + 1) // 2, n + n // 2))
        left -= n
        total.append(max(0, n * c["page"] - rng.randrange(c["page"])))
    return total


def _pool(c, num_pages, g):
    """Codes of one pool, [num_pages, kv_heads, page, dim] (a view of [num_pages, page, kv_heads, dim] for layout
    "token"), and the scale of each page and head: normal values, heads of different magnitude."""
    H, P, D = c["kv_heads"], c["page"], c["dim"]
    amp = torch.exp(0.5 * torch.randn(H, 1, 1, generator=g, device=DEV))
    x = torch.randn(num_pages, H, P, D, generator=g, device=DEV) * amp
    scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / 448)))
    x = (x / scale[:, :, None, None]).to(CODE)
    if c["layout"] == "token":
        x = x.transpose(1, 2).contiguous().transpose(1, 2)
    return x, scale


def _tables(c, totals, num_pages, rng):
    """The sequences' pages, scattered over the pool; -1 behind each sequence's last."""
    P = c["page"]
    cols = -(-max(totals) // P)
    ids = list(range(num_pages))
    rng.shuffle(ids)
    rows = []
    for t in totals:
        n = -(-t // P)
        rows.append([ids.pop() for _ in range(n)] + [-1] * (cols - n))
    return torch.tensor(rows, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    c, rng = case, random.Random(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"op": c["op"]}
    if c["op"] in ("attend", "append"):
        pairs = _lengths(c)
        rng.shuffle(pairs)
        new, total = zip(*pairs)
        need = sum(-(-t // c["page"]) for t in total)
        N = need + max(2, need // 16)
        s["table"] = _tables(c, total, N, rng)
        s["lens"] = torch.tensor(total, dtype=torch.int32, device=DEV)
        offs = [0]
        for n in new:
            offs.append(offs[-1] + n)
        T, dt = offs[-1], TYPES[c["type"]]
        s["offs"] = torch.tensor(offs, dtype=torch.int32, device=DEV) if c["new"] > 1 else None
        s["most"] = max(new)
        s["kp"], s["ks"] = _pool(c, N, g)
        s["vp"], s["vs"] = _pool(c, N, g)
        if c["op"] == "attend":
            s["scale"] = 1.0 / math.sqrt(c["dim"])
            s["q"] = (2 * torch.randn(T, c["q_heads"], c["dim"], generator=g, device=DEV)).to(dt)
            s["out"] = torch.zeros(T, c["q_heads"], c["dim"], dtype=dt, device=DEV)
        else:
            amp = torch.exp(0.5 * torch.randn(2, 1, c["kv_heads"], 1, generator=g, device=DEV))
            s["k"], s["v"] = (torch.randn(2, T, c["kv_heads"], c["dim"], generator=g, device=DEV) * amp).to(dt)
            # a program that fills pages knows on the host which of the new tokens opens which page
            firsts = []
            for b, n in enumerate(new):
                p0 = total[b] - n
                firsts += [offs[b] + i for i in range(n) if i == 0 or (p0 + i) % c["page"] == 0]
            s["firsts"] = torch.tensor(firsts, device=DEV)
    elif c["op"] == "copy":
        N = c["pages"]
        s["kp"], s["ks"] = _pool(c, N, g)
        s["vp"], s["vs"] = _pool(c, N, g)
        ids = list(range(N))
        rng.shuffle(ids)
        dst, rest = ids[:c["pairs"]], ids[c["pairs"]:]
        s["pairs"] = torch.tensor([[rng.choice(rest), d] for d in dst], dtype=torch.int32, device=DEV)
    else:
        N, P = c["pages"], c["page"]
        s["kp"], s["ks"] = _pool(c, N, g)
        s["vp"], s["vs"] = _pool(c, N, g)
        total = _held(c)
        rng.shuffle(total)
        s["table"] = _tables(c, [max(t, 1) for t in total], N, rng)
        s["lens"] = torch.tensor(total, dtype=torch.int32, device=DEV)
        s["new_table"] = torch.full_like(s["table"], -1)
        s["page_map"] = torch.zeros(N, dtype=torch.int32, device=DEV)
        s["live"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    if own:
        s["plan"] = _plan(s)
    return s


# ---- this library's calls -----------------------------------------------------------------------------------------

_library = []


def _plan(s):
    """The operator object a program keeps: the descriptor and the workspace of these shapes."""
    import operators_b200 as b200
    from operators_b200 import ops

    if not _library:
        lib = b200.open_lib()
        _library[:] = [lib, b200.create_handle(lib, b200.DeviceEnum.DEVICE_CUDA, 0)]
    lib, handle = _library
    cache = [s[n] for n in ("kp", "vp", "ks", "vs")]
    if s["op"] == "attend":
        return ops.PagedAttentionOp(lib, handle, s["out"], s["q"], *cache, s["table"], s["lens"], s["offs"], s["scale"])
    if s["op"] == "append":
        return ops.PagedCacheAppendOp(lib, handle, s["k"], s["v"], *cache, s["table"], s["lens"], s["offs"])
    if s["op"] == "copy":
        return ops.PagedCacheCopyOp(lib, handle, *cache, s["pairs"])
    return ops.PagedCacheCompactOp(lib, handle, *cache, s["new_table"], s["table"], s["lens"], s["page_map"], s["live"])


def _run_own(s):
    kp, vp, ks, vs = (s[n] for n in ("kp", "vp", "ks", "vs"))
    if s["op"] == "attend":
        s["plan"](s["out"], s["q"], kp, vp, ks, vs, s["table"], s["lens"], s["offs"])
        return s["out"]
    if s["op"] == "append":
        s["plan"](s["k"], s["v"], kp, vp, ks, vs, s["table"], s["lens"], s["offs"])
        return [kp, vp, ks, vs]
    if s["op"] == "copy":
        s["plan"](kp, vp, ks, vs, s["pairs"])
        return [kp, vp, ks, vs]
    s["plan"](kp, vp, ks, vs, s["new_table"], s["table"], s["lens"], s["page_map"], s["live"])
    return [kp, vp, ks, vs, s["new_table"], s["page_map"], s["live"]]


# ---- the plain form -----------------------------------------------------------------------------------------------

def _u8(x):
    return x.view(torch.uint8)


def _tokens_of(s, T):
    """Sequence and position of every new token."""
    t = torch.arange(T, device=DEV)
    if s["offs"] is None:
        return t, s["lens"].long() - 1
    offs = s["offs"].long()
    b = torch.searchsorted(offs, t, right=True) - 1
    n = offs[b + 1] - offs[b]
    return b, s["lens"].long()[b] - n + t - offs[b]


def _attend_plain(s):
    q, table, lens = s["q"], s["table"].long().clamp(min=0), s["lens"].long()
    T, HQ, D = q.shape
    B, S = table.shape
    _, H, P, _ = s["kp"].shape
    G, L, n_most = HQ // H, S * P, s["most"]
    offs = torch.arange(B + 1, device=DEV) if s["offs"] is None else s["offs"].long()
    n = offs[1:] - offs[:-1]
    i = torch.arange(n_most, device=DEV)
    rows = (offs[:-1, None] + i).clamp(max=T - 1)                                     # [B, n_most]
    pos = (lens - n)[:, None] + i
    def gather(pages, scales):
        x = _u8(pages)[table].view(CODE).float() * scales[table][..., None, None]    # [B, S, H, P, D]
        return x.permute(0, 2, 1, 3, 4).reshape(B, H, L, D)
    k, v = gather(s["kp"], s["ks"]), gather(s["vp"], s["vs"])
    inside = torch.arange(L, device=DEV) < lens[:, None]                              # [B, L]
    v = torch.where(inside[:, None, :, None], v, torch.zeros((), device=DEV))
    qq = q[rows].float().view(B, n_most, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * n_most, D)
    x = torch.matmul(qq, k.transpose(2, 3)).mul_(s["scale"]).view(B, H, G, n_most, L)
    seen = (torch.arange(L, device=DEV) <= pos[..., None])[:, None, None]             # [B, 1, 1, n_most, L]
    x.masked_fill_(~seen, -math.inf)
    m = x.amax(-1, keepdim=True)
    x.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = x.sum(-1, keepdim=True)
    y = torch.matmul(x.view(B, H, G * n_most, L), v).view(B, H, G, n_most, D)
    y = torch.where(total > 0, y / total, torch.zeros_like(y)).permute(0, 3, 1, 2, 4).reshape(B, n_most, HQ, D)
    out = torch.zeros_like(q)
    if n_most == 1:
        out[rows[:, 0]] = y[:, 0].to(q.dtype)
    else:
        keep = (i < n[:, None]).reshape(-1)
        # tokens beyond a sequence's own go to a row behind the last
        at = torch.where(keep, rows.reshape(-1), T)
        out = torch.cat([out, out[:1]])
        out[at] = y.reshape(B * n_most, HQ, D).to(q.dtype)
        out = out[:T]
    return out


def _encode(x):
    return x.clamp(-448.0, 448.0).to(CODE)


def _scale_of(amax):
    """The smallest power of two, not below 2 ** MIN_EXP, that brings amax to 448 or less."""
    f, e = torch.frexp(amax)
    e = torch.where(f <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e.clamp(min=MIN_EXP)), torch.full_like(amax, 2.0 ** MIN_EXP))


def _append_plain(s):
    T, H, D = s["k"].shape
    N, _, P, _ = s["kp"].shape
    b, pos = _tokens_of(s, T)
    page, slot = s["table"].long()[b, pos // P], pos % P
    first = s["firsts"]
    fp, keep = page[first], slot[first]                                               # each touched page, what it keeps
    for x, pages, scales in ((s["k"], s["kp"], s["ks"]), (s["v"], s["vp"], s["vs"])):
        xf = x.float()
        a = torch.where(xf.isfinite(), xf.abs(), torch.zeros((), device=DEV)).amax(-1)
        a = torch.zeros(N, H, device=DEV).index_reduce_(0, page, a, "amax")[fp]
        old = scales[fp]
        new = torch.maximum(_scale_of(a), torch.where((keep > 0)[:, None], old, torch.zeros_like(old)))
        kept = _encode(_u8(pages)[fp].view(CODE).float() * (old / new)[..., None, None])
        stays = (torch.arange(P, device=DEV) < keep[:, None])[:, None, :, None]
        _u8(pages)[fp] = torch.where(stays, _u8(kept), _u8(pages)[fp])
        scales[fp] = new
        _u8(pages)[page, :, slot] = _u8(_encode(xf / scales[page][..., None]))
    return [s["kp"], s["vp"], s["ks"], s["vs"]]


def _copy_plain(s):
    src, dst = s["pairs"].long().unbind(1)
    for pages, scales in ((s["kp"], s["ks"]), (s["vp"], s["vs"])):
        _u8(pages)[dst] = _u8(pages)[src]
        scales[dst] = scales[src]
    return [s["kp"], s["vp"], s["ks"], s["vs"]]


def _compact_plain(s):
    N, _, P, _ = s["kp"].shape
    table, lens = s["table"].long(), s["lens"].long()
    used = torch.arange(table.shape[1], device=DEV) * P < lens[:, None]
    mark = torch.zeros(N + 1, dtype=torch.bool, device=DEV)
    mark[torch.where(used, table, N)] = True
    live, ids = mark[:N], torch.arange(N, device=DEV)
    count = live.sum()
    src, dst = ids[live & (ids >= count)], ids[~live & (ids < count)]
    page_map = torch.where(live, ids, -1)
    page_map[src] = dst
    for pages, scales in ((s["kp"], s["ks"]), (s["vp"], s["vs"])):
        _u8(pages)[dst] = _u8(pages)[src]
        scales[dst] = scales[src]
    new_table = torch.where(used, page_map[table.clamp(min=0)], table)
    return [s["kp"], s["vp"], s["ks"], s["vs"], new_table.int(), page_map.int(), count.int().view(1)]


def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "attend":
        return _attend_plain(state)
    if state["op"] == "append":
        return _append_plain(state)
    if state["op"] == "copy":
        return _copy_plain(state)
    return _compact_plain(state)


# ---- 64 bits ------------------------------------------------------------------------------------------------------

def _exact_attend(c, s):
    """Sequence by sequence: softmax(scale * q k^T + mask) v over the sequence's own pages."""
    q, H, P, D = s["q"].double(), c["kv_heads"], c["page"], c["dim"]
    G, out, at = c["q_heads"] // H, torch.zeros_like(q), 0
    lens = s["lens"].tolist()
    counts = [1] * len(lens) if s["offs"] is None else [b - a for a, b in zip(s["offs"].tolist(), s["offs"].tolist()[1:])]
    for b, (n, total) in enumerate(zip(counts, lens)):
        ids = s["table"][b, : -(-total // P)].tolist()
        hidden = torch.ones(n, total, dtype=torch.bool, device=DEV).triu(total - n + 1)
        for h in range(H):
            def rows(pages, scales):
                x = pages[:, h].view(torch.uint8)[ids].view(CODE).double() * scales[ids, h].double()[:, None, None]
                return x.reshape(-1, D)[:total]
            k, v = rows(s["kp"], s["ks"]), rows(s["vp"], s["vs"])
            for j in range(h * G, h * G + G):
                w = (q[at:at + n, j] @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf)
                out[at:at + n, j] = torch.softmax(w, -1) @ v
        at += n
    return out


def _exact_append(c, s):
    """Sequence by sequence and page by page, on the host."""
    P, res = c["page"], []
    lens, table = s["lens"].tolist(), s["table"].tolist()
    counts = [1] * len(lens) if s["offs"] is None else [b - a for a, b in zip(s["offs"].tolist(), s["offs"].tolist()[1:])]
    for x, pages, scales in ((s["k"], s["kp"], s["ks"]), (s["v"], s["vp"], s["vs"])):
        x, codes, scales, at = x.double().cpu(), pages.cpu().double(), scales.double().cpu(), 0
        for b, (n, total) in enumerate(zip(counts, lens)):
            p = total - n
            while p < total:
                page, lo = table[b][p // P], p % P
                m = min(P - lo, total - p)
                new = x[at:at + m].transpose(0, 1)                                    # [H, m, D]
                want = torch.exp2(torch.ceil(torch.log2(new.abs().amax((1, 2)) / 448)).clamp(min=MIN_EXP))
                if lo:
                    want = torch.maximum(want, scales[page])
                    codes[page, :, :lo] = (codes[page, :, :lo] * (scales[page] / want)[:, None, None]).to(CODE).double()
                codes[page, :, lo:lo + m] = (new / want[:, None, None]).to(CODE).double()
                scales[page] = want
                p, at = p + m, at + m
        res.append((codes, scales))
    return [res[0][0], res[1][0], res[0][1], res[1][1]]


def _exact_moves(s, moves):
    kp, vp, ks, vs = (s[n].double() for n in ("kp", "vp", "ks", "vs"))
    src, dst = [a for a, _ in moves], [b for _, b in moves]
    for x in (kp, vp, ks, vs):
        x[dst] = x[src]
    return [kp, vp, ks, vs]


def _exact_compact(c, s):
    P, N = c["page"], c["pages"]
    lens, table = s["lens"].tolist(), s["table"].tolist()
    live = {row[i] for row, n in zip(table, lens) for i in range(-(-n // P))}
    to = {p: p for p in live}
    moves = list(zip(sorted(p for p in live if p >= len(live)), (p for p in range(len(live)) if p not in live)))
    to.update(moves)
    rows = [[to[p] if i < -(-n // P) else p for i, p in enumerate(row)] for row, n in zip(table, lens)]
    whole = [torch.tensor(x, dtype=torch.int32) for x in (rows, [to.get(p, -1) for p in range(N)], [len(live)])]
    return _exact_moves(s, moves) + whole


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "copy":
        return _exact_moves(s, [tuple(p) for p in s["pairs"].tolist()])
    return _exact_compact(case, s)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    c = case
    H, D, P = c["kv_heads"], c["dim"], c["page"]
    if c["op"] in ("attend", "append"):
        pairs = _lengths(c)
        tokens, pages = sum(n for n, _ in pairs), sum(-(-t // P) for _, t in pairs)
        if c["op"] == "attend":
            scores = c["q_heads"] * sum(n * t - n * (n - 1) // 2 for n, t in pairs)
            cached = H * (2 * D * sum(t for _, t in pairs) + 8 * pages)
            return {"bytes": cached + 4 * pages + 4 * tokens * c["q_heads"] * D, "flops": 4 * D * scores}
        touched = sum(-(-t // P) - (t - n) // P for n, t in pairs)
        return {"bytes": 6 * tokens * H * D + touched * (8 * H + 4), "flops": 6 * tokens * H * D}
    page = 2 * H * (P * D + 4)
    if c["op"] == "copy":
        return {"bytes": c["pairs"] * (2 * page + 8), "flops": 0}
    # pages are scattered evenly: of the live ones, the share that lies behind their number has to move
    live = sum(-(-t // P) for t in _held(c))
    return {"bytes": live * (1 - live / c["pages"]) * 2 * page + 8 * live + 4 * c["pages"], "flops": 0}
