"""Cases of the paged-cache and packed-prompt operators, with their plain forms.

``run`` makes one pass through one operator: in elementary torch operations in
32 bits where ``own`` is false, through ``joyomni_ops`` where it is true.

  layout   block tables, slots, positions and offsets from request lengths
  write    K and V rows of new tokens into their cache slots
  paged    attention of new tokens (one or a chunk) over a paged cache
  prompt   attention over whole packed prompts
"""
import math
import os
import random
import sys

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


def _jo():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "joyai-video-edit_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import joyomni_ops
    return joyomni_ops


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # the step of a server that answers 48 sessions with one token each
        {"name": "layout_decode", "op": "layout", "batch": 48, "new": 1, "even": True, "cached": 4096, "page": 64,
         "pad": 0, "shape": 1},
        # admission of a large ragged batch, some requests idle, token count padded for a captured graph
        {"name": "layout_admission", "op": "layout", "batch": 300, "new": 512, "even": False, "cached": 2000, "page": 16,
         "pad": 200, "shape": 2},
        # the same server's 48 new rows, some of them padding
        {"name": "write_decode", "op": "write", "tokens": 48, "kv_heads": 8, "dim": 128, "page": 64, "blocks": 600,
         "pad": 5, "dtype": "bf16", "shape": 3},
        # one video chunk (10530 image + 512 text tokens) of a rank that holds 10 of the 40 heads
        {"name": "write_chunk", "op": "write", "tokens": 11042, "kv_heads": 10, "dim": 128, "page": 128, "blocks": 260,
         "pad": 0, "dtype": "bf16", "shape": 4},
        # one token of one short request: latency
        {"name": "paged_one", "op": "paged", "batch": 1, "new": 1, "even": True, "cached": 300, "heads": 14, "kv_heads": 2,
         "dim": 64, "page": 16, "causal": True, "dtype": "f16", "shape": 5},
        # one token of each of 64 requests with histories of very different lengths
        {"name": "paged_decode", "op": "paged", "batch": 64, "new": 1, "even": True, "cached": 8190, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "causal": True, "dtype": "bf16", "shape": 6},
        # one token of one request with a very long history: the work is split along it
        {"name": "paged_long", "op": "paged", "batch": 1, "new": 1, "even": True, "cached": 131071, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 256, "causal": True, "dtype": "bf16", "shape": 7},
        # prompt chunks and single tokens together; pages that end inside a tile
        {"name": "paged_mixed", "op": "paged", "batch": 12, "new": 256, "even": False, "cached": 6000, "heads": 16,
         "kv_heads": 4, "dim": 128, "page": 48, "causal": True, "dtype": "bf16", "shape": 8},
        # one video chunk over the two cached ones, no mask, 10 of the 40 heads
        {"name": "paged_chunk", "op": "paged", "batch": 1, "new": 11042, "even": True, "cached": 21060, "heads": 10,
         "kv_heads": 10, "dim": 128, "page": 128, "causal": False, "dtype": "bf16", "shape": 9},
        # many short edit instructions packed together
        {"name": "prompt_short", "op": "prompt", "batch": 64, "len": 77, "heads": 16, "kv_heads": 4, "dim": 64,
         "causal": True, "dtype": "f16", "shape": 10},
        # a packed batch of prompts from a few tokens to thousands
        {"name": "prompt_ragged", "op": "prompt", "batch": 7, "len": 4096, "heads": 32, "kv_heads": 8, "dim": 128,
         "causal": True, "dtype": "bf16", "shape": 11},
        # one long prompt
        {"name": "prompt_long", "op": "prompt", "batch": 1, "len": 12288, "heads": 16, "kv_heads": 4, "dim": 128,
         "causal": True, "dtype": "bf16", "shape": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layout", "write", "paged", "paged", "paged", "prompt", "prompt"])
    shape = rng.randrange(1 << 20)
    dtype = rng.choice(["bf16", "f16"])
    dim = rng.choice([64, 128])
    page = rng.choice([16, 32, 48, 64, 80, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    if op == "layout":
        one = rng.random() < 0.4
        return {"op": op, "batch": _log(rng, 1, 600), "new": 1 if one else _log(rng, 2, 600), "even": one,
                "cached": _log(rng, 1, 20000), "page": page, "pad": rng.choice([0, 0, rng.randrange(1, 300)]),
                "shape": shape}
    if op == "write":
        tokens = _log(rng, 1, 11042)
        return {"op": op, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "page": page,
                "blocks": -(-tokens // page) + rng.randrange(1, 40), "pad": rng.choice([0, min(3, tokens - 1)]),
                "dtype": dtype, "shape": shape}
    if op == "paged":
        kind = rng.choice(["one", "few", "chunk"])
        new = 1 if kind == "one" else _log(rng, 2, 8) if kind == "few" else _log(rng, 9, 2048)
        batch = _log(rng, 1, 96 if kind != "chunk" else 12)
        # what the plain form holds: batch * heads * new * (cached + new) scores, batch * (cached + new) rows of K and V
        most = min(2 ** 31 // (batch * heads * new), 2 ** 30 // (batch * kv_heads * dim), 100000) - new
        cached = _log(rng, 1, max(2, most))
        return {"op": op, "batch": batch, "new": new, "even": kind == "one" or rng.random() < 0.5, "cached": cached,
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "causal": rng.random() < 0.75,
                "dtype": dtype, "shape": shape}
    batch = _log(rng, 1, 64)
    most = int(math.sqrt(2 ** 31 / (batch * heads)))
    return {"op": op, "batch": batch, "len": _log(rng, 1, min(most, 12288)), "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "causal": rng.random() < 0.8, "dtype": dtype, "shape": shape}


def _ragged(rng, n, hi, lo=0):
    """n lengths of lo..hi, the longest among them, spread over their logarithm."""
    got = [min(hi, max(lo, int(math.exp(rng.uniform(math.log(max(1, lo)), math.log(hi + 1)))) - (lo == 0))) for _ in range(n)]
    got[rng.randrange(n)] = hi
    return got


def _lengths(case):
    """(cached, new) of every request; the case's numbers alone decide them."""
    rng = random.Random(case["shape"])
    if case["op"] == "prompt":
        return [0] * case["batch"], _ragged(rng, case["batch"], case["len"], 1)
    cached = _ragged(rng, case["batch"], case["cached"])
    new = [case["new"]] * case["batch"] if case["even"] else _ragged(rng, case["batch"], case["new"], 0 if case["op"] == "layout" else 1)
    return cached, new


def _pages(n, page):
    return -(-n // page)


# ------------------------------------------------------------------ inputs --
def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device=DEV, dtype=DT[dtype])


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _starts(lens):
    got = [0]
    for n in lens:
        got.append(got[-1] + n)
    return got


def _tables(gen, lens, page, width, spare=3):
    """Random distinct blocks for the requests' tokens, -1 elsewhere; the blocks that are left."""
    counts = _ints([_pages(n, page) for n in lens])
    blocks = int(sum(_pages(n, page) for n in lens)) + spare
    ids = torch.randperm(blocks, generator=gen, device=DEV).to(torch.int32)
    first = torch.cumsum(counts, 0) - counts
    col = torch.arange(width, device=DEV)[None]
    at = first[:, None] + col
    table = torch.where(col < counts[:, None], ids[at.clamp(max=blocks - 1)], -1).to(torch.int32)
    return table.contiguous(), ids[blocks - spare:], blocks


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = {"op": case["op"], "case": case}
    if case["op"] == "layout":
        cached, new = _lengths(case)
        page = case["page"]
        width = max(_pages(c + n, page) for c, n in zip(cached, new)) + 1
        need = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new))
        s["table"], s["free"], _ = _tables(gen, cached, page, width, need + 7)
        s["cached"], s["new"] = _ints(cached), _ints(new)
        s["page"], s["tokens"] = page, sum(new) + case["pad"]
        s["keep"] = {}
    elif case["op"] == "write":
        T, H, D, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
        qkv = _randn(gen, (T, 3, H, D), case["dtype"])
        s["k"], s["v"] = qkv[:, 1], qkv[:, 2]
        s["kc"], s["vc"] = (torch.zeros((case["blocks"], page, H, D), dtype=DT[case["dtype"]], device=DEV) for _ in "kv")
        blocks = torch.randperm(case["blocks"], generator=gen, device=DEV)
        at = torch.arange(T, device=DEV)
        slots = blocks[at // page] * page + at % page
        slots[T - case["pad"]:] = -1
        s["slots"] = slots
    elif case["op"] == "paged":
        cached, new = _lengths(case)
        total = [c + n for c, n in zip(cached, new)]
        page, D = case["page"], case["dim"]
        s["table"], _, blocks = _tables(gen, total, page, max(_pages(n, page) for n in total) + 2)
        # blocks are reused: places that no token holds have the values of earlier requests
        s["kc"], s["vc"] = (_randn(gen, (blocks, page, case["kv_heads"], D), case["dtype"]) for _ in "kv")
        s["q"] = _randn(gen, (sum(new), case["heads"], D), case["dtype"])
        s["starts"], s["kv"] = _ints(_starts(new)), _ints(total)
        s["most_q"], s["most_k"] = max(new), max(total)
    else:
        _, lens = _lengths(case)
        H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
        qkv = _randn(gen, (sum(lens), H + 2 * Hk, D), case["dtype"])
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
        s["starts"], s["most_q"] = _ints(_starts(lens)), max(lens)
    return s


# ------------------------------------------------------------- plain forms --
def _plain_layout(s):
    page, T, table, free = s["page"], s["tokens"], s["table"], s["free"]
    cached, new = s["cached"].clamp(min=0), s["new"].clamp(min=0)
    kv = cached + new
    ends = torch.cumsum(new, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    first, last = (cached + page - 1) // page, (kv + page - 1) // page
    taken = torch.cumsum(last - first, 0)
    col = torch.arange(table.shape[1], device=table.device)[None]
    at = (taken - (last - first))[:, None] + col - first[:, None]
    fresh = torch.where(at < free.shape[0], free[at.clamp(0, free.shape[0] - 1)], -1)
    table.copy_(torch.where((col >= first[:, None]) & (col < last[:, None]), fresh, table))
    t = torch.arange(T, device=table.device)
    req = (t[:, None] >= ends[None]).sum(1)
    live = req < new.shape[0]
    req = req.clamp(max=new.shape[0] - 1)
    pos = torch.where(live, cached[req] + t - starts[req], 0)
    block = table[req, pos // page].to(torch.int64)
    slots = torch.where(live & (block >= 0), block * page + pos % page, -1)
    return {"table": table, "starts": starts, "kv": kv.to(torch.int32), "slots": slots, "positions": pos.to(torch.int32),
            "needed": taken[-1:].to(torch.int32)}


def _plain_write(s):
    live = s["slots"] >= 0
    at = s["slots"][live]
    for cache, rows in ((s["kc"], s["k"]), (s["vc"], s["v"])):
        cache.view(-1, *cache.shape[2:])[at] = rows[live]
    return [s["kc"], s["vc"]]


def _plain_attention(q, k, v, starts, kv, most_q, causal):
    """q [T, H, D]; k, v [B, K, Hk, D] in 32 bits, rows past kv[b] zero in v; requests side by side, padded to most_q rows."""
    T, H, D = q.shape
    B, K, Hk, _ = k.shape
    n = starts[1:] - starts[:-1]
    row = torch.arange(most_q, device=q.device)
    tok = (starts[:-1, None] + row).clamp(max=T - 1)
    qb = q.float()[tok].view(B, most_q, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, H // Hk * most_q, D)
    w = torch.matmul(qb, k.permute(0, 2, 3, 1)).view(B, Hk, H // Hk, most_q, K).mul_(1.0 / math.sqrt(D))
    last = (kv - n)[:, None] + row if causal else kv[:, None] - 1 + 0 * row
    seen = torch.arange(K, device=q.device) <= last.clamp(max=kv[:, None] - 1)[..., None]
    w.masked_fill_(~seen[:, None, None], -math.inf)
    w.sub_(w.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(B, Hk, -1, K), v.permute(0, 2, 1, 3)).view(B, Hk, H // Hk, most_q, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B * most_q, H, D)
    t = torch.arange(T, device=q.device)
    req = (t[:, None] >= starts[None, 1:]).sum(1)
    return o[req * most_q + t - starts[req]].to(q.dtype)


def _plain_paged(s):
    B = s["table"].shape[0]
    K = s["most_k"]
    blocks = s["table"].clamp(min=0).long()
    k, v = (c[blocks].view(B, -1, *c.shape[2:])[:, :K].float() for c in (s["kc"], s["vc"]))
    v.masked_fill_((torch.arange(K, device=v.device) >= s["kv"][:, None])[..., None, None], 0.0)
    return _plain_attention(s["q"], k, v, s["starts"], s["kv"], s["most_q"], s["case"]["causal"])


def _plain_prompt(s):
    L, starts = s["most_q"], s["starts"]
    n = starts[1:] - starts[:-1]
    row = torch.arange(L, device=starts.device)
    tok = (starts[:-1, None] + row).clamp(max=s["q"].shape[0] - 1)
    k, v = (x[tok].float() for x in (s["k"], s["v"]))
    v.masked_fill_((row >= n[:, None])[..., None, None], 0.0)
    return _plain_attention(s["q"], k, v, starts, n, L, s["case"]["causal"])


# --------------------------------------------------------------------- run --
def run(state):
    s = state
    if not own:
        return {"layout": _plain_layout, "write": _plain_write, "paged": _plain_paged, "prompt": _plain_prompt}[s["op"]](s)
    jo = s.get("jo")
    if jo is None:
        jo = s["jo"] = _jo()
    if s["op"] == "layout":
        out = s["keep"]["out"] = jo.paged_layout(s["cached"], s["new"], s["table"], s["free"], s["page"], s["tokens"],
                                                 out=s["keep"].get("out"))
        return {"table": s["table"], "starts": out.query_starts, "kv": out.kv_lens, "slots": out.slots,
                "positions": out.positions, "needed": out.blocks_needed}
    if s["op"] == "write":
        jo.paged_kv_write(s["k"], s["v"], s["kc"], s["vc"], s["slots"])
        return [s["kc"], s["vc"]]
    if s["op"] == "paged":
        return jo.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["starts"], s["kv"], causal=s["case"]["causal"],
                                  max_query_len=s["most_q"])
    return jo.prompt_attention(s["q"], s["k"], s["v"], s["starts"], causal=s["case"]["causal"])


# -------------------------------------------------------------------- work --
def _pairs(c, n, causal):
    return n * c + n * (n + 1) // 2 if causal else n * (c + n)


def work(case):
    if case["op"] == "write":
        row = case["kv_heads"] * case["dim"] * 2
        live = case["tokens"] - case["pad"]
        return {"bytes": 4 * live * row + 8 * case["tokens"], "flops": 0}
    cached, new = _lengths(case)
    B, T = len(new), sum(new)
    if case["op"] == "layout":
        page = case["page"]
        need = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new))
        return {"bytes": 8 * B + 8 * need + 4 * (2 * B + 1) + 12 * (T + case["pad"]) + 4, "flops": 0}
    total = sum(cached) + T
    row = case["dim"] * 2
    moved = 2 * T * case["heads"] * row + 2 * total * case["kv_heads"] * row + 4 * (2 * B + 1)
    if case["op"] == "paged":
        moved += 4 * sum(_pages(c + n, case["page"]) for c, n in zip(cached, new))
    return {"bytes": moved, "flops": 4 * case["dim"] * case["heads"] * sum(_pairs(c, n, case["causal"]) for c, n in zip(cached, new))}


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    """The definition in 64 bits, request by request and key head by key head."""
    if case["op"] == "layout":
        return None  # whole numbers: they have to be equal
    s = prepare(case, seed)
    if case["op"] == "write":
        got = []
        for cache, rows in ((s["kc"], s["k"]), (s["vc"], s["v"])):
            flat = cache.double().flatten(0, 1)
            n = case["tokens"] - case["pad"]
            flat.index_copy_(0, s["slots"][:n], rows[:n].double())
            got.append(flat.view(cache.shape))
        return got
    cached, new = _lengths(case)
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros((sum(new), H, D), dtype=torch.float64, device=DEV)
    t0 = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        if case["op"] == "paged":
            at = torch.arange(c + n, device=DEV)
            at = s["table"][b].long()[at // case["page"]] * case["page"] + at % case["page"]
        for h in range(Hk):
            if case["op"] == "paged":
                k, v = (x[:, :, h].reshape(-1, D)[at].double() for x in (s["kc"], s["vc"]))
            else:
                k, v = (x[t0:t0 + n, h].double() for x in (s["k"], s["v"]))
            for g in range(h * (H // Hk), (h + 1) * (H // Hk)):
                a = s["q"][t0:t0 + n, g].double() @ k.T / math.sqrt(D)
                if case["causal"]:
                    a = a + torch.full_like(a, -math.inf).triu_(c + 1)
                out[t0:t0 + n, g] = torch.softmax(a, 1) @ v
        t0 += n
    return out
