"""Performance cases of the attention operators and the paged key-value cache on one GPU, through the public Python API.

    decode   attention of one new token per sequence over a paged cache (ops.attention.decode_attention)
    prefill  attention of whole or chunked prompts, packed one behind the other (ops.attention.prefill_attention)
    write    new tokens' keys and values into their slots of one layer's pages (ops.kv_cache.PagedKVCache.write)
    branch   candidates forked from prompts, each advanced by a token, those of the step before dropped (free, fork, reserve)
    compact  the pages in use moved to the front of the cache, page tables rewritten (compact)

`listed()` are fixed cases, `draw(rng)` gives others of the same ranges. With `own` false `run` computes the operators in elementary
torch operations, in 32 bits, rounded once at the end. Lengths go by the case alone, values, page numbers and their order by the seed.
"""
from __future__ import annotations

import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # One chat session on an 8B-shaped model, short history: what counts is latency.
        {"name": "decode_one_short", "op": "decode", "batch": 1, "lo": 137, "hi": 137, "gaps": False, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "type": "bf16", "cache": "bf16"},
        # A continuous batch of a serving process: ragged histories, some slots of the batch empty.
        {"name": "decode_batch", "op": "decode", "batch": 61, "lo": 1, "hi": 4096, "gaps": True, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "type": "bf16", "cache": "bf16"},
        # Two agents with very long histories: few rows, a long axis to split; five query heads to a cache head.
        {"name": "decode_long", "op": "decode", "batch": 2, "lo": 131071, "hi": 131071, "gaps": False, "heads": 40, "kv_heads": 8, "dim": 128, "page": 64,
         "type": "fp16", "cache": "fp16"},
        # A large batch over an 8-bit cache.
        {"name": "decode_e4m3", "op": "decode", "batch": 128, "lo": 1000, "hi": 4096, "gaps": False, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "type": "bf16", "cache": "e4m3"},
        # Short prompts that arrive together.
        {"name": "prefill_short", "op": "prefill", "batch": 31, "lo": 5, "hi": 190, "past": 0, "causal": True, "heads": 32, "kv_heads": 8, "dim": 128,
         "type": "bf16"},
        # A mixed batch of prompts, small heads, seven query heads to a key head.
        {"name": "prefill_mixed", "op": "prefill", "batch": 12, "lo": 64, "hi": 1500, "past": 0, "causal": True, "heads": 28, "kv_heads": 4, "dim": 64,
         "type": "fp16"},
        # Chunks of long prompts: 512 new tokens each behind what is already there.
        {"name": "prefill_chunk", "op": "prefill", "batch": 4, "lo": 500, "hi": 512, "past": 5000, "causal": True, "heads": 32, "kv_heads": 8, "dim": 128,
         "type": "bf16"},
        # One long prompt.
        {"name": "prefill_8k", "op": "prefill", "batch": 1, "lo": 8192, "hi": 8192, "past": 0, "causal": True, "heads": 32, "kv_heads": 8, "dim": 128,
         "type": "bf16"},
        # A decode step's tokens: a few rows, latency.
        {"name": "write_step", "op": "write", "tokens": 61, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "pages": 4096, "type": "bf16", "cache": "bf16"},
        # A prompt's tokens, quantised on the way.
        {"name": "write_prompt_e4m3", "op": "write", "tokens": 8191, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "pages": 4096, "type": "bf16",
         "cache": "e4m3"},
        # Parallel sampling: seven candidates of each of 32 prompts, whose last pages are shared and partly filled; a tensor-parallel slice of heads.
        {"name": "branch", "op": "branch", "prompts": 32, "ways": 7, "lo": 200, "hi": 2000, "layers": 32, "kv_heads": 2, "dim": 128, "page": 16,
         "cache": "bf16"},
        # A cache half of whose pages have been freed, before its tail is given back.
        {"name": "compact", "op": "compact", "pages": 4096, "seqs": 64, "live": 0.5, "layers": 16, "kv_heads": 4, "dim": 128, "page": 16, "cache": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


HEADS = [(32, 8), (4, 1), (16, 16), (28, 4), (40, 8), (64, 4)]  # an 8B model, a slice of it, no groups, groups of 7, 5 and 16


def draw(rng):
    op = rng.choice(["decode", "decode", "decode", "prefill", "prefill", "prefill", "write", "branch", "compact"])
    heads, kv = rng.choice(HEADS)
    dim = rng.choice([64, 128, 128])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    page = rng.choice([16, 16, 32, 64, 128, 48])
    if op == "decode":
        batch = _log(rng, 1, 256)
        most = max(16, min(131072, (1 << 28) // (batch * kv * dim)))
        hi = _log(rng, 16, most)
        return {"op": op, "batch": batch, "lo": rng.choice([1, max(1, hi // 2), hi]), "hi": hi, "gaps": rng.random() < 0.3, "heads": heads, "kv_heads": kv,
                "dim": dim, "page": page, "type": kind, "cache": rng.choice([kind, kind, "e4m3"])}
    if op == "prefill":
        past = rng.choice([0, 0, _log(rng, 1, 6000)])
        batch = _log(rng, 1, 32)
        most = 8192
        while batch * heads * most * (most + past) > 1 << 30:
            most = most * 3 // 4
        hi = _log(rng, min(16, most), most)
        return {"op": op, "batch": batch, "lo": rng.choice([1, max(1, hi // 3), hi]), "hi": hi, "past": past, "causal": rng.random() < 0.8,
                "heads": heads, "kv_heads": kv, "dim": dim, "type": kind}
    if op == "write":
        tokens = _log(rng, 1, 8192)
        pages = -(-tokens * 5 // (4 * page)) + 8
        return {"op": op, "tokens": tokens, "heads": heads, "kv_heads": kv, "dim": dim, "page": page, "pages": pages, "type": kind,
                "cache": rng.choice([kind, kind, "e4m3"])}
    layers, kv = _log(rng, 1, 32), rng.choice([1, 2, 4])
    if op == "branch":
        prompts, ways, hi = _log(rng, 1, 32), rng.randrange(1, 8), _log(rng, 16, 2000)
        return {"op": op, "prompts": prompts, "ways": ways, "lo": max(1, hi // 10), "hi": hi, "layers": layers, "kv_heads": min(kv, 2), "dim": dim,
                "page": rng.choice([16, 32]), "cache": rng.choice([kind, "e4m3"])}
    pages = _log(rng, 64, 4096)
    return {"op": op, "pages": pages, "seqs": _log(rng, 1, min(64, pages // 16)), "live": rng.choice([0.2, 0.5, 0.9]), "layers": min(layers, 16),
            "kv_heads": kv, "dim": dim, "page": 16, "cache": kind}


# ------------------------------------------------------------------------------------------------ inputs


def _lengths(c, count, empty=False):
    r = random.Random("%d %d %d" % (count, c["lo"], c["hi"]))
    got = [r.randint(c["lo"], c["hi"]) for _ in range(count)]
    if got:
        got[0] = c["hi"]
    return [0 if empty and i % 9 == 4 else n for i, n in enumerate(got)]


def _tables(lengths, page, width, order):
    """Page table [len(lengths), width] and the pages that it takes from `order` (a tensor of page numbers on the GPU); -1 where there is none."""
    need = [-(-n // page) for n in lengths]
    where = torch.full((len(lengths), width), -1, dtype=torch.int64)
    at = 0
    for i, n in enumerate(need):
        where[i, :n] = torch.arange(at, at + n)
        at += n
    where = where.to(order.device)
    return torch.where(where >= 0, order[where.clamp(min=0)], -1).to(torch.int32), at


def _fill(shape, kind, gen):
    """Normal values of a type. An 8-bit cache holds x / scale with scale = 1 / 100, about what keeps 4.5 sigma inside the type's range."""
    x = torch.empty(shape, dtype=torch.bfloat16 if kind == "e4m3" else TYPES[kind], device="cuda").normal_(generator=gen)
    return (x * 100).clamp_(-448, 448).to(torch.float8_e4m3fn) if kind == "e4m3" else x


def _scales(heads, gen):
    return (1 + torch.rand(heads, generator=gen, device="cuda")) / 100


def prepare(case, seed):
    c, gen = case, torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] == "decode":
        lengths = _lengths(c, c["batch"], c["gaps"])
        width = max(1, -(-c["hi"] // c["page"]))
        used = sum(-(-n // c["page"]) for n in lengths)
        pages = used + used // 8 + 1
        s["table"], _ = _tables(lengths, c["page"], width, torch.randperm(pages, generator=gen, device="cuda"))
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        data = _fill((pages, 2, c["kv_heads"], c["page"], c["dim"]), c["cache"], gen)
        s["k_pages"], s["v_pages"] = data[:, 0], data[:, 1]
        # what the projections give for a sharp and for a flat head: logits of a few units
        s["q"] = _fill((c["batch"], c["heads"], c["dim"]), c["type"], gen) * 1.5
        s["k_scale"], s["v_scale"] = (_scales(c["kv_heads"], gen), _scales(c["kv_heads"], gen)) if c["cache"] == "e4m3" else (None, None)
    elif c["op"] == "prefill":
        new = _lengths(c, c["batch"])
        old = _lengths({"lo": c["past"] // 2, "hi": c["past"]}, c["batch"])
        cu = [[0], [0]]
        for n, p in zip(new, old):
            cu[0].append(cu[0][-1] + n)
            cu[1].append(cu[1][-1] + n + p)
        s["cu_q"], s["cu_k"] = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in cu)
        s["most"] = (max(new), max(n + p for n, p in zip(new, old)))
        s["q"] = _fill((cu[0][-1], c["heads"], c["dim"]), c["type"], gen) * 1.5
        s["k"], s["v"] = (_fill((cu[1][-1], c["kv_heads"], c["dim"]), c["type"], gen) for _ in range(2))
    elif c["op"] == "write":
        s["data"] = _fill((1, c["pages"], 2, c["kv_heads"], c["page"], c["dim"]), c["cache"], gen)
        # the rows of one fused projection of queries, keys and values
        qkv = _fill((c["tokens"], c["heads"] + 2 * c["kv_heads"], c["dim"]), c["type"], gen)
        s["k"], s["v"] = qkv[:, c["heads"]:c["heads"] + c["kv_heads"]], qkv[:, c["heads"] + c["kv_heads"]:]
        # a prompt's tokens lie one behind the other in pages that lie anywhere
        n = -(-c["tokens"] // c["page"])
        got = torch.randperm(c["pages"], generator=gen, device="cuda")[:n]
        s["slots"] = (got[:, None] * c["page"] + torch.arange(c["page"], device="cuda")).reshape(-1)[:c["tokens"]].contiguous()
        s["k_scale"], s["v_scale"] = (_scales(c["kv_heads"], gen), _scales(c["kv_heads"], gen)) if c["cache"] == "e4m3" else (None, None)
        s["table"] = torch.full((1, 1), -1, dtype=torch.int32, device="cuda")
        s["lengths"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["refs"] = torch.zeros(c["pages"], dtype=torch.int32, device="cuda")
    elif c["op"] == "branch":
        lengths = _lengths(c, c["prompts"])
        forks = c["prompts"] * c["ways"]
        used = sum(-(-n // c["page"]) for n in lengths)
        pages = used + used // 8 + forks + 1
        order = torch.randperm(used + used // 8, generator=gen, device="cuda")
        s["table"], used = _tables(lengths + [0] * forks, c["page"], c["hi"] // c["page"] + 2, order)
        s["lengths"] = torch.tensor(lengths + [0] * forks, dtype=torch.int32, device="cuda")
        s["refs"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
        s["refs"][order[:used]] = 1
        s["data"] = _fill((c["layers"], pages, 2, c["kv_heads"], c["page"], c["dim"]), c["cache"], gen)
        s["src"] = torch.arange(c["prompts"], dtype=torch.int32, device="cuda").repeat_interleave(c["ways"])
        s["dst"] = torch.arange(c["prompts"], c["prompts"] + forks, dtype=torch.int32, device="cuda")
        s["counts"] = torch.ones(forks, dtype=torch.int32, device="cuda")
    else:
        live = max(c["seqs"], int(c["pages"] * c["live"]))
        each = [live // c["seqs"] + (i < live % c["seqs"]) for i in range(c["seqs"])]
        order = torch.randperm(c["pages"], generator=gen, device="cuda")
        s["given"], _ = _tables([n * c["page"] for n in each], c["page"], max(each), order)
        s["lengths"] = torch.tensor([n * c["page"] for n in each], dtype=torch.int32, device="cuda")
        s["given_refs"] = torch.zeros(c["pages"], dtype=torch.int32, device="cuda")
        s["given_refs"][order[:live]] = 1
        s["table"], s["refs"] = s["given"].clone(), s["given_refs"].clone()
        s["data"] = _fill((c["layers"], c["pages"], 2, c["kv_heads"], c["page"], c["dim"]), c["cache"], gen)
    return s


# ------------------------------------------------------------------------------------------------ a pass


def _attend(q, k, v, hidden):
    """softmax(q k^T) v in 32 bits over the places that `hidden` leaves; rows without any give zeros."""
    p = q @ k.transpose(-1, -2)
    p.masked_fill_(hidden, float("-inf"))
    top = p.amax(-1, keepdim=True)
    top.masked_fill_(top == float("-inf"), 0.0)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return (p @ v) / total.clamp(min=1e-37)


def _pick(pages, table):
    """The pages of a table's rows, [rows, heads, positions, dim], in 32 bits."""
    bits = pages.view(torch.uint8) if pages.dtype == torch.float8_e4m3fn else pages
    got = bits[table.clamp(min=0).long()]
    got = (got.view(pages.dtype) if got.dtype != pages.dtype else got).float()
    return got.permute(0, 2, 1, 3, 4).reshape(got.shape[0], got.shape[2], -1, got.shape[4])


def _plain_decode(s):
    c, q = s["case"], s["q"]
    k, v = _pick(s["k_pages"], s["table"]), _pick(s["v_pages"], s["table"])
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][:, None, None], v * s["v_scale"][:, None, None]
    q32 = q.float().view(c["batch"], c["kv_heads"], -1, c["dim"]) * c["dim"] ** -0.5
    hidden = torch.arange(k.shape[2], device="cuda") >= s["lengths"][:, None, None, None]
    return _attend(q32, k, v, hidden).reshape(q.shape).to(q.dtype)


def _plain_prefill(s):
    c, q = s["case"], s["q"]
    group = c["heads"] // c["kv_heads"]
    most_q, most_k = s["most"]
    first_q, first_k = s["cu_q"][:-1].long(), s["cu_k"][:-1].long()
    len_q, len_k = s["cu_q"].diff().long(), s["cu_k"].diff().long()
    at_q, at_k = torch.arange(most_q, device="cuda"), torch.arange(most_k, device="cuda")
    rows = (first_q[:, None] + at_q).clamp(max=q.shape[0] - 1)
    cols = (first_k[:, None] + at_k).clamp(max=s["k"].shape[0] - 1)
    q32 = (q[rows].float() * c["dim"] ** -0.5).view(-1, most_q, c["kv_heads"], group, c["dim"]).permute(0, 2, 3, 1, 4).reshape(-1, c["kv_heads"], group * most_q, c["dim"])
    k, v = (s[x][cols].float().transpose(1, 2) for x in ("k", "v"))
    hidden = (at_k >= len_k[:, None])[:, None, :]
    if c["causal"]:
        hidden = hidden | (at_k > (at_q + (len_k - len_q)[:, None])[:, :, None])
    hidden = hidden.expand(-1, most_q, -1)[:, None].repeat(1, 1, group, 1)
    got = _attend(q32, k, v, hidden).view(-1, c["kv_heads"], group, most_q, c["dim"]).permute(0, 3, 1, 2, 4).reshape(-1, c["heads"], c["dim"])
    place = torch.searchsorted(s["cu_q"], torch.arange(q.shape[0], device="cuda"), right=True) - 1
    return got[place * most_q + torch.arange(q.shape[0], device="cuda") - first_q[place]].to(q.dtype)


def _plain_write(s):
    c, data = s["case"], s["data"]
    page, off = s["slots"] // c["page"], s["slots"] % c["page"]
    k, v = s["k"], s["v"]
    if s["k_scale"] is not None:
        k, v = ((x.float() * (1 / y)[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) for x, y in ((k, s["k_scale"]), (v, s["v_scale"])))
        data = data.view(torch.uint8)
    data[0, page, 0, :, off] = k
    data[0, page, 1, :, off] = v
    return s["data"]


def _plain_branch(s):
    c, table, lengths, refs, data = s["case"], s["table"], s["lengths"], s["refs"], s["data"]
    page, src, dst = c["page"], s["src"].long(), s["dst"].long()
    at = torch.arange(table.shape[1], device="cuda")
    # free
    gone = table[dst].long()
    refs.index_add_(0, gone.clamp(min=0).reshape(-1), -(gone >= 0).to(torch.int32).reshape(-1))
    # fork
    kept = table[src]
    refs.index_add_(0, kept.clamp(min=0).long().reshape(-1), (kept >= 0).to(torch.int32).reshape(-1))
    table[dst], lengths[dst] = kept, lengths[src]
    # reserve: pages in ascending order, one more where the last page is shared and partly filled
    old = lengths[dst].long()
    new = old + s["counts"]
    first, last = -(-old // page), -(-new // page)
    tail = kept.gather(1, (first - 1)[:, None])[:, 0].long()
    copied = (old % page > 0) & (refs[tail] > 1)
    need = last - first + copied
    base = need.cumsum(0) - need
    free = torch.argsort((refs > 0).to(torch.int8), stable=True)
    fresh = (at >= first[:, None]) & (at < last[:, None])
    moved = copied[:, None] & (at == first[:, None] - 1)
    pick = torch.where(moved, base[:, None], (base + copied)[:, None] + at - first[:, None])
    took = free[pick.clamp(0, refs.shape[0] - 1)]
    taken = fresh | moved
    table[dst] = torch.where(taken, took, kept).to(torch.int32)
    refs.index_add_(0, took.reshape(-1), taken.to(torch.int32).reshape(-1))
    refs.index_add_(0, tail, -copied.to(torch.int32))
    lengths[dst] = new.to(torch.int32)
    # the filled rows of the pages that were shared
    to = torch.where(copied, free[base.clamp(max=refs.shape[0] - 1)], tail)
    bits = data.view(torch.uint8) if data.dtype == torch.float8_e4m3fn else data
    rows = (torch.arange(page, device="cuda") < (old % page)[:, None])[None, :, None, None, :, None]
    bits[:, to] = torch.where(rows, bits[:, tail], bits[:, to])
    # slots of the new tokens
    begin = s["counts"].cumsum(0) - s["counts"]
    token = torch.arange(dst.shape[0], device="cuda")  # one each
    i = torch.searchsorted(begin, token, right=True) - 1
    place = old[i] + token - begin[i]
    slots = table[dst[i], place // page].long() * page + place % page
    return [slots, table, lengths, refs, data]


def _plain_compact(s):
    s["table"].copy_(s["given"])  # what the scheduler hands in
    s["refs"].copy_(s["given_refs"])
    refs, table = s["refs"], s["table"]
    live, at = refs > 0, torch.arange(refs.shape[0], device="cuda")
    n = live.sum()
    come, go = (live & (at >= n)).nonzero()[:, 0], (~live & (at < n)).nonzero()[:, 0]
    bits = s["data"].view(torch.uint8) if s["data"].dtype == torch.float8_e4m3fn else s["data"]
    bits[:, go] = bits[:, come]
    remap = torch.where(live, at, -1)
    remap[come] = go
    table.copy_(torch.where(table >= 0, remap[table.clamp(min=0).long()], -1))
    refs[go] = refs[come]
    refs[come] = 0
    return [remap.to(torch.int32), table, refs, s["data"]]


def _cache(s):
    """The handle that a program keeps for its cache."""
    from memfabric_hybrid_b200.ops.kv_cache import PagedKVCache

    if "handle" not in s:
        s["handle"] = PagedKVCache(s["data"], s["table"], s["lengths"], s["refs"])
    return s["handle"]


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        with torch.no_grad():
            return {"decode": _plain_decode, "prefill": _plain_prefill, "write": _plain_write, "branch": _plain_branch, "compact": _plain_compact}[op](s)
    from memfabric_hybrid_b200.ops import attention

    if op == "decode":
        return attention.decode_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if op == "prefill":
        return attention.prefill_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["case"]["causal"])
    cache = _cache(s)
    if op == "write":
        cache.write(0, s["k"], s["v"], s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return s["data"]
    if op == "branch":
        cache.free(s["dst"])
        cache.fork(s["src"], s["dst"])
        slots = cache.reserve(s["dst"], s["counts"], s["dst"].shape[0])
        return [slots, s["table"], s["lengths"], s["refs"], s["data"]]
    s["table"].copy_(s["given"])  # what the scheduler hands in
    s["refs"].copy_(s["given_refs"])
    return [cache.compact(), s["table"], s["refs"], s["data"]]


# ------------------------------------------------------------------------------------------------ work and exact results


def work(case):
    c = case
    wide = 1 if c.get("cache") == "e4m3" else 2
    if c["op"] == "decode":
        seen = sum(_lengths(c, c["batch"], c["gaps"]))
        ends = 4 * c["batch"] * c["heads"] * c["dim"]
        return {"bytes": 2 * seen * c["kv_heads"] * c["dim"] * wide + ends + 4 * seen // c["page"], "flops": 4 * seen * c["heads"] * c["dim"]}
    if c["op"] == "prefill":
        new, old = _lengths(c, c["batch"]), _lengths({"lo": c["past"] // 2, "hi": c["past"]}, c["batch"])
        pairs = sum(n * p + (n * (n + 1) // 2 if c["causal"] else n * n) for n, p in zip(new, old))
        rows = 2 * sum(new) * c["heads"] + 2 * (sum(new) + sum(old)) * c["kv_heads"]
        return {"bytes": 2 * rows * c["dim"], "flops": 4 * pairs * c["heads"] * c["dim"]}
    row = 2 * c["kv_heads"] * c["dim"]  # values of a token's key and value
    if c["op"] == "write":
        return {"bytes": c["tokens"] * (row * (2 + wide) + 8), "flops": 2 * c["tokens"] * row if wide == 1 else 0}
    if c["op"] == "branch":
        lengths = _lengths(c, c["prompts"])
        moved = c["ways"] * sum(n % c["page"] for n in lengths)
        entries = 2 * c["ways"] * sum(-(-n // c["page"]) for n in lengths)  # table entries dropped and set, counts changed
        return {"bytes": 2 * moved * c["layers"] * row * wide + 16 * entries, "flops": 0}
    live = max(c["seqs"], int(c["pages"] * c["live"]))
    moved = live * (c["pages"] - live) // c["pages"]  # on average: the live pages behind the first `live` ones
    return {"bytes": 2 * max(1, moved) * c["layers"] * row * c["page"] * wide + 12 * c["pages"] + 16 * live, "flops": 0}


def _exact_rows(q, k, v, hidden):
    """One sequence, one key head, in 64 bits: q [rows, dim], hidden [rows, keys]."""
    logits = torch.where(hidden, float("-inf"), (q @ k.T) * q.shape[-1] ** -0.5)
    if not logits.shape[1]:
        return torch.zeros_like(q)
    weights = torch.nan_to_num(torch.exp(logits - logits.max(1, keepdim=True).values), nan=0.0)
    return weights @ v / weights.sum(1, keepdim=True).clamp(min=1e-300)


def exact(case, seed):
    c = case
    if c["op"] in ("branch", "compact") or (c["op"] == "write" and c["cache"] != "e4m3"):
        return None  # page numbers and copies: nothing is computed that 64 bits would change
    s = prepare(c, seed)
    if c["op"] == "write":
        out = s["data"].double()
        for which, name in enumerate(("k", "v")):
            x = s[name].double() / s[name + "_scale"].double()[:, None]
            step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)  # three bits behind the leading one, down to 2^-6
            out[0, s["slots"] // c["page"], which, :, s["slots"] % c["page"]] = (torch.round(x / step) * step).clamp(-448, 448)
        return out
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if c["op"] == "decode":
        for b, n in enumerate(s["lengths"].tolist()):
            pages = s["table"][b, :-(-n // c["page"])].long()
            for h in range(c["kv_heads"]):
                k, v = (s[x][:, h].view(torch.uint8)[pages].view(s[x].dtype).double().reshape(-1, c["dim"])[:n] if c["cache"] == "e4m3"
                        else s[x][pages, h].double().reshape(-1, c["dim"])[:n] for x in ("k_pages", "v_pages"))
                if c["cache"] == "e4m3":
                    k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
                rows = slice(h * group, (h + 1) * group)
                out[b, rows] = _exact_rows(s["q"][b, rows].double(), k, v, torch.zeros(group, n, dtype=torch.bool, device="cuda"))
        return out
    cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
    for b in range(c["batch"]):
        n, m = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        hidden = torch.zeros(n, m, dtype=torch.bool, device="cuda")
        if c["causal"]:
            hidden = torch.arange(m, device="cuda") > torch.arange(n, device="cuda")[:, None] + (m - n)
        for h in range(c["heads"]):
            out[cu_q[b]:cu_q[b + 1], h] = _exact_rows(s["q"][cu_q[b]:cu_q[b + 1], h].double(), s["k"][cu_k[b]:cu_k[b + 1], h // group].double(),
                                                      s["v"][cu_k[b]:cu_k[b + 1], h // group].double(), hidden)
    return out
